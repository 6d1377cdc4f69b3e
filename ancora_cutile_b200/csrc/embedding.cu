// Embedding lookup with scaling, and the embedding's gradient by sorted tokens.
//
//   lookup    out[t,:] = round(scale * W[id_t,:])                        zero row where id_t < 0
//   gradient  dW[v,:]  = round(scale * sum_{t: id_t = v} dY[t,:])        "write": every row of the table
//             dW[v,:]  = round(dW[v,:] + scale * sum_{...} dY[t,:])      "add": only rows some token names
//
// Sums are float32, products and sums round to nearest even, the result is rounded once to its type.
// A negative id is padding: zero row, no gradient.  An id at or above V sets status bit 0x8 and is then
// treated as padding, so no address outside the table is ever formed.
//
// The gradient is deterministic: no float atomics.  The tokens are sorted by id (stable, so a row's
// tokens keep their order), the sorted list is cut into equal pieces, each piece sums its runs of equal
// ids, and runs that cross a piece's border are joined from the pieces' partial sums in order.  The work is balanced
// however often one token occurs.
#include <algorithm>
#include <cuda_bf16.h>
#include <initializer_list>
#include <math.h>
#include <type_traits>
#include <mutex>
#include "anc_internal.h"
#include "philox.cuh"
#include "pred_load.cuh"

namespace {

// ------------------------------------------------------------------ rows in registers
// Eight columns of a row as they lie in memory: eight neighbouring ones, in one access, where rows are vectors
// of eight aligned to their size (kVec: 16 bytes of bf16, 32 of f32), else every L-th column.
template <bool kF32, bool kVec>
struct Oct {
  uint32_t w[(kF32 || !kVec) ? 8 : 4];
};

// p: address of the first column; cols: columns from there to the row's end
template <bool kF32, bool kVec>
__device__ __forceinline__ void load_oct(Oct<kF32, kVec> &r, const uint8_t *p, int cols, int L, bool on) {
  if constexpr (kVec) {
    on = on && cols > 0;
    if constexpr (kF32) ld_v8(r.w, p, on);
    else ld_v4(r.w[0], r.w[1], r.w[2], r.w[3], p, on);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (kF32) ld_1(r.w[k], (const float *)p + k * L, on && k * L < cols);
      else ld_h(r.w[k], (const uint16_t *)p + k * L, on && k * L < cols);
    }
  }
}

template <bool kF32, bool kVec>
__device__ __forceinline__ float elem(const Oct<kF32, kVec> &r, int k) {
  if constexpr (kF32) return __uint_as_float(r.w[k]);
  else if constexpr (!kVec) return __uint_as_float(r.w[k] << 16);
  else return __uint_as_float((k & 1) ? (r.w[k >> 1] & 0xFFFF0000u) : (r.w[k >> 1] << 16));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <bool kF32, bool kVec>
__device__ __forceinline__ void store_oct(uint8_t *p, int cols, int L, const float (&x)[8]) {
  if constexpr (kVec) {
    if (cols <= 0) return;
    if constexpr (kF32) st_v8(p, x);
    else
      *reinterpret_cast<uint4 *>(p) =
          make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k * L < cols) {
        if constexpr (kF32) ((float *)p)[k * L] = x[k];
        else ((uint16_t *)p)[k * L] = (uint16_t)bf16_rne(x[k]);
      }
  }
}

__device__ __forceinline__ int64_t load_id(const void *ids, int ids64, int64_t t) {
  return ids64 ? ((const int64_t *)ids)[t] : (int64_t)((const int32_t *)ids)[t];
}

// ------------------------------------------------------------------ lookup
// Bound by memory once two latencies (id, then row) are covered: 32768 rows of 1024 bf16, 91 MB of distinct rows,
// ids and output, take 14.4 us on the device, 131072 rows 59 us (ids by a 1 / rank law).  A warp takes 32 / L rows side by side, L lanes a
// row, and every lane up to four octets: kOcts of a row, of 4 / kOcts rows; rows longer than four octets a lane
// are cut into slices as equal as that allows (53579 rows of 1303 bf16: two slices of three octets 62 us, of four
// and two 76).  Warps do one unit and leave: resident ones that went on to further rows, with the next ids read
// ahead, were slower (131072 rows of 1024 bf16: 70 against 59 us; 32768: 20.4 against 18.7).
constexpr int kLookupThreads = 128;

struct LookupArgs {
  const uint8_t *table;
  const void *ids;
  uint8_t *out;
  uint32_t table_pitch, out_pitch;      // bytes from row to row
  uint32_t T, V, units;
  int ids64, D, L;
  float scale;
  uint32_t *status;
};

// A warp per unit: unit u is rows [u, u + 1) * kRows * 32 / L; blockIdx.y: slice of 8 * kOcts * L columns.
template <bool kTabF32, bool kOutF32, bool kVec, int kOcts>
__global__ void __launch_bounds__(kLookupThreads)
embedding_lookup_kernel(LookupArgs a) {
  constexpr int kRows = 4 / kOcts, kTB = kTabF32 ? 4 : 2, kOB = kOutF32 ? 4 : 2;
  const int L = a.L, lane = threadIdx.x & 31, l = lane & (L - 1);
  const uint32_t u = blockIdx.x * (kLookupThreads / 32) + (threadIdx.x >> 5);
  if (u >= a.units) return;
  const int c0 = (int)blockIdx.y * (8 * kOcts) * L + (kVec ? l * 8 : l);
  const int cols = a.D - c0;            // from this lane's first column to the row's end
  const uint32_t t0 = u * kRows * (32 / L) + lane / L, t_step = 32 / L;
  Oct<kTabF32, kVec> x[kRows][kOcts] = {};
  int64_t id[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const uint32_t t = t0 + r * t_step;
    id[r] = load_id(a.ids, a.ids64, t < a.T ? t : a.T - 1);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const bool live = id[r] >= 0 && id[r] < a.V;
    const uint8_t *row = a.table + (int64_t)c0 * kTB + (uint64_t)(live ? (uint32_t)id[r] : 0u) * a.table_pitch;
#pragma unroll
    for (int q = 0; q < kOcts; ++q)
      load_oct<kTabF32, kVec>(x[r][q], row + q * 8 * L * kTB, cols - q * 8 * L, L, live);
    if (id[r] >= a.V && l == 0 && blockIdx.y == 0) atomicOr(a.status, ANC_DEV_BAD_INDEX);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const uint32_t t = t0 + r * t_step;
    uint8_t *row = a.out + (int64_t)c0 * kOB + (uint64_t)t * a.out_pitch;
    const float scale = id[r] >= 0 && id[r] < a.V ? a.scale : 0.f;      // a negative one would make -0 of a zero row
#pragma unroll
    for (int q = 0; q < kOcts; ++q) {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = __fmul_rn(elem(x[r][q], k), scale);
      store_oct<kOutF32, kVec>(row + q * 8 * L * kOB, t < a.T ? cols - q * 8 * L : 0, L, f);
    }
  }
}

// ------------------------------------------------------------------ sort
// Stable least-significant-digit radix sort of (id, token) by one cluster of CTAs, up to nine bits a pass:
// two passes for tables of up to 2^18 rows.  Per pass every warp counts the digits of its stretch of the list,
// the cluster exchanges its CTAs' digit counts through distributed shared memory, and every warp then
// writes its stretch to the places the counts give.  Padding sorts behind the last row of the table as id V.
// The passes are bound by latency, not by bytes: hence many CTAs with short stretches, all loads of a stretch
// before their first use, and the ranks of a stretch of up to eight rounds kept in registers from the
// counting to the writing.  Lanes of equal digit find each other by a word per digit in shared memory (nine
// ballots or the match instruction took two to four times as long).  65536 tokens: 18.5 us, 16384: 14.4, 2048: 8.3.
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortThreads = kDigits;              // a thread per digit
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortRounds = 8;
constexpr uint32_t kMaxCluster = 16;

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ uint4 ld_cluster(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct SortArgs {
  const void *ids;
  int ids64;
  uint32_t T;
  int64_t V, padding_idx;
  uint2 *list[2];                // (id, token)
  int passes;
  uint32_t *clear;               // words to clear: flags of the sums
  uint32_t n_clear;
  uint32_t *status;
};

__device__ __forceinline__ uint32_t key_of(int64_t id, int64_t V, int64_t padding_idx) {
  return (id < 0 || id >= V || id == padding_idx) ? (uint32_t)V : (uint32_t)id;
}

// The order of the list: the last row of the table first, padding at the end.  Vocabularies have their frequent
// tokens at the front; the long runs of those are the cheap pieces, and come last (65536 tokens, rows of 1024 bf16
// added to f32, id = rank in frequency: 75 us against 82 in ascending order).
__device__ __forceinline__ uint32_t reversed(uint32_t key, uint32_t V) { return key == V ? V : V - 1u - key; }

struct SortShared {
  uint32_t cnt[kSortWarps][kDigits];     // per warp: counts, then places of the warp's first keys
  uint32_t lanes[kSortWarps][kDigits];   // per warp: the lanes that hold a digit, one round at a time
  uint32_t tot[kDigits];                 // this CTA's digit counts, read by the whole cluster
  uint32_t off[kDigits];                 // first place of a digit's keys of this CTA
  uint32_t share[2][4][kDigits];         // counts of a quarter of the cluster: all, and those before this CTA
  uint32_t wsum[kSortWarps];
  uint2 list[kSortThreads * kSortRounds];   // the list between passes when one CTA sorts
};

__global__ void __launch_bounds__(kSortThreads, 1)
embedding_sort_kernel(SortArgs a, uint32_t n_ctas) {
  extern __shared__ __align__(16) uint8_t sort_smem[];
  SortShared &sh = *reinterpret_cast<SortShared *>(sort_smem);
  pdl_trigger();
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x;
  for (uint32_t i = rank * kSortThreads + tid; i < a.n_clear; i += n_ctas * kSortThreads) a.clear[i] = 0u;
  // every warp's stretch: the same number of whole rounds of 32 keys
  const uint32_t rounds = (a.T + n_ctas * kSortThreads - 1) / (n_ctas * kSortThreads);
  const uint64_t lo64 = (uint64_t)(rank * kSortWarps + warp) * rounds * 32;
  const uint32_t lo = lo64 < a.T ? (uint32_t)lo64 : a.T;
  const uint32_t hi = a.T - lo < rounds * 32 ? a.T : lo + rounds * 32;
  const bool short_stretch = rounds <= kSortRounds;
  const bool single = n_ctas == 1 && short_stretch;      // the list stays in shared memory between passes
  uint32_t *mine = sh.cnt[warp], *lanes = sh.lanes[warp];
  // kSortRounds rounds of the list, all loads before the first use (places past the end repeat the last one);
  // the first pass reads the ids.  Returns whether one of this lane's ids lies outside the table.
  auto fetch = [&](uint2 (&e)[kSortRounds], const uint2 *in, bool first, uint32_t i0) {
    bool bad = false;
    if (first) {
      int64_t id[kSortRounds];
#pragma unroll
      for (int r = 0; r < kSortRounds; ++r) {
        const uint32_t i = i0 + r * 32 + lane;
        id[r] = load_id(a.ids, a.ids64, i < a.T ? i : a.T - 1);
      }
#pragma unroll
      for (int r = 0; r < kSortRounds; ++r) {
        e[r] = make_uint2(reversed(key_of(id[r], a.V, a.padding_idx), (uint32_t)a.V), i0 + r * 32 + lane);
        bad = bad || id[r] >= a.V;
      }
    } else {
#pragma unroll
      for (int r = 0; r < kSortRounds; ++r) {
        const uint32_t i = i0 + r * 32 + lane;
        const uint32_t j = i < a.T ? i : a.T - 1;
        if (single) e[r] = sh.list[j < kSortThreads * kSortRounds ? j : 0];
        else e[r] = __ldcg(in + j);
      }
    }
    return bad;
  };
  // Places of this lane's keys among the warp's keys of the same digit so far.  The lanes of equal digit find
  // each other by setting their bits in a word per digit.
  auto rank_in = [&](uint32_t (&place)[kSortRounds], const uint2 (&e)[kSortRounds], int shift, uint32_t i0) {
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (i0 + r * 32 >= hi) break;
      const bool on = i0 + r * 32 + lane < hi;
      const uint32_t d = (e[r].x >> shift) & (kDigits - 1);
      if (on) atomicOr(lanes + d, 1u << lane);
      __syncwarp();
      const uint32_t peers = lanes[d], at = mine[d];
      __syncwarp();
      if (on && lane == (uint32_t)(__ffs(peers) - 1)) {
        mine[d] = at + __popc(peers);
        lanes[d] = 0u;
      }
      __syncwarp();
      place[r] = at + __popc(peers & ((1u << lane) - 1u));
    }
  };
  for (uint32_t d = lane * 4; d < kDigits; d += 128) *reinterpret_cast<uint4 *>(lanes + d) = make_uint4(0u, 0u, 0u, 0u);
  for (int p = 0; p < a.passes; ++p) {
    const bool odd = p & 1, last = p + 1 == a.passes;
    const uint2 *in = odd ? a.list[0] : a.list[1];
    uint2 *out = odd ? a.list[1] : a.list[0];
    const int shift = p * kDigitBits;
    auto put = [&](uint32_t dst, uint2 e, bool on) {
      if (on) {
        if (last) e.x = reversed(e.x, (uint32_t)a.V);
        if (single && !last) sh.list[dst] = e;
        else out[dst] = e;
      }
    };
    for (uint32_t d = lane * 4; d < kDigits; d += 128) *reinterpret_cast<uint4 *>(mine + d) = make_uint4(0u, 0u, 0u, 0u);
    __syncwarp();
    uint2 e[kSortRounds];
    uint32_t place[kSortRounds];
    for (uint32_t i0 = lo; i0 < hi; i0 += 32 * kSortRounds) {
      if (fetch(e, in, p == 0, i0)) atomicOr(a.status, ANC_DEV_BAD_INDEX);
      if (short_stretch) {
        rank_in(place, e, shift, i0);
      } else {
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r)
          if (i0 + r * 32 + lane < hi) atomicAdd(mine + ((e[r].x >> shift) & (kDigits - 1)), 1u);
      }
    }
    __syncthreads();
    uint32_t all = 0, before = 0, run = 0, c[kSortWarps];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) c[w] = sh.cnt[w][tid];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      sh.cnt[w][tid] = run;
      run += c[w];
    }
    if (!single) {
      sh.tot[tid] = run;
      cluster_sync();
    }
    if (single) {
      all = run;
    } else {
      // a quarter of the threads per quarter of the cluster, four digits each
      const uint32_t quad = tid & 127, quarter = tid >> 7;
      const uint32_t slot = (uint32_t)__cvta_generic_to_shared(sh.tot + quad * 4);
      uint4 v[kMaxCluster / 4];
#pragma unroll
      for (uint32_t j = 0; j < kMaxCluster / 4; ++j) {
        const uint32_t q = j * 4 + quarter;
        v[j] = ld_cluster(peer_smem(slot, q < n_ctas ? q : rank));
      }
      uint4 sum_all = make_uint4(0u, 0u, 0u, 0u), sum_before = sum_all;
#pragma unroll
      for (uint32_t j = 0; j < kMaxCluster / 4; ++j) {
        const uint32_t q = j * 4 + quarter, in_all = q < n_ctas ? 0xFFFFFFFFu : 0u, in_before = q < rank ? 0xFFFFFFFFu : 0u;
        sum_all.x += v[j].x & in_all; sum_all.y += v[j].y & in_all;
        sum_all.z += v[j].z & in_all; sum_all.w += v[j].w & in_all;
        sum_before.x += v[j].x & in_before; sum_before.y += v[j].y & in_before;
        sum_before.z += v[j].z & in_before; sum_before.w += v[j].w & in_before;
      }
      *reinterpret_cast<uint4 *>(&sh.share[0][quarter][quad * 4]) = sum_all;
      *reinterpret_cast<uint4 *>(&sh.share[1][quarter][quad * 4]) = sum_before;
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        all += sh.share[0][q][tid];
        before += sh.share[1][q][tid];
      }
    }
    uint32_t sum = all;      // exclusive scan of the digit totals
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      if (lane >= (uint32_t)o) sum += u;
    }
    if (lane == 31) sh.wsum[warp] = sum;
    __syncthreads();
    uint32_t base = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSortWarps; ++w)
      if (w < warp) base += sh.wsum[w];
    sh.off[tid] = base + sum - all + before;
    __syncthreads();
    if (short_stretch) {
      if (lo < hi) {
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r) {
          if (lo + r * 32 >= hi) break;
          const uint32_t d = (e[r].x >> shift) & (kDigits - 1);
          put(sh.off[d] + mine[d] + place[r], e[r], lo + r * 32 + lane < hi);
        }
      }
    } else {
      for (uint32_t i0 = lo; i0 < hi; i0 += 32 * kSortRounds) {
        fetch(e, in, p == 0, i0);
        rank_in(place, e, shift, i0);
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r) {
          if (i0 + r * 32 >= hi) break;
          put(sh.off[(e[r].x >> shift) & (kDigits - 1)] + place[r], e[r], i0 + r * 32 + lane < hi);
        }
      }
    }
    __syncwarp();
    if (single) __syncthreads();
    else cluster_sync();     // the next pass reads what other CTAs wrote, and overwrites tot
  }
}

// ------------------------------------------------------------------ zeros
struct ZeroArgs {
  uint8_t *dw;
  int64_t row_bytes, pitch, V;
  int64_t rows, bytes;           // of one part: whole rows, or where rows leave no gaps `bytes` of the table
  uint32_t parts;
};

// zeros in n bytes at p by the threads of one block, 16 at a time between the first and the last 16-byte boundary
__device__ __forceinline__ void zero_bytes(uint8_t *p, int64_t n) {
  const int64_t to_16 = (16 - ((uintptr_t)p & 15)) & 15, head = to_16 < n ? to_16 : n;
  const int64_t vecs = (n - head) / 16, tail = head + vecs * 16;
  uint4 *q = reinterpret_cast<uint4 *>(p + head);
  for (int64_t i = threadIdx.x; i < vecs; i += blockDim.x) q[i] = make_uint4(0u, 0u, 0u, 0u);
  const int64_t mine = (int64_t)threadIdx.x * 2;
  if (mine < head) *reinterpret_cast<uint16_t *>(p + mine) = 0;
  if (tail + mine < n) *reinterpret_cast<uint16_t *>(p + tail + mine) = 0;
}

__device__ __forceinline__ void zero_part(const ZeroArgs &z, int64_t k) {
  if (z.pitch == z.row_bytes) {
    const int64_t lo = k * z.bytes, left = z.V * z.row_bytes - lo;
    zero_bytes(z.dw + lo, left < z.bytes ? left : z.bytes);
  } else {
    const int64_t v1 = (k + 1) * z.rows < z.V ? (k + 1) * z.rows : z.V;
    for (int64_t v = k * z.rows; v < v1; ++v) zero_bytes(z.dw + v * z.pitch, z.row_bytes);
  }
}

// Up to kRankT tokens a token's place in the list is counted: keys below its own, and equal ones of earlier
// tokens. Every CTA holds all keys in shared memory, every warp counts for two tokens at a time, four keys per
// lane and step.  T^2 comparisons on all SMs, but no step waits for another CTA: 300 tokens 4.8 us, 2048 5.3, 4096
// 6.6, against 6.0, 8.0 and 10.5 by the sort above (whole calls: 5000 tokens 20.2 against 20.7, 6500: 22.9 against
// 22.4).  The CTAs write the zeros of a small table too, which saves a launch (2048 tokens, 1 MB: 13.6 us against
// 15.9 a call; 16 MB: 15.4 against 16.8, 65 MB: 23.5 against 22.1, where the zeros hide the sort beside them).
constexpr int kRankT = 4096;
constexpr int kRankThreads = 512;
constexpr int kRankTokens = 2;      // neighbours, one step of 128 keys holds both

__global__ void __launch_bounds__(kRankThreads)
embedding_rank_kernel(SortArgs a, ZeroArgs z) {
  extern __shared__ __align__(16) uint32_t rank_keys[];
  pdl_trigger();
  const uint32_t tid = threadIdx.x, lane = tid & 31;
  for (uint32_t i = blockIdx.x * kRankThreads + tid; i < a.n_clear; i += gridDim.x * kRankThreads) a.clear[i] = 0u;
  const uint32_t steps = (a.T + 127) / 128;
  constexpr int kAtOnce = 8;
  for (uint32_t i0 = tid; i0 < steps * 128; i0 += kRankThreads * kAtOnce) {
    int64_t id[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const uint32_t i = i0 + k * kRankThreads;
      id[k] = load_id(a.ids, a.ids64, i < a.T ? i : a.T - 1);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const uint32_t i = i0 + k * kRankThreads;
      if (i < steps * 128)      // behind the last key: above every other
        rank_keys[i] = i < a.T ? reversed(key_of(id[k], a.V, a.padding_idx), (uint32_t)a.V) : 0xFFFFFFFFu;
      if (id[k] >= a.V && blockIdx.x == 0) atomicOr(a.status, ANC_DEV_BAD_INDEX);
    }
  }
  for (int64_t k = blockIdx.x; k < z.parts; k += gridDim.x) zero_part(z, k);
  __syncthreads();
  const uint32_t n_warps = gridDim.x * (kRankThreads / 32);
  for (uint32_t t0 = (blockIdx.x * (kRankThreads / 32) + (tid >> 5)) * kRankTokens; t0 < a.T;
       t0 += n_warps * kRankTokens) {
    const uint4 *keys = reinterpret_cast<const uint4 *>(rank_keys) + lane;
    uint32_t key[kRankTokens], n[kRankTokens] = {};
#pragma unroll
    for (int b = 0; b < kRankTokens; ++b) key[b] = rank_keys[t0 + b];
    auto count = [&](uint32_t s, uint32_t equal) {       // equal: 1 where equal keys count too
      const uint4 k = keys[s * 32];
#pragma unroll
      for (int b = 0; b < kRankTokens; ++b) {
        const uint32_t below = key[b] + equal;
        n[b] += (k.x < below) + (k.y < below) + (k.z < below) + (k.w < below);
      }
    };
    const uint32_t mid = t0 / 128;
#pragma unroll 4
    for (uint32_t s = 0; s < mid; ++s) count(s, 1u);
#pragma unroll 4
    for (uint32_t s = mid; s < steps; ++s) count(s, 0u);
    const uint4 k = keys[mid * 32];                      // equal keys of earlier tokens in the middle step
    const uint32_t s0 = mid * 128 + lane * 4;
#pragma unroll
    for (int b = 0; b < kRankTokens; ++b) {
      n[b] += (k.x == key[b] && s0 < t0 + b) + (k.y == key[b] && s0 + 1 < t0 + b) + (k.z == key[b] && s0 + 2 < t0 + b) +
              (k.w == key[b] && s0 + 3 < t0 + b);
      n[b] = __reduce_add_sync(0xFFFFFFFFu, n[b]);
      if (lane == (uint32_t)b && t0 + b < a.T) a.list[0][n[b]] = make_uint2(reversed(key[b], (uint32_t)a.V), t0 + b);
    }
  }
}

constexpr int kZeroThreads = 256;

// When the whole table is written, what the SMs that do not sort do meanwhile.  Launched behind the sort without
// waiting for it; it waits for the sort only before it ends, so that whoever waits for this kernel has the
// sorted list too.  311 MB of zeros: 48 us alone, 6.5 TB/s.  (Reading dy into L2 at that time
// cost 9 us of 66 beside the zeros.)
__global__ void __launch_bounds__(kZeroThreads)
embedding_zero_kernel(ZeroArgs z) {
  pdl_trigger();
  zero_part(z, blockIdx.x);
  pdl_wait();
}

// ------------------------------------------------------------------ sums of runs
constexpr int kRedThreads = 256;
constexpr int kMaxPiece = 512;       // sorted places per block
constexpr uint32_t kWaitPolls = 1u << 20;
constexpr uint32_t kAheadBlocks = 296, kAheadPiece = 8192;

struct RedArgs {
  const uint8_t *dy;
  const uint8_t *ahead;          // bytes of dy to read into L2 while the list is made
  uint64_t ahead_bytes;
  uint8_t *dw;
  uint32_t dy_pitch, dw_pitch;   // bytes from row to row
  int64_t T;
  const uint2 *list;             // sorted (id, token)
  float *partial;                // [piece][slices * columns of a slice], register layout
  uint32_t V;
  int D, slices;
  int L;                         // lanes that share a row's slice: a power of two up to 32
  int per_part;                  // sorted places per group of L lanes
  float scale;
  uint32_t *flags;               // [piece][slice]: the partial sum of the run open at the piece's end is there
  uint32_t raised, polls;        // what a raised flag holds (the self-test of the wait: 0), reads of a flag at most
  uint32_t *status;
};

// A lane's columns of a slice: sixteen in two octets, all lanes' first octets before their second ones, or
// eight where rows are not vectors.  Sums are pairs of floats (one instruction adds two).
template <bool kVec>
struct Cols {
  static constexpr int kOcts = kVec ? 2 : 1, kEach = 8 * kOcts;
};
template <bool kVec>
struct Sum {
  uint64_t p[Cols<kVec>::kEach / 2];
  __device__ __forceinline__ float get(int k) const {
    return __uint_as_float((uint32_t)((k & 1) ? p[k >> 1] >> 32 : p[k >> 1]));
  }
  __device__ __forceinline__ void add_pair(int i, float lo, float hi) {
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tadd.rn.f32x2 %0, %0, t;\n\t}" : "+l"(p[i]) : "f"(lo), "f"(hi));
  }
  __device__ __forceinline__ void set_pair(int i, float lo, float hi) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(p[i]) : "f"(lo), "f"(hi));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < Cols<kVec>::kEach / 2; ++i) p[i] = 0ull;
  }
  // as kEach floats `pitch` apart
  __device__ __forceinline__ void put(float *d, int pitch) const {
#pragma unroll
    for (int k = 0; k < Cols<kVec>::kEach; ++k) d[k * pitch] = get(k);
  }
  __device__ __forceinline__ void set(const float *d, int pitch) {
#pragma unroll
    for (int i = 0; i < Cols<kVec>::kEach / 2; ++i) set_pair(i, d[2 * i * pitch], d[(2 * i + 1) * pitch]);
  }
  __device__ __forceinline__ void add(const float *d, int pitch) {
#pragma unroll
    for (int i = 0; i < Cols<kVec>::kEach / 2; ++i) add_pair(i, d[2 * i * pitch], d[(2 * i + 1) * pitch]);
  }
};

template <bool kF32, bool kVec>
struct Row {
  Oct<kF32, kVec> o[Cols<kVec>::kOcts];
  __device__ __forceinline__ void load(const uint8_t *p, int cols, int L, bool on) {
#pragma unroll
    for (int q = 0; q < Cols<kVec>::kOcts; ++q)
      load_oct<kF32, kVec>(o[q], p + q * 8 * L * (kF32 ? 4 : 2), cols - q * 8 * L, L, on);
  }
  __device__ __forceinline__ void add_to(Sum<kVec> &s) const {
#pragma unroll
    for (int q = 0; q < Cols<kVec>::kOcts; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) s.add_pair(q * 4 + i, elem(o[q], 2 * i), elem(o[q], 2 * i + 1));
  }
};

// One lane's view of the rows: its first column, and the columns from there to the row's end.
template <bool kDyF32, bool kDwF32, bool kVec, bool kAdd, bool kWide>
struct Lane {
  const uint8_t *dy;
  uint8_t *dw;
  int cols, L;
  __device__ __forceinline__ Lane(const RedArgs &a, int slice, int l) {
    L = kWide ? 32 : a.L;
    const int c = slice * Cols<kVec>::kEach * L + (kVec ? l * 8 : l);
    cols = kWide ? Cols<kVec>::kEach * 32 : a.D - c;
    dy = a.dy + (int64_t)c * (kDyF32 ? 4 : 2);
    dw = a.dw + (int64_t)c * (kDwF32 ? 4 : 2);
  }
  __device__ __forceinline__ const uint8_t *dy_row(const RedArgs &a, uint32_t t) const {
    return dy + (uint64_t)t * a.dy_pitch;
  }
  __device__ __forceinline__ uint8_t *dw_row(const RedArgs &a, uint32_t v) const {
    return dw + (uint64_t)v * a.dw_pitch;
  }
  // the finished sum of row v into the table
  __device__ __forceinline__ void finish(const RedArgs &a, uint32_t v, const Sum<kVec> &s,
                                         const Row<kDwF32, kVec> &old) const {
    uint8_t *p = dw_row(a, v);
#pragma unroll
    for (int q = 0; q < Cols<kVec>::kOcts; ++q) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] = __fmul_rn(a.scale, s.get(q * 8 + k));
        if (kAdd) x[k] = __fadd_rn(elem(old.o[q], k), x[k]);
      }
      store_oct<kDwF32, kVec>(p + q * 8 * L * (kDwF32 ? 4 : 2), cols - q * 8 * L, L, x);
    }
  }
  __device__ __forceinline__ void flush(const RedArgs &a, uint32_t v, const Sum<kVec> &s) const {
    Row<kDwF32, kVec> old = {};
    old.load(dw_row(a, v), cols, L, kAdd);
    finish(a, v, s, old);
  }
};

// A block takes one piece of the sorted list and one slice of columns; each of its groups of L lanes
// takes per_part places of the piece.  A run inside a part goes straight to the table.  The sums of runs
// that are open at a part's start or end are left in shared memory and joined in order by the group in whose
// part the run starts.  A run that is open at the piece's end leaves its sum in `partial`, raises the
// piece's flag, and is finished by the block in whose piece it ends: that block waits for the flags of the pieces
// before it (blocks start in index order, and a block raises its flag before it waits for anything; the
// wait is bounded) and adds their sums in order.
//
// Bound by memory latency unless enough rows are in flight.  Rows that are vectors go through a ring in
// shared memory: every warp has asynchronous copies of the rows of the next kDepth places on the way and,
// with "add", of the old table rows of the runs that end there (12 KB per warp, 192 KB per SM).  Loads ahead into
// registers did not get there: they share six scoreboards, so waiting for one row waited for the newest
// one too (accumulating 65536 rows of 1024, 209 MB read and 44 written: 63 us that way, 50 us by the ring, 5.1 TB/s).
//
// kWide: 32 lanes per row and whole slices, so that nothing about columns is left to compute in the loop (198
// instructions per place and warp without it, 140 with it).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <bool kDyF32, bool kDwF32, bool kVec, bool kAdd>
struct Stage {
  static constexpr int kCols = 32 * Cols<true>::kEach;                  // columns a warp holds
  static constexpr int kDy = kCols * (kDyF32 ? 4 : 2), kOld = kAdd ? kCols * (kDwF32 ? 4 : 2) : 0;
  static constexpr int kDepth = 12288 / (kDy + kOld) < 8 ? 12288 / (kDy + kOld) : 8;
  static constexpr uint32_t kWarp = kDepth * (kDy + kOld);
  // afterwards the same memory holds the open sums of all parts
  static constexpr uint32_t kRing = kRedThreads / 32 * kWarp, kOpen = 2 * kRedThreads * Cols<kVec>::kEach * 4;
  static constexpr uint32_t kBytes = kVec && kRing > kOpen ? kRing : kOpen;
};

template <bool kDyF32, bool kDwF32, bool kVec, bool kAdd, bool kWide>
__global__ void __launch_bounds__(kRedThreads, 2)
embedding_reduce_kernel(RedArgs a) {
  using St = Stage<kDyF32, kDwF32, kVec, kAdd>;
  constexpr int kEach = Cols<kVec>::kEach;
  constexpr uint32_t kEnds = 0x80000000u;             // in a token number: the run ends here
  extern __shared__ __align__(128) uint8_t stage_smem[];
  __shared__ uint32_t open_key[2][kRedThreads];       // V: nothing open
  __shared__ uint8_t through[kRedThreads];            // the part is one run, open at both ends (slot 0)
  __shared__ uint2 list[kMaxPiece + 1];               // the place before the piece, the piece's places
  __shared__ uint32_t s_first;
  const int L = kWide ? 32 : a.L, l = threadIdx.x & (L - 1), part = threadIdx.x / L, parts = kRedThreads / L;
  const int span = kEach * L;
  float *const open_head = reinterpret_cast<float *>(stage_smem);      // [part][span], after the loop: the run open at
  float *const open_tail = open_head + kRedThreads * kEach;            // the part's start, and at its end only
  const uint32_t piece = blockIdx.x / a.slices;
  const int slice = (int)(blockIdx.x - piece * a.slices);
  const Lane<kDyF32, kDwF32, kVec, kAdd, kWide> lane(a, slice, l);
  const int len = parts * a.per_part;
  const int64_t p0 = (int64_t)piece * len;
  for (int i = threadIdx.x; i < 2 * parts; i += kRedThreads) open_key[i & 1][i >> 1] = a.V;
  if (l == 0) through[part] = 0;
  if (kAdd && threadIdx.x == 0 && blockIdx.x < kAheadBlocks) {
    const uint64_t step = (uint64_t)(gridDim.x < kAheadBlocks ? gridDim.x : kAheadBlocks) * kAheadPiece;
    for (uint64_t o = (uint64_t)blockIdx.x * kAheadPiece; o < a.ahead_bytes; o += step) {
      const uint32_t n = (uint32_t)(a.ahead_bytes - o < kAheadPiece ? a.ahead_bytes - o : kAheadPiece);
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.ahead + o), "r"(n) : "memory");
    }
  }
  pdl_wait();
  int live = 0;      // the padding lies behind the last run
  for (int i0 = 0; i0 < len + 1; i0 += kRedThreads) {
    const int i = i0 + threadIdx.x;
    const int64_t g = p0 + i - 1;
    uint2 e = make_uint2(a.V, 0u);
    if (i < len + 1 && g >= 0 && g < a.T) {
      e = __ldcg(a.list + g);
      const uint32_t next = g + 1 < a.T ? __ldcg(&a.list[g + 1].x) : a.V;
      if (next != e.x) e.y |= kEnds;
    }
    if (i < len + 1) list[i] = e;
    live += __syncthreads_count(i >= 1 && i <= len && e.x < a.V);
  }
  const uint2 *mine = list + 1 + part * a.per_part;
  int n = live - part * a.per_part;
  n = n < 0 ? 0 : n > a.per_part ? a.per_part : n;
  const uint32_t prev = mine[-1].x;
  Sum<kVec> acc, own;        // the run so far; the run from before the part (later: the piece), where it ends here
  acc.clear();
  own.clear();
  bool has_own = false, open = false;
  // the end of place e in its run, with acc holding the run's sum
  auto end_run = [&](uint2 e, const Row<kDwF32, kVec> &old) {
    if (e.x != prev) {
      lane.finish(a, e.x, acc, old);
    } else {
      own = acc;
      has_own = true;
    }
    acc.clear();
    open = false;
  };
  if constexpr (kVec) {
    constexpr int kYB = kDyF32 ? 4 : 2, kWB = kDwF32 ? 4 : 2, kYChunks = kEach * kYB / 16, kWChunks = kEach * kWB / 16;
    const int c0 = slice * span, group = (threadIdx.x & 31) / L;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(stage_smem) + (threadIdx.x >> 5) * St::kWarp;
    const uint8_t *ring_ptr = stage_smem + (threadIdx.x >> 5) * St::kWarp;
    const uint8_t *dy = a.dy + (int64_t)c0 * kYB, *dw = a.dw + (int64_t)c0 * kWB;
    const int y_bytes = (a.D - c0) * kYB, w_bytes = (a.D - c0) * kWB;
    // chunk q of a row: 16 bytes per lane, the group's lanes side by side
    auto fetch = [&](uint32_t slot, int j) {
      if (j < n) {
        const uint2 e = mine[j];
        const uint8_t *src = dy + (uint64_t)(e.y & ~kEnds) * a.dy_pitch + l * 16;
        const uint32_t dst = ring + slot * (St::kDy + St::kOld) + group * (span * kYB) + l * 16;
#pragma unroll
        for (int q = 0; q < kYChunks; ++q)
          if (kWide || (q * L + l) * 16 < y_bytes) cp_async16(dst + q * L * 16, src + q * L * 16);
        if (kAdd && (e.y & kEnds) && e.x != prev) {
          const uint8_t *old = dw + (uint64_t)e.x * a.dw_pitch + l * 16;
          const uint32_t od = ring + slot * (St::kDy + St::kOld) + St::kDy + group * (span * kWB) + l * 16;
#pragma unroll
          for (int q = 0; q < kWChunks; ++q)
            if (kWide || (q * L + l) * 16 < w_bytes) cp_async16(od + q * L * 16, old + q * L * 16);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto take = [&](auto &row, const uint8_t *p, auto f32) {      // this lane's octets of a staged row
#pragma unroll
      for (int q = 0; q < Cols<true>::kOcts; ++q) {
        const uint4 *v = reinterpret_cast<const uint4 *>(p + (q * 8 * L + l * 8) * (f32.value ? 4 : 2));
        const uint4 w = v[0];
        row.o[q].w[0] = w.x; row.o[q].w[1] = w.y; row.o[q].w[2] = w.z; row.o[q].w[3] = w.w;
        if constexpr (f32.value) {
          const uint4 u = v[1];
          row.o[q].w[4] = u.x; row.o[q].w[5] = u.y; row.o[q].w[6] = u.z; row.o[q].w[7] = u.w;
        }
      }
    };
    // all groups of a warp go round together, the longest sets the count
    int rounds = n;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rounds = max(rounds, __shfl_xor_sync(0xFFFFFFFFu, rounds, o));
#pragma unroll
    for (int d = 0; d < St::kDepth; ++d) fetch(d, d);
    uint32_t slot = 0;
    for (int j = 0; j < rounds; ++j) {
      asm volatile("cp.async.wait_group %0;" ::"n"(St::kDepth - 1) : "memory");
      __syncwarp();
      if (j < n) {
        const uint8_t *st = ring_ptr + slot * (St::kDy + St::kOld);
        const uint2 e = mine[j];
        Row<kDyF32, kVec> x;
        take(x, st + group * (span * kYB), std::integral_constant<bool, kDyF32>());
        x.add_to(acc);
        open = true;
        if (e.y & kEnds) {
          Row<kDwF32, kVec> old = {};
          if (kAdd && e.x != prev) take(old, st + St::kDy + group * (span * kWB), std::integral_constant<bool, kDwF32>());
          end_run(e, old);
        }
      }
      __syncwarp();
      fetch(slot, j + St::kDepth);
      if (++slot == St::kDepth) slot = 0;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else {
    constexpr int kAhead = 4;
    for (int j0 = 0; j0 < n; j0 += kAhead) {
      Row<kDyF32, kVec> x[kAhead] = {};
      Row<kDwF32, kVec> old[kAhead] = {};
#pragma unroll
      for (int b = 0; b < kAhead; ++b) {
        const uint2 e = mine[j0 + b < n ? j0 + b : 0];
        x[b].load(lane.dy_row(a, e.y & ~kEnds), lane.cols, L, j0 + b < n);
        if (kAdd) old[b].load(lane.dw_row(a, e.x), lane.cols, L, j0 + b < n && (e.y & kEnds) && e.x != prev);
      }
#pragma unroll
      for (int b = 0; b < kAhead; ++b) {
        if (j0 + b >= n) break;
        const uint2 e = mine[j0 + b];
        x[b].add_to(acc);
        open = true;
        if (e.y & kEnds) end_run(e, old[b]);
      }
    }
  }
  __syncthreads();
  if (has_own) own.put(open_head + part * span + l, L);
  if (open) acc.put((mine[n - 1].x == prev ? open_head : open_tail) + part * span + l, L);
  if (l == 0) {
    if (has_own) open_key[0][part] = prev;
    if (open) {
      const uint32_t k = mine[n - 1].x;
      open_key[k == prev ? 0 : 1][part] = k;
      if (k == prev) through[part] = 1;
    }
  }
  __syncthreads();
  // [piece][slice][span]: the sum of the run that is open at the piece's end, over this piece
  float *partial = a.partial + (int64_t)slice * span + l;
  const int64_t pitch = (int64_t)a.slices * span;
  auto publish = [&](const Sum<kVec> &sum) {
    sum.put(partial + piece * pitch, L);
    __syncwarp(L == 32 ? 0xFFFFFFFFu : ((1u << L) - 1u) << (threadIdx.x & 31 & ~(L - 1)));
    if (l == 0) {
      __threadfence();
      asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(a.flags + (int64_t)piece * a.slices + slice), "r"(a.raised)
                   : "memory");
    }
  };
  // the run this part starts and leaves open
  const uint32_t ko = open_key[1][part];
  if (ko != a.V) {
    Sum<kVec> sum;
    sum.set(open_tail + part * span + l, L);
    bool open = true;
    for (int q = part + 1; q < parts && open; ++q) {
      sum.add(open_head + q * span + l, L);
      open = through[q];
    }
    if (!open) lane.flush(a, ko, sum);
    else publish(sum);
  }
  // the run that was open before the piece
  const uint32_t kb = open_key[0][0];
  if (kb == a.V) return;
  int n_through = 0;
  while (n_through < parts && through[n_through]) ++n_through;
  if (part == 0) {
    own.set(open_head + l, L);
    for (int q = 1; q <= n_through && q < parts; ++q) own.add(open_head + q * span + l, L);
    if (n_through == parts) publish(own);
  }
  if (n_through == parts) return;
  // It ends here.  First piece: going back, pieces before which the list holds the same id.
  if (threadIdx.x < 32) {
    uint32_t first = piece - 1;
    for (int64_t q0 = first;; q0 -= 32) {
      const int64_t q = q0 - threadIdx.x;
      const bool same = q > 0 && __ldcg(&a.list[q * len - 1].x) == kb;
      const uint32_t m = __ballot_sync(0xFFFFFFFFu, same);
      const uint32_t run = m == 0xFFFFFFFFu ? 32u : (uint32_t)__ffs(~m) - 1u;
      first -= run;
      if (run < 32u) break;
    }
    if (threadIdx.x == 0) s_first = first;
  }
  __syncthreads();
  const uint32_t first = s_first;
  bool ok = true;
  for (uint32_t q = first + threadIdx.x; q < piece; q += kRedThreads) {
    uint32_t seen = 0;
    for (uint32_t i = 0; i < a.polls && !seen; ++i)
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];"
                   : "=r"(seen)
                   : "l"(a.flags + (int64_t)q * a.slices + slice)
                   : "memory");
    ok = ok && seen;
  }
  if (!__syncthreads_and(ok)) {
    if (!ok) atomicOr(a.status, ANC_DEV_TIMEOUT_DEP);
    return;
  }
  // group i adds the sums of every parts-th piece from the i-th, group 0 then the groups' sums
  acc.clear();
  for (uint32_t q = first + part; q < piece; q += parts) {
    float t[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) t[k] = __ldcg(partial + q * pitch + k * L);
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) acc.add_pair(i, t[2 * i], t[2 * i + 1]);
  }
  acc.put(open_tail + part * span + l, L);
  __syncthreads();
  if (part != 0) return;
  for (int w = 1; w < parts && (uint32_t)w < piece - first; ++w) acc.add(open_tail + w * span + l, L);
#pragma unroll
  for (int i = 0; i < kEach / 2; ++i) acc.add_pair(i, own.get(2 * i), own.get(2 * i + 1));
  lane.flush(a, kb, acc);
}

// ------------------------------------------------------------------ few tokens
// Up to kSmallT tokens need no sort: every CTA links the equal ids of the list in shared memory, and
// the group of lanes of each id's first token adds the rows along the links.  One launch.
constexpr int kSmallT = 128;

template <bool kDyF32, bool kDwF32, bool kVec, bool kAdd>
__global__ void __launch_bounds__(kRedThreads)
embedding_small_kernel(RedArgs a, const void *__restrict__ ids, int ids64, int64_t padding_idx, uint32_t *status) {
  __shared__ uint32_t key[kSmallT];
  __shared__ int16_t link[kSmallT];            // next token with the same id, -1: none
  __shared__ uint8_t head[kSmallT];
  constexpr int kBatch = 4;
  const int T = (int)a.T;
  if ((int)threadIdx.x < T) {
    const int64_t id = load_id(ids, ids64, threadIdx.x);
    key[threadIdx.x] = key_of(id, a.V, padding_idx);
    if (id >= (int64_t)a.V && blockIdx.x == 0) atomicOr(status, ANC_DEV_BAD_INDEX);
  }
  __syncthreads();
  if ((int)threadIdx.x < T) {
    const uint32_t k = key[threadIdx.x];
    int next = -1;
    bool first = k < a.V;
    for (int t = T - 1; t >= 0; --t) {
      const bool same = key[t] == k;
      if (same && t > (int)threadIdx.x) next = t;
      if (same && t < (int)threadIdx.x) first = false;
    }
    link[threadIdx.x] = (int16_t)next;
    head[threadIdx.x] = first;
  }
  __syncthreads();
  pdl_wait();      // the zeros of the table, when the whole table is written
  const int L = a.L, l = threadIdx.x & (L - 1);
  const int64_t u = (int64_t)blockIdx.x * (kRedThreads / L) + threadIdx.x / L;
  const int64_t t0 = u / a.slices;
  if (t0 >= T || !head[t0]) return;
  const Lane<kDyF32, kDwF32, kVec, kAdd, false> lane(a, (int)(u - t0 * a.slices), l);
  Row<kDwF32, kVec> old = {};
  old.load(lane.dw_row(a, key[t0]), lane.cols, L, kAdd);
  Sum<kVec> acc;
  acc.clear();
  for (int t = (int)t0; t >= 0;) {
    Row<kDyF32, kVec> x[kBatch] = {};
    int m = 0;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      x[b].load(lane.dy_row(a, t < 0 ? 0 : t), lane.cols, L, t >= 0);
      if (t >= 0) {
        t = link[t];
        m = b + 1;
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (b < m) x[b].add_to(acc);
  }
  lane.finish(a, key[t0], acc, old);
}

// ------------------------------------------------------------------ host side
// Lanes per row at least, however short the rows: fewer lanes are more and shorter parts, and joining the runs of a
// block goes from part to part (rows of 8 f32: 3085 tokens 15.6 us against 26.9 with one lane a row, 131072 43
// against 64; rows of 56: 41 against 43, with 16 lanes 46).
constexpr int kMinLanes = 8;
// Adding, the blocks of the sums that are resident while the list is made read dy into L2, where dy is no more than
// three quarters of it (rows of 1024 bf16 added to f32: 16384 tokens 32.3 us against 35.0, 32768 46.8 against 48.9, of
// bf16 48000 50.0 against 53.1; above it goes either way: 117 MB -2 and +2 us, 134 MB -3 and +5).
constexpr int64_t kAheadMost = 94 << 20;
constexpr int kMinPart = 4;                  // places per part at least
constexpr int64_t kResident = 296;           // blocks of the sums that are resident at once, two per SM
constexpr int kSortTarget = 4;               // rounds of 32 keys per warp the sort aims at
constexpr int64_t kZeroBytes = 128 << 10;    // zeros per block at most
constexpr int64_t kZeroParts = 592;          // blocks a small table's zeros are spread over (0.5 MB: 13 us, in four blocks 17)
constexpr int64_t kRankZeroBytes = 32 << 20; // zeros the counting kernel writes itself; more hide a sort beside them
struct Shape {
  int L, slices, per_part, span;      // span: columns of a slice
  int64_t pieces, max_pieces;
};

Shape shape_of(int64_t T, int64_t D, bool vec) {
  const int each = vec ? Cols<true>::kEach : Cols<false>::kEach;
  Shape s;
  s.L = kMinLanes;
  while (s.L < 32 && s.L * each < D) s.L *= 2;
  s.span = s.L * each;
  s.slices = (int)((D + s.span - 1) / s.span);
  // As many places per part as fill the GPU's resident blocks evenly, in as few waves as the list of a piece
  // allows: a block has a start and an end without rows in flight (accumulating 65536 rows of 1024,
  // sort included: 293 blocks 72.7 us, 1024 blocks 81 us).
  const int64_t parts_per_cta = kRedThreads / s.L, longest = kMaxPiece / parts_per_cta;
  const int64_t wave = std::max<int64_t>(1, kResident / s.slices);
  const int64_t waves = (T + wave * kMaxPiece - 1) / (wave * kMaxPiece);
  int64_t places = waves > 0 ? (T + waves * wave * parts_per_cta - 1) / (waves * wave * parts_per_cta) : 1;
  const int64_t least = std::min<int64_t>(longest, kMinPart);
  s.per_part = (int)std::max(least, std::min(longest, places));
  s.pieces = (T + parts_per_cta * s.per_part - 1) / (parts_per_cta * s.per_part);
  // at least the pieces of any smaller T, so that the workspace for T serves every smaller one
  s.max_pieces = std::max((waves + 1) * wave, s.pieces);
  return s;
}

struct Workspace {
  size_t list[2], clear, partial, total;
  uint32_t n_flags;                // words at `clear`
};

Workspace workspace_of(int64_t T, int64_t D) {
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  size_t flags = 0, partial = 0;       // whether rows are vectors is not known yet
  for (bool vec : {false, true}) {
    const Shape s = shape_of(T, D, vec);
    flags = std::max(flags, (size_t)s.max_pieces * s.slices);
    partial = std::max(partial, (size_t)s.max_pieces * s.slices * s.span * sizeof(float));
  }
  Workspace w;
  size_t at = 0;
  for (int i = 0; i < 2; ++i) {
    w.list[i] = at;
    at += up((size_t)T * sizeof(uint2));
  }
  w.n_flags = (uint32_t)flags;
  w.clear = at;
  at += up((size_t)w.n_flags * 4);
  w.partial = at;
  at += up(partial);
  w.total = at ? at : 256;
  return w;
}

constexpr int64_t kMaxLd = 1 << 29;          // row strides in bytes stay below 2^32
constexpr int64_t kMaxT = 0x7FFFFFFF - 1024, kMaxV = 0x7FFFFFFE, kMaxD = 1 << 24;

int check_sizes(int64_t T, int64_t V, int64_t D) {
  ANC_REQUIRE(T >= 0 && T <= kMaxT, "token count %lld out of range", (long long)T);
  ANC_REQUIRE(V >= 1 && V <= kMaxV, "table of %lld rows out of range", (long long)V);
  ANC_REQUIRE(D >= 1 && D <= kMaxD, "row length %lld out of range", (long long)D);
  return ANC_OK;
}

int check_dtype(int d, const char *what) {
  ANC_REQUIRE(d == ANC_GRAD_BF16 || d == ANC_GRAD_F32, "bad %s %d", what, d);
  return ANC_OK;
}

// Largest cluster the sort can use on a device (0: an error is set), and the kernels' shared-memory limits;
// once per device.
uint32_t sort_cluster(int device) {
  static std::mutex mu;
  static uint32_t most[64] = {};
  std::lock_guard<std::mutex> lock(mu);
  if (device >= 0 && device < 64 && most[device]) return most[device];
  cudaError_t e = cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortShared));
#define ANC_REDUCE_SMEM(Y, W, ADD)                                                                         \
  for (auto k : {embedding_reduce_kernel<Y, W, true, ADD, false>, embedding_reduce_kernel<Y, W, true, ADD, true>}) \
    if (e == cudaSuccess)                                                                                  \
      e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Stage<Y, W, true, ADD>::kBytes)
  ANC_REDUCE_SMEM(false, false, false);
  ANC_REDUCE_SMEM(false, false, true);
  ANC_REDUCE_SMEM(false, true, false);
  ANC_REDUCE_SMEM(false, true, true);
  ANC_REDUCE_SMEM(true, false, false);
  ANC_REDUCE_SMEM(true, false, true);
  ANC_REDUCE_SMEM(true, true, false);
  ANC_REDUCE_SMEM(true, true, true);
#undef ANC_REDUCE_SMEM
  uint32_t found = 8;                // the portable size
  for (uint32_t c = kMaxCluster; e == cudaSuccess && c > 8; c /= 2) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = sizeof(SortShared);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = c;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, embedding_sort_kernel, &cfg) == cudaSuccess && n > 0) {
      found = c;
      break;
    }
    cudaGetLastError();
  }
  if (e != cudaSuccess) {
    anc_cuda_fail(e, "embedding kernel attributes");
    return 0;
  }
  if (device >= 0 && device < 64) most[device] = found;
  return found;
}

// bytes from the first to the last element of an array of rows
int64_t row_span(int64_t rows, int64_t ld, int bytes, int64_t D) { return ((rows - 1) * ld + D) * bytes; }

// whether an array of rows and `n` bytes at b share a byte
bool overlap(const void *a, int64_t rows, int64_t ld, int bytes, int64_t D, const void *b, int64_t n) {
  const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  return a0 < b0 + (uintptr_t)n && b0 < a0 + (uintptr_t)row_span(rows, ld, bytes, D);
}

bool rows_are_vectors(const void *p, int64_t ld, int f32, int64_t D) {
  const int64_t align = f32 ? 32 : 16;       // of eight elements
  return (uintptr_t)p % align == 0 && D % 8 == 0 && ld % 8 == 0;
}

// anc_embedding_grad; raised, polls: of the wait between blocks (RedArgs)
int grad_impl(anc_ctx *ctx, const void *dy, int dy_dtype, int64_t dy_ld, const void *ids, int ids_dtype, void *dw,
              int dw_dtype, int64_t dw_ld, int64_t T, int64_t V, int64_t D, float scale, int mode, int64_t padding_idx,
              void *work, uint64_t work_bytes, void *stream, uint32_t raised, uint32_t polls) {
  ANC_REQUIRE(ctx && dw, "NULL argument");
  int rc = check_sizes(T, V, D);
  if (!rc) rc = check_dtype(dy_dtype, "dy_dtype");
  if (!rc) rc = check_dtype(dw_dtype, "dw_dtype");
  if (rc) return rc;
  ANC_REQUIRE(ids_dtype == ANC_IDS_I32 || ids_dtype == ANC_IDS_I64, "bad ids_dtype %d", ids_dtype);
  ANC_REQUIRE(isfinite(scale), "scale must be finite");
  ANC_REQUIRE(mode == ANC_EMBED_WRITE || mode == ANC_EMBED_ADD, "bad mode %d", mode);
  if (dy_ld == 0) dy_ld = D;
  if (dw_ld == 0) dw_ld = D;
  ANC_REQUIRE(dy_ld >= D && dw_ld >= D && dy_ld <= kMaxLd && dw_ld <= kMaxLd,
              "row strides must be at least the row length and at most 2^29");
  const int yf = dy_dtype == ANC_GRAD_F32, wf = dw_dtype == ANC_GRAD_F32, i64 = ids_dtype == ANC_IDS_I64;
  ANC_REQUIRE(((uintptr_t)dw & (wf ? 3 : 1)) == 0, "dw not aligned to its element size");
  if (T > 0) {
    ANC_REQUIRE(dy && ids && work, "NULL argument");
    ANC_REQUIRE(((uintptr_t)dy & (yf ? 3 : 1)) == 0 && ((uintptr_t)ids & (i64 ? 7 : 3)) == 0,
                "pointer not aligned to its element size");
    ANC_REQUIRE(((uintptr_t)work & 15) == 0, "workspace not aligned to 16 bytes");
    ANC_REQUIRE(!overlap(dw, V, dw_ld, wf ? 4 : 2, D, dy, row_span(T, dy_ld, yf ? 4 : 2, D)) &&
                    !overlap(dw, V, dw_ld, wf ? 4 : 2, D, ids, T * (i64 ? 8 : 4)) &&
                    !overlap(dw, V, dw_ld, wf ? 4 : 2, D, work, (int64_t)workspace_of(T, D).total) &&
                    !overlap(dy, T, dy_ld, yf ? 4 : 2, D, work, (int64_t)workspace_of(T, D).total) &&
                    !overlap(ids, 1, 0, i64 ? 8 : 4, T, work, (int64_t)workspace_of(T, D).total),
                "dw or the workspace overlaps another buffer");
  }
  const Workspace ws = workspace_of(T, D);
  ANC_REQUIRE(T == 0 || work_bytes >= ws.total, "workspace of %llu bytes, %llu are needed",
              (unsigned long long)work_bytes, (unsigned long long)ws.total);
  if (T == 0 && mode == ANC_EMBED_ADD) return ANC_OK;
  anc_device_guard guard(ctx->device);
  cudaStream_t st = anc_pick_stream(ctx, stream);
  ZeroArgs za = {};
  za.dw = (uint8_t *)dw;
  za.row_bytes = D * (wf ? 4 : 2);
  za.pitch = dw_ld * (wf ? 4 : 2);
  za.V = V;
  const int64_t zeros = V * za.row_bytes, even = (zeros + kZeroParts - 1) / kZeroParts;
  za.bytes = std::min(kZeroBytes, (even + 4095) / 4096 * 4096);
  za.rows = std::max<int64_t>(1, za.bytes / za.row_bytes);
  const int64_t parts = za.pitch == za.row_bytes ? (zeros + za.bytes - 1) / za.bytes : (V + za.rows - 1) / za.rows;
  ANC_REQUIRE(parts <= 0x7FFFFFFF, "V x D too large");
  za.parts = (uint32_t)parts;
  const bool write = mode == ANC_EMBED_WRITE, small = T <= kSmallT;
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  auto launch_zero = [&](int n_attrs) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(za.parts);
    cfg.blockDim = dim3(kZeroThreads);
    cfg.stream = st;
    cfg.attrs = pdl;
    cfg.numAttrs = n_attrs;
    return cudaLaunchKernelEx(&cfg, embedding_zero_kernel, za);
  };
  if (write && small) ANC_CUDA(launch_zero(0));
  if (T == 0) return ANC_OK;
  uint8_t *wp = (uint8_t *)work;
  const bool vec = rows_are_vectors(dy, dy_ld, yf, D) && rows_are_vectors(dw, dw_ld, wf, D);
  const Shape sh = shape_of(T, D, vec);
  RedArgs ra = {};
  ra.dy = (const uint8_t *)dy; ra.dw = (uint8_t *)dw; ra.T = T;
  ra.dy_pitch = (uint32_t)(dy_ld * (yf ? 4 : 2)); ra.dw_pitch = (uint32_t)(dw_ld * (wf ? 4 : 2));
  ra.partial = (float *)(wp + ws.partial);
  ra.V = (uint32_t)V; ra.D = (int)D; ra.slices = sh.slices; ra.L = sh.L; ra.per_part = sh.per_part; ra.scale = scale;
  ra.status = ctx->d_status;
  ra.raised = raised; ra.polls = polls;
  const int64_t blocks =
      small ? (T * sh.slices + kRedThreads / sh.L - 1) / (kRedThreads / sh.L) : sh.pieces * sh.slices;
  ANC_REQUIRE(blocks <= 0x7FFFFFFF, "T x D too large");
  int n_attrs = write ? 1 : 0;
  const int64_t dy_bytes = T * D * (yf ? 4 : 2), skip = (16 - ((uintptr_t)dy & 15)) & 15;
  if (dy_ld == D && dy_bytes <= kAheadMost && dy_bytes >= 32) {
    ra.ahead = (const uint8_t *)dy + skip;
    ra.ahead_bytes = (uint64_t)(dy_bytes - skip) / 16 * 16;
  }
  if (!small) {
    SortArgs sa = {};
    sa.ids = ids; sa.ids64 = i64; sa.T = (uint32_t)T; sa.V = V; sa.padding_idx = padding_idx;
    for (int i = 0; i < 2; ++i) sa.list[i] = (uint2 *)(wp + ws.list[i]);
    int bits = 0;
    while (((uint64_t)V >> bits) != 0) ++bits;
    sa.passes = (bits + kDigitBits - 1) / kDigitBits;
    sa.status = ctx->d_status;
    sa.clear = (uint32_t *)(wp + ws.clear);
    sa.n_clear = (uint32_t)blocks;
    ra.flags = sa.clear;
    const uint32_t most = sort_cluster(ctx->device);
    if (!most) return ANC_E_CUDA;
    if (T <= kRankT && (!write || V * za.row_bytes <= kRankZeroBytes)) {
      ra.list = sa.list[0];
      const int64_t per_cta = kRankThreads / 32 * kRankTokens, want = (T + per_cta - 1) / per_cta;
      const unsigned grid = (unsigned)(write || want > ctx->sm_count ? ctx->sm_count : want);
      if (!write) za.parts = 0;
      const size_t keys = (T + 127) / 128 * 128 * sizeof(uint32_t);
      embedding_rank_kernel<<<grid, kRankThreads, keys, st>>>(sa, za);
      ANC_CUDA(cudaGetLastError());
    } else {
      ra.list = sa.list[(sa.passes - 1) & 1];
      // one CTA as long as the list stays in its shared memory (4096 tokens: 10.3 us, two CTAs 12.4)
      uint32_t n_ctas = 1;
      while (T > kSortThreads * kSortRounds && n_ctas < most && (int64_t)n_ctas * kSortThreads * kSortTarget < T) n_ctas *= 2;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(n_ctas);
      cfg.blockDim = dim3(kSortThreads);
      cfg.dynamicSmemBytes = sizeof(SortShared);
      cfg.stream = st;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = n_ctas;
      at[0].val.clusterDim.y = 1;
      at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      ANC_CUDA(cudaLaunchKernelEx(&cfg, embedding_sort_kernel, sa, n_ctas));
      if (write) ANC_CUDA(launch_zero(1));
    }
    n_attrs = 1;
  }
  // these launches start while their predecessor drains and wait for it on the device
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kRedThreads);
  cfg.stream = st;
  cfg.attrs = pdl;
  cfg.numAttrs = n_attrs;
#define ANC_REDUCE_W(Y, W, VEC, ADD, WIDE)                                                           \
  do {                                                                                               \
    cfg.dynamicSmemBytes = Stage<Y, W, VEC, ADD>::kBytes;                                            \
    ANC_CUDA(cudaLaunchKernelEx(&cfg, embedding_reduce_kernel<Y, W, VEC, ADD, WIDE>, ra));           \
  } while (0)
#define ANC_REDUCE_A(Y, W, VEC, ADD)                                                                 \
  do {                                                                                               \
    if (small)                                                                                       \
      ANC_CUDA(cudaLaunchKernelEx(&cfg, embedding_small_kernel<Y, W, VEC, ADD>, ra, ids, i64, padding_idx, \
                                  ctx->d_status));                                                   \
    else if (VEC && sh.L == 32 && D % sh.span == 0)                                                  \
      ANC_REDUCE_W(Y, W, VEC, ADD, VEC);                                                             \
    else                                                                                             \
      ANC_REDUCE_W(Y, W, VEC, ADD, false);                                                           \
  } while (0)
#define ANC_REDUCE(Y, W, VEC)                    \
  do {                                           \
    if (write) ANC_REDUCE_A(Y, W, VEC, false);   \
    else ANC_REDUCE_A(Y, W, VEC, true);          \
  } while (0)
#define ANC_REDUCE_V(Y, W)                \
  do {                                    \
    if (vec) ANC_REDUCE(Y, W, true);      \
    else ANC_REDUCE(Y, W, false);         \
  } while (0)
  if (yf && wf) ANC_REDUCE_V(true, true);
  else if (yf) ANC_REDUCE_V(true, false);
  else if (wf) ANC_REDUCE_V(false, true);
  else ANC_REDUCE_V(false, false);
#undef ANC_REDUCE_V
#undef ANC_REDUCE
#undef ANC_REDUCE_A
#undef ANC_REDUCE_W
  ANC_CUDA(cudaGetLastError());
  return ANC_OK;
}

}  // namespace

extern "C" {

int anc_embedding_lookup(anc_ctx *ctx, const void *table, int table_dtype, int64_t table_ld, const void *ids,
                         int ids_dtype, void *out, int out_dtype, int64_t out_ld, int64_t T, int64_t V, int64_t D,
                         float scale, void *stream) {
  ANC_REQUIRE(ctx, "ctx is NULL");
  int rc = check_sizes(T, V, D);
  if (!rc) rc = check_dtype(table_dtype, "table_dtype");
  if (!rc) rc = check_dtype(out_dtype, "out_dtype");
  if (rc) return rc;
  ANC_REQUIRE(ids_dtype == ANC_IDS_I32 || ids_dtype == ANC_IDS_I64, "bad ids_dtype %d", ids_dtype);
  ANC_REQUIRE(isfinite(scale), "scale must be finite");
  if (T == 0) return ANC_OK;
  ANC_REQUIRE(table && ids && out, "NULL argument");
  if (table_ld == 0) table_ld = D;
  if (out_ld == 0) out_ld = D;
  ANC_REQUIRE(table_ld >= D && out_ld >= D && table_ld <= kMaxLd && out_ld <= kMaxLd,
              "row strides must be at least the row length and at most 2^29");
  const int tf = table_dtype == ANC_GRAD_F32, of = out_dtype == ANC_GRAD_F32, i64 = ids_dtype == ANC_IDS_I64;
  ANC_REQUIRE(((uintptr_t)table & (tf ? 3 : 1)) == 0 && ((uintptr_t)out & (of ? 3 : 1)) == 0 &&
                  ((uintptr_t)ids & (i64 ? 7 : 3)) == 0,
              "pointer not aligned to its element size");
  ANC_REQUIRE(!overlap(table, V, table_ld, tf ? 4 : 2, D, out, row_span(T, out_ld, of ? 4 : 2, D)) &&
                  !overlap(out, T, out_ld, of ? 4 : 2, D, ids, T * (i64 ? 8 : 4)),
              "the output overlaps an input");
  anc_device_guard guard(ctx->device);
  cudaStream_t st = anc_pick_stream(ctx, stream);
  const bool vec = rows_are_vectors(table, table_ld, tf, D) && rows_are_vectors(out, out_ld, of, D);
  LookupArgs a = {};
  a.table = (const uint8_t *)table; a.ids = ids; a.out = (uint8_t *)out;
  a.table_pitch = (uint32_t)(table_ld * (tf ? 4 : 2)); a.out_pitch = (uint32_t)(out_ld * (of ? 4 : 2));
  a.T = (uint32_t)T; a.V = (uint32_t)V; a.ids64 = i64; a.D = (int)D; a.scale = scale; a.status = ctx->d_status;
  a.L = 1;
  while (a.L < 32 && a.L * 8 < D) a.L *= 2;
  const int64_t per_lane = (D + 8 * a.L - 1) / (8 * a.L);        // octets of a row
  const int64_t slices = (per_lane + 3) / 4;
  const int octs = (int)((per_lane + slices - 1) / slices);
  ANC_REQUIRE(slices <= 65535, "row length %lld out of range", (long long)D);
  const int64_t rows = (int64_t)(32 / a.L) * (4 / octs);         // per unit
  a.units = (uint32_t)((T + rows - 1) / rows);
  const dim3 blocks((unsigned)((a.units + kLookupThreads / 32 - 1) / (kLookupThreads / 32)), (unsigned)slices);
#define ANC_LOOKUP(F, O, VEC, OCTS) \
  embedding_lookup_kernel<F, O, VEC, OCTS><<<blocks, kLookupThreads, 0, st>>>(a)
#define ANC_LOOKUP_O(F, O, VEC)                         \
  do {                                                  \
    if (octs == 4) ANC_LOOKUP(F, O, VEC, 4);            \
    else if (octs == 3) ANC_LOOKUP(F, O, VEC, 3);       \
    else if (octs == 2) ANC_LOOKUP(F, O, VEC, 2);       \
    else ANC_LOOKUP(F, O, VEC, 1);                      \
  } while (0)
#define ANC_LOOKUP_V(F, O)                              \
  do {                                                  \
    if (vec) ANC_LOOKUP_O(F, O, true);                  \
    else ANC_LOOKUP_O(F, O, false);                     \
  } while (0)
  if (tf && of) ANC_LOOKUP_V(true, true);
  else if (tf) ANC_LOOKUP_V(true, false);
  else if (of) ANC_LOOKUP_V(false, true);
  else ANC_LOOKUP_V(false, false);
#undef ANC_LOOKUP_V
#undef ANC_LOOKUP_O
#undef ANC_LOOKUP
  ANC_CUDA(cudaGetLastError());
  return ANC_OK;
}

int anc_embedding_grad_workspace(int64_t T, int64_t V, int64_t D, uint64_t *bytes) {
  ANC_REQUIRE(bytes, "bytes is NULL");
  int rc = check_sizes(T, V, D);
  if (rc) return rc;
  *bytes = workspace_of(T, D).total;
  return ANC_OK;
}

int anc_embedding_grad(anc_ctx *ctx, const void *dy, int dy_dtype, int64_t dy_ld, const void *ids, int ids_dtype,
                       void *dw, int dw_dtype, int64_t dw_ld, int64_t T, int64_t V, int64_t D, float scale, int mode,
                       int64_t padding_idx, void *work, uint64_t work_bytes, void *stream) {
  return grad_impl(ctx, dy, dy_dtype, dy_ld, ids, ids_dtype, dw, dw_dtype, dw_ld, T, V, D, scale, mode, padding_idx, work,
                   work_bytes, stream, 1u, kWaitPolls);
}

int anc_embedding_wait_selftest(anc_ctx *ctx, const float *dy, const int64_t *ids, float *dw, int64_t T, int64_t V,
                                int64_t D, void *work, uint64_t work_bytes, uint32_t polls, void *stream) {
  ANC_REQUIRE(polls > 0 && polls <= (1u << 14), "polls %u outside 1..2^14", polls);
  return grad_impl(ctx, dy, ANC_GRAD_F32, 0, ids, ANC_IDS_I64, dw, ANC_GRAD_F32, 0, T, V, D, 1.f, ANC_EMBED_ADD, -1, work,
                   work_bytes, stream, 0u, polls);
}

}  // extern "C"
