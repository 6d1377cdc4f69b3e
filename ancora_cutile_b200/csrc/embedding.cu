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
#include <cuda_bf16.h>
#include "anc_internal.h"
#include "philox.cuh"

namespace {

// ------------------------------------------------------------------ rows in registers
// A warp holds a slice of kSliceCols columns of a row, eight per lane: eight neighbouring ones where rows
// are 16-byte aligned vectors of eight (kVec), else every 32nd.
constexpr int kSliceCols = 256;

template <bool kVec>
__device__ __forceinline__ int col_of(int c0, int lane, int k) {
  return kVec ? c0 + lane * 8 + k : c0 + k * 32 + lane;
}

template <bool kF32, bool kVec>
__device__ __forceinline__ void load8(const void *row, int c0, int lane, int D, float x[8]) {
  if constexpr (kVec) {
    const int c = c0 + lane * 8;
    if (c >= D) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = 0.f;
    } else if constexpr (kF32) {
      const float4 a = *reinterpret_cast<const float4 *>((const float *)row + c);
      const float4 b = *reinterpret_cast<const float4 *>((const float *)row + c + 4);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
      const uint4 r = *reinterpret_cast<const uint4 *>((const uint16_t *)row + c);
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = __uint_as_float(w[k] << 16);
        x[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = c0 + k * 32 + lane;
      x[k] = 0.f;
      if (c < D) {
        if constexpr (kF32) x[k] = ((const float *)row)[c];
        else x[k] = __uint_as_float((uint32_t)((const uint16_t *)row)[c] << 16);
      }
    }
  }
}

template <bool kF32, bool kVec>
__device__ __forceinline__ void store8(void *row, int c0, int lane, int D, const float x[8]) {
  if constexpr (kVec) {
    const int c = c0 + lane * 8;
    if (c >= D) return;
    if constexpr (kF32) {
      float4 *d = reinterpret_cast<float4 *>((float *)row + c);
      d[0] = make_float4(x[0], x[1], x[2], x[3]);
      d[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      uint32_t h[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) h[k] = bf16_rne(x[k]);
      *reinterpret_cast<uint4 *>((uint16_t *)row + c) =
          make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = c0 + k * 32 + lane;
      if (c < D) {
        if constexpr (kF32) ((float *)row)[c] = x[k];
        else ((uint16_t *)row)[c] = (uint16_t)bf16_rne(x[k]);
      }
    }
  }
}

__device__ __forceinline__ int64_t load_id(const void *ids, int ids64, int64_t t) {
  return ids64 ? ((const int64_t *)ids)[t] : (int64_t)((const int32_t *)ids)[t];
}

template <bool kF32>
__device__ __forceinline__ const void *row_ptr(const void *base, int64_t row, int64_t ld) {
  return (const uint8_t *)base + row * ld * (kF32 ? 4 : 2);
}
template <bool kF32>
__device__ __forceinline__ void *row_ptr(void *base, int64_t row, int64_t ld) {
  return (uint8_t *)base + row * ld * (kF32 ? 4 : 2);
}

// ------------------------------------------------------------------ lookup
constexpr int kLookupWarps = 8;

// One warp per (token, slice of kSliceCols columns).
template <bool kTabF32, bool kOutF32, bool kVec>
__global__ void __launch_bounds__(kLookupWarps * 32)
embedding_lookup_kernel(const void *__restrict__ table, int64_t table_ld, const void *__restrict__ ids, int ids64,
                        void *__restrict__ out, int64_t out_ld, int64_t T, int64_t V, int D, int slices, float scale,
                        uint32_t *status) {
  const int lane = threadIdx.x & 31;
  const int64_t units = T * slices;
  for (int64_t u = (int64_t)blockIdx.x * kLookupWarps + (threadIdx.x >> 5); u < units;
       u += (int64_t)gridDim.x * kLookupWarps) {
    const int64_t t = u / slices;
    const int c0 = (int)(u - t * slices) * kSliceCols;
    const int64_t id = load_id(ids, ids64, t);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (id >= 0 && id < V) {
      load8<kTabF32, kVec>(row_ptr<kTabF32>(table, id, table_ld), c0, lane, D, x);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = __fmul_rn(x[k], scale);
    } else if (id >= V && lane == 0) {
      atomicOr(status, ANC_DEV_BAD_INDEX);
    }
    store8<kOutF32, kVec>(row_ptr<kOutF32>(out, t, out_ld), c0, lane, D, x);
  }
}

// ------------------------------------------------------------------ sort
// Stable least-significant-digit radix sort of (id, token) by one cluster of CTAs, nine bits a pass: two
// passes for tables of up to 2^18 rows.  Per pass every warp counts the digits of its stretch of the list,
// the cluster exchanges its CTAs' digit counts through distributed shared memory, and every warp then
// writes its stretch in order to the places the counts give.  Padding sorts behind the last row of
// the table as id V.
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr size_t kSortSmem = (size_t)(kSortWarps * kDigits + 2 * kDigits + 64) * 4;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

struct SortArgs {
  const void *ids;
  int ids64;
  int64_t T, V, padding_idx;
  uint32_t *key[2], *pos[2];
  int passes;
  uint32_t *status;
};

__device__ __forceinline__ uint32_t key_of(const SortArgs &a, int64_t t, bool report) {
  const int64_t id = load_id(a.ids, a.ids64, t);
  if (id >= a.V && report) atomicOr(a.status, ANC_DEV_BAD_INDEX);
  return (id < 0 || id >= a.V || id == a.padding_idx) ? (uint32_t)a.V : (uint32_t)id;
}

__global__ void __launch_bounds__(kSortThreads, 1)
embedding_sort_kernel(SortArgs a, uint32_t n_ctas) {
  extern __shared__ uint32_t sm[];
  uint32_t *cnt = sm;                                // [warp][digit]
  uint32_t *tot = sm + kSortWarps * kDigits;         // this CTA's digit counts, read by the whole cluster
  uint32_t *off = tot + kDigits;                     // first place of a digit's keys of this CTA
  uint32_t *wsum = off + kDigits;
  const uint32_t rank = cluster_rank();
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // stretches: whole rounds of 32 keys per warp
  const int64_t per = ((a.T + (int64_t)n_ctas * kSortThreads - 1) / ((int64_t)n_ctas * kSortThreads)) * 32;
  const int64_t lo = ((int64_t)rank * kSortWarps + warp) * per;
  const int64_t hi = lo + per < a.T ? lo + per : a.T;
  for (int p = 0; p < a.passes; ++p) {
    const bool odd = p & 1;
    const uint32_t *ik = odd ? a.key[0] : a.key[1], *ip = odd ? a.pos[0] : a.pos[1];
    uint32_t *ok = odd ? a.key[1] : a.key[0], *op = odd ? a.pos[1] : a.pos[0];
    const int shift = p * kDigitBits;
    for (uint32_t d = tid; d < kSortWarps * kDigits; d += kSortThreads) cnt[d] = 0u;
    __syncthreads();
    for (int64_t i = lo + lane; i < hi; i += 32) {
      const uint32_t key = p == 0 ? key_of(a, i, true) : __ldcg(ik + i);
      atomicAdd(&cnt[warp * kDigits + ((key >> shift) & (kDigits - 1))], 1u);
    }
    __syncthreads();
    if (tid < kDigits) {
      uint32_t run = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = cnt[w * kDigits + tid];
        cnt[w * kDigits + tid] = run;
        run += c;
      }
      tot[tid] = run;
    }
    cluster_sync();
    uint32_t before = 0, all = 0;
    if (tid < kDigits) {
      const uint32_t mine = (uint32_t)__cvta_generic_to_shared(tot + tid);
      for (uint32_t c = 0; c < n_ctas; ++c) {
        const uint32_t v = ld_cluster(peer_smem(mine, c));
        if (c < rank) before += v;
        all += v;
      }
      // exclusive scan of the digit totals
      uint32_t s = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, s, o);
        if (lane >= (uint32_t)o) s += v;
      }
      if (lane == 31) wsum[warp] = s;
      off[tid] = s - all + before;
    }
    __syncthreads();
    if (tid < kDigits) {
      uint32_t base = 0;
      for (uint32_t w = 0; w < warp; ++w) base += wsum[w];
      off[tid] += base;
    }
    __syncthreads();
    for (int64_t i0 = lo; i0 < hi; i0 += 32) {
      const int64_t i = i0 + lane;
      const bool on = i < hi;
      const uint32_t active = __ballot_sync(0xFFFFFFFFu, on);
      if (on) {
        const uint32_t key = p == 0 ? key_of(a, i, false) : __ldcg(ik + i);
        const uint32_t pos = p == 0 ? (uint32_t)i : __ldcg(ip + i);
        const uint32_t d = (key >> shift) & (kDigits - 1);
        const uint32_t peers = __match_any_sync(active, d);
        const uint32_t at = cnt[warp * kDigits + d];
        __syncwarp(active);
        if (lane == (uint32_t)(__ffs(peers) - 1)) cnt[warp * kDigits + d] = at + __popc(peers);
        __syncwarp(active);
        const uint32_t dst = off[d] + at + __popc(peers & ((1u << lane) - 1u));
        ok[dst] = key;
        op[dst] = pos;
      }
    }
    __syncwarp();
    cluster_sync();     // the next pass reads what other CTAs wrote, and overwrites tot
  }
}

__global__ void __launch_bounds__(256)
embedding_zero_kernel(uint8_t *dw, int64_t row_bytes, int64_t pitch, int64_t V, int vec) {
  const int64_t stride = (int64_t)gridDim.x * 256, i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (vec) {
    const int64_t n = row_bytes / 16, total = n * V;
    for (int64_t i = i0; i < total; i += stride)
      *reinterpret_cast<uint4 *>(dw + (pitch == row_bytes ? i * 16 : (i / n) * pitch + (i % n) * 16)) =
          make_uint4(0u, 0u, 0u, 0u);
  } else {
    const int64_t n = row_bytes / 2, total = n * V;
    for (int64_t i = i0; i < total; i += stride)
      *reinterpret_cast<uint16_t *>(dw + (i / n) * pitch + (i % n) * 2) = 0;
  }
}

// ------------------------------------------------------------------ sums of runs
constexpr int kRedWarps = 8;

struct RedArgs {
  const void *dy;
  void *dw;
  int64_t dy_ld, dw_ld, T;
  const uint32_t *key, *pos;     // sorted
  float *partial;                // [piece][open at its start, open at its end][slices * 256], register layout
  uint32_t V;
  int D, slices;
  int per_warp;                  // sorted places per warp, at most 32
  float scale;
  int add;
};

template <bool kDwF32, bool kVec>
__device__ __forceinline__ void flush_row(const RedArgs &a, uint32_t v, int c0, int lane, const float acc[8]) {
  void *row = row_ptr<kDwF32>(a.dw, v, a.dw_ld);
  float x[8];
  if (a.add) {
    load8<kDwF32, kVec>(row, c0, lane, a.D, x);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __fadd_rn(x[k], __fmul_rn(a.scale, acc[k]));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __fmul_rn(a.scale, acc[k]);
  }
  store8<kDwF32, kVec>(row, c0, lane, a.D, x);
}

// A CTA takes one piece of kRedWarps * per_warp sorted places and one slice of columns; its warps take
// equal parts.  A run inside a warp's part goes straight to the table.  The sums of runs that are open at
// a part's start or end are left in shared memory and joined in order; what is still open at the
// piece's start or end goes to `partial`.
template <bool kDyF32, bool kDwF32, bool kVec>
__global__ void __launch_bounds__(kRedWarps * 32)
embedding_reduce_kernel(RedArgs a) {
  __shared__ float open_sum[kRedWarps][2][kSliceCols];
  __shared__ uint32_t open_key[kRedWarps][2];      // V: nothing open
  __shared__ uint32_t through[kRedWarps];          // the part is one run, open at both ends (slot 0)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t piece = blockIdx.x / a.slices;
  const int slice = (int)(blockIdx.x - piece * a.slices), c0 = slice * kSliceCols;
  const int64_t p0 = piece * (kRedWarps * (int64_t)a.per_warp), w0 = p0 + (int64_t)warp * a.per_warp;
  const int n = (int)(a.T - w0 < a.per_warp ? (a.T - w0 > 0 ? a.T - w0 : 0) : a.per_warp);
  uint32_t key = a.V, pos = 0, prev = a.V, next = a.V;
  if (lane < n) {
    key = __ldg(a.key + w0 + lane);
    pos = __ldg(a.pos + w0 + lane);
  }
  if (n > 0) {
    if (w0 > 0) prev = __ldg(a.key + w0 - 1);
    if (w0 + n < a.T) next = __ldg(a.key + w0 + n);
  }
  if (lane < 2) open_key[warp][lane] = a.V;
  if (lane == 0) through[warp] = 0u;
  __syncwarp();
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  bool from_before = n > 0 && __shfl_sync(0xFFFFFFFFu, key, 0) == prev;
  constexpr int kBatch = 4;
  for (int j0 = 0; j0 < n; j0 += kBatch) {
    float x[kBatch][8];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int j = j0 + b;
      const uint32_t k = __shfl_sync(0xFFFFFFFFu, key, j & 31), t = __shfl_sync(0xFFFFFFFFu, pos, j & 31);
      if (j < n && k < a.V) load8<kDyF32, kVec>(row_ptr<kDyF32>(a.dy, t, a.dy_ld), c0, lane, a.D, x[b]);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int j = j0 + b;
      const uint32_t k = __shfl_sync(0xFFFFFFFFu, key, j & 31);
      const uint32_t kn = j + 1 < n ? __shfl_sync(0xFFFFFFFFu, key, (j + 1) & 31) : next;
      if (j >= n || k >= a.V) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = __fadd_rn(acc[e], x[b][e]);
      if (j + 1 < n && kn == k) continue;
      const bool goes_on = j + 1 >= n && kn == k;
      if (!from_before && !goes_on) {
        flush_row<kDwF32, kVec>(a, k, c0, lane, acc);
      } else {
        const int s = from_before ? 0 : 1;
#pragma unroll
        for (int e = 0; e < 8; ++e) open_sum[warp][s][e * 32 + lane] = acc[e];
        if (lane == 0) {
          open_key[warp][s] = k;
          if (from_before && goes_on) through[warp] = 1u;
        }
      }
      from_before = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    }
  }
  __syncthreads();
  // Join the parts in order; warp 0, each lane its eight columns of every part.
  if (warp != 0) return;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  bool have = false, started_before = false;
  float *part = a.partial + (piece * 2 * a.slices + slice) * (int64_t)kSliceCols;
  const int64_t slot = (int64_t)a.slices * kSliceCols;
  for (int w = 0; w < kRedWarps; ++w) {
    const uint32_t k0 = open_key[w][0];
    if (k0 != a.V) {
      if (!have) started_before = true;       // only the piece's first part can continue an unseen run
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = have ? __fadd_rn(sum[e], open_sum[w][0][e * 32 + lane]) : open_sum[w][0][e * 32 + lane];
      have = true;
      if (!through[w]) {
        if (started_before) {
#pragma unroll
          for (int e = 0; e < 8; ++e) part[e * 32 + lane] = sum[e];
        } else {
          flush_row<kDwF32, kVec>(a, k0, c0, lane, sum);
        }
        have = started_before = false;
      }
    }
    if (open_key[w][1] != a.V) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = open_sum[w][1][e * 32 + lane];
      have = true;
    }
  }
  if (have) {
    float *p = part + (started_before ? 0 : slot);
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e * 32 + lane] = sum[e];
  }
}

// Runs that cross pieces.  A CTA takes one piece and one slice; if a run starts in the piece and is still
// open at its end, its warps add the partial sums of the pieces it covers, each warp a stretch, and the
// stretches are added in order.
template <bool kDwF32, bool kVec>
__global__ void __launch_bounds__(kRedWarps * 32)
embedding_join_kernel(RedArgs a, int64_t pieces) {
  __shared__ float sums[kRedWarps][kSliceCols];
  __shared__ int64_t s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t piece = blockIdx.x / a.slices;
  const int slice = (int)(blockIdx.x - piece * a.slices), c0 = slice * kSliceCols;
  const int64_t len = kRedWarps * (int64_t)a.per_warp, p0 = piece * len, p1 = p0 + len;
  if (p1 >= a.T) return;
  const uint32_t k = __ldg(a.key + p1 - 1);
  if (k >= a.V || __ldg(a.key + p1) != k) return;
  if (p0 > 0 && __ldg(a.key + p0 - 1) == k) return;        // the run starts in an earlier piece
  if (warp == 0) {      // last piece of the run: pieces start with k up to there
    int64_t last = piece;
    for (int64_t q0 = piece + 1; q0 < pieces; q0 += 32) {
      const bool same = q0 + lane < pieces && __ldg(a.key + (q0 + lane) * len) == k;
      const uint32_t m = __ballot_sync(0xFFFFFFFFu, same);
      last += __popc(m);
      if (m != 0xFFFFFFFFu) break;
    }
    if (lane == 0) s_last = last;
  }
  __syncthreads();
  const int64_t last = s_last, count = last - piece;      // pieces piece + 1 .. last
  const int64_t slot = (int64_t)a.slices * kSliceCols;
  const float *base = a.partial + (int64_t)slice * kSliceCols + lane;
  const int64_t q0 = piece + 1 + count * warp / kRedWarps, q1 = piece + 1 + count * (warp + 1) / kRedWarps;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int64_t q = q0; q < q1; ++q) {
    const float *p = base + q * 2 * slot;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = __fadd_rn(acc[e], p[e * 32]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[warp][e * 32 + lane] = acc[e];
  __syncthreads();
  if (warp != 0) return;
  const float *first = base + (piece * 2 + 1) * slot;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    acc[e] = first[e * 32];
    for (int w = 0; w < kRedWarps; ++w) acc[e] = __fadd_rn(acc[e], sums[w][e * 32 + lane]);
  }
  flush_row<kDwF32, kVec>(a, k, c0, lane, acc);
}

// ------------------------------------------------------------------ host side
struct Shape {
  int slices, per_warp;
  int64_t pieces;
};

Shape shape_of(int64_t T, int64_t D) {
  Shape s;
  s.slices = (int)((D + kSliceCols - 1) / kSliceCols);
  s.per_warp = 32;
  s.pieces = (T + kRedWarps * s.per_warp - 1) / (kRedWarps * s.per_warp);
  return s;
}

struct Workspace {
  size_t key[2], pos[2], partial, total;
};

Workspace workspace_of(int64_t T, int64_t D) {
  const Shape s = shape_of(T, D);
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  Workspace w;
  size_t at = 0;
  for (int i = 0; i < 2; ++i) {
    w.key[i] = at;
    at += up((size_t)T * 4);
    w.pos[i] = at;
    at += up((size_t)T * 4);
  }
  w.partial = at;
  at += up((size_t)s.pieces * 2 * s.slices * kSliceCols * 4);
  w.total = at ? at : 256;
  return w;
}

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

bool rows_are_vectors(const void *p, int64_t ld, int f32, int64_t D) {
  return ((uintptr_t)p & 15) == 0 && D % 8 == 0 && (ld * (f32 ? 4 : 2)) % 16 == 0;
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
  if (T == 0) return ANC_OK;
  ANC_REQUIRE(table && ids && out, "NULL argument");
  if (table_ld == 0) table_ld = D;
  if (out_ld == 0) out_ld = D;
  ANC_REQUIRE(table_ld >= D && out_ld >= D, "row strides must be at least the row length");
  const int tf = table_dtype == ANC_GRAD_F32, of = out_dtype == ANC_GRAD_F32, i64 = ids_dtype == ANC_IDS_I64;
  ANC_REQUIRE(((uintptr_t)table & (tf ? 3 : 1)) == 0 && ((uintptr_t)out & (of ? 3 : 1)) == 0 &&
                  ((uintptr_t)ids & (i64 ? 7 : 3)) == 0,
              "pointer not aligned to its element size");
  anc_device_guard guard(ctx->device);
  cudaStream_t st = anc_pick_stream(ctx, stream);
  const int slices = (int)((D + kSliceCols - 1) / kSliceCols);
  int64_t blocks = (T * slices + kLookupWarps - 1) / kLookupWarps;
  const int64_t cap = (int64_t)ctx->sm_count * 64;
  if (blocks > cap) blocks = cap;
  const bool vec = rows_are_vectors(table, table_ld, tf, D) && rows_are_vectors(out, out_ld, of, D);
#define ANC_LOOKUP(F, O, VEC)                                                                             \
  embedding_lookup_kernel<F, O, VEC><<<(unsigned)blocks, kLookupWarps * 32, 0, st>>>(                     \
      table, table_ld, ids, i64, out, out_ld, T, V, (int)D, slices, scale, ctx->d_status)
#define ANC_LOOKUP_V(F, O)                \
  do {                                    \
    if (vec) ANC_LOOKUP(F, O, true);      \
    else ANC_LOOKUP(F, O, false);         \
  } while (0)
  if (tf && of) ANC_LOOKUP_V(true, true);
  else if (tf) ANC_LOOKUP_V(true, false);
  else if (of) ANC_LOOKUP_V(false, true);
  else ANC_LOOKUP_V(false, false);
#undef ANC_LOOKUP_V
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
  ANC_REQUIRE(ctx && dw, "NULL argument");
  int rc = check_sizes(T, V, D);
  if (!rc) rc = check_dtype(dy_dtype, "dy_dtype");
  if (!rc) rc = check_dtype(dw_dtype, "dw_dtype");
  if (rc) return rc;
  ANC_REQUIRE(ids_dtype == ANC_IDS_I32 || ids_dtype == ANC_IDS_I64, "bad ids_dtype %d", ids_dtype);
  ANC_REQUIRE(mode == ANC_EMBED_WRITE || mode == ANC_EMBED_ADD, "bad mode %d", mode);
  if (dy_ld == 0) dy_ld = D;
  if (dw_ld == 0) dw_ld = D;
  ANC_REQUIRE(dy_ld >= D && dw_ld >= D, "row strides must be at least the row length");
  const int yf = dy_dtype == ANC_GRAD_F32, wf = dw_dtype == ANC_GRAD_F32, i64 = ids_dtype == ANC_IDS_I64;
  ANC_REQUIRE(((uintptr_t)dw & (wf ? 3 : 1)) == 0, "dw not aligned to its element size");
  if (T > 0) {
    ANC_REQUIRE(dy && ids && work, "NULL argument");
    ANC_REQUIRE(((uintptr_t)dy & (yf ? 3 : 1)) == 0 && ((uintptr_t)ids & (i64 ? 7 : 3)) == 0,
                "pointer not aligned to its element size");
    ANC_REQUIRE(((uintptr_t)work & 15) == 0, "workspace not aligned to 16 bytes");
  }
  const Workspace ws = workspace_of(T, D);
  ANC_REQUIRE(T == 0 || work_bytes >= ws.total, "workspace of %llu bytes, %llu are needed",
              (unsigned long long)work_bytes, (unsigned long long)ws.total);
  if (T == 0 && mode == ANC_EMBED_ADD) return ANC_OK;
  anc_device_guard guard(ctx->device);
  cudaStream_t st = anc_pick_stream(ctx, stream);
  if (mode == ANC_EMBED_WRITE) {
    const int64_t row = D * (wf ? 4 : 2), pitch = dw_ld * (wf ? 4 : 2);
    const int vec = ((uintptr_t)dw & 15) == 0 && pitch % 16 == 0 && row % 16 == 0;
    const int64_t items = V * (row / (vec ? 16 : 2));
    int64_t blocks = (items + 255) / 256;
    const int64_t cap = (int64_t)ctx->sm_count * 16;
    if (blocks > cap) blocks = cap;
    embedding_zero_kernel<<<(unsigned)blocks, 256, 0, st>>>((uint8_t *)dw, row, pitch, V, vec);
    ANC_CUDA(cudaGetLastError());
  }
  if (T == 0) return ANC_OK;
  uint8_t *wp = (uint8_t *)work;
  SortArgs sa;
  sa.ids = ids; sa.ids64 = i64; sa.T = T; sa.V = V; sa.padding_idx = padding_idx;
  for (int i = 0; i < 2; ++i) {
    sa.key[i] = (uint32_t *)(wp + ws.key[i]);
    sa.pos[i] = (uint32_t *)(wp + ws.pos[i]);
  }
  int bits = 0;
  while (((uint64_t)V >> bits) != 0) ++bits;
  sa.passes = (bits + kDigitBits - 1) / kDigitBits;
  sa.status = ctx->d_status;
  const uint32_t n_ctas = T <= 4096 ? 1 : T <= 8192 ? 2 : T <= 16384 ? 4 : 8;
  {
    ANC_CUDA(cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSortSmem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_ctas);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = kSortSmem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = n_ctas;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    ANC_CUDA(cudaLaunchKernelEx(&cfg, embedding_sort_kernel, sa, n_ctas));
  }
  const Shape sh = shape_of(T, D);
  RedArgs ra;
  ra.dy = dy; ra.dw = dw; ra.dy_ld = dy_ld; ra.dw_ld = dw_ld; ra.T = T;
  ra.key = sa.key[(sa.passes - 1) & 1];
  ra.pos = sa.pos[(sa.passes - 1) & 1];
  ra.partial = (float *)(wp + ws.partial);
  ra.V = (uint32_t)V; ra.D = (int)D; ra.slices = sh.slices; ra.per_warp = sh.per_warp; ra.scale = scale;
  ra.add = mode == ANC_EMBED_ADD;
  const int64_t grid = sh.pieces * sh.slices;
  ANC_REQUIRE(grid <= 0x7FFFFFFF, "T x D too large");
  const bool vec = rows_are_vectors(dy, dy_ld, yf, D) && rows_are_vectors(dw, dw_ld, wf, D);
#define ANC_REDUCE(Y, W, VEC)                                                                        \
  do {                                                                                               \
    embedding_reduce_kernel<Y, W, VEC><<<(unsigned)grid, kRedWarps * 32, 0, st>>>(ra);               \
    if (sh.pieces > 1) embedding_join_kernel<W, VEC><<<(unsigned)grid, kRedWarps * 32, 0, st>>>(ra, sh.pieces); \
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
  ANC_CUDA(cudaGetLastError());
  return ANC_OK;
}

}  // extern "C"
