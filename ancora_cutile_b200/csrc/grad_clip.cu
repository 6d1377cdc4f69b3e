// Global gradient norm over many tensors, and clipping.
//
//   sumsq  = sum_i sum_j g_ij^2
//   norm   = scale * sqrt(sumsq)
//   factor = scale * min(1, max_norm / (norm + eps))        NaN stays NaN, inf gives 0
//   out_ij = round(g_ij * factor)                           one float32 product, one rounding
//
// norm and factor stay in device memory: the clipping sweep, and the optimizer sweeps that apply the
// factor to the gradient as they load it, read it there, so a clipped step needs no host round trip and
// can be captured into a graph.
//
// Arithmetic.  Eight squares are added in float32 (bf16 squares are exact in float32) and every such group
// is added in float64: a float32 sum of 6e8 squares would lose half its digits.  A group whose sum leaves
// [2^-90, 2^120] is summed again in float64, so that gradients of 1e-25 or 1e25 keep their norm; only
// a true infinity or NaN in a gradient makes the norm infinite or NaN.
//
// Order.  Thread sums, the shuffle tree, the warps of a block, the blocks: all in an order that depends on the
// table, the number of SMs and the call (norm or clip) alone, never on timing.  The last block to finish (an
// integer ticket) adds the block sums in index order, so one launch gives the norm.
//
// Launches.  The norm is one launch of resident blocks that share the vectors of all tensors piece by piece.
// Clipping reads the gradients twice (the factor is known only after all of them), in two launches; what
// fits the registers of the resident blocks is read once, in one launch whose blocks wait for one
// another between the two halves.
#include <algorithm>
#include <cuda_bf16.h>
#include <math.h>
#include <new>
#include <vector>
#include "anc_internal.h"
#include "philox.cuh"
#include "pred_load.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kVecPerThread = 4;                              // vectors of 8 elements a thread has in flight
constexpr int kChunkVec = kThreads * kVecPerThread;           // vectors per chunk of the scaling sweep
constexpr int kChunkElems = kChunkVec * 8;
constexpr uint64_t kPieceVec = 2 * kChunkVec;                 // vectors per piece of the norm
constexpr uint64_t kMostVec = 1u << 30;                        // a piece fits an int
constexpr uint64_t kManyBytes = 400u << 20;                   // gradients from which a clip's norm has more blocks
constexpr uint32_t kWaitPolls = 1u << 22;                     // of the one-launch clip; about a second
constexpr uint32_t kGaveUp = 1u << 31;                        // in its ticket; above any count of blocks
constexpr uint32_t kTestPolls = 1u << 14;

// One tensor.  The norm reads elements [head, head + 8 * nvec) as vectors of eight aligned to their size (16
// bytes of bf16, 32 of f32), and the up to 7 on either side one by one.  The scaling sweep wants input and output
// aligned together: from shead on, snvec vectors; without a common alignment snvec is 0 and all elements go one by
// one.
struct Entry {
  const void *g;
  void *out;
  uint64_t numel;
  uint64_t vec0;        // vectors of the tensors before this one (a tensor counts one at least)
  uint64_t nvec, snvec;
  uint32_t chunk0;      // chunks of the tensors before this one
  uint16_t head, shead;
};
static_assert(sizeof(Entry) == 56, "table entry");

template <bool kF32>
__device__ __forceinline__ float load1(const void *p, uint64_t i) {
  if constexpr (kF32) return ((const float *)p)[i];
  else return __uint_as_float((uint32_t)((const uint16_t *)p)[i] << 16);
}

// eight elements as they lie in memory
template <bool kF32>
struct Raw {
  uint32_t w[kF32 ? 8 : 4];
};
template <bool kF32>
__device__ __forceinline__ void load_raw(Raw<kF32> &r, const void *p, uint64_t i, bool on) {
  const uint8_t *q = (const uint8_t *)p + i * (kF32 ? 4 : 2);
  if constexpr (kF32) ld_v8(r.w, q, on);
  else ld_v4(r.w[0], r.w[1], r.w[2], r.w[3], q, on);
}
template <bool kF32>
__device__ __forceinline__ void widen(const Raw<kF32> &r, float x[8]) {
  if constexpr (kF32) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(r.w[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = __uint_as_float(r.w[k] << 16);
      x[2 * k + 1] = __uint_as_float(r.w[k] & 0xFFFF0000u);
    }
  }
}

template <bool kF32>
__device__ __forceinline__ double sumsq8(const Raw<kF32> &r) {
  float x[8];
  widen<kF32>(r, x);
  float s = x[0] * x[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) s = fmaf(x[k], x[k], s);
  if (s >= 8.0779357e-28f && s <= 1.3292280e36f) return (double)s;     // 2^-90, 2^120
  uint32_t any = 0;
#pragma unroll
  for (int k = 0; k < (kF32 ? 8 : 4); ++k) any |= r.w[k];
  if (any == 0) return 0.0;            // rows of an embedding that no token named
  double d = 0.0;
#pragma unroll
  for (int k = 0; k < 8; ++k) d = fma((double)x[k], (double)x[k], d);
  return d;
}

// Index of the tensor that holds place `c` of the space whose starts `start(i)` gives: every warp narrows the
// table 32-fold per round, all lanes' loads at once.
template <typename F>
__device__ __forceinline__ uint32_t find_entry(uint32_t n, uint64_t c, F start) {
  uint32_t lo = 0;
  while (n > 1) {
    const uint32_t step = (n + 31) / 32, i = (threadIdx.x & 31) * step;
    const bool le = i < n && start(lo + i) <= c;
    const uint32_t k = __popc(__ballot_sync(0xFFFFFFFFu, le)) - 1;      // starts ascend: the last that is <= c
    lo += k * step;
    n = n - k * step < step ? n - k * step : step;
  }
  return lo;
}

// the elements of a tensor outside its vectors: fewer than 8 on either side
template <bool kF32>
__device__ __forceinline__ double loose_sumsq(const Entry &e, uint32_t head, uint64_t nvec) {
  double acc = 0.0;
  const uint64_t after = head + nvec * 8;
  if (threadIdx.x < head) {
    const double x = load1<kF32>(e.g, threadIdx.x);
    acc = fma(x, x, acc);
  }
  for (uint64_t i = after + threadIdx.x; i < e.numel; i += kThreads) {
    const double x = load1<kF32>(e.g, i);
    acc = fma(x, x, acc);
  }
  return acc;
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int k = 1; k < kThreads / 32; ++k) v += part[k];
  __syncthreads();
  return v;
}

struct NormOut {
  double *sumsq;
  float *result;        // {norm, factor}
  float scale, max_norm, eps;
};

__device__ __forceinline__ void finish_norm(const NormOut &o, double sumsq) {
  const double norm = (double)o.scale * sqrt(sumsq);
  const double den = norm + (double)o.eps;
  double c = (double)o.max_norm / den;
  // max_norm = inf never clips, whatever the gradients hold, and all-zero gradients need no clipping;
  // otherwise a NaN norm gives a NaN factor
  if (isinf(o.max_norm) || den == 0.0 || c > 1.0) c = 1.0;
  o.result[0] = (float)norm;
  o.result[1] = (float)((double)o.scale * c);
}

__device__ __forceinline__ double sum_partials(const double *partial, uint32_t n) {
  double acc = 0.0;
  for (uint32_t b = threadIdx.x; b < n; b += kThreads) acc += __ldcg(partial + b);
  return block_sum(acc);
}

// the thread sums of all blocks into the norm, by the last block to get here
__device__ __forceinline__ void reduce_blocks(double acc, double *partial, uint32_t *ticket, const NormOut &o,
                                              int finish) {
  acc = block_sum(acc);
  __shared__ bool last;
  if (threadIdx.x == 0) {
    partial[blockIdx.x] = acc;
    __threadfence();
    last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  acc = sum_partials(partial, gridDim.x);
  if (threadIdx.x == 0) {
    *ticket = 0u;                        // ready for the next launch
    *o.sumsq = acc;
    if (finish) finish_norm(o, acc);
  }
}

// Bound by the read of the gradients: 1.19 GB of bf16 in 176 us a call, 6.8 TB/s.  Resident blocks go through the arena in
// pieces, in address order as far as they keep step, which DRAM likes better than one long share per block
// (150 M bf16: 50.8 us against 52.5, 596 M: 172 against 181; pieces half or twice as long: 186 and 173).
template <bool kF32>
__global__ void __launch_bounds__(kThreads)
grad_sumsq_kernel(const Entry *__restrict__ tab, uint32_t n_tab, uint64_t n_vec, uint64_t piece,
                  double *__restrict__ partial, uint32_t *ticket, NormOut o, int finish) {
  constexpr uint32_t kBytes = kF32 ? 32 : 16;                    // of a vector
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  double acc = 0.0;
  Entry e;
  uint32_t ti = 0;
  uint64_t end = 0;                                              // of tensor ti, 0: none yet
  for (uint64_t v0 = blockIdx.x * piece; v0 < n_vec; v0 += gridDim.x * piece) {
    const uint64_t v1 = v0 + piece < n_vec ? v0 + piece : n_vec;
    for (uint64_t v = v0; v < v1;) {
      if (v >= end) {
        ti = v == end && end ? ti + 1 : find_entry(n_tab, v, [&](uint32_t i) { return tab[i].vec0; });
        e = tab[ti];
        end = e.vec0 + (e.nvec ? e.nvec : 1);
      }
      const uint64_t a = v - e.vec0, stop = end < v1 ? end : v1;
      if (a == 0) acc += loose_sumsq<kF32>(e, e.head, e.nvec);
      if (e.nvec) {
        const uint8_t *p = (const uint8_t *)e.g + e.head * (kBytes / 8) + (a + threadIdx.x) * kBytes;
        for (int left = (int)(stop - v) - (int)threadIdx.x; left > 0; left -= kChunkVec, p += kChunkVec * kBytes) {
          Raw<kF32> r[kVecPerThread] = {};
#pragma unroll
          for (int k = 0; k < kVecPerThread; ++k) load_raw<kF32>(r[k], p + k * kThreads * kBytes, 0, left > k * kThreads);
#pragma unroll
          for (int k = 0; k < kVecPerThread; ++k) acc += sumsq8<kF32>(r[k]);
        }
      }
      v = stop;
    }
  }
  reduce_blocks(acc, partial, ticket, o, finish);
}

__global__ void grad_norm_finish_kernel(NormOut o) { finish_norm(o, *o.sumsq); }

template <bool kOutF32>
__device__ __forceinline__ void store1(void *p, uint64_t i, float x) {
  if constexpr (kOutF32) ((float *)p)[i] = x;
  else ((uint16_t *)p)[i] = (uint16_t)bf16_rne(x);
}

// One chunk of one tensor in registers, between its load and its scaled store.
template <bool kF32, bool kOutF32>
struct Chunk {
  Entry e;
  uint64_t local;        // chunk within the tensor
  Raw<kF32> r[kVecPerThread];

  __device__ __forceinline__ uint64_t vec(int k) const { return local * kChunkVec + threadIdx.x + (uint64_t)k * kThreads; }

  __device__ __forceinline__ void find(const Entry *__restrict__ tab, uint32_t n_tab, uint32_t c) {
    e = tab[find_entry(n_tab, c, [&](uint32_t i) { return (uint64_t)tab[i].chunk0; })];
    local = c - e.chunk0;
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int k = 0; k < kVecPerThread; ++k) {
      r[k] = Raw<kF32>{};
      load_raw<kF32>(r[k], e.g, e.shead + vec(k) * 8, vec(k) < e.snvec);
    }
  }
  // elements that are not in vectors: the ends of the tensor, or all of the chunk
  template <typename F>
  __device__ __forceinline__ void loose(F f) const {
    if (e.snvec == 0) {
      const uint64_t end = e.numel < (local + 1) * kChunkElems ? e.numel : (local + 1) * kChunkElems;
#pragma unroll 4
      for (uint64_t i = local * kChunkElems + threadIdx.x; i < end; i += kThreads) f(i);
    } else if (local == 0) {
      const uint64_t after = e.shead + e.snvec * 8;
      if (threadIdx.x < e.shead) f((uint64_t)threadIdx.x);
      if (after + threadIdx.x < e.numel) f(after + threadIdx.x);
    }
  }
  __device__ __forceinline__ double sumsq() const {
    double acc = 0.0;
#pragma unroll
    for (int k = 0; k < kVecPerThread; ++k) acc += sumsq8<kF32>(r[k]);
    loose([&](uint64_t i) {
      const double x = load1<kF32>(e.g, i);
      acc = fma(x, x, acc);
    });
    return acc;
  }
  __device__ __forceinline__ void store(float f) const {
#pragma unroll
    for (int k = 0; k < kVecPerThread; ++k) {
      if (vec(k) >= e.snvec) break;
      const uint64_t i = e.shead + vec(k) * 8;
      float x[8];
      widen<kF32>(r[k], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(x[j], f);
      if constexpr (kOutF32) {
        st_v8((float *)e.out + i, x);
      } else {
        uint32_t h[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = bf16_rne(x[j]);
        *reinterpret_cast<uint4 *>((uint16_t *)e.out + i) =
            make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
      }
    }
    loose([&](uint64_t i) { store1<kOutF32>(e.out, i, __fmul_rn(load1<kF32>(e.g, i), f)); });
  }
};

// The norm of what fits a resident block per chunk: many small tensors are then read side by side, where
// the pieces of a block walk through them one after another (25 tensors, 2.5 M elements: 6.4 against
// 9.3 us).
template <bool kF32>
__global__ void __launch_bounds__(kThreads)
grad_sumsq_chunk_kernel(const Entry *__restrict__ tab, uint32_t n_tab, double *partial, uint32_t *ticket, NormOut o,
                        int finish) {
  Chunk<kF32, false> ch;
  ch.find(tab, n_tab, blockIdx.x);
  ch.load();
  reduce_blocks(ch.sumsq(), partial, ticket, o, finish);
}

// A block per chunk, not resident blocks with a loop: blocks that start in address order keep DRAM streaming
// (1.19 GB of bf16 in and out: 342 us, 7.0 TB/s, against 395-408 with 1184 resident blocks, 366 for a memcpy).
//
// Behind a norm the sweep starts at the end of the arena, which the norm read last (`reverse`): 109 M bf16 134 us
// against 136, 25 M f32 115 against 120.  From 400 MiB on the norm then has eight waves of blocks with a share each,
// which keep closer to address order: 218 M f32 to bf16 321 us against 329, 0.6 GB 273 against 278; but 0.26 GB 124
// against 115.
template <bool kF32, bool kOutF32>
__global__ void __launch_bounds__(kThreads)
grad_scale_kernel(const Entry *__restrict__ tab, uint32_t n_tab, const float *result, int in_place,
                  int reverse) {
  const uint32_t c = reverse ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  Chunk<kF32, kOutF32> ch;
  if (!in_place) {                       // the gradients are the norm's input too: they may be read beside it
    ch.find(tab, n_tab, c);
    ch.load();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    ch.store(result[1]);
    return;
  }
  const float f = result[1];
  if (f == 1.0f) return;                 // every element would be written back as it is
  ch.find(tab, n_tab, c);
  ch.load();
  ch.store(f);
}

__device__ __forceinline__ uint32_t ld_acquire(const uint32_t *p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// Whether all blocks of the grid have counted themselves in `ticket`: the same answer in every block.  The first block
// that gives up marks the ticket, which it can only while a block is missing; from then on the answer is no,
// also for the blocks that arrive later.
__device__ __forceinline__ bool all_arrived(uint32_t *ticket, uint32_t polls) {
  uint32_t seen = 0;
  for (uint32_t i = 0; i < polls; ++i) {
    seen = ld_acquire(ticket);
    if (seen >= gridDim.x) return seen == gridDim.x;
  }
  while (seen < gridDim.x) {             // every round that fails is one more block in the ticket, or its mark
    const uint32_t old = atomicCAS(ticket, seen, seen | kGaveUp);
    if (old == seen) seen |= kGaveUp;
    else seen = old;
  }
  __threadfence();
  return seen == gridDim.x;
}

// Norm and scaling in one launch: a block per chunk, all resident at once (a cooperative launch), the
// chunk in registers while the blocks wait for one another's sums: 2.5 M elements of bf16 8.2 us against 14.3 by two
// launches.  From 3.6 M elements on the chunks are too many and there are two launches.  The wait is
// bounded, and the blocks decide together: when it runs out, status bit 0x10 is set, norm and factor are NaN and no
// gradient is written.  kLate, for the self-test: block `late` comes only after another one gave up.  Three blocks an
// SM: left to itself the compiler takes registers that leave room for two.
template <bool kF32, bool kOutF32, bool kLate>
__global__ void __launch_bounds__(kThreads, 3)
grad_clip_fused_kernel(const Entry *__restrict__ tab, uint32_t n_tab, double *partial, uint32_t *ticket, NormOut o,
                       int in_place, uint32_t *status, uint32_t polls, uint32_t late) {
  Chunk<kF32, kOutF32> ch;
  ch.find(tab, n_tab, blockIdx.x);
  ch.load();
  double acc = block_sum(ch.sumsq());
  __shared__ bool ok;
  if (threadIdx.x == 0) {
    if constexpr (kLate) {
      if (blockIdx.x == late)
        for (uint32_t i = 0; i < 64 * kTestPolls && !(ld_acquire(ticket) & kGaveUp); ++i) {}
    }
    partial[blockIdx.x] = acc;
    __threadfence();
    atomicAdd(ticket, 1u);
    ok = all_arrived(ticket, polls);
    // the last block to leave makes the counters ready for the next launch
    if (atomicAdd(ticket + 1, 1u) == gridDim.x - 1) {
      ticket[0] = 0u;
      ticket[1] = 0u;
    }
    if (!ok) {
      atomicOr(status, ANC_DEV_TIMEOUT_DEP);
      o.result[0] = o.result[1] = __int_as_float(0x7FFFFFFF);
    }
  }
  __syncthreads();
  if (!ok) return;
  acc = sum_partials(partial, gridDim.x);
  __shared__ float s_f;
  if (threadIdx.x == 0) {
    float res[2];
    NormOut mine = o;
    mine.result = res;
    finish_norm(mine, acc);
    s_f = res[1];
    if (blockIdx.x == 0) {
      *o.sumsq = acc;
      o.result[0] = res[0];
      o.result[1] = res[1];
    }
  }
  __syncthreads();
  if (in_place && s_f == 1.0f) return;
  ch.store(s_f);
}

}  // namespace

struct anc_clip_plan {
  anc_ctx *ctx;
  int grad_f32, out_f32, in_place;
  uint32_t n_tab;
  uint64_t n_vec, n_chunks;
  uint32_t grid, clip_grid;  // blocks of the norm alone, and in front of the scaling sweep
  int fused;                 // all chunks resident at once: one launch clips
  uint8_t *d_mem;            // one allocation: table, block sums, sum of squares, ticket, result
  Entry *d_tab;
  double *d_partial, *d_sumsq;
  uint32_t *d_ticket;
  float *d_result;
};

namespace {

struct Span {            // bytes of one tensor
  uintptr_t lo, hi;
  bool written;
};

NormOut norm_out(const anc_clip_plan *pl, float scale, float max_norm, float eps) {
  NormOut o;
  o.sumsq = pl->d_sumsq; o.result = pl->d_result;
  o.scale = scale; o.max_norm = max_norm; o.eps = eps;
  return o;
}

int check_scalars(float scale, float max_norm, float eps) {
  ANC_REQUIRE(isfinite(scale) && scale > 0.f, "scale must be finite and positive");
  ANC_REQUIRE(max_norm >= 0.f, "max_norm must not be negative or NaN");      // +inf: never clips
  ANC_REQUIRE(isfinite(eps) && eps >= 0.f, "eps must be finite and not negative");
  return ANC_OK;
}

int launch_sumsq(const anc_clip_plan *pl, uint32_t grid, uint64_t piece, const NormOut &o, int finish, cudaStream_t st) {
  if (pl->fused) {
    if (pl->grad_f32)
      grad_sumsq_chunk_kernel<true><<<(unsigned)pl->n_chunks, kThreads, 0, st>>>(pl->d_tab, pl->n_tab, pl->d_partial,
                                                                                 pl->d_ticket, o, finish);
    else
      grad_sumsq_chunk_kernel<false><<<(unsigned)pl->n_chunks, kThreads, 0, st>>>(pl->d_tab, pl->n_tab, pl->d_partial,
                                                                                  pl->d_ticket, o, finish);
  } else if (pl->grad_f32)
    grad_sumsq_kernel<true><<<grid, kThreads, 0, st>>>(pl->d_tab, pl->n_tab, pl->n_vec, piece, pl->d_partial,
                                                       pl->d_ticket, o, finish);
  else
    grad_sumsq_kernel<false><<<grid, kThreads, 0, st>>>(pl->d_tab, pl->n_tab, pl->n_vec, piece, pl->d_partial,
                                                        pl->d_ticket, o, finish);
  ANC_CUDA(cudaGetLastError());
  return ANC_OK;
}

// Vectors per piece of the norm: kPieceVec, which keeps pieces on DRAM's boundaries (596 M bf16: 172 us, 175 with
// pieces a little shorter), or with few rounds of the resident blocks what makes all rounds full (5 M bf16: 12.6 us
// against 14.5, 40 M f32: 31.5 against 32.5).
uint64_t piece_of(const anc_clip_plan *pl) {
  const uint64_t rounds = (pl->n_vec + pl->grid * kPieceVec - 1) / (pl->grid * kPieceVec);
  if (rounds > 4) return kPieceVec;
  return rounds ? (pl->n_vec + pl->grid * rounds - 1) / (pl->grid * rounds) : 1;
}

using ScaleKernel = void (*)(const Entry *, uint32_t, const float *, int, int);
using FusedKernel = void (*)(const Entry *, uint32_t, double *, uint32_t *, NormOut, int, uint32_t *, uint32_t, uint32_t);

ScaleKernel scale_kernel(const anc_clip_plan *pl) {
  if (pl->grad_f32) return pl->out_f32 ? grad_scale_kernel<true, true> : grad_scale_kernel<true, false>;
  return pl->out_f32 ? grad_scale_kernel<false, true> : grad_scale_kernel<false, false>;
}
template <bool kLate>
FusedKernel fused_kernel(const anc_clip_plan *pl) {
  if (pl->grad_f32)
    return pl->out_f32 ? grad_clip_fused_kernel<true, true, kLate> : grad_clip_fused_kernel<true, false, kLate>;
  return pl->out_f32 ? grad_clip_fused_kernel<false, true, kLate> : grad_clip_fused_kernel<false, false, kLate>;
}

int launch_fused(const anc_clip_plan *pl, FusedKernel kernel, const NormOut &o, uint32_t polls, uint32_t late,
                 cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)pl->n_chunks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  ANC_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const Entry *)pl->d_tab, pl->n_tab, pl->d_partial, pl->d_ticket, o,
                              pl->in_place, pl->ctx->d_status, polls, late));
  return ANC_OK;
}

// behind_norm: backwards and, unless in place, started while the norm's last blocks run (27 M f32 to bf16 45.5 us
// against 49.7, 71 M bf16 81.5 against 85.0, 596 M 531 against 535)
int launch_scale(const anc_clip_plan *pl, int behind_norm, cudaStream_t st) {
  if (pl->n_chunks == 0) return ANC_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)pl->n_chunks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = behind_norm && !pl->in_place ? 1 : 0;
  ANC_CUDA(cudaLaunchKernelEx(&cfg, scale_kernel(pl), (const Entry *)pl->d_tab, pl->n_tab,
                              (const float *)pl->d_result, pl->in_place, behind_norm));
  return ANC_OK;
}

}  // namespace

extern "C" {

int anc_clip_plan_create(anc_ctx *ctx, const anc_clip_tensor *tensors, int n_tensors, int grad_dtype, int out_dtype,
                         float *result, anc_clip_plan **out) {
  ANC_REQUIRE(ctx && out && (tensors || n_tensors == 0), "NULL argument");
  ANC_REQUIRE(n_tensors >= 0, "n_tensors < 0");
  ANC_REQUIRE(grad_dtype == ANC_GRAD_BF16 || grad_dtype == ANC_GRAD_F32, "bad grad_dtype %d", grad_dtype);
  ANC_REQUIRE(out_dtype == ANC_GRAD_BF16 || out_dtype == ANC_GRAD_F32, "bad out_dtype %d", out_dtype);
  ANC_REQUIRE(((uintptr_t)result & 3) == 0, "result not aligned to 4 bytes");
  *out = nullptr;
  const uint64_t gs = grad_dtype == ANC_GRAD_F32 ? 4 : 2, os = out_dtype == ANC_GRAD_F32 ? 4 : 2;
  bool all_in_place = true;
  uint64_t chunks = 0, vecs = 0;
  std::vector<Entry> tab;
  std::vector<Span> spans;
  try {
    tab.reserve((size_t)n_tensors + 1);
    for (int i = 0; i < n_tensors; ++i) {
      const anc_clip_tensor &t = tensors[i];
      if (t.numel == 0) continue;
      ANC_REQUIRE(t.g, "tensor %d has a NULL pointer", i);
      ANC_REQUIRE(t.numel <= (1ull << 48), "tensor %d: numel out of range", i);
      ANC_REQUIRE(((uintptr_t)t.g & (gs - 1)) == 0 && ((uintptr_t)t.out & (os - 1)) == 0,
                  "tensor %d: pointer not aligned to its element size", i);
      Entry e;
      e.g = t.g;
      e.out = t.out ? t.out : const_cast<void *>(t.g);
      ANC_REQUIRE(e.out != e.g || gs == os, "tensor %d: in place needs equal gradient and output types", i);
      all_in_place = all_in_place && e.out == e.g;
      e.numel = t.numel;
      e.vec0 = vecs;
      e.chunk0 = (uint32_t)chunks;
      e.head = (uint16_t)((8 * gs - (uintptr_t)e.g % (8 * gs)) % (8 * gs) / gs);
      e.nvec = t.numel >= e.head + 8u ? (t.numel - e.head) / 8 : 0;
      if (!e.nvec) e.head = 0;
      e.shead = 0;
      e.snvec = 0;
      for (uint32_t h = 0; h < 8; ++h) {
        if (((uintptr_t)e.g + h * gs) % (8 * gs) || ((uintptr_t)e.out + h * os) % (8 * os)) continue;
        if (t.numel >= h + 8) {
          e.shead = (uint16_t)h;
          e.snvec = (t.numel - h) / 8;
        }
        break;
      }
      // what a call reads and writes: outputs lie over nothing else of the call
      spans.push_back({(uintptr_t)e.g, (uintptr_t)e.g + t.numel * gs, e.out == e.g});
      if (e.out != e.g) spans.push_back({(uintptr_t)e.out, (uintptr_t)e.out + t.numel * os, true});
      vecs += e.nvec ? e.nvec : 1;
      chunks += e.snvec ? (e.snvec + kChunkVec - 1) / kChunkVec : (t.numel + kChunkElems - 1) / kChunkElems;
      ANC_REQUIRE(chunks <= 0x7FFFFFFF, "tensors too large for one plan");
      tab.push_back(e);
    }
    if (result) spans.push_back({(uintptr_t)result, (uintptr_t)result + 2 * sizeof(float), true});
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.lo < b.lo; });
    Span reach = {0, 0, false}, written = {0, 0, false};     // furthest-reaching spans so far: any, written
    for (const Span &s : spans) {
      ANC_REQUIRE(!(s.written && s.lo < reach.hi) && s.lo >= written.hi,
                  "a clipped tensor or the result would overlap another tensor of the plan");
      if (s.hi > reach.hi) reach = s;
      if (s.written && s.hi > written.hi) written = s;
    }
  } catch (const std::bad_alloc &) {
    anc_set_error("out of host memory");
    return ANC_E_NOMEM;
  }
  anc_device_guard guard(ctx->device);
  anc_clip_plan *pl = new (std::nothrow) anc_clip_plan();
  if (!pl) {
    anc_set_error("out of host memory");
    return ANC_E_NOMEM;
  }
  memset(pl, 0, sizeof(*pl));
  pl->ctx = ctx;
  pl->grad_f32 = grad_dtype == ANC_GRAD_F32;
  pl->out_f32 = out_dtype == ANC_GRAD_F32;
  pl->in_place = all_in_place ? 1 : 0;
  pl->n_tab = (uint32_t)tab.size();
  pl->n_chunks = chunks;
  pl->n_vec = vecs;
  // the norm's blocks: as many as are resident at once, each with four vectors per thread at least
  int norm_per_sm = 0, fused_per_sm = 0;
  cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(
      &norm_per_sm, pl->grad_f32 ? grad_sumsq_kernel<true> : grad_sumsq_kernel<false>, kThreads, 0);
  if (e == cudaSuccess)
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fused_per_sm, fused_kernel<false>(pl), kThreads, 0);
  if (e != cudaSuccess) {
    delete pl;
    return anc_cuda_fail(e, "clip kernel occupancy");
  }
  const uint64_t cap = (uint64_t)ctx->sm_count * (norm_per_sm > 0 ? norm_per_sm : 1);
  const uint64_t want = (vecs + kChunkVec - 1) / kChunkVec;
  pl->grid = (uint32_t)(want < cap ? (want ? want : 1) : cap);
  pl->clip_grid = vecs * 8 * gs >= kManyBytes ? pl->grid * 8 : pl->grid;
  pl->fused = chunks > 0 && chunks <= (uint64_t)fused_per_sm * ctx->sm_count;
  const uint64_t n_part = pl->fused && chunks > pl->clip_grid ? chunks : pl->clip_grid;
  const size_t tab_bytes = (tab.size() * sizeof(Entry) + 255) / 256 * 256;
  const size_t part_bytes = ((size_t)n_part * sizeof(double) + 255) / 256 * 256;
  e = cudaMalloc((void **)&pl->d_mem, tab_bytes + part_bytes + 256);
  if (e == cudaSuccess && !tab.empty())
    e = cudaMemcpy(pl->d_mem, tab.data(), tab.size() * sizeof(Entry), cudaMemcpyHostToDevice);
  if (e == cudaSuccess) e = cudaMemset(pl->d_mem + tab_bytes + part_bytes, 0, 256);
  if (e == cudaSuccess) e = anc_finish_setup();
  if (e != cudaSuccess) {
    if (pl->d_mem) cudaFree(pl->d_mem);
    delete pl;
    return anc_cuda_fail(e, "clip plan memory");
  }
  pl->d_tab = (Entry *)pl->d_mem;
  pl->d_partial = (double *)(pl->d_mem + tab_bytes);
  uint8_t *small = pl->d_mem + tab_bytes + part_bytes;
  pl->d_sumsq = (double *)small;
  pl->d_ticket = (uint32_t *)(small + 64);
  pl->d_result = result ? result : (float *)(small + 128);
  *out = pl;
  return ANC_OK;
}

int anc_clip_plan_result(anc_clip_plan *plan, float **result, double **sumsq) {
  ANC_REQUIRE(plan, "plan is NULL");
  if (result) *result = plan->d_result;
  if (sumsq) *sumsq = plan->d_sumsq;
  return ANC_OK;
}

int anc_grad_norm(anc_clip_plan *plan, float scale, float max_norm, float eps, void *stream) {
  ANC_REQUIRE(plan, "plan is NULL");
  int rc = check_scalars(scale, max_norm, eps);
  if (rc) return rc;
  anc_device_guard guard(plan->ctx->device);
  return launch_sumsq(plan, plan->grid, piece_of(plan), norm_out(plan, scale, max_norm, eps), 1, anc_pick_stream(plan->ctx, stream));
}

int anc_grad_sumsq(anc_clip_plan *plan, void *stream) {
  ANC_REQUIRE(plan, "plan is NULL");
  anc_device_guard guard(plan->ctx->device);
  return launch_sumsq(plan, plan->grid, piece_of(plan), norm_out(plan, 1.f, INFINITY, 0.f), 0, anc_pick_stream(plan->ctx, stream));
}

int anc_grad_norm_finish(anc_clip_plan *plan, float scale, float max_norm, float eps, void *stream) {
  ANC_REQUIRE(plan, "plan is NULL");
  int rc = check_scalars(scale, max_norm, eps);
  if (rc) return rc;
  anc_device_guard guard(plan->ctx->device);
  grad_norm_finish_kernel<<<1, 1, 0, anc_pick_stream(plan->ctx, stream)>>>(norm_out(plan, scale, max_norm, eps));
  ANC_CUDA(cudaGetLastError());
  return ANC_OK;
}

int anc_grad_apply(anc_clip_plan *plan, void *stream) {
  ANC_REQUIRE(plan, "plan is NULL");
  anc_device_guard guard(plan->ctx->device);
  return launch_scale(plan, 0, anc_pick_stream(plan->ctx, stream));
}

int anc_grad_clip(anc_clip_plan *plan, float scale, float max_norm, float eps, void *stream) {
  ANC_REQUIRE(plan, "plan is NULL");
  int rc = check_scalars(scale, max_norm, eps);
  if (rc) return rc;
  anc_device_guard guard(plan->ctx->device);
  cudaStream_t st = anc_pick_stream(plan->ctx, stream);
  const NormOut o = norm_out(plan, scale, max_norm, eps);
  if (!plan->fused) {
    const uint64_t share = std::min((plan->n_vec + plan->clip_grid - 1) / plan->clip_grid, kMostVec);
    rc = launch_sumsq(plan, plan->clip_grid, plan->clip_grid == plan->grid ? piece_of(plan) : share, o, 1, st);
    return rc ? rc : launch_scale(plan, 1, st);
  }
  return launch_fused(plan, fused_kernel<false>(plan), o, kWaitPolls, 0, st);
}

int anc_clip_wait_selftest(anc_clip_plan *plan, float max_norm, uint32_t polls, uint32_t late, void *stream) {
  ANC_REQUIRE(plan, "plan is NULL");
  ANC_REQUIRE(polls > 0 && polls <= kTestPolls, "polls %u outside 1..2^14", polls);
  int rc = check_scalars(1.f, max_norm, 0.f);
  if (rc) return rc;
  ANC_REQUIRE(plan->fused && plan->n_chunks > 1 && late < plan->n_chunks,
              "needs a plan of several blocks that one launch clips, and one of its blocks");
  anc_device_guard guard(plan->ctx->device);
  const FusedKernel kernel = fused_kernel<true>(plan);
  int per_sm = 0;
  ANC_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, 0));
  ANC_REQUIRE(plan->n_chunks <= (uint64_t)per_sm * plan->ctx->sm_count, "plan too large for the self-test");
  return launch_fused(plan, kernel, norm_out(plan, 1.f, max_norm, 0.f), polls, late, anc_pick_stream(plan->ctx, stream));
}

int anc_clip_plan_destroy(anc_clip_plan *plan) {
  if (!plan) return ANC_OK;
  anc_device_guard guard(plan->ctx->device);
  if (plan->d_mem) cudaFree(plan->d_mem);       // waits for the device: no launch still uses the table
  delete plan;
  return ANC_OK;
}

}  // extern "C"
