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
// Order.  Thread sums, the shuffle tree, the warps of a block, the blocks: all in an order that depends on
// the table and the number of SMs alone, never on timing.  The last block to finish (an integer ticket)
// adds the block sums in index order, so one launch gives the norm.
#include <algorithm>
#include <cuda_bf16.h>
#include <math.h>
#include <new>
#include <vector>
#include "anc_internal.h"
#include "philox.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kVecPerThread = 4;                              // vectors of 8 elements a thread has in flight
constexpr int kChunkVec = kThreads * kVecPerThread;           // vectors per chunk
constexpr int kChunkElems = kChunkVec * 8;
constexpr int kCtasPerSm = 8;

// One tensor.  Elements [head, head + 8 * nvec) are read as 16-byte aligned vectors, the up to 7 before
// and after them one by one.  Without a common alignment of input and output nvec is 0 and all elements
// go one by one.
struct Entry {
  const void *g;
  void *out;
  uint64_t numel;
  uint64_t chunk0;      // chunks of the tensors before this one
  uint64_t nvec;
  uint32_t head;
  uint32_t _pad;
};
static_assert(sizeof(Entry) == 48, "table entry");

template <bool kF32>
__device__ __forceinline__ float load1(const void *p, uint64_t i) {
  if constexpr (kF32) return __ldg((const float *)p + i);
  else return __uint_as_float((uint32_t)__ldg((const uint16_t *)p + i) << 16);
}

// eight elements as they lie in memory
template <bool kF32>
struct Raw {
  uint4 a, b;
};
template <>
struct Raw<false> {
  uint4 a;
};
template <bool kF32>
__device__ __forceinline__ Raw<kF32> load_raw(const void *p, uint64_t i) {
  Raw<kF32> r;
  if constexpr (kF32) {
    r.a = __ldg(reinterpret_cast<const uint4 *>((const float *)p + i));
    r.b = __ldg(reinterpret_cast<const uint4 *>((const float *)p + i) + 1);
  } else {
    r.a = __ldg(reinterpret_cast<const uint4 *>((const uint16_t *)p + i));
  }
  return r;
}
template <bool kF32>
__device__ __forceinline__ void widen(const Raw<kF32> &r, float x[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
  if constexpr (kF32) {
    const uint32_t u[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = __uint_as_float(w[k]);
      x[4 + k] = __uint_as_float(u[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = __uint_as_float(w[k] << 16);
      x[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
    }
  }
}

__device__ __forceinline__ double sumsq8(const float x[8]) {
  float s = x[0] * x[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) s = fmaf(x[k], x[k], s);
  if (s >= 8.0779357e-28f && s <= 1.3292280e36f) return (double)s;     // 2^-90, 2^120
  double d = 0.0;
#pragma unroll
  for (int k = 0; k < 8; ++k) d = fma((double)x[k], (double)x[k], d);
  return d;
}

// index of the tensor that holds chunk c (the table is never empty and c is below the number of chunks)
__device__ __forceinline__ uint32_t find_entry(const Entry *__restrict__ tab, uint32_t n, uint64_t c) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (tab[mid].chunk0 <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <bool kF32>
__device__ __forceinline__ double chunk_sumsq(const Entry &e, uint64_t local) {
  double acc = 0.0;
  if (e.nvec) {
    const uint64_t v0 = local * kChunkVec + threadIdx.x;
    Raw<kF32> r[kVecPerThread];
#pragma unroll
    for (int k = 0; k < kVecPerThread; ++k)
      if (v0 + (uint64_t)k * kThreads < e.nvec) r[k] = load_raw<kF32>(e.g, e.head + (v0 + (uint64_t)k * kThreads) * 8);
#pragma unroll
    for (int k = 0; k < kVecPerThread; ++k)
      if (v0 + (uint64_t)k * kThreads < e.nvec) {
        float x[8];
        widen<kF32>(r[k], x);
        acc += sumsq8(x);
      }
    if (local == 0) {      // the elements outside the vectors: fewer than 8 on either side
      const uint64_t after = e.head + e.nvec * 8;
      if (threadIdx.x < e.head) {
        const double x = load1<kF32>(e.g, threadIdx.x);
        acc = fma(x, x, acc);
      }
      if (after + threadIdx.x < e.numel) {
        const double x = load1<kF32>(e.g, after + threadIdx.x);
        acc = fma(x, x, acc);
      }
    }
  } else {
    const uint64_t end = e.numel < (local + 1) * kChunkElems ? e.numel : (local + 1) * kChunkElems;
    for (uint64_t i = local * kChunkElems + threadIdx.x; i < end; i += kThreads) {
      const double x = load1<kF32>(e.g, i);
      acc = fma(x, x, acc);
    }
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

template <bool kF32>
__global__ void __launch_bounds__(kThreads)
grad_sumsq_kernel(const Entry *__restrict__ tab, uint32_t n_tab, uint64_t n_chunks, double *__restrict__ partial,
                  uint32_t *ticket, NormOut o, int finish) {
  // this block's chunks: a contiguous share, so that one search finds the first tensor
  const uint64_t c0 = n_chunks * blockIdx.x / gridDim.x, c1 = n_chunks * (blockIdx.x + 1ull) / gridDim.x;
  double acc = 0.0;
  if (c0 < c1) {
    uint32_t ti = find_entry(tab, n_tab, c0);
    Entry e = tab[ti];
    uint64_t next = ti + 1 < n_tab ? tab[ti + 1].chunk0 : n_chunks;
    for (uint64_t c = c0; c < c1; ++c) {
      while (c >= next) {
        e = tab[++ti];
        next = ti + 1 < n_tab ? tab[ti + 1].chunk0 : n_chunks;
      }
      acc += chunk_sumsq<kF32>(e, c - e.chunk0);
    }
  }
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
  acc = 0.0;
  for (uint32_t b = threadIdx.x; b < gridDim.x; b += kThreads) acc += __ldcg(partial + b);
  acc = block_sum(acc);
  if (threadIdx.x == 0) {
    *ticket = 0u;                        // ready for the next launch
    *o.sumsq = acc;
    if (finish) finish_norm(o, acc);
  }
}

__global__ void grad_norm_finish_kernel(NormOut o) { finish_norm(o, *o.sumsq); }

template <bool kOutF32>
__device__ __forceinline__ void store1(void *p, uint64_t i, float x) {
  if constexpr (kOutF32) ((float *)p)[i] = x;
  else ((uint16_t *)p)[i] = (uint16_t)bf16_rne(x);
}

template <bool kF32, bool kOutF32>
__global__ void __launch_bounds__(kThreads)
grad_scale_kernel(const Entry *__restrict__ tab, uint32_t n_tab, uint64_t n_chunks, const float *__restrict__ result,
                  int in_place) {
  const float f = result[1];
  if (in_place && f == 1.0f) return;     // every element would be written back as it is
  const uint64_t c0 = n_chunks * blockIdx.x / gridDim.x, c1 = n_chunks * (blockIdx.x + 1ull) / gridDim.x;
  if (c0 >= c1) return;
  uint32_t ti = find_entry(tab, n_tab, c0);
  Entry e = tab[ti];
  uint64_t next = ti + 1 < n_tab ? tab[ti + 1].chunk0 : n_chunks;
  for (uint64_t c = c0; c < c1; ++c) {
    while (c >= next) {
      e = tab[++ti];
      next = ti + 1 < n_tab ? tab[ti + 1].chunk0 : n_chunks;
    }
    const uint64_t local = c - e.chunk0;
    if (e.nvec) {
      const uint64_t v0 = local * kChunkVec + threadIdx.x;
      Raw<kF32> r[kVecPerThread];
#pragma unroll
      for (int k = 0; k < kVecPerThread; ++k)
        if (v0 + (uint64_t)k * kThreads < e.nvec) r[k] = load_raw<kF32>(e.g, e.head + (v0 + (uint64_t)k * kThreads) * 8);
#pragma unroll
      for (int k = 0; k < kVecPerThread; ++k)
        if (v0 + (uint64_t)k * kThreads < e.nvec) {
          const uint64_t i = e.head + (v0 + (uint64_t)k * kThreads) * 8;
          float x[8];
          widen<kF32>(r[k], x);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(x[j], f);
          if constexpr (kOutF32) {
            float4 *d = reinterpret_cast<float4 *>((float *)e.out + i);
            d[0] = make_float4(x[0], x[1], x[2], x[3]);
            d[1] = make_float4(x[4], x[5], x[6], x[7]);
          } else {
            uint32_t h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = bf16_rne(x[j]);
            *reinterpret_cast<uint4 *>((uint16_t *)e.out + i) =
                make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
          }
        }
      if (local == 0) {
        const uint64_t after = e.head + e.nvec * 8;
        if (threadIdx.x < e.head) store1<kOutF32>(e.out, threadIdx.x, __fmul_rn(load1<kF32>(e.g, threadIdx.x), f));
        if (after + threadIdx.x < e.numel)
          store1<kOutF32>(e.out, after + threadIdx.x, __fmul_rn(load1<kF32>(e.g, after + threadIdx.x), f));
      }
    } else {
      const uint64_t end = e.numel < (local + 1) * kChunkElems ? e.numel : (local + 1) * kChunkElems;
      for (uint64_t i = local * kChunkElems + threadIdx.x; i < end; i += kThreads)
        store1<kOutF32>(e.out, i, __fmul_rn(load1<kF32>(e.g, i), f));
    }
  }
}

}  // namespace

struct anc_clip_plan {
  anc_ctx *ctx;
  int grad_f32, out_f32, in_place;
  uint32_t n_tab;
  uint64_t n_chunks;
  uint32_t grid;
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

int launch_sumsq(const anc_clip_plan *pl, const NormOut &o, int finish, cudaStream_t st) {
  if (pl->grad_f32)
    grad_sumsq_kernel<true><<<pl->grid, kThreads, 0, st>>>(pl->d_tab, pl->n_tab, pl->n_chunks, pl->d_partial,
                                                           pl->d_ticket, o, finish);
  else
    grad_sumsq_kernel<false><<<pl->grid, kThreads, 0, st>>>(pl->d_tab, pl->n_tab, pl->n_chunks, pl->d_partial,
                                                            pl->d_ticket, o, finish);
  ANC_CUDA(cudaGetLastError());
  return ANC_OK;
}

int launch_scale(const anc_clip_plan *pl, cudaStream_t st) {
  if (pl->n_chunks == 0) return ANC_OK;
#define ANC_SCALE(F, O) \
  grad_scale_kernel<F, O><<<pl->grid, kThreads, 0, st>>>(pl->d_tab, pl->n_tab, pl->n_chunks, pl->d_result, pl->in_place)
  if (pl->grad_f32 && pl->out_f32) ANC_SCALE(true, true);
  else if (pl->grad_f32) ANC_SCALE(true, false);
  else if (pl->out_f32) ANC_SCALE(false, true);
  else ANC_SCALE(false, false);
#undef ANC_SCALE
  ANC_CUDA(cudaGetLastError());
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
  uint64_t chunks = 0;
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
      ANC_REQUIRE(t.out || gs == os, "tensor %d: in place needs equal gradient and output types", i);
      Entry e;
      e.g = t.g;
      e.out = t.out ? t.out : const_cast<void *>(t.g);
      all_in_place = all_in_place && e.out == e.g;
      e.numel = t.numel;
      e.chunk0 = chunks;
      e.head = 0;
      e.nvec = 0;
      e._pad = 0;
      for (uint32_t h = 0; h < 8; ++h) {
        if ((((uintptr_t)e.g + h * gs) & 15) || (((uintptr_t)e.out + h * os) & 15)) continue;
        if (t.numel >= h + 8) {
          e.head = h;
          e.nvec = (t.numel - h) / 8;
        }
        break;
      }
      // what a call reads and writes: outputs lie over nothing else of the call
      spans.push_back({(uintptr_t)e.g, (uintptr_t)e.g + t.numel * gs, e.out == e.g});
      if (e.out != e.g) spans.push_back({(uintptr_t)e.out, (uintptr_t)e.out + t.numel * os, true});
      chunks += e.nvec ? (e.nvec + kChunkVec - 1) / kChunkVec : (t.numel + kChunkElems - 1) / kChunkElems;
      tab.push_back(e);
    }
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.lo < b.lo; });
    Span reach = {0, 0, false}, written = {0, 0, false};     // furthest-reaching spans so far: any, written
    for (const Span &s : spans) {
      ANC_REQUIRE(!(s.written && s.lo < reach.hi) && s.lo >= written.hi,
                  "a clipped tensor would overlap another tensor of the plan");
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
  const uint64_t cap = (uint64_t)ctx->sm_count * kCtasPerSm;
  pl->grid = (uint32_t)(chunks < cap ? (chunks ? chunks : 1) : cap);
  const size_t tab_bytes = (tab.size() * sizeof(Entry) + 255) / 256 * 256;
  const size_t part_bytes = ((size_t)pl->grid * sizeof(double) + 255) / 256 * 256;
  cudaError_t e = cudaMalloc((void **)&pl->d_mem, tab_bytes + part_bytes + 256);
  if (e == cudaSuccess && !tab.empty())
    e = cudaMemcpy(pl->d_mem, tab.data(), tab.size() * sizeof(Entry), cudaMemcpyHostToDevice);
  if (e == cudaSuccess) e = cudaMemset(pl->d_mem + tab_bytes + part_bytes, 0, 256);
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
  return launch_sumsq(plan, norm_out(plan, scale, max_norm, eps), 1, anc_pick_stream(plan->ctx, stream));
}

int anc_grad_sumsq(anc_clip_plan *plan, void *stream) {
  ANC_REQUIRE(plan, "plan is NULL");
  anc_device_guard guard(plan->ctx->device);
  return launch_sumsq(plan, norm_out(plan, 1.f, INFINITY, 0.f), 0, anc_pick_stream(plan->ctx, stream));
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
  return launch_scale(plan, anc_pick_stream(plan->ctx, stream));
}

int anc_grad_clip(anc_clip_plan *plan, float scale, float max_norm, float eps, void *stream) {
  int rc = anc_grad_norm(plan, scale, max_norm, eps, stream);
  return rc ? rc : anc_grad_apply(plan, stream);
}

int anc_clip_plan_destroy(anc_clip_plan *plan) {
  if (!plan) return ANC_OK;
  anc_device_guard guard(plan->ctx->device);
  if (plan->d_mem) cudaFree(plan->d_mem);       // waits for the device: no launch still uses the table
  delete plan;
  return ANC_OK;
}

}  // extern "C"
