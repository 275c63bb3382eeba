// Cross entropy of a language-model head straight from its hidden states: the passes around the product that makes the
// logits (gemm_tcgen05.cu, epilogue_ce), which never exist in memory.
//
//   l_rv = x_r . w_v        loss_r = log sum_v e^{l_rv} - l_rt        d_rv = g_r (e^{l_rv} / Z_r - [v = t])
//   dX = d W                dW = d^T X                                 (t = target of row r, rows without one: 0)
//
// The product's epilogue leaves e_rv = exp(l_rv - m_r) in bf16 and, per column tile, their fp32 sums S_r without the
// target's column.  The reference m_r is the target's own logit, an H-long dot product that is known beforehand: then
//   loss_r = log1p(S_r),  1 - p_t = S_r / (1 + S_r),  Z_r = 1 + S_r
// hold to fp32 precision however sure the row is of its target.  (A row whose largest logit is more than 40 above its
// target's is computed again against that maximum M: Z_r = S_r + e^{l_t - M}, loss_r = log Z_r + M - l_t.)
//
// The gradient needs no pass over the [rows, V] exponentials: d_rv = f_r E_rv with E = e except in the target's column,
// where E_rt = -S_r, and f_r = g_r / Z_r, one factor for the row.  dX takes f_r in its product's epilogue (fp32); dW
// takes it with the rows of X (xs = bf16(f_r x_r), one rounding).  E_rt is rounded to bf16 like every other entry, but
// it is the largest of its row by far, and its rounding would be common to the whole row of the gradient: f_r is made
// from the rounded value, f_r = g_r (S_r / Z_r) / |bf16(S_r)|, so the target's part f_r E_rt is exact and the other
// entries carry the (at most 2^-8 relative) difference like one more rounding.
#include <cfloat>
#include <cmath>

#include "olb_api.h"
#include "ptx.cuh"

namespace olb {

constexpr int LCE_THREADS = 256;
constexpr int LCE_WARPS = LCE_THREADS / 32;

// How many of the whole batch's n targets lie in [0, V): integers, so their order does not matter.
__device__ __forceinline__ void lce_count(const long long* __restrict__ targets, long long n, int V, float* __restrict__ count,
                                          float* __restrict__ inv_count) {
  __shared__ int s[LCE_WARPS];
  int c = 0;  // n < 2^31
#pragma unroll 16
  for (long long i = threadIdx.x; i < n; i += LCE_THREADS) {
    const long long t = targets[i];
    c += (t >= 0 && t < V) ? 1 : 0;
  }
  c = __reduce_add_sync(0xffffffffu, c);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    int total = 0;
    for (int i = 0; i < LCE_WARPS; ++i) total += s[i];
    *count = static_cast<float>(total);
    *inv_count = total > 0 ? 1.f / static_cast<float>(total) : 0.f;
  }
}

// What the tensor cores' running sum loses on average of a logit whose x has `vecs` vectors of 8 channels that are not all
// zero, relative to it (see epilogue_ce); the first 16 channels are added to nothing.  Never 0, so that -inf stays -inf.
__device__ __forceinline__ float lce_grow(int vecs) { return fmaxf(0.7e-8f * (vecs - 2), 1e-30f); }

// ref[r] = x_r . w_t: one warp per row, or the block's eight for one row when there are few (a single row of 4096:
// 6.7 us with one warp).  The last block counts the targets (`count` set).
template <bool FEW>
__global__ void __launch_bounds__(LCE_THREADS)
lce_prep_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, const __nv_bfloat16* __restrict__ w, long long ldw,
                const long long* __restrict__ targets, int rows, int H, int V, float* __restrict__ ref,
                float* __restrict__ grow, unsigned* __restrict__ ce_max, int* __restrict__ ce_flags, unsigned* __restrict__ ticket,
                const long long* __restrict__ all_targets, long long n_all, float* __restrict__ count) {
  // the product may start: nothing of it but its epilogue needs what this kernel writes
  grid_launch_dependents();
  if (count != nullptr && blockIdx.x == gridDim.x - 1) {
    lce_count(all_targets, n_all, V, count, count + 1);
    return;
  }
  __shared__ float s_part[LCE_WARPS];
  __shared__ int s_used[LCE_WARPS];
  const int warp = threadIdx.x >> 5, lane = FEW ? threadIdx.x : threadIdx.x & 31;
  constexpr int LANES = FEW ? LCE_THREADS : 32;
  const int row = FEW ? blockIdx.x : blockIdx.x * LCE_WARPS + warp;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    ce_flags[0] = 0;
    *ticket = 0;
  }
  if (row >= rows) return;
  const long long t = targets[row];
  float acc = 0.f;
  int used = 0;
  if (t >= 0 && t < V) {
    const uint4* a = reinterpret_cast<const uint4*>(x + row * ldx);
    const uint4* b = reinterpret_cast<const uint4*>(w + t * ldw);
    const int vecs = H / 8;
    float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll 4
    for (int i = lane; i < vecs; i += LANES) {
      const uint4 u = a[i], v = b[i];
      used += ((u.x | u.y | u.z | u.w) & 0x7fff7fffu) != 0;
      s0 = fma2(unpack_bf16(u.x), unpack_bf16(v.x), s0);
      s1 = fma2(unpack_bf16(u.y), unpack_bf16(v.y), s1);
      s0 = fma2(unpack_bf16(u.z), unpack_bf16(v.z), s0);
      s1 = fma2(unpack_bf16(u.w), unpack_bf16(v.w), s1);
    }
    acc = warp_sum((s0.x + s0.y) + (s1.x + s1.y));
    used = __reduce_add_sync(0xffffffffu, used);
  }
  if (FEW) {
    if ((threadIdx.x & 31) == 0) {
      s_part[warp] = acc;
      s_used[warp] = used;
    }
    __syncthreads();
    acc = 0.f;
    used = 0;
#pragma unroll
    for (int i = 0; i < LCE_WARPS; ++i) {
      acc += s_part[i];
      used += s_used[i];
    }
  }
  if (lane == 0) {
    ref[row] = acc;
    grow[row] = lce_grow(used);
    ce_max[row] = 0;
    if (row % 128 == 0) ce_flags[1 + row / 128] = 0;
  }
}

// xs[row, :] = bf16(f * x[row, :]), by one warp.  A row without a target (f = 0) gives zeros whatever it holds.
__device__ __forceinline__ void lce_scale_row(const void* x, long long ldx, void* xs, long long row, int H, float f, int lane) {
  const int vecs = H / 8;
  uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(xs) + row * H);
  if (f == 0.f) {
    for (int i = lane; i < vecs; i += 32) dst[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(x) + row * ldx);
#pragma unroll 4
  for (int i = lane; i < vecs; i += 32) {
    const uint4 u = src[i];
    const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), e = unpack_bf16(u.w);
    dst[i] = make_uint4(pack_bf16(f * a.x, f * a.y), pack_bf16(f * b.x, f * b.y), pack_bf16(f * c.x, f * c.y),
                        pack_bf16(f * e.x, f * e.y));
  }
}

// The target's entry of a row of exponentials and the row's factor, from S (without the target) and the row's 1 / Z.
__device__ __forceinline__ float lce_patch_row(__nv_bfloat16* entry, float S, float inv_z) {
  const __nv_bfloat16 q = __float2bfloat16_rn(-S);
  *entry = q;
  const float rounded = -__bfloat162float(q);
  return rounded > 0.f && rounded <= FLT_MAX ? inv_z * (S / rounded) : inv_z;
}

// Block: 8 rows (a 32-byte sector of every tile's sums) x 32 tiles at a time; eight threads finish the rows, then each
// warp scales one row of X.  (32 rows per block left half of the SMs without one: 29 us for 8192 x 2048, V = 50304.)
// With few rows one per block (one row of 2292 sums: 7 us with eight).
template <int LCE_ROWS>
__global__ void __launch_bounds__(LCE_THREADS)
lce_finish_kernel(const olb_lce_finish_desc d) {
  constexpr int TILES = LCE_THREADS / LCE_ROWS;
  __shared__ float s_sum[LCE_WARPS][LCE_ROWS];
  __shared__ float s_factor[LCE_ROWS];
  __shared__ double s_total[LCE_WARPS];
  __shared__ bool s_last;
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.x * LCE_ROWS;
  const int sub = threadIdx.x % LCE_ROWS, row = row0 + sub;
  const bool ok = row < d.rows;
  const long long t = ok ? d.targets[row] : -1;
  {
    float s = 0.f;
    if (t >= 0 && t < d.V) {
      const float* p = d.part + row;
#pragma unroll 8
      for (int i = threadIdx.x / LCE_ROWS; i < d.ntiles; i += TILES) s += p[i * d.part_ld];
    }
#pragma unroll
    for (int o = 16; o >= LCE_ROWS; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane < LCE_ROWS) s_sum[warp][sub] = s;
  }
  __syncthreads();
  if (threadIdx.x < LCE_ROWS) {
    float factor = 0.f;
    if (ok) {
      float loss = 0.f, sum = 0.f, base = 0.f, inv_z = 0.f;
      if (t >= 0 && t < d.V) {
        float S = 0.f;
#pragma unroll
        for (int i = 0; i < LCE_WARPS; ++i) S += s_sum[i][sub];
        const float lt = d.ref[row];
        const unsigned m = d.ce_max[row];
        float z;
        if (m == 0) {  // the exponentials are relative to the target's logit
          z = 1.f + S;
          loss = log1pf(S);
          base = lt;
        } else {       // ... to the row's maximum
          base = __uint_as_float((m & 0x80000000u) ? (m & 0x7fffffffu) : ~m);
          z = S + expf(lt - base);
          loss = logf(z) + (base - lt);
        }
        sum = S;
        inv_z = 1.f / z;
        if (d.scale) inv_z *= *d.scale;
        if (d.E) factor = lce_patch_row(static_cast<__nv_bfloat16*>(d.E) + row * d.lde + t, S, inv_z);
      }
      d.loss[row] = loss;
      if (d.sum) {
        d.sum[row] = sum;
        d.base[row] = base;
        d.inv_z[row] = inv_z;
      }
      if (d.factor) d.factor[row] = factor;
    }
    s_factor[sub] = factor;
  }
  __syncthreads();
  if (d.xs) {
    static_assert(LCE_ROWS <= LCE_WARPS, "a warp per row");
    if (warp < LCE_ROWS && row0 + warp < d.rows) lce_scale_row(d.x, d.ldx, d.xs, row0 + warp, d.H, s_factor[warp], lane);
  }
  if (d.total == nullptr) return;
  // the last block to arrive sums the rows' losses, in a fixed order
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(d.ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double acc = 0.0;  // a long batch has many losses of one sign
#pragma unroll 16
  for (long long i = threadIdx.x; i < d.n_all; i += LCE_THREADS) acc += __ldcg(d.loss_all + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) s_total[warp] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int i = 0; i < LCE_WARPS; ++i) sum += s_total[i];
    // a division, as a mean is defined: 0 / 0 where no row has a target
    *d.total = static_cast<float>(d.total_scale ? sum / *d.total_scale : sum);
  }
}

__global__ void __launch_bounds__(LCE_THREADS)
lce_patch_kernel(const float* __restrict__ sum, const float* __restrict__ inv_z, const long long* __restrict__ targets, int rows,
                 int V, float* __restrict__ factor, int v0, int cols, __nv_bfloat16* __restrict__ E, long long lde) {
  const int row = blockIdx.x * LCE_THREADS + threadIdx.x;
  if (row >= rows) return;
  const long long t = targets[row];
  __nv_bfloat16 entry;
  float f = 0.f;
  if (t >= 0 && t < V) {
    f = lce_patch_row(&entry, sum[row], inv_z[row]);
    if (E && t >= v0 && t < v0 + cols) E[row * lde + (t - v0)] = entry;
  }
  if (factor) factor[row] = f;
}

// One warp per row.
__global__ void __launch_bounds__(LCE_THREADS)
lce_scale_rows_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, const float* __restrict__ factor,
                      const float* __restrict__ grad, long long grad_stride, int rows, int H, float* __restrict__ row_factor,
                      __nv_bfloat16* __restrict__ xs) {
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * LCE_WARPS + (threadIdx.x >> 5);
  if (row >= rows) return;
  const float f0 = factor[row];
  const float f = f0 == 0.f ? 0.f : f0 * grad[row * grad_stride];
  if (lane == 0) row_factor[row] = f;
  if (xs) lce_scale_row(x, ldx, xs, row, H, f, lane);
}

// 8 columns per thread.
__global__ void __launch_bounds__(LCE_THREADS)
lce_round_rows_kernel(const float4* __restrict__ src, int rows, int H, const float* __restrict__ row_factor,
                      uint4* __restrict__ out) {
  const int vecs = H / 8;
  const long long total = static_cast<long long>(rows) * vecs;
  for (long long i = blockIdx.x * static_cast<long long>(LCE_THREADS) + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * LCE_THREADS) {
    const float4 a = __ldcs(src + 2 * i), b = __ldcs(src + 2 * i + 1);
    const float f = row_factor[i / vecs];
    out[i] = make_uint4(pack_bf16(f * a.x, f * a.y), pack_bf16(f * a.z, f * a.w), pack_bf16(f * b.x, f * b.y),
                        pack_bf16(f * b.z, f * b.w));
  }
}

template <bool SRC_BF16, bool ACCUMULATE>
__global__ void __launch_bounds__(LCE_THREADS)
lce_scale_out_kernel(const void* __restrict__ src_, long long vecs, const float* __restrict__ grad, uint4* __restrict__ dst) {
  const float g = *grad;
  for (long long i = blockIdx.x * static_cast<long long>(LCE_THREADS) + threadIdx.x; i < vecs;
       i += static_cast<long long>(gridDim.x) * LCE_THREADS) {
    float f[8];
    if (SRC_BF16) {
      const uint4 u = static_cast<const uint4*>(src_)[i];
      const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), e = unpack_bf16(u.w);
      f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = e.x; f[7] = e.y;
    } else {
      const float4 u = __ldcs(static_cast<const float4*>(src_) + 2 * i), v = __ldcs(static_cast<const float4*>(src_) + 2 * i + 1);
      f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w; f[4] = v.x; f[5] = v.y; f[6] = v.z; f[7] = v.w;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] *= g;
    if (ACCUMULATE) {
      const uint4 o = dst[i];
      const float2 a = unpack_bf16(o.x), b = unpack_bf16(o.y), c = unpack_bf16(o.z), e = unpack_bf16(o.w);
      f[0] += a.x; f[1] += a.y; f[2] += b.x; f[3] += b.y; f[4] += c.x; f[5] += c.y; f[6] += e.x; f[7] += e.y;
    }
    dst[i] = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
}

static bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
// A launch that may begin before the one before it on the stream has ended: the kernel waits for that itself.
template <typename... P, typename... A>
static int launch_waiting(void (*kernel)(P...), int grid, cudaStream_t stream, A... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(LCE_THREADS);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...) == cudaSuccess ? 0 : -2;
}
static int launched() { return cudaGetLastError() == cudaSuccess ? 0 : -2; }

}  // namespace olb

using namespace olb;

extern "C" int olb_lce_prep(const void* x, long long ldx, const void* w, long long ldw, const long long* targets, int rows,
                            int H, int V, float* ref, float* grow, unsigned* ce_max, int* ce_flags, unsigned* ticket,
                            const long long* all_targets, long long n_all, float* count, cudaStream_t stream) {
  if (H % 8 || ldx % 8 || ldw % 8 || misaligned(x) || misaligned(w) || n_all >= (1ll << 31)) return -1;
  if (rows <= 0) return 0;
  const auto* xb = static_cast<const __nv_bfloat16*>(x);
  const auto* wb = static_cast<const __nv_bfloat16*>(w);
  const int extra = count != nullptr ? 1 : 0;
  if (rows <= 148 * 8)
    lce_prep_kernel<true><<<rows + extra, LCE_THREADS, 0, stream>>>(xb, ldx, wb, ldw, targets, rows, H, V, ref, grow, ce_max,
                                                                    ce_flags, ticket, all_targets, n_all, count);
  else
    lce_prep_kernel<false><<<(rows + LCE_WARPS - 1) / LCE_WARPS + extra, LCE_THREADS, 0, stream>>>(
        xb, ldx, wb, ldw, targets, rows, H, V, ref, grow, ce_max, ce_flags, ticket, all_targets, n_all, count);
  return launched();
}

extern "C" int olb_lce_finish(const olb_lce_finish_desc* d, cudaStream_t stream) {
  if ((d->xs && (d->H % 8 || d->ldx % 8 || misaligned(d->x) || misaligned(d->xs))) || (d->total && !d->ticket) ||
      (d->sum && (!d->base || !d->inv_z)))
    return -1;
  if (d->rows <= 0) return 0;
  if (d->rows <= 148 * 2) return launch_waiting(lce_finish_kernel<1>, d->rows, stream, *d);
  return launch_waiting(lce_finish_kernel<8>, (d->rows + 7) / 8, stream, *d);
}

extern "C" int olb_lce_patch(const float* sum, const float* inv_z, const long long* targets, int rows, int V, float* factor,
                             int v0, int cols, void* E, long long lde, cudaStream_t stream) {
  if (rows <= 0) return 0;
  lce_patch_kernel<<<(rows + LCE_THREADS - 1) / LCE_THREADS, LCE_THREADS, 0, stream>>>(
      sum, inv_z, targets, rows, V, factor, v0, cols, static_cast<__nv_bfloat16*>(E), lde);
  return launched();
}

extern "C" int olb_lce_scale_rows(const void* x, long long ldx, const float* factor, const float* grad, long long grad_stride,
                                  int rows, int H, float* row_factor, void* xs, cudaStream_t stream) {
  if (H % 8 || ldx % 8 || misaligned(x) || misaligned(xs)) return -1;
  if (rows <= 0) return 0;
  lce_scale_rows_kernel<<<(rows + LCE_WARPS - 1) / LCE_WARPS, LCE_THREADS, 0, stream>>>(
      static_cast<const __nv_bfloat16*>(x), ldx, factor, grad, grad_stride, rows, H, row_factor, static_cast<__nv_bfloat16*>(xs));
  return launched();
}

extern "C" int olb_lce_round_rows(const float* src, int rows, int H, const float* row_factor, void* out, cudaStream_t stream) {
  if (H % 8 || misaligned(src) || misaligned(out)) return -1;
  if (rows <= 0) return 0;
  const long long blocks = (static_cast<long long>(rows) * (H / 8) + LCE_THREADS - 1) / LCE_THREADS;
  lce_round_rows_kernel<<<static_cast<int>(blocks < 148 * 16 ? blocks : 148 * 16), LCE_THREADS, 0, stream>>>(
      reinterpret_cast<const float4*>(src), rows, H, row_factor, static_cast<uint4*>(out));
  return launched();
}

extern "C" int olb_lce_scale_out(const void* src, int src_bf16, long long n, const float* grad, void* dst, int accumulate,
                                 cudaStream_t stream) {
  if (n % 8 || misaligned(src) || misaligned(dst)) return -1;
  if (n <= 0) return 0;
  const long long vecs = n / 8, blocks = (vecs + LCE_THREADS - 1) / LCE_THREADS;
  const int grid = static_cast<int>(blocks < 148 * 16 ? blocks : 148 * 16);
  uint4* out = static_cast<uint4*>(dst);
  if (src_bf16) {
    if (accumulate) lce_scale_out_kernel<true, true><<<grid, LCE_THREADS, 0, stream>>>(src, vecs, grad, out);
    else lce_scale_out_kernel<true, false><<<grid, LCE_THREADS, 0, stream>>>(src, vecs, grad, out);
  } else {
    if (accumulate) lce_scale_out_kernel<false, true><<<grid, LCE_THREADS, 0, stream>>>(src, vecs, grad, out);
    else lce_scale_out_kernel<false, false><<<grid, LCE_THREADS, 0, stream>>>(src, vecs, grad, out);
  }
  return launched();
}
