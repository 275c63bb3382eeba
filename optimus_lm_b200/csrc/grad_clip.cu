// Norm over a list of gradient tensors and their scaling to a maximum norm.
//
//   norm = sqrt(sum_i sum_j g_ij^2)  (or max |g_ij|)        g_ij *= min(1, max_norm / (norm + eps))
//
// Two launches read the list from their own parameters (pointer, length and first piece of every tensor, up to 2040 of
// them), so that a call needs no table in device memory and no copy, and a captured graph carries everything it uses.
// Tensors are cut into pieces of 32 KB on 16-byte boundaries; a block owns a contiguous run of pieces, eight 16-byte
// loads of a thread in flight.  Bound by HBM: 2 N bytes to read for the norm, 2 N to read and 2 N to write for the
// scaling, which walks every block's run backwards, so that it starts on what the first launch left in the L2.
//
// Squares are summed in fp32 over one 16-byte vector and in fp64 beyond it: one fp64 addition for 8 (4) elements costs
// nothing against the loads, and neither the number of elements nor the order of sizes shows in the result.  A vector
// whose fp32 sum leaves [1e-30, 1e30] is squared in fp64.  Fixed pieces, fixed runs, a fixed tree: the same bits every run.
// The second launch sums the first one's block results itself, in every block (a few hundred values from the L2).
#include <cmath>
#include <cstdint>

#include "olb_api.h"
#include "ptx.cuh"

namespace olb {

constexpr int CLIP_THREADS = 256;
constexpr int CLIP_VECS = 8;                                        // 16-byte vectors per thread and piece
constexpr long long CLIP_PIECE = 16ll * CLIP_THREADS * CLIP_VECS;   // bytes

// n: elements, bit 31 set for fp32; first: number of this tensor's first piece in the launch
struct ClipEntry {
  unsigned long long ptr;
  unsigned n, first;
};
template <int CAP>
struct ClipTable {
  ClipEntry e[CAP];
  int count;
  unsigned pieces;
};
// Launch parameters of 4, 13 and 32 KB: every launch copies all of them (300 tensors took 8 us longer in the largest form
// than 250 in the smallest).
constexpr int CLIP_SMALL = 250, CLIP_MIDDLE = 800, CLIP_LARGE = 2040;

template <int CAP>
__device__ __forceinline__ int clip_find(const ClipTable<CAP>& t, unsigned piece) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first <= piece) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The aligned base of a piece and the byte range of it that belongs to the tensor.
struct ClipPiece {
  unsigned long long base;
  int lo, hi;   // bytes from base; whole piece: 0, CLIP_PIECE
  bool fp32;
};
__device__ __forceinline__ ClipPiece clip_piece(const ClipEntry& e, unsigned piece) {
  ClipPiece p;
  p.fp32 = (e.n >> 31) != 0;
  const unsigned long long end = e.ptr + static_cast<unsigned long long>(e.n & 0x7fffffffu) * (p.fp32 ? 4 : 2);
  p.base = (e.ptr & ~15ull) + static_cast<unsigned long long>(piece - e.first) * CLIP_PIECE;
  p.lo = e.ptr > p.base ? static_cast<int>(e.ptr - p.base) : 0;
  p.hi = end - p.base < CLIP_PIECE ? static_cast<int>(end - p.base) : static_cast<int>(CLIP_PIECE);
  return p;
}

// A 16-byte vector at byte `at` of a piece: the elements outside [lo, hi) read as zero.
__device__ __forceinline__ uint4 clip_load_part(const ClipPiece& p, int at) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (p.fp32) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + 4 * i >= p.lo && at + 4 * i < p.hi) w[i] = *reinterpret_cast<const uint32_t*>(p.base + at + 4 * i);
    v = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + 2 * i >= p.lo && at + 2 * i < p.hi)
        w[i >> 1] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p.base + at + 2 * i)) << (16 * (i & 1));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
__device__ __forceinline__ void clip_store_part(const ClipPiece& p, int at, const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if (p.fp32) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + 4 * i >= p.lo && at + 4 * i < p.hi) *reinterpret_cast<uint32_t*>(p.base + at + 4 * i) = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + 2 * i >= p.lo && at + 2 * i < p.hi)
        *reinterpret_cast<uint16_t*>(p.base + at + 2 * i) = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
  }
}
__device__ __forceinline__ void clip_load(const ClipPiece& p, uint4 (&v)[CLIP_VECS]) {
  if (p.lo == 0 && p.hi == CLIP_PIECE) {
#pragma unroll
    for (int i = 0; i < CLIP_VECS; ++i)
      v[i] = *reinterpret_cast<const uint4*>(p.base + 16 * (i * CLIP_THREADS + threadIdx.x));
    return;
  }
#pragma unroll
  for (int i = 0; i < CLIP_VECS; ++i) {
    const int at = 16 * (i * CLIP_THREADS + static_cast<int>(threadIdx.x));
    v[i] = make_uint4(0, 0, 0, 0);
    if (at >= p.lo && at + 16 <= p.hi) v[i] = *reinterpret_cast<const uint4*>(p.base + at);
    else if (at + 16 > p.lo && at < p.hi) v[i] = clip_load_part(p, at);
  }
}

__device__ __forceinline__ float clip_lo_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float clip_hi_bf16(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ double clip_squares(const uint4& v, bool fp32) {
  float f[8];
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float s = 0.f;
  if (fp32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = __uint_as_float(w[i]);
      f[4 + i] = 0.f;
      s = fmaf(f[i], f[i], s);
    }
  } else {
    float s1 = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = clip_lo_bf16(w[i]);
      f[2 * i + 1] = clip_hi_bf16(w[i]);
      s = fmaf(f[2 * i], f[2 * i], s);
      s1 = fmaf(f[2 * i + 1], f[2 * i + 1], s1);
    }
    s += s1;
  }
  if (s >= 1e-30f && s <= 1e30f) return static_cast<double>(s);
  if (((w[0] | w[1] | w[2] | w[3]) & (fp32 ? 0x7fffffffu : 0x7fff7fffu)) == 0) return 0.0;  // a row without a gradient
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) d += static_cast<double>(f[i]) * static_cast<double>(f[i]);
  return d;
}
// Largest absolute value as a bit pattern: the order of non-negative floats is that of their bits, and a NaN is above
// all of them.
__device__ __forceinline__ unsigned clip_largest(const uint4& v, bool fp32, unsigned m) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (fp32) {
      m = max(m, w[i] & 0x7fffffffu);
    } else {
      m = max(m, (w[i] << 16) & 0x7fff0000u);
      m = max(m, w[i] & 0x7fff0000u);
    }
  }
  return m;
}

__device__ __forceinline__ double clip_block_sum(double v, double* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < CLIP_THREADS / 32; ++i) v += s[i];
  return v;
}
__device__ __forceinline__ unsigned clip_block_max(unsigned v, unsigned* s) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < CLIP_THREADS / 32; ++i) v = max(v, s[i]);
  return v;
}

// partial[block]: sum of squares (fp64), or the largest absolute value's bits in the lower half.
template <int CAP, bool INF>
__global__ void __launch_bounds__(CLIP_THREADS, 4)
grad_norm_kernel(const __grid_constant__ ClipTable<CAP> t, unsigned per_block, double* __restrict__ partial) {
  grid_launch_dependents();
  __shared__ double s[CLIP_THREADS / 32];
  const unsigned begin = blockIdx.x * per_block, end = min(begin + per_block, t.pieces);
  double sum = 0.0;
  unsigned top = 0;
  int k = begin < end ? clip_find(t, begin) : 0;
  for (unsigned piece = begin; piece < end; ++piece) {
    while (k + 1 < t.count && t.e[k + 1].first <= piece) ++k;
    const ClipPiece p = clip_piece(t.e[k], piece);
    uint4 v[CLIP_VECS];
    clip_load(p, v);
#pragma unroll
    for (int i = 0; i < CLIP_VECS; ++i) {
      if (INF) top = clip_largest(v[i], p.fp32, top);
      else sum += clip_squares(v[i], p.fp32);
    }
  }
  if (INF) {
    top = clip_block_max(top, reinterpret_cast<unsigned*>(s));
    if (threadIdx.x == 0) partial[blockIdx.x] = __longlong_as_double(static_cast<long long>(top));
  } else {
    sum = clip_block_sum(sum, s);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
  }
}

// `partial` comes from the launch before, under which grad_scale_kernel starts: loads from the L2, which stay behind the wait.
template <bool INF>
__device__ __forceinline__ float clip_norm(const double* partial, int nparts, double* s) {
  if (INF) {
    unsigned top = 0;
    for (int i = threadIdx.x; i < nparts; i += CLIP_THREADS)
      top = max(top, static_cast<unsigned>(__double_as_longlong(__ldcg(partial + i))));
    return __uint_as_float(clip_block_max(top, reinterpret_cast<unsigned*>(s)));
  }
  double sum = 0.0;
  for (int i = threadIdx.x; i < nparts; i += CLIP_THREADS) sum += __ldcg(partial + i);
  return static_cast<float>(sqrt(clip_block_sum(sum, s)));
}

template <bool INF>
__global__ void __launch_bounds__(CLIP_THREADS)
grad_norm_finish_kernel(const double* partial, int nparts, float* norm_out) {
  __shared__ double s[CLIP_THREADS / 32];
  const float norm = clip_norm<INF>(partial, nparts, s);
  if (threadIdx.x == 0) *norm_out = norm;
}

template <int CAP, bool INF>
__global__ void __launch_bounds__(CLIP_THREADS, 4)
grad_scale_kernel(const __grid_constant__ ClipTable<CAP> t, unsigned per_block, const double* partial, int nparts,
                  float max_norm, float eps, float* norm_out) {
  grid_dependency_wait();
  __shared__ double s[CLIP_THREADS / 32];
  const float norm = clip_norm<INF>(partial, nparts, s);
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) *norm_out = norm;
  const float factor = max_norm / (norm + eps);
  if (factor >= 1.f) return;   // nothing to scale (a NaN is not: it reaches the gradients, as a product would)
  const unsigned begin = blockIdx.x * per_block, end = min(begin + per_block, t.pieces);
  if (begin >= end) return;
  int k = clip_find(t, end - 1);
  for (unsigned piece = end; piece-- > begin;) {
    while (t.e[k].first > piece) --k;
    const ClipPiece p = clip_piece(t.e[k], piece);
    uint4 v[CLIP_VECS];
    clip_load(p, v);
    const bool whole = p.lo == 0 && p.hi == CLIP_PIECE;
#pragma unroll
    for (int i = 0; i < CLIP_VECS; ++i) {
      uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = p.fp32 ? __float_as_uint(factor * __uint_as_float(w[j]))
                      : pack_bf16(factor * clip_lo_bf16(w[j]), factor * clip_hi_bf16(w[j]));
      v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      const int at = 16 * (i * CLIP_THREADS + static_cast<int>(threadIdx.x));
      if (whole || (at >= p.lo && at + 16 <= p.hi)) *reinterpret_cast<uint4*>(p.base + at) = v[i];
      else if (at + 16 > p.lo && at < p.hi) clip_store_part(p, at, v[i]);
    }
  }
}

static int clip_grid(unsigned pieces, unsigned* per_block) {
  const unsigned most = 148 * 4;
  *per_block = (pieces + most - 1) / most;
  return static_cast<int>((pieces + *per_block - 1) / *per_block);
}

// Fills the table with tensors from *next on; returns the number of pieces (0: none left).
template <int CAP>
static unsigned clip_fill(ClipTable<CAP>& t, const olb_clip_tensor* list, int n, int* next, long long* done) {
  constexpr long long MOST = 1ll << 30;  // elements of one entry; longer tensors take several
  t.count = 0;
  unsigned long long pieces = 0;
  while (*next < n && t.count < CAP && pieces < (1ull << 30)) {
    const olb_clip_tensor& x = list[*next];
    const long long left = x.n - *done;
    if (left > 0) {
      const int es = x.fp32 ? 4 : 2;
      const long long take = left < MOST ? left : MOST;
      const unsigned long long ptr = reinterpret_cast<unsigned long long>(x.ptr) + static_cast<unsigned long long>(*done) * es;
      t.e[t.count].ptr = ptr;
      t.e[t.count].n = static_cast<unsigned>(take) | (x.fp32 ? 0x80000000u : 0u);
      t.e[t.count].first = static_cast<unsigned>(pieces);
      ++t.count;
      pieces += ((ptr & 15) + static_cast<unsigned long long>(take) * es + CLIP_PIECE - 1) / CLIP_PIECE;
      *done += take;
    }
    if (*done >= x.n) {
      ++*next;
      *done = 0;
    }
  }
  t.pieces = static_cast<unsigned>(pieces);
  return t.pieces;
}

template <int CAP, bool INF>
static int clip_run(const olb_clip_tensor* list, int n, int scale, float max_norm, float eps, double* partial, int room,
                    float* norm_out, cudaStream_t stream) {
  static thread_local ClipTable<CAP> t;  // 32 KB: not on the stack of whatever thread calls
  unsigned per = 0;
  int nparts = 0, next = 0;
  long long done = 0;
  while (clip_fill(t, list, n, &next, &done)) {
    const int grid = clip_grid(t.pieces, &per);
    if (nparts + grid > room) return -2;
    grad_norm_kernel<CAP, INF><<<grid, CLIP_THREADS, 0, stream>>>(t, per, partial + nparts);
    nparts += grid;
  }
  if (!scale || nparts == 0) {
    grad_norm_finish_kernel<INF><<<1, CLIP_THREADS, 0, stream>>>(partial, nparts, norm_out);
  } else {
    next = 0;
    done = 0;
    float* out = norm_out;
    while (clip_fill(t, list, n, &next, &done)) {
      const int grid = clip_grid(t.pieces, &per);
      // the first one is put in place under the last of the norm's launches
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr.val.programmaticStreamSerializationAllowed = out != nullptr;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(grid);
      cfg.blockDim = dim3(CLIP_THREADS);
      cfg.stream = stream;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      if (cudaLaunchKernelEx(&cfg, grad_scale_kernel<CAP, INF>, t, per, static_cast<const double*>(partial), nparts, max_norm,
                             eps, out) != cudaSuccess)
        return -3;
      out = nullptr;
    }
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace olb

using namespace olb;

extern "C" int olb_grad_clip_parts(const olb_clip_tensor* list, int n) {
  // an entry takes at most 2^30 elements and a launch at most CLIP_SMALL entries (the smaller table)
  long long entries = 0;
  for (int i = 0; i < n; ++i) entries += list[i].n > 0 ? (list[i].n + (1ll << 30) - 1) >> 30 : 0;
  return static_cast<int>((entries / CLIP_SMALL + 1) * 148 * 4);
}

extern "C" int olb_grad_clip(const olb_clip_tensor* list, int n, int inf_norm, int scale, float max_norm, float eps,
                             double* partial, int room, float* norm_out, cudaStream_t stream) {
  if (n < 0 || norm_out == nullptr || partial == nullptr) return -1;
  for (int i = 0; i < n; ++i)
    if (list[i].n < 0 || (reinterpret_cast<uintptr_t>(list[i].ptr) & (list[i].fp32 ? 3 : 1))) return -1;
  if (n <= CLIP_SMALL)
    return inf_norm ? clip_run<CLIP_SMALL, true>(list, n, scale, max_norm, eps, partial, room, norm_out, stream)
                    : clip_run<CLIP_SMALL, false>(list, n, scale, max_norm, eps, partial, room, norm_out, stream);
  if (n <= CLIP_MIDDLE)
    return inf_norm ? clip_run<CLIP_MIDDLE, true>(list, n, scale, max_norm, eps, partial, room, norm_out, stream)
                    : clip_run<CLIP_MIDDLE, false>(list, n, scale, max_norm, eps, partial, room, norm_out, stream);
  return inf_norm ? clip_run<CLIP_LARGE, true>(list, n, scale, max_norm, eps, partial, room, norm_out, stream)
                  : clip_run<CLIP_LARGE, false>(list, n, scale, max_norm, eps, partial, room, norm_out, stream);
}
