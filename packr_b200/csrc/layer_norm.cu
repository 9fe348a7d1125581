// Layer norm over the last dimension, forward and backward, with an optional
// residual added to the input first:
//   s = x + residual                      (f32, never rounded)
//   h = (s - mean(s)) * rstd,  rstd = 1 / sqrt(mean((s - mean)^2) + eps)
//   y = h * weight + bias
//   g = dy * weight;  dx = dresidual = rstd * (g - mean(g) - h * mean(g * h))
//   dweight[n] = sum over rows of dy * h;  dbias[n] = sum over rows of dy
// x, residual, y, dy, dx share one type (bf16 or f32), weight, bias and their
// gradients another; sums and statistics are f32.
//
// Bound by HBM: one read of each input and one write of each output.  A row
// lives in the registers of `blockDim.x` threads, E elements each, so mean and
// centred variance are two exact passes over registers; `blockDim.y` rows are
// in flight per CTA and the next row's loads are issued before the current
// row's reductions.  The backward recomputes h from x and residual instead of
// a stored sum: the sum would have to be rounded (bf16) or read back at twice
// the width, for the same number of bytes.  Its CTAs are persistent: a thread
// owns the same E columns in every row it visits and carries their dweight /
// dbias sums in registers (E = 16: in its own shared-memory words); the CTAs'
// sums go to the workspace and a second launch adds them in a fixed order, so
// results do not depend on timing.  Rows wider than the register path are
// walked in strides of the CTA, three passes over L2-resident data.
#include "common.cuh"

namespace packr {
namespace norm {

constexpr int kMaxRowThreads = 1024;
constexpr long long kMaxRegN = 16LL * kMaxRowThreads;  // widest row held in registers
constexpr int kMaxGroups = 8;                          // rows in flight per CTA (named barriers 1..8)

template <class T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<uint16_t> {  // bf16 bit pattern
  static __device__ __forceinline__ float get(uint16_t v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ uint16_t put(float v) { return (uint16_t)(pack_bf16x2_rne(v, 0.0f) & 0xFFFFu); }
};

// One thread's E elements of a row.  VEC: vectors of VW = 16 / sizeof(x type)
// elements, vector v of thread t covering columns (v * nt + t) * VW ..; else
// element e is column e * nt + t (any N, any alignment; still coalesced).
template <class T, int E>
struct Raw {
  static constexpr int kWords = E * (int)sizeof(T) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ float at(int e) const {
    if (sizeof(T) == 4) return __uint_as_float(w[e]);
    return __uint_as_float((e & 1) ? (w[e >> 1] & 0xFFFF0000u) : (w[e >> 1] << 16));
  }
  __device__ __forceinline__ void set_scalar(int e, T v) {
    if (sizeof(T) == 4) {
      w[e] = __float_as_uint(Elem<T>::get(v));
    } else if (e & 1) {
      w[e >> 1] |= __float_as_uint(Elem<T>::get(v));
    } else {
      w[e >> 1] = __float_as_uint(Elem<T>::get(v)) >> 16;
    }
  }
};

// Columns of a thread's elements when the x type has XB bytes.
template <int XB, int E, bool VEC>
struct Cols {
  static constexpr int VW = 16 / XB;
  static __device__ __forceinline__ int col(int e, int t, int nt) {
    return VEC ? ((e / VW) * nt + t) * VW + e % VW : e * nt + t;
  }
  static __device__ __forceinline__ bool valid(int e, int t, int nt, int N) { return col(e, t, nt) < N; }
};

// Loads the thread's E elements of row p (P: element type, XB: bytes of the x
// type, which sets the column layout).  Elements past N read as zero.
template <class P, int XB, int E, bool VEC, bool STREAM>
__device__ __forceinline__ void load_row(Raw<P, E>& r, const P* __restrict__ p, int t, int nt, int N) {
  using C = Cols<XB, E, VEC>;
#pragma unroll
  for (int i = 0; i < Raw<P, E>::kWords; ++i) r.w[i] = 0u;
  if (VEC) {
    constexpr int VW = C::VW;
    constexpr int kWordsPerVec = VW * (int)sizeof(P) / 4;  // 2, 4 or 8
#pragma unroll
    for (int v = 0; v < E / VW; ++v) {
      const int c = (v * nt + t) * VW;
      if (c >= N) continue;
      uint32_t* d = r.w + v * kWordsPerVec;
      if constexpr (kWordsPerVec == 2) {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(p + c));
        d[0] = q.x; d[1] = q.y;
      } else {
#pragma unroll
        for (int k = 0; k < kWordsPerVec; k += 4) {
          const uint4* src = reinterpret_cast<const uint4*>(p + c) + k / 4;
          const uint4 q = STREAM ? __ldcs(src) : __ldg(src);
          d[k] = q.x; d[k + 1] = q.y; d[k + 2] = q.z; d[k + 3] = q.w;
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * nt + t;
      if (c < N) r.set_scalar(e, STREAM ? __ldcs(p + c) : __ldg(p + c));
    }
  }
}

template <class T, int E, bool VEC>
__device__ __forceinline__ void store_row(T* __restrict__ p, const float* v, int t, int nt, int N) {
  using C = Cols<(int)sizeof(T), E, VEC>;
  if (VEC) {
    constexpr int VW = C::VW;
#pragma unroll
    for (int k = 0; k < E / VW; ++k) {
      const int c = (k * nt + t) * VW;
      if (c >= N) continue;
      const float* s = v + k * VW;
      uint4 q;
      if (sizeof(T) == 4) {
        q = make_uint4(__float_as_uint(s[0]), __float_as_uint(s[1]), __float_as_uint(s[2]), __float_as_uint(s[3]));
      } else {
        q = make_uint4(pack_bf16x2_rne(s[0], s[1]), pack_bf16x2_rne(s[2], s[3]),
                       pack_bf16x2_rne(s[VW - 4], s[VW - 3]), pack_bf16x2_rne(s[VW - 2], s[VW - 1]));
      }
      __stcs(reinterpret_cast<uint4*>(p + c), q);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * nt + t;
      if (c < N) p[c] = Elem<T>::put(v[e]);
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

// Barrier of one row group (blockDim.x threads, a multiple of 32).
__device__ __forceinline__ void group_sync(int group, int nt) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(nt) : "memory");
}

// Sum over the row group's threads, the same value in each; `buf` holds one
// float per warp of the group.  The caller alternates two buffers.
__device__ __forceinline__ float group_sum(float v, float* buf, int group, int nt, int t) {
  v = warp_sum(v);
  if (nt == 32) return v;
  if ((t & 31) == 0) buf[t >> 5] = v;
  group_sync(group, nt);
  const int lane = t & 31;
  return warp_sum(lane < (nt >> 5) ? buf[lane] : 0.0f);
}

template <class T, class W, int E, bool VEC, bool RES>
__global__ void __launch_bounds__(kMaxRowThreads, 1)
    fwd_kernel(const T* __restrict__ x, const T* __restrict__ res, const W* __restrict__ weight,
               const W* __restrict__ bias, float eps, T* __restrict__ y, float* __restrict__ mean_out,
               float* __restrict__ rstd_out, long long M, int N) {
  using C = Cols<(int)sizeof(T), E, VEC>;
  __shared__ float bufs[kMaxGroups][2][32];
  const int t = threadIdx.x, nt = blockDim.x, group = threadIdx.y;
  const long long step = (long long)gridDim.x * blockDim.y;
  long long row = (long long)blockIdx.x * blockDim.y + group;
  if (row >= M) return;  // named barriers count this group's threads only
  Raw<T, E> rx, rr;
  load_row<T, sizeof(T), E, VEC, true>(rx, x + row * N, t, nt, N);
  if (RES) load_row<T, sizeof(T), E, VEC, true>(rr, res + row * N, t, nt, N);
  Raw<W, E> rw, rb;
  if (weight) load_row<W, sizeof(T), E, VEC, false>(rw, weight, t, nt, N);
  if (bias) load_row<W, sizeof(T), E, VEC, false>(rb, bias, t, nt, N);
  const float inv_n = 1.0f / (float)N;
  for (; row < M; row += step) {
    float v[E];
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = RES ? __fadd_rn(rx.at(e), rr.at(e)) : rx.at(e);
      sum += v[e];
    }
    if (row + step < M) {  // the next row's loads, in flight during this row's reductions
      load_row<T, sizeof(T), E, VEC, true>(rx, x + (row + step) * N, t, nt, N);
      if (RES) load_row<T, sizeof(T), E, VEC, true>(rr, res + (row + step) * N, t, nt, N);
    }
    const float mean = group_sum(sum, bufs[group][0], group, nt, t) * inv_n;
    float m2 = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] -= mean;
      if (C::valid(e, t, nt, N)) m2 = fmaf(v[e], v[e], m2);
    }
    const float var = group_sum(m2, bufs[group][1], group, nt, t) * inv_n;
    const float rstd = 1.0f / sqrtf(var + eps);
    if (t == 0) {
      if (mean_out) mean_out[row] = mean;
      if (rstd_out) rstd_out[row] = rstd;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float h = v[e] * rstd;
      v[e] = weight ? (bias ? fmaf(h, rw.at(e), rb.at(e)) : h * rw.at(e)) : (bias ? h + rb.at(e) : h);
    }
    store_row<T, E, VEC>(y + row * N, v, t, nt, N);
  }
}

// Any width: three passes of one CTA over its row.
template <class T, class W, bool RES>
__global__ void __launch_bounds__(256) fwd_wide_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                       const W* __restrict__ weight, const W* __restrict__ bias,
                                                       float eps, T* __restrict__ y, float* __restrict__ mean_out,
                                                       float* __restrict__ rstd_out, long long M, long long N) {
  __shared__ float bufs[2][32];
  const int t = threadIdx.x, nt = blockDim.x;
  for (long long row = blockIdx.x; row < M; row += gridDim.x) {
    const T* xr = x + row * N;
    const T* rr = RES ? res + row * N : nullptr;
    auto at = [&](long long c) {
      const float v = Elem<T>::get(__ldg(xr + c));
      return RES ? __fadd_rn(v, Elem<T>::get(__ldg(rr + c))) : v;
    };
    float sum = 0.0f;
    for (long long c = t; c < N; c += nt) sum += at(c);
    const float mean = group_sum(sum, bufs[0], 0, nt, t) / (float)N;
    float m2 = 0.0f;
    for (long long c = t; c < N; c += nt) {
      const float d = at(c) - mean;
      m2 = fmaf(d, d, m2);
    }
    const float rstd = 1.0f / sqrtf(group_sum(m2, bufs[1], 0, nt, t) / (float)N + eps);
    if (t == 0) {
      if (mean_out) mean_out[row] = mean;
      if (rstd_out) rstd_out[row] = rstd;
    }
    for (long long c = t; c < N; c += nt) {
      const float h = (at(c) - mean) * rstd;
      const float w = weight ? Elem<W>::get(__ldg(weight + c)) : 1.0f;
      const float b = bias ? Elem<W>::get(__ldg(bias + c)) : 0.0f;
      y[row * N + c] = Elem<T>::put(fmaf(h, w, b));
    }
  }
}

// dx, and this CTA's column sums: partial[blockIdx.x][0][n] = sum of dy * h,
// [1][n] = sum of dy over the CTA's rows (PARAMS).  ACC_SMEM: the column sums
// are kept in dynamic shared memory, two floats per element, each touched by
// its owner alone.  Dynamic shared memory: [groups][2][E][nt] floats, also the
// buffer in which the groups of a CTA are added.
template <class T, class W, int E, bool VEC, bool RES, bool PARAMS, bool ACC_SMEM>
__global__ void __launch_bounds__((E <= 8 && !ACC_SMEM) ? 512 : kMaxRowThreads, 1)
    bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ res,
               const W* __restrict__ weight, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
               T* __restrict__ dx, float* __restrict__ partial, long long M, int N) {
  using C = Cols<(int)sizeof(T), E, VEC>;
  __shared__ float bufs[kMaxGroups][2][2][32];
  extern __shared__ float acc_s[];
  const int t = threadIdx.x, nt = blockDim.x, group = threadIdx.y, groups = blockDim.y;
  const long long step = (long long)gridDim.x * groups;
  long long row = (long long)blockIdx.x * groups + group;
  float aw[ACC_SMEM ? 1 : E], ab[ACC_SMEM ? 1 : E];
  float* my = acc_s + (size_t)group * 2 * E * nt + t;  // + (which * E + e) * nt
  if (PARAMS) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (ACC_SMEM) {
        my[e * nt] = 0.0f;
        my[(E + e) * nt] = 0.0f;
      } else {
        aw[e] = 0.0f;
        ab[e] = 0.0f;
      }
    }
  }
  const float inv_n = 1.0f / (float)N;
  Raw<W, E> rw;
  if (weight) load_row<W, sizeof(T), E, VEC, false>(rw, weight, t, nt, N);
  Raw<T, E> rx, rr, rd;
  float mean_n = 0.0f, rstd_n = 0.0f;
  if (row < M) {
    load_row<T, sizeof(T), E, VEC, true>(rx, x + row * N, t, nt, N);
    if (RES) load_row<T, sizeof(T), E, VEC, true>(rr, res + row * N, t, nt, N);
    load_row<T, sizeof(T), E, VEC, true>(rd, dy + row * N, t, nt, N);
    mean_n = __ldg(mean_in + row);
    rstd_n = __ldg(rstd_in + row);
  }
  for (int parity = 0; row < M; row += step, parity ^= 1) {
    const float mean = mean_n, rstd = rstd_n;
    float h[E], g[E];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float v = RES ? __fadd_rn(rx.at(e), rr.at(e)) : rx.at(e);
      const float d = rd.at(e);  // zero past N: no sum sees those columns
      h[e] = C::valid(e, t, nt, N) ? (v - mean) * rstd : 0.0f;
      g[e] = weight ? d * rw.at(e) : d;
      s1 += g[e];
      s2 = fmaf(g[e], h[e], s2);
      if (PARAMS) {
        if (ACC_SMEM) {
          my[e * nt] = fmaf(d, h[e], my[e * nt]);
          my[(E + e) * nt] += d;
        } else {
          aw[e] = fmaf(d, h[e], aw[e]);
          ab[e] += d;
        }
      }
    }
    if (row + step < M) {
      load_row<T, sizeof(T), E, VEC, true>(rx, x + (row + step) * N, t, nt, N);
      if (RES) load_row<T, sizeof(T), E, VEC, true>(rr, res + (row + step) * N, t, nt, N);
      load_row<T, sizeof(T), E, VEC, true>(rd, dy + (row + step) * N, t, nt, N);
      mean_n = __ldg(mean_in + row + step);
      rstd_n = __ldg(rstd_in + row + step);
    }
    if (dx) {
      s1 = warp_sum(s1);
      s2 = warp_sum(s2);
      if (nt > 32) {
        float* b1 = bufs[group][parity][0];
        float* b2 = bufs[group][parity][1];
        if ((t & 31) == 0) {
          b1[t >> 5] = s1;
          b2[t >> 5] = s2;
        }
        group_sync(group, nt);
        const int lane = t & 31;
        s1 = warp_sum(lane < (nt >> 5) ? b1[lane] : 0.0f);
        s2 = warp_sum(lane < (nt >> 5) ? b2[lane] : 0.0f);
      }
      const float m1 = s1 * inv_n, m2 = s2 * inv_n;
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] = rstd * (g[e] - fmaf(h[e], m2, m1));
      store_row<T, E, VEC>(dx + row * N, h, t, nt, N);
    }
  }
  if (!PARAMS) return;
  if (!ACC_SMEM && groups > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      my[e * nt] = aw[e];
      my[(E + e) * nt] = ab[e];
    }
  }
  if (groups > 1) __syncthreads();
  if (group != 0) return;
  float* out = partial + (size_t)blockIdx.x * 2 * N;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float a, b;
    if (ACC_SMEM || groups > 1) {
      a = my[e * nt];
      b = my[(E + e) * nt];
      for (int q = 1; q < groups; ++q) {
        a += my[((size_t)q * 2 * E + e) * nt];
        b += my[((size_t)q * 2 * E + E + e) * nt];
      }
    } else {
      a = aw[e];
      b = ab[e];
    }
    const int c = C::col(e, t, nt);
    if (c < N) {
      out[c] = a;
      out[N + c] = b;
    }
  }
}

// Any width: dx in two passes of one CTA over its row.
template <class T, class W, bool RES>
__global__ void __launch_bounds__(256)
    bwd_wide_kernel(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ res,
                    const W* __restrict__ weight, const float* __restrict__ mean_in,
                    const float* __restrict__ rstd_in, T* __restrict__ dx, long long M, long long N) {
  __shared__ float bufs[2][32];
  const int t = threadIdx.x, nt = blockDim.x;
  for (long long row = blockIdx.x; row < M; row += gridDim.x) {
    const float mean = mean_in[row], rstd = rstd_in[row];
    auto hat = [&](long long c) {
      float v = Elem<T>::get(__ldg(x + row * N + c));
      if (RES) v = __fadd_rn(v, Elem<T>::get(__ldg(res + row * N + c)));
      return (v - mean) * rstd;
    };
    auto grad = [&](long long c) {
      const float d = Elem<T>::get(__ldg(dy + row * N + c));
      return weight ? d * Elem<W>::get(__ldg(weight + c)) : d;
    };
    float s1 = 0.0f, s2 = 0.0f;
    for (long long c = t; c < N; c += nt) {
      const float g = grad(c);
      s1 += g;
      s2 = fmaf(g, hat(c), s2);
    }
    const float m1 = group_sum(s1, bufs[0], 0, nt, t) / (float)N;
    const float m2 = group_sum(s2, bufs[1], 0, nt, t) / (float)N;
    for (long long c = t; c < N; c += nt)
      dx[row * N + c] = Elem<T>::put(rstd * (grad(c) - fmaf(hat(c), m2, m1)));
  }
}

// Any width: column sums of a slab of rows, one column per thread.
template <class T, bool RES>
__global__ void __launch_bounds__(256)
    bwd_wide_cols_kernel(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ res,
                         const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                         float* __restrict__ partial, long long M, long long N) {
  const long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= N) return;
  float a = 0.0f, b = 0.0f;
  for (long long row = blockIdx.y; row < M; row += gridDim.y) {
    float v = Elem<T>::get(__ldg(x + row * N + c));
    if (RES) v = __fadd_rn(v, Elem<T>::get(__ldg(res + row * N + c)));
    const float d = Elem<T>::get(__ldg(dy + row * N + c));
    a = fmaf(d, (v - __ldg(mean_in + row)) * __ldg(rstd_in + row), a);
    b += d;
  }
  float* out = partial + (size_t)blockIdx.y * 2 * N;
  out[c] = a;
  out[N + c] = b;
}

// out0[n] / out1[n] = sum over slabs of partial[slab][0 / 1][n] (`planes` 1:
// only out0): 32 columns per CTA, 16 warps each adding every 16th slab, then
// the 16 sums in order.
template <class W>
__global__ void __launch_bounds__(512) reduce_cols_kernel(const float* __restrict__ partial, int slabs, int planes,
                                                          long long N, W* __restrict__ out0, W* __restrict__ out1) {
  __shared__ float s[16][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane;
  const int which = blockIdx.y;
  W* out = which ? out1 : out0;
  if (out == nullptr) return;
  float a = 0.0f;
  if (c < N)
    for (int q = warp; q < slabs; q += 16) a += __ldcg(partial + ((size_t)q * planes + which) * N + c);
  s[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && c < N) {
    float v = s[0][lane];
#pragma unroll
    for (int q = 1; q < 16; ++q) v += s[q][lane];
    out[c] = Elem<W>::put(v);
  }
}

// ------------------------------------------------------------------ host
template <class W>
int reduce_cols(const float* partial, int slabs, int planes, long long N, W* out0, W* out1, cudaStream_t st) {
  reduce_cols_kernel<W><<<dim3((unsigned)((N + 31) / 32), (unsigned)planes), 512, 0, st>>>(partial, slabs, planes, N,
                                                                                           out0, out1);
  return launch_status();
}

constexpr int kSlabs = 148 * 2;  // upper bound of the CTAs that leave column sums (workspace)

struct Shape {
  int nt, groups, e;
};
// Threads per row (E = 8 elements each, 16 beyond 8192 columns) and rows per
// CTA (CTAs of about `target` threads).
inline Shape shape(long long N, int target) {
  Shape s{};
  s.e = N <= 8LL * kMaxRowThreads ? 8 : 16;
  s.nt = (int)(((N + s.e - 1) / s.e + 31) / 32 * 32);
  s.groups = target / s.nt;
  s.groups = s.groups < 1 ? 1 : s.groups > kMaxGroups ? kMaxGroups : s.groups;
  return s;
}

inline int grid_rows(long long M, int groups, int per_sm) {
  const long long want = (M + groups - 1) / groups;
  const long long cap = (long long)sm_count() * per_sm;
  return (int)(want < cap ? want : cap);
}

template <class T, class W, int E, bool VEC, bool RES>
int launch_fwd(const Shape& s, const void* x, const void* res, const void* w, const void* b, float eps, void* y,
               float* mean, float* rstd, long long M, long long N, cudaStream_t st) {
  const int threads = s.nt * s.groups;
  const int grid = grid_rows(M, s.groups, 2048 / threads > 0 ? 2048 / threads : 1);
  fwd_kernel<T, W, E, VEC, RES><<<grid, dim3(s.nt, s.groups), 0, st>>>(
      static_cast<const T*>(x), static_cast<const T*>(res), static_cast<const W*>(w), static_cast<const W*>(b), eps,
      static_cast<T*>(y), mean, rstd, M, (int)N);
  return launch_status();
}

template <class T, class W>
int forward(const void* x, const void* res, const void* w, const void* b, float eps, void* y, float* mean, float* rstd,
            long long M, long long N, cudaStream_t st) {
  if (N > kMaxRegN) {
    const int grid = grid_rows(M, 1, 8);
    if (res)
      fwd_wide_kernel<T, W, true><<<grid, 256, 0, st>>>(static_cast<const T*>(x), static_cast<const T*>(res),
                                                        static_cast<const W*>(w), static_cast<const W*>(b), eps,
                                                        static_cast<T*>(y), mean, rstd, M, N);
    else
      fwd_wide_kernel<T, W, false><<<grid, 256, 0, st>>>(static_cast<const T*>(x), nullptr,
                                                         static_cast<const W*>(w), static_cast<const W*>(b), eps,
                                                         static_cast<T*>(y), mean, rstd, M, N);
    return launch_status();
  }
  const bool vec = N % (16 / (int)sizeof(T)) == 0 && aligned(x, 16) && aligned(res, 16) && aligned(y, 16) &&
                   aligned(w, 16) && aligned(b, 16);
  const Shape s = shape(N, 256);
#define PACKR_NORM_FWD(E, V, R) \
  return launch_fwd<T, W, E, V, R>(s, x, res, w, b, eps, y, mean, rstd, M, N, st)
  if (s.e == 8) {
    if (vec) { if (res) PACKR_NORM_FWD(8, true, true); else PACKR_NORM_FWD(8, true, false); }
    if (res) PACKR_NORM_FWD(8, false, true); else PACKR_NORM_FWD(8, false, false);
  }
  if (vec) { if (res) PACKR_NORM_FWD(16, true, true); else PACKR_NORM_FWD(16, true, false); }
  if (res) PACKR_NORM_FWD(16, false, true); else PACKR_NORM_FWD(16, false, false);
#undef PACKR_NORM_FWD
}

template <class T, class W, int E, bool VEC, bool RES, bool PARAMS, bool ACC_SMEM>
int launch_bwd(const Shape& s, const void* dy, const void* x, const void* res, const void* w, const float* mean,
               const float* rstd, void* dx, float* partial, int slabs, long long M, long long N, cudaStream_t st) {
  auto kern = bwd_kernel<T, W, E, VEC, RES, PARAMS, ACC_SMEM>;
  const size_t smem = PARAMS && (ACC_SMEM || s.groups > 1) ? (size_t)s.groups * 2 * E * s.nt * sizeof(float) : 0;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    cudaGetLastError();
    return PACKR_ERR_CUDA;
  }
  kern<<<slabs, dim3(s.nt, s.groups), smem, st>>>(static_cast<const T*>(dy), static_cast<const T*>(x),
                                                  static_cast<const T*>(res), static_cast<const W*>(w), mean, rstd,
                                                  static_cast<T*>(dx), partial, M, (int)N);
  return launch_status();
}

// CTAs of the backward, each leaving one slab of column sums.
inline int bwd_slabs(long long M, long long N) {
  if (N > kMaxRegN) return (int)(M < 64 ? M : 64);
  const Shape s = shape(N, 512);
  const int n = grid_rows(M, s.groups, s.nt * s.groups <= 512 ? 2 : 1);
  return n < kSlabs ? n : kSlabs;
}

template <class T, class W, bool RES>
int backward_res(const void* dy, const void* x, const void* res, const void* w, const float* mean, const float* rstd,
                 void* dx, void* dw, void* db, float* partial, long long M, long long N, cudaStream_t st) {
  const bool params = dw != nullptr || db != nullptr;
  const int slabs = bwd_slabs(M, N);
  int rc = PACKR_OK;
  if (N > kMaxRegN) {
    if (dx) {
      bwd_wide_kernel<T, W, RES><<<grid_rows(M, 1, 8), 256, 0, st>>>(
          static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const T*>(res), static_cast<const W*>(w),
          mean, rstd, static_cast<T*>(dx), M, N);
      if ((rc = launch_status()) != PACKR_OK) return rc;
    }
    if (params) {
      bwd_wide_cols_kernel<T, RES><<<dim3((unsigned)((N + 255) / 256), (unsigned)slabs), 256, 0, st>>>(
          static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const T*>(res), mean, rstd, partial, M, N);
      if ((rc = launch_status()) != PACKR_OK) return rc;
    }
  } else {
    const bool vec = N % (16 / (int)sizeof(T)) == 0 && aligned(dy, 16) && aligned(x, 16) && aligned(res, 16) &&
                     aligned(dx, 16) && aligned(w, 16);
    const Shape s = shape(N, 512);
#define PACKR_NORM_BWD(E, V, P, A) \
  rc = launch_bwd<T, W, E, V, RES, P, A>(s, dy, x, res, w, mean, rstd, dx, partial, slabs, M, N, st)
#define PACKR_NORM_BWD_P(E, V, A)                                            \
  do {                                                                       \
    if (params) PACKR_NORM_BWD(E, V, true, A); else PACKR_NORM_BWD(E, V, false, A); \
  } while (0)
    if (s.nt <= 512 && s.e == 8) {
      if (vec) PACKR_NORM_BWD_P(8, true, false); else PACKR_NORM_BWD_P(8, false, false);
    } else if (s.e == 8) {
      if (vec) PACKR_NORM_BWD_P(8, true, true); else PACKR_NORM_BWD_P(8, false, true);
    } else {
      if (vec) PACKR_NORM_BWD_P(16, true, true); else PACKR_NORM_BWD_P(16, false, true);
    }
#undef PACKR_NORM_BWD_P
#undef PACKR_NORM_BWD
    if (rc != PACKR_OK) return rc;
  }
  if (!params) return PACKR_OK;
  return reduce_cols(partial, slabs, 2, N, static_cast<W*>(dw), static_cast<W*>(db), st);
}

template <class T, class W>
int backward(const void* dy, const void* x, const void* res, const void* w, const float* mean, const float* rstd,
             void* dx, void* dw, void* db, float* partial, long long M, long long N, cudaStream_t st) {
  return res ? backward_res<T, W, true>(dy, x, res, w, mean, rstd, dx, dw, db, partial, M, N, st)
             : backward_res<T, W, false>(dy, x, res, w, mean, rstd, dx, dw, db, partial, M, N, st);
}

inline int check(long long M, long long N, int x_dtype, int w_dtype, const void* const* xs, int nx,
                 const void* const* ws, int nw) {
  if (M < 0 || N < 1 || M > 0x7FFFFFFFll || N > 0x7FFFFFFFll) return PACKR_ERR_SHAPE;
  if ((x_dtype != PACKR_DTYPE_F32 && x_dtype != PACKR_DTYPE_BF16) ||
      (w_dtype != PACKR_DTYPE_F32 && w_dtype != PACKR_DTYPE_BF16))
    return PACKR_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < nx; ++i)
    if (!aligned(xs[i], x_dtype == PACKR_DTYPE_F32 ? 4 : 2)) return PACKR_ERR_ALIGNMENT;
  for (int i = 0; i < nw; ++i)
    if (!aligned(ws[i], w_dtype == PACKR_DTYPE_F32 ? 4 : 2)) return PACKR_ERR_ALIGNMENT;
  return PACKR_OK;
}

}  // namespace norm
}  // namespace packr

extern "C" int packr_layer_norm_forward(const void* x, const void* residual, int x_dtype, const void* weight,
                                        const void* bias, int w_dtype, float eps, void* y, float* mean, float* rstd,
                                        int64_t M, int64_t N, void* stream) {
  using namespace packr;
  const void* xs[] = {x, residual, y};
  const void* ws[] = {weight, bias};
  int st = norm::check(M, N, x_dtype, w_dtype, xs, 3, ws, 2);
  if (st != PACKR_OK) return st;
  if (!(eps >= 0.0f)) return PACKR_ERR_INVALID_ARGUMENT;
  if (M > 0 && (x == nullptr || y == nullptr)) return PACKR_ERR_INVALID_ARGUMENT;
  if (!aligned(mean, 4) || !aligned(rstd, 4)) return PACKR_ERR_ALIGNMENT;
  if ((st = check_device()) != PACKR_OK) return st;
  if (M == 0) return PACKR_OK;
  cudaStream_t s = as_stream(stream);
  const bool xf = x_dtype == PACKR_DTYPE_F32, wf = w_dtype == PACKR_DTYPE_F32;
  if (xf && wf) return norm::forward<float, float>(x, residual, weight, bias, eps, y, mean, rstd, M, N, s);
  if (xf) return norm::forward<float, uint16_t>(x, residual, weight, bias, eps, y, mean, rstd, M, N, s);
  if (wf) return norm::forward<uint16_t, float>(x, residual, weight, bias, eps, y, mean, rstd, M, N, s);
  return norm::forward<uint16_t, uint16_t>(x, residual, weight, bias, eps, y, mean, rstd, M, N, s);
}

extern "C" size_t packr_layer_norm_backward_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0 || M > 0x7FFFFFFFll || N > 0x7FFFFFFFll) return 0;
  return (size_t)packr::norm::bwd_slabs(M, N) * 2 * (size_t)N * sizeof(float);
}

extern "C" int packr_layer_norm_backward(const void* dy, const void* x, const void* residual, int x_dtype,
                                         const void* weight, int w_dtype, const float* mean, const float* rstd,
                                         void* dx, void* dweight, void* dbias, int64_t M, int64_t N, void* workspace,
                                         size_t workspace_bytes, void* stream) {
  using namespace packr;
  const void* xs[] = {dy, x, residual, dx};
  const void* ws[] = {weight, dweight, dbias};
  int st = norm::check(M, N, x_dtype, w_dtype, xs, 4, ws, 3);
  if (st != PACKR_OK) return st;
  if (M > 0 && (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr)) return PACKR_ERR_INVALID_ARGUMENT;
  if (!aligned(mean, 4) || !aligned(rstd, 4)) return PACKR_ERR_ALIGNMENT;
  if ((st = check_device()) != PACKR_OK) return st;
  cudaStream_t s = as_stream(stream);
  const bool xf = x_dtype == PACKR_DTYPE_F32, wf = w_dtype == PACKR_DTYPE_F32;
  if (M == 0) {  // empty batch: zero gradients
    const size_t bytes = (size_t)N * (wf ? 4 : 2);
    if (dweight && cudaMemsetAsync(dweight, 0, bytes, s) != cudaSuccess) return PACKR_ERR_CUDA;
    if (dbias && cudaMemsetAsync(dbias, 0, bytes, s) != cudaSuccess) return PACKR_ERR_CUDA;
    return PACKR_OK;
  }
  if (dx == nullptr && dweight == nullptr && dbias == nullptr) return PACKR_OK;
  if (dweight != nullptr || dbias != nullptr) {
    if (workspace == nullptr || workspace_bytes < packr_layer_norm_backward_workspace_bytes(M, N) ||
        !aligned(workspace, 16))
      return PACKR_ERR_WORKSPACE;
  }
  float* partial = static_cast<float*>(workspace);
  if (xf && wf)
    return norm::backward<float, float>(dy, x, residual, weight, mean, rstd, dx, dweight, dbias, partial, M, N, s);
  if (xf)
    return norm::backward<float, uint16_t>(dy, x, residual, weight, mean, rstd, dx, dweight, dbias, partial, M, N, s);
  if (wf)
    return norm::backward<uint16_t, float>(dy, x, residual, weight, mean, rstd, dx, dweight, dbias, partial, M, N, s);
  return norm::backward<uint16_t, uint16_t>(dy, x, residual, weight, mean, rstd, dx, dweight, dbias, partial, M, N,
                                            s);
}
