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
// Bound by HBM: one read of each input and one write of each output.
// * A row lives in the registers of `blockDim.x` threads, E elements each, so
//   mean and centred variance are two exact passes over registers;
//   `blockDim.y` rows are in flight per CTA, and CTAs are persistent.
// * Loads: each thread copies its own 16-byte chunks of the following rows into
//   its own shared-memory slots with cp.async, `stages` deep (no barrier: a
//   thread reads only what it copied).  Registers alone held 32 KB in flight
//   per SM at 4096 columns, 70 % of HBM's rate.
// * Rows of any length use the same 16-byte chunks: chunks are laid on the
//   16-byte grid of the tensor, so a row may begin and end inside one (its
//   phase).  The rows of a CTA are a multiple of 8 (f32: 4) apart, which gives
//   them one phase, so a thread's columns, weights and column sums stay its
//   own over the whole launch; elements of neighbouring rows in the two edge
//   chunks are loaded and dropped, and never read past the tensor's end.
// * The backward recomputes h from x and residual instead of a stored sum: the
//   sum would have to be rounded (bf16) or read back at twice the width, for
//   the same number of bytes.  A thread carries its columns' dweight / dbias
//   sums in registers (rows beyond 8192 columns: in its own shared-memory
//   words); the CTAs' sums go to the workspace and a second launch adds them in
//   a fixed order, so results do not depend on timing.
// Rows wider than 16384, and tensors that do not start on a 16-byte boundary,
// are walked by one CTA per row in passes over L2-resident data.
#include <atomic>

#include "activation.cuh"
#include "common.cuh"
#include "layer_norm_shape.cuh"

namespace packr {
namespace norm {

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

// Pairs of f32 (first element in the low half) for the packed add, multiply and
// fma: the kernels are within 2x of the issue rate when each element takes an
// instruction of its own.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pk2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void upk2(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 sub2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 splat(float a) { return pk2(a, a); }
__device__ __forceinline__ float both(f32x2 v) {
  float a, b;
  upk2(v, a, b);
  return a + b;
}

// A 16-byte chunk as pairs.
__device__ __forceinline__ void unpack(const uint4 q, f32x2* v, float) {
  v[0] = pk2(__uint_as_float(q.x), __uint_as_float(q.y));
  v[1] = pk2(__uint_as_float(q.z), __uint_as_float(q.w));
}
__device__ __forceinline__ void unpack(const uint4 q, f32x2* v, uint16_t) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = pk2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
}
__device__ __forceinline__ uint4 pack(const f32x2* v, float) {
  uint4 q;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(q.x), "=r"(q.y) : "l"(v[0]));
  asm("mov.b64 {%0, %1}, %2;" : "=r"(q.z), "=r"(q.w) : "l"(v[1]));
  return q;
}
__device__ __forceinline__ uint32_t pack_pair(f32x2 v) {
  float a, b;
  upk2(v, a, b);
  return pack_bf16x2_rne(a, b);
}
__device__ __forceinline__ uint4 pack(const f32x2* v, uint16_t) {
  return make_uint4(pack_pair(v[0]), pack_pair(v[1]), pack_pair(v[2]), pack_pair(v[3]));
}

// Which elements a thread holds: chunk v of thread t covers VW = 16 /
// sizeof(T) columns from (v * nt + t) * VW - phase.  Rows of whole chunks
// (RAGGED false) have phase 0 and chunks that are inside or outside as a whole.
template <class T, int E, bool RAGGED>
struct Layout {
  static constexpr int VW = 16 / (int)sizeof(T);
  static constexpr int NV = E / VW;
  static constexpr uint32_t kFull = E == 32 ? 0xFFFFFFFFu : (1u << (E & 31)) - 1u;
  int t, nt, phase, N;
  uint32_t mask;  // elements inside the row
  bool full;
  __device__ __forceinline__ Layout(int t_, int nt_, long long row, int N_) : t(t_), nt(nt_), phase(0), N(N_), mask(0) {
    if (RAGGED) phase = (int)(row * N % VW);
#pragma unroll
    for (int e = 0; e < E; ++e) mask |= (uint32_t)(col(e) >= 0 && col(e) < N) << e;
    full = mask == kFull;
  }
  __device__ __forceinline__ int col(int e) const { return ((e / VW) * nt + t) * VW + e % VW - phase; }
  __device__ __forceinline__ bool inside(int e) const { return mask >> e & 1u; }
  __device__ __forceinline__ bool any(int v) const { return (mask >> (v * VW) & ((1u << VW) - 1u)) != 0; }
  __device__ __forceinline__ bool whole(int v) const {
    return RAGGED ? (~mask >> (v * VW) & ((1u << VW) - 1u)) == 0 : any(v);
  }
  __device__ __forceinline__ void clear_outside(f32x2* x) const {
    if (!full) {
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float a, b;
        upk2(x[e / 2], a, b);
        x[e / 2] = pk2(inside(e) ? a : 0.0f, inside(e + 1) ? b : 0.0f);
      }
    }
  }
  // the thread's values of a [N] vector, `absent` where there is none
  __device__ __forceinline__ void load_vector(const void* p, int f32, float absent, f32x2* x) const {
    if (!RAGGED && p != nullptr && aligned(p, 16)) {  // whole chunks: 8- or 16-byte loads
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int k = 0; k < VW; k += 4) {
          f32x2* d = x + (v * VW + k) / 2;
          d[0] = d[1] = splat(absent);
          if (!any(v)) continue;
          if (f32) {
            unpack(__ldcg(reinterpret_cast<const uint4*>(static_cast<const float*>(p) + col(v * VW) + k)), d, float());
          } else {
            const uint2 q = __ldcg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + col(v * VW) + k));
            d[0] = pk2(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xFFFF0000u));
            d[1] = pk2(__uint_as_float(q.y << 16), __uint_as_float(q.y & 0xFFFF0000u));
          }
        }
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      float a = absent, b = absent;
      if (p != nullptr && inside(e)) a = load_io_late(p, col(e), f32);
      if (p != nullptr && inside(e + 1)) b = load_io_late(p, col(e + 1), f32);
      x[e / 2] = pk2(a, b);
    }
  }
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {  // the rest of the 16 bytes: zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait(int ahead) {  // all but the newest `ahead` groups have landed
  if (ahead >= 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (ahead == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// This thread's chunks of NT tensors, row after row: `at` is the element index
// of its first chunk in the current row, the same in every tensor (chunk v lies
// v * nt * VW further).  RING: the rows pass through shared memory, `stages`
// deep; slot of stage s, tensor a, chunk v: ((s * NT + a) * NV + v) * pitch from
// the thread's first.  Without RING chunks are loaded when they are read.
template <class T, int E, bool RAGGED, int NT, bool RING>
struct Rows {
  using L = Layout<T, E, RAGGED>;
  const T* p[NT];
  long long at, stride;   // elements; stride: to the thread's next row
  long long total;        // elements of each tensor
  uint32_t smem, pitch;
  // bytes of a chunk, from element i on, that lie inside the tensor
  __device__ __forceinline__ int bytes_in(long long i) const {
    const long long n = (total - i) * (long long)sizeof(T);
    return n < 16 ? (int)n : 16;
  }
  // copies the row `ahead` rows on into stage `stage`; `last`: its last chunk may pass the tensor's end
  __device__ __forceinline__ void issue(const L& l, int ahead, int stage, bool last) const {
    const long long i0 = at + ahead * stride;
    const uint32_t dst = smem + stage * (NT * L::NV) * pitch;
#pragma unroll
    for (int v = 0; v < L::NV; ++v) {
      if (!l.any(v)) continue;  // its slots hold zeros from the start
      const long long i = i0 + (long long)v * l.nt * L::VW;
      const int n = RAGGED && last ? bytes_in(i) : 16;
#pragma unroll
      for (int a = 0; a < NT; ++a) cp16(dst + (a * L::NV + v) * pitch, p[a] + i, n);
    }
  }
  // zeros in the slots of chunks outside the row, which no copy writes
  __device__ __forceinline__ void clear(const L& l, int stages) const {
#pragma unroll
    for (int v = 0; v < L::NV; ++v) {
      if (l.any(v)) continue;
      for (int k = 0; k < stages * NT; ++k)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem + (k * L::NV + v) * pitch), "r"(0) : "memory");
    }
  }
  template <bool ADD>  // ADD: onto x
  __device__ __forceinline__ void get(const L& l, int stage, int a, f32x2* x) const {
#pragma unroll
    for (int v = 0; v < L::NV; ++v) {
      uint4 q = make_uint4(0, 0, 0, 0);
      if (RING) {
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                     : "r"(smem + ((stage * NT + a) * L::NV + v) * pitch)
                     : "memory");
      } else if (l.any(v)) {
        const long long i = at + (long long)v * l.nt * L::VW;
        if (!RAGGED || bytes_in(i) == 16) {
          q = __ldcs(reinterpret_cast<const uint4*>(p[a] + i));
        } else {
          f32x2 f[L::VW / 2];
#pragma unroll
          for (int j = 0; j < L::VW; j += 2)
            f[j / 2] = pk2(i + j < total ? Elem<T>::get(__ldcg(p[a] + i + j)) : 0.0f,
                           i + j + 1 < total ? Elem<T>::get(__ldcg(p[a] + i + j + 1)) : 0.0f);
          q = pack(f, T());
        }
      }
      if (ADD) {
        f32x2 r[L::VW / 2];
        unpack(q, r, T());
#pragma unroll
        for (int j = 0; j < L::VW / 2; ++j) x[v * (L::VW / 2) + j] = add2(x[v * (L::VW / 2) + j], r[j]);
      } else {
        unpack(q, x + v * (L::VW / 2), T());
      }
    }
  }
};

// at: element index of the thread's first chunk.
template <class T, int E, bool RAGGED>
__device__ __forceinline__ void store_row(const Layout<T, E, RAGGED>& l, T* __restrict__ out, long long at,
                                          const f32x2* x) {
  using L = Layout<T, E, RAGGED>;
#pragma unroll
  for (int k = 0; k < L::NV; ++k) {
    T* p = out + at + (long long)k * l.nt * L::VW;
    if (l.whole(k)) {
      __stcs(reinterpret_cast<uint4*>(p), pack(x + k * (L::VW / 2), T()));
    } else if (RAGGED && l.any(k)) {
#pragma unroll
      for (int j = 0; j < L::VW; j += 2) {
        float a, b;
        upk2(x[(k * L::VW + j) / 2], a, b);
        if (l.inside(k * L::VW + j)) p[j] = Elem<T>::put(a);
        if (l.inside(k * L::VW + j + 1)) p[j + 1] = Elem<T>::put(b);
      }
    }
  }
}

template <int n>
__device__ __forceinline__ float sum_all(const f32x2* x) {
  f32x2 s = x[0];
#pragma unroll
  for (int k = 1; k < n; ++k) s = add2(s, x[k]);
  return both(s);
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
// float per warp of the group, 32 in all, zeros past the last.  The caller
// alternates two buffers.
__device__ __forceinline__ float group_sum(float v, float* buf, int group, int nt, int t) {
  v = warp_sum(v);
  if (nt == 32) return v;
  if ((t & 31) == 0) buf[t >> 5] = v;
  group_sync(group, nt);
  const float4* b = reinterpret_cast<const float4*>(buf);
  float s = 0.0f;
  for (int i = 0; i * 128 < nt; ++i) {
    const float4 q = b[i];
    s += (q.x + q.y) + (q.z + q.w);
  }
  return s;
}

template <class T, int E, bool RAGGED, bool RES, int TMAX>
__global__ void __launch_bounds__(TMAX, ctas_per_sm(false, E, TMAX))
    fwd_kernel(const T* __restrict__ x, const T* __restrict__ res, const void* __restrict__ weight,
               const void* __restrict__ bias, int wf, float eps, T* __restrict__ y, float* __restrict__ mean_out,
               float* __restrict__ rstd_out, long long M, int N, int stages) {
  using L = Layout<T, E, RAGGED>;
  constexpr bool RING = true;
  constexpr int P = E / 2;  // pairs
  __shared__ __align__(16) float bufs[kMaxGroups][2][32];
  extern __shared__ __align__(16) uint8_t ring[];
  // may start before the kernel in front of it ends, and lets the next one start
  wait_previous_kernel();
  let_next_kernel_start();
  const int t = threadIdx.x, nt = blockDim.x, group = threadIdx.y;
  const long long step = (long long)gridDim.x * blockDim.y;
  long long row = (long long)blockIdx.x * blockDim.y + group;
  if (row >= M) return;  // named barriers count this group's threads only
  const L l(t, nt, row, N);
  Rows<T, E, RAGGED, RES ? 2 : 1, RING> in;
  in.p[0] = x;
  if (RES) in.p[RES ? 1 : 0] = res;
  in.at = row * N + l.col(0);
  in.stride = step * N;
  in.total = M * N;
  in.pitch = (uint32_t)(nt * blockDim.y) * 16;
  in.smem = (uint32_t)__cvta_generic_to_shared(ring) + (uint32_t)(group * nt + t) * 16;
  int left = (int)((M - 1 - row) / step);        // rows after this one
  const bool ends = (M - 1 - row - left * step) * N < L::VW;  // the last of them shares the tensor's last chunk
  if (RING) {
    in.clear(l, stages);
    for (int s = 0; s < stages - 1; ++s) {
      if (s <= left) in.issue(l, s, s, ends && s == left);
      cp_commit();
    }
  }
  for (int k = t; k < 64; k += nt) bufs[group][0][k] = 0.0f;  // both buffers
  group_sync(group, nt);
  f32x2 w[P], b[P];
  l.load_vector(weight, wf, 1.0f, w);
  l.load_vector(bias, wf, 0.0f, b);
  const float inv_n = 1.0f / (float)N;
  for (int s = 0;; row += step, in.at += in.stride, --left) {
    if (RING) {
      if (stages - 1 <= left) in.issue(l, stages - 1, s == 0 ? stages - 1 : s - 1, ends && stages - 1 == left);
      cp_commit();
      cp_wait(stages - 1);
    }
    f32x2 v[P];
    in.template get<false>(l, s, 0, v);
    if (RES) in.template get<true>(l, s, RES ? 1 : 0, v);
    if (RAGGED) l.clear_outside(v);  // whole chunks outside the row read as zero
    const float mean = group_sum(sum_all<P>(v), bufs[group][0], group, nt, t) * inv_n;
    const f32x2 mean2 = splat(mean);
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = sub2(v[k], mean2);
    l.clear_outside(v);
    f32x2 m2 = mul2(v[0], v[0]);
#pragma unroll
    for (int k = 1; k < P; ++k) m2 = fma2(v[k], v[k], m2);
    const float rstd = rsqrtf(fmaf(group_sum(both(m2), bufs[group][1], group, nt, t), inv_n, eps));
    if (t == 0) {
      if (mean_out) mean_out[row] = mean;
      if (rstd_out) rstd_out[row] = rstd;
    }
    const f32x2 rstd2 = splat(rstd);
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = fma2(mul2(v[k], rstd2), w[k], b[k]);
    store_row<T, E, RAGGED>(l, y, in.at, v);
    if (left == 0) break;
    s = s + 1 == stages ? 0 : s + 1;
  }
}

// Any width and alignment: three passes of one CTA over its row.  The types
// are run-time values; the speed of this path is L2's, not the conversions'.
__global__ void __launch_bounds__(512) fwd_wide_kernel(const void* __restrict__ x, const void* __restrict__ res, int xf,
                                                       const void* __restrict__ weight, const void* __restrict__ bias,
                                                       int wf, float eps, void* __restrict__ y,
                                                       float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                       long long M, long long N) {
  __shared__ __align__(16) float bufs[2][32];
  const int t = threadIdx.x, nt = blockDim.x;
  for (long long row = blockIdx.x; row < M; row += gridDim.x) {
    auto at = [&](long long c) {
      const float v = load_io(x, row * N + c, xf);
      return res ? __fadd_rn(v, load_io(res, row * N + c, xf)) : v;
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
    for (long long c = t; c < N; c += nt)
      store_io(y, row * N + c, xf,
               fmaf((at(c) - mean) * rstd, weight ? load_io(weight, c, wf) : 1.0f, bias ? load_io(bias, c, wf) : 0.0f));
  }
}

// dx, and with `partial` this CTA's column sums: partial[blockIdx.x][0][n] =
// sum of dy * h, [1][n] = sum of dy over the CTA's rows.  CTAs of more than 512
// threads have no registers to spare for a ring's bookkeeping and the column
// sums: they load rows directly and keep the sums in dynamic shared memory,
// [2][E][nt] floats, each touched by its owner alone.  Otherwise dynamic shared
// memory is the ring, then (several groups) [2][N] floats for their sums.
template <class T, int E, bool RAGGED, bool RES, int TMAX>
__global__ void __launch_bounds__(TMAX, ctas_per_sm(true, E, TMAX))
    bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ res,
               const void* __restrict__ weight, int wf, const float* __restrict__ mean_in,
               const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ partial, long long M, int N,
               int stages) {
  using L = Layout<T, E, RAGGED>;
  constexpr int NT = RES ? 3 : 2;
  constexpr int P = E / 2;  // pairs
  constexpr bool RING = TMAX <= 512, ACC_SMEM = !RING;
  __shared__ __align__(16) float bufs[kMaxGroups][2][2][32];
  extern __shared__ __align__(16) uint8_t ring[];
  const int t = threadIdx.x, nt = blockDim.x, group = threadIdx.y, groups = blockDim.y;
  const long long step = (long long)gridDim.x * groups;
  const long long row0 = (long long)blockIdx.x * groups + group;
  wait_previous_kernel();
  let_next_kernel_start();
  const L l(t, nt, row0, N);  // the same phase in every row of this group
  Rows<T, E, RAGGED, NT, RING> in;
  in.p[0] = dy;
  in.p[1] = x;
  if (RES) in.p[RES ? 2 : 0] = res;
  in.at = row0 * N + l.col(0);
  in.stride = step * N;
  in.total = M * N;
  in.pitch = (uint32_t)(nt * groups) * 16;
  in.smem = (uint32_t)__cvta_generic_to_shared(ring) + (uint32_t)(group * nt + t) * 16;
  int left = row0 < M ? (int)((M - 1 - row0) / step) : -1;  // rows after the first, -1: no row at all
  const bool ends = left >= 0 && (M - 1 - row0 - left * step) * N < L::VW;  // the last row shares the tensor's last chunk
  if (RING) {
    in.clear(l, stages);
    for (int s = 0; s < stages - 1; ++s) {
      if (s <= left) in.issue(l, s, s, ends && s == left);
      cp_commit();
    }
  }
  for (int k = t; k < 128; k += nt) bufs[group][0][0][k] = 0.0f;
  group_sync(group, nt);
  float* acc_s = reinterpret_cast<float*>(ring + (RING ? (size_t)stages * NT * L::NV * in.pitch : 0));
  f32x2* my = reinterpret_cast<f32x2*>(acc_s) + t;  // ACC_SMEM (one group): + (which * P + k) * nt
  f32x2 aw[ACC_SMEM ? 1 : P], ab[ACC_SMEM ? 1 : P];
#pragma unroll
  for (int k = 0; k < P; ++k) {
    if (ACC_SMEM) {
      my[k * nt] = 0ull;
      my[(P + k) * nt] = 0ull;
    } else {
      aw[k] = 0ull;
      ab[k] = 0ull;
    }
  }
  const float inv_n = 1.0f / (float)N;
  f32x2 w[P];
  l.load_vector(weight, wf, 1.0f, w);
  const float *mean_p = mean_in + row0, *rstd_p = rstd_in + row0;
  float mean_n = left >= 0 ? __ldcg(mean_p) : 0.0f, rstd_n = left >= 0 ? __ldcg(rstd_p) : 0.0f;
  int parity = 0;
  for (int s = 0; left >= 0; in.at += in.stride, --left, parity ^= 1) {
    if (RING) {
      if (stages - 1 <= left) in.issue(l, stages - 1, s == 0 ? stages - 1 : s - 1, ends && stages - 1 == left);
      cp_commit();
      cp_wait(stages - 1);
    }
    const f32x2 mean = splat(mean_n), rstd = splat(rstd_n);
    if (left > 0) {
      mean_p += step;
      rstd_p += step;
      mean_n = __ldcg(mean_p);
      rstd_n = __ldcg(rstd_p);
    }
    f32x2 h[P], g[P];
    in.template get<false>(l, s, 0, g);
    in.template get<false>(l, s, 1, h);
    if (RES) in.template get<true>(l, s, RES ? 2 : 0, h);
#pragma unroll
    for (int k = 0; k < P; ++k) h[k] = mul2(sub2(h[k], mean), rstd);
    if (RAGGED) l.clear_outside(g);  // whole chunks outside the row read as zero
    l.clear_outside(h);  // -mean * rstd there, whose product with g's zeros may be a NaN
    f32x2 s1 = 0ull, s2 = 0ull;
#pragma unroll
    for (int k = 0; k < P; ++k) {
      if (ACC_SMEM) {
        my[k * nt] = fma2(g[k], h[k], my[k * nt]);
        my[(P + k) * nt] = add2(my[(P + k) * nt], g[k]);
      } else {
        aw[k] = fma2(g[k], h[k], aw[k]);
        ab[k] = add2(ab[k], g[k]);
      }
      g[k] = mul2(g[k], w[k]);
      s1 = add2(s1, g[k]);
      s2 = fma2(g[k], h[k], s2);
    }
    if (dx) {
      float m1 = warp_sum(both(s1)), m2 = warp_sum(both(s2));
      if (nt > 32) {
        float* b1 = bufs[group][parity][0];
        float* b2 = bufs[group][parity][1];
        if ((t & 31) == 0) {
          b1[t >> 5] = m1;
          b2[t >> 5] = m2;
        }
        group_sync(group, nt);
        m1 = m2 = 0.0f;
        for (int i = 0; i * 128 < nt; ++i) {
          const float4 q1 = reinterpret_cast<const float4*>(b1)[i], q2 = reinterpret_cast<const float4*>(b2)[i];
          m1 += (q1.x + q1.y) + (q1.z + q1.w);
          m2 += (q2.x + q2.y) + (q2.z + q2.w);
        }
      }
      const f32x2 a1 = splat(m1 * inv_n), a2 = splat(m2 * inv_n);
#pragma unroll
      for (int k = 0; k < P; ++k) h[k] = mul2(rstd, sub2(g[k], fma2(h[k], a2, a1)));
      store_row<T, E, RAGGED>(l, dx, in.at, h);
    }
    s = s + 1 == stages ? 0 : s + 1;
  }
  if (partial == nullptr) return;
  // Groups of a CTA have different phases when rows are not whole chunks, so
  // their sums are added per column: each group in turn into [2][N] floats.
  float* out = partial + (size_t)blockIdx.x * 2 * N;
  for (int q = 0; q < groups; ++q) {
    if (groups > 1) __syncthreads();
    if (group != q) continue;
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const f32x2 av = ACC_SMEM ? my[k * nt] : aw[ACC_SMEM ? 0 : k];
      const f32x2 bv = ACC_SMEM ? my[(P + k) * nt] : ab[ACC_SMEM ? 0 : k];
      float a[2], b[2];
      upk2(av, a[0], a[1]);
      upk2(bv, b[0], b[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int c = l.col(2 * k + j);
        if (!l.inside(2 * k + j)) continue;
        if (groups == 1) {
          out[c] = a[j];
          out[N + c] = b[j];
        } else {
          acc_s[c] = q == 0 ? a[j] : acc_s[c] + a[j];
          acc_s[N + c] = q == 0 ? b[j] : acc_s[N + c] + b[j];
        }
      }
    }
  }
  if (groups == 1) return;
  __syncthreads();
  for (int c = group * nt + t; c < 2 * N; c += nt * groups) out[c] = acc_s[c];
}

// Any width and alignment: dx in two passes of one CTA over its row.
__global__ void __launch_bounds__(512)
    bwd_wide_kernel(const void* __restrict__ dy, const void* __restrict__ x, const void* __restrict__ res, int xf,
                    const void* __restrict__ weight, int wf, const float* __restrict__ mean_in,
                    const float* __restrict__ rstd_in, void* __restrict__ dx, long long M, long long N) {
  __shared__ __align__(16) float bufs[2][32];
  const int t = threadIdx.x, nt = blockDim.x;
  for (long long row = blockIdx.x; row < M; row += gridDim.x) {
    const float mean = mean_in[row], rstd = rstd_in[row];
    auto hat = [&](long long c) {
      float v = load_io(x, row * N + c, xf);
      if (res) v = __fadd_rn(v, load_io(res, row * N + c, xf));
      return (v - mean) * rstd;
    };
    auto grad = [&](long long c) {
      const float d = load_io(dy, row * N + c, xf);
      return weight ? d * load_io(weight, c, wf) : d;
    };
    float s1 = 0.0f, s2 = 0.0f;
    for (long long c = t; c < N; c += nt) {
      const float g = grad(c);
      s1 += g;
      s2 = fmaf(g, hat(c), s2);
    }
    const float m1 = group_sum(s1, bufs[0], 0, nt, t) / (float)N;
    const float m2 = group_sum(s2, bufs[1], 0, nt, t) / (float)N;
    for (long long c = t; c < N; c += nt) store_io(dx, row * N + c, xf, rstd * (grad(c) - fmaf(hat(c), m2, m1)));
  }
}

// Any width and alignment: column sums of every gridDim.y-th row, one column
// per thread.
__global__ void __launch_bounds__(256)
    bwd_wide_cols_kernel(const void* __restrict__ dy, const void* __restrict__ x, const void* __restrict__ res, int xf,
                         const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                         float* __restrict__ partial, long long M, long long N) {
  const long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= N) return;
  float a = 0.0f, b = 0.0f;
#pragma unroll 4
  for (long long row = blockIdx.y; row < M; row += gridDim.y) {
    float v = load_io(x, row * N + c, xf);
    if (res) v = __fadd_rn(v, load_io(res, row * N + c, xf));
    const float d = load_io(dy, row * N + c, xf);
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
  wait_previous_kernel();
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
  return launch_overlapped(reduce_cols_kernel<W>, dim3((unsigned)((N + 31) / 32), (unsigned)planes), dim3(512), 0, st,
                           partial, slabs, planes, N, out0, out1);
}

constexpr int kWideSlabs = 64;  // row slabs of bwd_wide_cols_kernel

// CTAs of the backward, each leaving one slab of column sums.
inline int bwd_slabs(long long M, long long N, int esize, bool res, bool vec) {
  if (!vec || wide(N)) return (int)(M < kWideSlabs ? M : kWideSlabs);
  return shape(M, N, esize, res ? 3 : 2, true, sm_count()).grid;
}

// Raises a kernel's dynamic shared-memory limit to kMaxSmem, once per device
// (`done`: the kernel's own flags; relaxed: concurrent first calls set the same
// attribute).
template <class K>
int allow_smem(K kern, size_t smem, std::atomic<int>* done) {
  if (smem <= 40 * 1024) return PACKR_OK;  // the default limit less the static buffers
  int dev = 0;
  cudaGetDevice(&dev);
  if (done[dev & 63].load(std::memory_order_relaxed)) return PACKR_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) != cudaSuccess) {
    cudaGetLastError();
    return PACKR_ERR_CUDA;
  }
  done[dev & 63].store(1, std::memory_order_relaxed);
  return PACKR_OK;
}

template <class T, int E, bool RES, int TMAX>
int launch_fwd(const Shape& s, const void* x, const void* res, const void* w, const void* b, int wf, float eps, void* y,
               float* mean, float* rstd, long long M, long long N, cudaStream_t st) {
  auto kern = s.ragged ? fwd_kernel<T, E, true, RES, TMAX> : fwd_kernel<T, E, false, RES, TMAX>;
  static std::atomic<int> done[2][64];
  if (s.tmax > TMAX) return PACKR_ERR_LAUNCH;  // the rule and the dispatch disagree
  const int rc = allow_smem(kern, s.smem, done[s.ragged]);
  if (rc != PACKR_OK) return rc;
  return launch_overlapped(kern, dim3((unsigned)s.grid), dim3(s.nt, s.groups), s.smem, st, static_cast<const T*>(x),
                           static_cast<const T*>(res), w, b, wf, eps, static_cast<T*>(y), mean, rstd, M, (int)N, s.stages);
}

template <class T>
int forward(const void* x, const void* res, const void* w, const void* b, int wf, float eps, void* y, float* mean,
            float* rstd, long long M, long long N, cudaStream_t st) {
  const bool vec = aligned(x, 16) && aligned(res, 16) && aligned(y, 16);
  if (!vec || wide(N)) {
    const long long cap = 4LL * sm_count();
    fwd_wide_kernel<<<(int)(M < cap ? M : cap), N >= 4096 ? 512 : 128, 0, st>>>(x, res, sizeof(T) == 4, w, b, wf, eps, y,
                                                                               mean, rstd, M, N);
    return launch_status();
  }
  const Shape s = shape(M, N, sizeof(T), res ? 2 : 1, false, sm_count());
#define PACKR_NORM_FWD(E, TMAX)                                                              \
  return res ? launch_fwd<T, E, true, TMAX>(s, x, res, w, b, wf, eps, y, mean, rstd, M, N, st) \
             : launch_fwd<T, E, false, TMAX>(s, x, res, w, b, wf, eps, y, mean, rstd, M, N, st)
  if (s.e == 8) PACKR_NORM_FWD(8, 256);
  if (s.e == 16) PACKR_NORM_FWD(16, 256);
  if (s.tmax == 256) PACKR_NORM_FWD(32, 256);
  PACKR_NORM_FWD(32, 512);
#undef PACKR_NORM_FWD
}

template <class T, int E, bool RES, int TMAX>
int launch_bwd(const Shape& s, const void* dy, const void* x, const void* res, const void* w, int wf, const float* mean,
               const float* rstd, void* dx, float* partial, long long M, long long N, cudaStream_t st) {
  auto kern = s.ragged ? bwd_kernel<T, E, true, RES, TMAX> : bwd_kernel<T, E, false, RES, TMAX>;
  static std::atomic<int> done[2][64];
  if (s.tmax > TMAX) return PACKR_ERR_LAUNCH;  // the rule and the dispatch disagree
  const int rc = allow_smem(kern, s.smem, done[s.ragged]);
  if (rc != PACKR_OK) return rc;
  return launch_overlapped(kern, dim3((unsigned)s.grid), dim3(s.nt, s.groups), s.smem, st, static_cast<const T*>(dy),
                           static_cast<const T*>(x), static_cast<const T*>(res), w, wf, mean, rstd, static_cast<T*>(dx),
                           partial, M, (int)N, s.stages);
}

template <class T>
int backward(const void* dy, const void* x, const void* res, const void* w, int wf, const float* mean,
             const float* rstd, void* dx, void* dw, void* db, void* workspace, size_t workspace_bytes, long long M,
             long long N, cudaStream_t st) {
  const bool params = dw != nullptr || db != nullptr;
  const bool vec = aligned(dy, 16) && aligned(x, 16) && aligned(res, 16) && aligned(dx, 16);
  const int slabs = bwd_slabs(M, N, sizeof(T), res != nullptr, vec);
  float* partial = params ? static_cast<float*>(workspace) : nullptr;
  if (params && (workspace == nullptr || workspace_bytes < (size_t)slabs * 2 * N * sizeof(float) || !aligned(workspace, 16)))
    return PACKR_ERR_WORKSPACE;
  int rc = PACKR_OK;
  if (!vec || wide(N)) {
    const int xf = sizeof(T) == 4;
    if (dx) {
      const long long cap = 4LL * sm_count();
      bwd_wide_kernel<<<(int)(M < cap ? M : cap), N >= 4096 ? 512 : 128, 0, st>>>(dy, x, res, xf, w, wf, mean, rstd, dx, M,
                                                                                  N);
      if ((rc = launch_status()) != PACKR_OK) return rc;
    }
    if (params) {
      bwd_wide_cols_kernel<<<dim3((unsigned)((N + 255) / 256), (unsigned)slabs), 256, 0, st>>>(dy, x, res, xf, mean, rstd,
                                                                                               partial, M, N);
      rc = launch_status();
    }
  } else {
    const Shape s = shape(M, N, sizeof(T), res ? 3 : 2, true, sm_count());
#define PACKR_NORM_BWD(E, TMAX)                                                                  \
  rc = res ? launch_bwd<T, E, true, TMAX>(s, dy, x, res, w, wf, mean, rstd, dx, partial, M, N, st) \
           : launch_bwd<T, E, false, TMAX>(s, dy, x, res, w, wf, mean, rstd, dx, partial, M, N, st)
    if (s.e == 8)
      PACKR_NORM_BWD(8, 256);
    else if (s.tmax == 256)
      PACKR_NORM_BWD(16, 256);
    else if (s.tmax == 512)
      PACKR_NORM_BWD(16, 512);
    else
      PACKR_NORM_BWD(16, 1024);
#undef PACKR_NORM_BWD
  }
  if (rc != PACKR_OK || !params) return rc;
  return wf ? reduce_cols(partial, slabs, 2, N, static_cast<float*>(dw), static_cast<float*>(db), st)
            : reduce_cols(partial, slabs, 2, N, static_cast<uint16_t*>(dw), static_cast<uint16_t*>(db), st);
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
  return xf ? norm::forward<float>(x, residual, weight, bias, wf, eps, y, mean, rstd, M, N, s)
            : norm::forward<uint16_t>(x, residual, weight, bias, wf, eps, y, mean, rstd, M, N, s);
}

extern "C" size_t packr_layer_norm_backward_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0 || M > 0x7FFFFFFFll || N > 0x7FFFFFFFll) return 0;
  // the most of any type, residual and alignment
  int slabs = 0;
  for (int i = 0; i < 5; ++i) {
    const int n = packr::norm::bwd_slabs(M, N, i & 1 ? 2 : 4, (i & 2) != 0, i != 4);
    slabs = n > slabs ? n : slabs;
  }
  return (size_t)slabs * 2 * (size_t)N * sizeof(float);
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
  return xf ? norm::backward<float>(dy, x, residual, weight, wf, mean, rstd, dx, dweight, dbias, workspace,
                                    workspace_bytes, M, N, s)
            : norm::backward<uint16_t>(dy, x, residual, weight, wf, mean, rstd, dx, dweight, dbias, workspace,
                                       workspace_bytes, M, N, s);
}
