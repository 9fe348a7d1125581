// The linear layer with bias, activation and residual in its epilogue:
//   z = x @ W + bias,  out = act(z) + residual,  W = bf16(W_f + bf16(lut[W_p]))
//   dz = dout * act'(z);  dX = dz @ W^T;  dW_f = x^T @ dz;  dbias = column sums
//   of dz;  dlut = W_p-binned sums of dW_f / (count + 1e-8);  dresidual = dout
// x bf16 or f32 (rounded to bf16, the tensor cores' operand); residual, out, z
// and dout of one type.  z, the only tensor kept for the backward besides x,
// is stored in that type: its rounding moves act'(z) by at most the half step
// of the type, which is what a bf16 layer followed by a bf16 activation keeps.
//
// Routes (forward): 1 and 2 rows the CUDA-core GEMV; 3..16, and 1 or 2 with a long
// reduction, the mma.sync kernel and 17..128 the skinny tcgen05 GEMM, each with its
// reduction.  Where W's rows do not allow TMA (N % 16 != 0 or a misaligned base), up
// to 16 rows take the GEMV if it can (gemv::eligible: even N, W aligned to a lane's
// load, a CTA's share of x in shared memory).  Everything else, and from 129 rows on
// every width: W is decoded once into the workspace, with rows padded to a multiple
// of 8, and read by TMA, so that odd widths take the same tensor-core GEMM as even
// ones.  The backward takes dz in one pass over dout and z (bf16 operand, optional
// residual part of the split, column sums), then the existing dX and dW GEMMs.  A W
// that the caller decoded (the _decoded entries) takes the place of either decode.
#include "activation.cuh"

namespace packr {
namespace linear_act {

using linear::Carve;
using linear::round8;

// ------------------------------------------------------------------ decode of any W
// W [K, N] -> bf16 [K, ldw], ldw = round8(N), pad columns zero.  One thread per
// 8 consecutive columns of a row: byte and 16-bit loads (rows start at any
// address), one 16-byte store.  Bound by load instructions, not bytes; it
// serves the widths that the streaming decode (16-byte rows) cannot.
__global__ void __launch_bounds__(256) decode_any_kernel(const uint8_t* __restrict__ W_p,
                                                         const uint16_t* __restrict__ W_f,
                                                         const float* __restrict__ lut, uint4* __restrict__ out,
                                                         long long K, int N, int chunks_per_row) {
  __shared__ uint16_t lut_s[256];
  lut_s[threadIdx.x] = (uint16_t)f32_to_bf16_rne(__ldg(lut + threadIdx.x));
  __syncthreads();
  const long long total = K * chunks_per_row;
  for (long long c = (long long)blockIdx.x * 256 + threadIdx.x; c < total; c += (long long)gridDim.x * 256) {
    const long long r = c / chunks_per_row;
    const int n0 = (int)(c - r * chunks_per_row) * 8;
    const long long off = r * N + n0;
    uint32_t f[8], p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = n0 + j < N;
      f[j] = in ? __ldg(W_f + off + j) : 0u;
      p[j] = in ? __ldg(W_p + off + j) : 0u;
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = gemm::bf16x2_add(f[2 * j] | (f[2 * j + 1] << 16),
                              (uint32_t)lut_s[p[2 * j]] | ((uint32_t)lut_s[p[2 * j + 1]] << 16));
      if (n0 + 2 * j >= N) w[j] = 0u;
      else if (n0 + 2 * j + 1 >= N) w[j] &= 0xFFFFu;
    }
    out[c] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// bf16 W [K, round8(N)] for the plain GEMMs.
int decode(const uint8_t* W_p, const uint16_t* W_f, const float* lut, uint16_t* out, long long K, long long N,
           cudaStream_t st) {
  if (gemm::wtma_ok(W_p, W_f, N)) return gemm::predecode(W_p, W_f, lut, out, K, N, st);
  const int cpr = (int)(round8(N) / 8);
  const long long blocks = (K * cpr + 255) / 256;
  const long long cap = 16LL * sm_count();
  decode_any_kernel<<<(int)(blocks < cap ? blocks : cap), 256, 0, st>>>(W_p, W_f, lut, reinterpret_cast<uint4*>(out), K,
                                                                        (int)N, cpr);
  return launch_status();
}

// ------------------------------------------------------------------ dz
// dz = dout * act'(z) for a slab of rows:
//   hi[r, c] = bf16(dz), lo[r, c] = bf16(dz - hi) (optional; the difference is
//   exact in f32), colsum[slab][c] = sum over the slab's rows of dz (optional).
// A thread owns 8 columns and walks its slab's rows; sums of different slabs
// are added in order by a second launch.
// hi == nullptr: only the column sums (a bf16 dout without activation is the
// GEMMs' operand as it stands).
// Bound by HBM (2 + 2 bytes in, 2 out per element with bf16): raw loads of
// kDzUnroll rows are issued before the first is used.
constexpr int kDzUnroll = 4;
template <bool F32>
struct DzRow {  // 8 elements as loaded
  uint4 q[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* src, long long off, bool vec, int nc) {
    if (vec) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(src) + off * (F32 ? 4 : 2));
#pragma unroll
      for (int k = 0; k < (F32 ? 2 : 1); ++k) q[k] = __ldcs(p + k);
    } else {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = j < nc ? __float_as_uint(load_io(src, off + j, F32)) : 0u;
      if (F32) {
        q[0] = make_uint4(w[0], w[1], w[2], w[3]);
        q[F32 ? 1 : 0] = make_uint4(w[4], w[5], w[6], w[7]);
      } else {
        q[0] = make_uint4(w[0] >> 16 | w[1], w[2] >> 16 | w[3], w[4] >> 16 | w[5], w[6] >> 16 | w[7]);
      }
    }
  }
  __device__ __forceinline__ void get(float* v) const {
    if (F32) {
      const uint4 a = q[0], b = q[F32 ? 1 : 0];
      v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
      v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
    } else {
      const uint32_t w[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  }
};

template <bool F32, int ACT>
__global__ void __launch_bounds__(256) dz_kernel(const void* __restrict__ dout, const void* __restrict__ z, int M,
                                                 int N, int rows_per_slab, uint16_t* __restrict__ hi,
                                                 uint16_t* __restrict__ lo, long long ld, int vec,
                                                 float* __restrict__ colsum) {
  let_next_kernel_start();
  const long long c0 = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 8;
  if (c0 >= N) return;
  const int r0 = blockIdx.y * rows_per_slab;
  const int r1 = min(M, r0 + rows_per_slab);
  const int nc = (int)min(8ll, (long long)N - c0);
  const bool v8 = vec && nc == 8;
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int r = r0; r < r1; r += kDzUnroll) {
    DzRow<F32> rd[kDzUnroll], rz[kDzUnroll];
#pragma unroll
    for (int u = 0; u < kDzUnroll; ++u) {
      if (r + u < r1) {
        rd[u].load(dout, (long long)(r + u) * N + c0, v8, nc);
        if (ACT != PACKR_ACT_NONE) rz[u].load(z, (long long)(r + u) * N + c0, v8, nc);
      }
    }
#pragma unroll
    for (int u = 0; u < kDzUnroll; ++u) {
      if (r + u >= r1) break;
      float d[8];
      rd[u].get(d);
      if (ACT != PACKR_ACT_NONE) {
        float zz[8];
        rz[u].get(zz);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] *= act::slope<ACT>(zz[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += d[j];
      if (hi == nullptr) continue;
      uint32_t h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = pack_bf16x2_rne(d[2 * j], d[2 * j + 1]);
      // ld is a multiple of 8: the padding of a ragged row is written as zero
      const long long o = (long long)(r + u) * ld + c0;
      *reinterpret_cast<uint4*>(hi + o) = make_uint4(h[0], h[1], h[2], h[3]);
      if (lo != nullptr) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          l[j] = pack_bf16x2_rne(__fsub_rn(d[2 * j], __uint_as_float(h[j] << 16)),
                                 __fsub_rn(d[2 * j + 1], __uint_as_float(h[j] & 0xFFFF0000u)));
        *reinterpret_cast<uint4*>(lo + o) = make_uint4(l[0], l[1], l[2], l[3]);
      }
    }
  }
  if (colsum != nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < nc) colsum[(long long)blockIdx.y * N + c0 + j] = acc[j];
  }
}

struct DzPlan {
  int threads, slabs, rows_per_slab;
  unsigned col_blocks;
};
// About four CTAs of 256 threads' worth per SM, at least 8 rows a slab.
inline DzPlan dz_plan(long long M, long long N) {
  DzPlan p{};
  const long long chunks = (N + 7) / 8;
  p.threads = (int)(chunks >= 256 ? 256 : (chunks + 31) / 32 * 32);
  p.col_blocks = (unsigned)((chunks + p.threads - 1) / p.threads);
  long long want = 4LL * sm_count() * 256 / ((long long)p.col_blocks * p.threads);
  const long long most = (M + 7) / 8;
  if (want > most) want = most;
  if (want > 1024) want = 1024;
  if (want < 1) want = 1;
  p.rows_per_slab = (int)((M + want - 1) / want);
  p.slabs = (int)((M + p.rows_per_slab - 1) / p.rows_per_slab);
  return p;
}

template <bool F32>
int dz_launch(int a, const void* dout, const void* z, long long M, long long N, uint16_t* hi, uint16_t* lo,
              long long ld, float* colsum, cudaStream_t st) {
  const DzPlan p = dz_plan(M, N);
  const dim3 grid(p.col_blocks, (unsigned)p.slabs);
  const int vec = (N & 7) == 0 && aligned(dout, 16) && aligned(z, 16);
#define PACKR_DZ(A)                                                                                                  \
  dz_kernel<F32, A><<<grid, p.threads, 0, st>>>(dout, z, (int)M, (int)N, p.rows_per_slab, hi, lo, ld, vec, colsum)
  switch (a) {
    case PACKR_ACT_RELU: PACKR_DZ(PACKR_ACT_RELU); break;
    case PACKR_ACT_GELU: PACKR_DZ(PACKR_ACT_GELU); break;
    case PACKR_ACT_GELU_TANH: PACKR_DZ(PACKR_ACT_GELU_TANH); break;
    case PACKR_ACT_SILU: PACKR_DZ(PACKR_ACT_SILU); break;
    default: PACKR_DZ(PACKR_ACT_NONE); break;
  }
#undef PACKR_DZ
  return launch_status();
}

// ------------------------------------------------------------------ plans
enum Route { GEMV, SKINNY_MMA, SKINNY, PLAIN };
// The mma.sync route's rows, where W's layout allows its TMA.  Measured (us in a
// graph; 11008 -> 4096 / 4096 -> 11008 / 1024 -> 4096): 16 rows 29.3 / 28.7 / 8.4
// with it, 40.2 / 40.4 / 12.0 with the tcgen05 skinny GEMM (24 rows in a four-group
// instance: 46.9 against 42.3); 3 rows 27.4 / 27.1 / 7.3 with it, 40.8 / 32.0 / 8.7
// with the GEMV.  2 rows 27.3 / 27.1 / 7.3 and 34.3 / 27.4 / 7.3, 1 row 27.2 / 27.1 /
// 7.1 and 29.7 / 25.1 / 6.7: the GEMV cuts K over at most 16 CTAs, which a long
// reduction leaves uneven (16384 -> 256, 1 row: 12.9 and 17.3; 8192 -> 2048: 14.2 and
// 17.0), and is ahead where it is one launch's latency that counts (1024 x 1024, 2
// rows: 5.8 and 5.0; 4096 x 4096: 14.4 and 16.1).
// Widths that TMA cannot read, GEMV / decode and GEMM: 1024 -> 1002 3 rows 5.7 / 25.1,
// 16 rows 8.7 / 25.6; 4096 -> 4100 4 rows 18.8 / 64.1, 8 rows 24.7 / 64.3; 4096 -> 11004
// 8 rows 73 / 98.
constexpr long long kSkinnyMmaMaxM = 16;
inline bool skinny_mma_pays(long long M, long long K, long long N) {
  if (M > kSkinnyMmaMaxM) return false;
  if (M >= 3) return true;
  return M == 2 ? K >= 8192 || K * N >= 1 << 23 : K >= 8192 && K >= 2 * N;
}

inline Route route(long long M, long long K, long long N, const uint8_t* W_p, const uint16_t* W_f) {
  if (skinny_mma_pays(M, K, N) && gemm::wtma_ok(W_p, W_f, N)) return SKINNY_MMA;
  if (linear::skinny_eligible(M, N) && gemm::wtma_ok(W_p, W_f, N)) return SKINNY;
  if (gemv::eligible(M, K, N, W_p, W_f)) return GEMV;
  return PLAIN;
}

struct Fwd {
  uint16_t *xh, *wd;
  float *part, *skp;
  int* skf;
};

size_t plan_forward(Carve& c, Fwd& p, Route r, long long M, long long K, long long N, int x_dtype, int io_f32,
                    bool wd_given = false) {
  p = Fwd{};
  if (r == GEMV) return 0;
  p.xh = linear::x_needs_copy(x_dtype, K) ? c.take<uint16_t>((size_t)M * round8(K)) : nullptr;
  if (r == SKINNY_MMA) {
    p.part = c.take<float>(gemm::sm_partial_bytes(M, K, N) / sizeof(float));
  } else if (r == SKINNY) {
    p.part = c.take<float>(gemm::skinny_partial_bytes(M, K, N, io_f32 ? gemm::kSegBlocks : 0) / sizeof(float));
  } else {
    p.wd = wd_given ? nullptr : c.take<uint16_t>((size_t)K * round8(N));
    p.skp = c.take<float>(gemm::sk_partial_bytes(linear::sk_pairs(), gemm::epi_msub(M, K, io_f32)) / sizeof(float));
    p.skf = c.take<int>(gemm::sk_flag_bytes(linear::sk_pairs(), 16) / sizeof(int));
  }
  return c.off;
}

struct Bwd {
  uint16_t *dh, *dl, *xh, *xl, *wd;
  float *part, *skp, *colsum, *dlut_sum;
  int *skf, *tiles;
  int32_t* counts;
};

size_t plan_backward(Carve& c, Bwd& p, long long M, long long K, long long N, int x_dtype, int flags, bool direct,
                     bool skinny, bool dx, bool dw, bool dlut, bool dbias, bool have_counts, bool wd_given = false) {
  p = Bwd{};
  const bool need_x = dw || dlut;
  const bool split = (flags & PACKR_BWD_DW_SPLIT) != 0 && need_x;
  if (dx && skinny) {
    p.part = c.take<float>(gemm::skinny_partial_bytes(M, N, K) / sizeof(float));
  } else if (dx) {
    p.wd = wd_given ? nullptr : c.take<uint16_t>((size_t)K * round8(N));
    p.skp = c.take<float>(gemm::sk_partial_bytes(linear::sk_pairs(), linear::plain_msub(M)) / sizeof(float));
    p.skf = c.take<int>(gemm::sk_flag_bytes(linear::sk_pairs()) / sizeof(int));
  }
  p.dh = direct ? nullptr : c.take<uint16_t>((size_t)M * round8(N));
  p.dl = split && !direct ? c.take<uint16_t>((size_t)M * round8(N)) : nullptr;
  p.xh = need_x && linear::x_needs_copy(x_dtype, K) ? c.take<uint16_t>((size_t)M * round8(K)) : nullptr;
  p.xl = need_x && split && x_dtype == PACKR_DTYPE_F32 ? c.take<uint16_t>((size_t)M * round8(K)) : nullptr;
  p.colsum = dbias ? c.take<float>((size_t)dz_plan(M, N).slabs * N) : nullptr;
  p.dlut_sum = dlut ? c.take<float>(256) : nullptr;
  p.counts = dlut && !have_counts ? c.take<int32_t>(256) : nullptr;
  p.tiles = dw ? c.take<int>(1) : nullptr;
  return c.off;
}

// Output tiles (256 * msub rows, 256 columns) of a GEMM.
inline long long tiles_of(long long rows, long long cols, int msub) {
  return (rows + 256LL * msub - 1) / (256 * msub) * ((cols + 255) / 256);
}

// Largest dimension: tiles and slabs of rows that start inside it end within an int.
constexpr long long kMaxDim = 0x7F000000ll;

int check_args(const void* x, int x_dtype, const uint8_t* W_p, const uint16_t* W_f, const float* lut, long long M,
               long long K, long long N) {
  if (M > kMaxDim || K > kMaxDim || N > kMaxDim) return PACKR_ERR_SHAPE;
  return linear::check_common(x, x_dtype, W_p, W_f, lut, M, K, N);
}

inline bool act_ok(int a) { return a >= PACKR_ACT_NONE && a <= PACKR_ACT_SILU; }
inline bool io_ok(int d) { return d == PACKR_DTYPE_F32 || d == PACKR_DTYPE_BF16; }
inline size_t io_size(int d) { return d == PACKR_DTYPE_F32 ? 4 : 2; }

// x [M, K] -> hi = bf16(x) and, for the split dW, lo = bf16(x - hi), rows padded
// to a multiple of 8 with zeros.  One thread per 8 consecutive elements of a
// row, any row length and alignment.
__global__ void __launch_bounds__(256) operand_kernel(const void* __restrict__ x, int f32, long long M, int K,
                                                      int chunks_per_row, int vec, uint4* __restrict__ hi,
                                                      uint4* __restrict__ lo) {
  const long long total = M * chunks_per_row;
  for (long long c = (long long)blockIdx.x * 256 + threadIdx.x; c < total; c += (long long)gridDim.x * 256) {
    const long long r = c / chunks_per_row;
    const int k0 = (int)(c - r * chunks_per_row) * 8;
    const long long off = r * K + k0;
    float v[8];
    if (vec) {  // f32 rows of whole chunks
      const float4 a = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(x) + off));
      const float4 b = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(x) + off) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k0 + j < K ? load_io(x, off + j, f32) : 0.0f;
    }
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[j] = pack_bf16x2_rne(v[2 * j], v[2 * j + 1]);
      l[j] = pack_bf16x2_rne(__fsub_rn(v[2 * j], __uint_as_float(h[j] << 16)),
                             __fsub_rn(v[2 * j + 1], __uint_as_float(h[j] & 0xFFFF0000u)));
    }
    hi[c] = make_uint4(h[0], h[1], h[2], h[3]);
    if (lo != nullptr) lo[c] = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

// x as the GEMMs' bf16 operand (a copy in xh, with its residual part in xl,
// when its type or row length needs one).
int operand_x(const void* x, int x_dtype, long long M, long long K, uint16_t* xh, uint16_t* xl, const void** a,
              long long* lda, cudaStream_t s) {
  *a = x;
  *lda = K;
  if (xh == nullptr) return PACKR_OK;
  *a = xh;
  *lda = round8(K);
  const int cpr = (int)(round8(K) / 8), f32 = x_dtype == PACKR_DTYPE_F32;
  const long long blocks = (M * cpr + 255) / 256, cap = 16LL * sm_count();
  operand_kernel<<<(int)(blocks < cap ? blocks : cap), 256, 0, s>>>(x, f32, M, (int)K, cpr, f32 && (K & 7) == 0 && aligned(x, 16),
                                                                   reinterpret_cast<uint4*>(xh),
                                                                   reinterpret_cast<uint4*>(xl));
  return launch_status();
}

}  // namespace linear_act
}  // namespace packr

extern "C" size_t packr_linear_act_workspace_bytes(int64_t M, int64_t K, int64_t N, int x_dtype, int out_dtype,
                                                   const uint8_t* W_p, const uint16_t* W_f) {
  using namespace packr;
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  linear::Carve c{nullptr};
  linear_act::Fwd p;
  return linear_act::plan_forward(c, p, linear_act::route(M, K, N, W_p, W_f), M, K, N, x_dtype,
                                  out_dtype == PACKR_DTYPE_F32);
}

namespace packr {
namespace linear_act {
// The forward of checked W (W_p, W_f, lut), or of W decoded by the caller (Wd, N %
// 8 == 0), which then goes to the GEMM over a decoded W at every M.
int forward_impl(const void* x, int x_dtype, const uint8_t* W_p, const uint16_t* W_f, const float* lut,
                 const uint16_t* Wd, const void* bias, int bias_dtype, int activation, const void* residual, void* out,
                 void* z, int out_dtype, long long M, long long K, long long N, void* workspace, size_t workspace_bytes,
                 void* stream) {
  int st;
  if (!act_ok(activation) || !io_ok(out_dtype) || (bias != nullptr && !io_ok(bias_dtype)))
    return PACKR_ERR_INVALID_ARGUMENT;
  if (M > 0 && out == nullptr) return PACKR_ERR_INVALID_ARGUMENT;
  const size_t ob = io_size(out_dtype);
  if (!aligned(out, ob) || !aligned(residual, ob) || !aligned(z, ob) ||
      (bias != nullptr && !aligned(bias, io_size(bias_dtype))))
    return PACKR_ERR_ALIGNMENT;
  if ((st = check_device()) != PACKR_OK) return st;
  if (M == 0) return PACKR_OK;
  cudaStream_t s = as_stream(stream);
  const Route r = Wd != nullptr ? PLAIN : route(M, K, N, W_p, W_f);
  Carve c{static_cast<uint8_t*>(workspace)};
  Fwd p;
  const size_t need = linear_act::plan_forward(c, p, r, M, K, N, x_dtype, out_dtype == PACKR_DTYPE_F32, Wd != nullptr);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, linear::kAlign)))
    return PACKR_ERR_WORKSPACE;
  Epilogue e{};
  e.residual = residual;
  e.out = out;
  e.z = z;
  e.io_f32 = out_dtype == PACKR_DTYPE_F32;
  e.act = activation;
  e.vec = aligned(out, 16) && aligned(residual, 16) && aligned(z, 16) && (N * ob) % 16 == 0;
  const int bias_f32 = bias_dtype == PACKR_DTYPE_F32;
  if (r == GEMV)
    return gemv::forward_epi(x, x_dtype == PACKR_DTYPE_F32, W_p, W_f, lut, bias, bias_f32, e, M, K, N, s);
  const void* a;
  long long lda;
  if ((st = operand_x(x, x_dtype, M, K, p.xh, nullptr, &a, &lda, s)) != PACKR_OK) return st;
  if (r == SKINNY_MMA)
    return gemm::skinny_mma_forward(static_cast<const uint16_t*>(a), lda, W_p, W_f, lut, bias, bias_f32, e, M, K, N,
                                    p.part, s);
  if (r == SKINNY)
    return gemm::skinny_forward_epi(static_cast<const uint16_t*>(a), lda, W_p, W_f, lut, bias, bias_f32, e, M, K, N,
                                    p.part, s);
  gemm::Maps maps;
  if ((st = gemm::make_map(&maps.a[0], a, K, M, lda * 2, gemm::BM)) != PACKR_OK) return st;
  if ((st = gemm::make_map(&maps.b[0], Wd != nullptr ? Wd : p.wd, N, K, round8(N) * 2, 64)) != PACKR_OK) return st;
  if (Wd == nullptr && (st = decode(W_p, W_f, lut, p.wd, K, N, s)) != PACKR_OK) return st;
  gemm::Params P{};
  P.Mg = (int)M;
  P.Ng = (int)N;
  P.Kg = (int)K;
  P.nseg = 1;
  P.ld_out = N;
  P.bias = bias;
  P.bias_f32 = bias_f32;
  P.epi = e;
  const int msub = gemm::epi_msub(M, K, e.io_f32);
  gemm::set_split(P, p.skp, p.skf, linear::sk_pairs(), tiles_of(M, N, msub), msub);
  return gemm::launch_plain_epi(P, maps, s);
}
}  // namespace linear_act
}  // namespace packr

extern "C" int packr_linear_act_forward(const void* x, int x_dtype, const uint8_t* W_p, const uint16_t* W_f,
                                        const float* lut, const void* bias, int bias_dtype, int activation,
                                        const void* residual, void* out, void* z, int out_dtype, int64_t M, int64_t K,
                                        int64_t N, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = linear_act::check_args(x, x_dtype, W_p, W_f, lut, M, K, N);
  if (st != PACKR_OK) return st;
  return linear_act::forward_impl(x, x_dtype, W_p, W_f, lut, nullptr, bias, bias_dtype, activation, residual, out, z,
                                  out_dtype, M, K, N, workspace, workspace_bytes, stream);
}

extern "C" size_t packr_linear_act_forward_decoded_workspace_bytes(int64_t M, int64_t K, int64_t N, int x_dtype,
                                                                   int out_dtype) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  linear::Carve c{nullptr};
  linear_act::Fwd p;
  return linear_act::plan_forward(c, p, linear_act::PLAIN, M, K, N, x_dtype, out_dtype == PACKR_DTYPE_F32, true);
}

extern "C" int packr_linear_act_forward_decoded(const void* x, int x_dtype, const uint16_t* Wd, const void* bias,
                                                int bias_dtype, int activation, const void* residual, void* out, void* z,
                                                int out_dtype, int64_t M, int64_t K, int64_t N, void* workspace,
                                                size_t workspace_bytes, void* stream) {
  if ((N & 7) != 0 && N > 0) return PACKR_ERR_SHAPE;  // Wd rows must be 16-byte multiples for TMA
  // Wd in the places of what it was decoded from, for the checks of pointers
  const int st = linear_act::check_args(x, x_dtype, reinterpret_cast<const uint8_t*>(Wd), Wd,
                                        reinterpret_cast<const float*>(Wd), M, K, N);
  if (st != PACKR_OK) return st;
  if (!aligned(Wd, 16)) return PACKR_ERR_ALIGNMENT;
  return linear_act::forward_impl(x, x_dtype, nullptr, nullptr, nullptr, Wd, bias, bias_dtype, activation, residual, out,
                                  z, out_dtype, M, K, N, workspace, workspace_bytes, stream);
}

extern "C" size_t packr_linear_act_backward_workspace_bytes(int64_t M, int64_t K, int64_t N, int x_dtype, int flags,
                                                            const uint8_t* W_p, const uint16_t* W_f) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  linear::Carve c{nullptr};
  linear_act::Bwd p;
  const bool skinny = linear::skinny_dx_eligible(M, N) && gemm::wtma_ok(W_p, W_f, N);
  return linear_act::plan_backward(c, p, M, K, N, x_dtype, flags, false, skinny, true, true, true, true, false);
}

namespace packr {
namespace linear_act {
// The backward; wd_given (nullable) is W as the caller decoded it, used by the plain
// dX GEMM in place of a decode of its own.
int backward_impl(const void* dout, const void* z, int out_dtype, int activation, const void* x, int x_dtype,
                  const uint8_t* W_p, const uint16_t* W_f, const float* lut, const uint16_t* wd_given,
                  const int32_t* lut_counts, void* dX, uint16_t* dW_f, float* dlut, void* dbias, int dbias_dtype,
                  long long M, long long K, long long N, int flags, void* workspace, size_t workspace_bytes,
                  void* stream) {
  int st = check_args(x, x_dtype, W_p, W_f, lut, M, K, N);
  if (st != PACKR_OK) return st;
  if (!act_ok(activation) || !io_ok(out_dtype) || (dbias != nullptr && !io_ok(dbias_dtype)) ||
      (flags & ~PACKR_BWD_DW_SPLIT) != 0)
    return PACKR_ERR_INVALID_ARGUMENT;
  if (M > 0 && (dout == nullptr || (activation != PACKR_ACT_NONE && z == nullptr))) return PACKR_ERR_INVALID_ARGUMENT;
  const size_t ob = io_size(out_dtype);
  if (!aligned(dout, ob) || !aligned(z, ob) || !aligned(dX, io_size(x_dtype)) || !aligned(dW_f, 2) ||
      !aligned(dlut, 4) || !aligned(lut_counts, 4) || (dbias != nullptr && !aligned(dbias, io_size(dbias_dtype))))
    return PACKR_ERR_ALIGNMENT;
  if ((st = check_device()) != PACKR_OK) return st;
  cudaStream_t s = as_stream(stream);
  const bool dx = dX != nullptr, dw = dW_f != nullptr, dl = dlut != nullptr, db = dbias != nullptr;
  if (M == 0) {  // empty batch: every gradient is zero
    if (dw && cudaMemsetAsync(dW_f, 0, (size_t)K * N * 2, s) != cudaSuccess) return PACKR_ERR_CUDA;
    if (dl && cudaMemsetAsync(dlut, 0, 256 * 4, s) != cudaSuccess) return PACKR_ERR_CUDA;
    if (db && cudaMemsetAsync(dbias, 0, (size_t)N * io_size(dbias_dtype), s) != cudaSuccess) return PACKR_ERR_CUDA;
    return PACKR_OK;
  }
  if (!dx && !dw && !dl && !db) return PACKR_OK;
  // a bf16 dout without activation is the GEMMs' operand as it stands (and
  // its split residual part is zero)
  const bool direct = activation == PACKR_ACT_NONE && out_dtype == PACKR_DTYPE_BF16 && (N & 7) == 0 && aligned(dout, 16);
  const bool skinny = linear::skinny_dx_eligible(M, N) && gemm::wtma_ok(W_p, W_f, N);
  Carve c{static_cast<uint8_t*>(workspace)};
  Bwd p;
  const size_t need = linear_act::plan_backward(c, p, M, K, N, x_dtype, flags, direct, skinny, dx, dw, dl, db,
                                                lut_counts != nullptr, wd_given != nullptr);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, linear::kAlign)))
    return PACKR_ERR_WORKSPACE;
  const long long ldN = round8(N);
  const uint16_t* dh = direct ? static_cast<const uint16_t*>(dout) : p.dh;
  if (!direct || db) {
    const void* zz = activation != PACKR_ACT_NONE ? z : nullptr;
    st = out_dtype == PACKR_DTYPE_F32 ? dz_launch<true>(activation, dout, zz, M, N, p.dh, p.dl, ldN, p.colsum, s)
                                      : dz_launch<false>(activation, dout, zz, M, N, p.dh, p.dl, ldN, p.colsum, s);
    if (st != PACKR_OK) return st;
  }
  if (db) {
    const int slabs = dz_plan(M, N).slabs;
    st = dbias_dtype == PACKR_DTYPE_F32
             ? norm::reduce_cols(p.colsum, slabs, 1, N, static_cast<float*>(dbias), static_cast<float*>(nullptr), s)
             : norm::reduce_cols(p.colsum, slabs, 1, N, static_cast<uint16_t*>(dbias),
                                 static_cast<uint16_t*>(nullptr), s);
    if (st != PACKR_OK) return st;
  }
  if (dx && skinny) {
    st = gemm::skinny_dx(dh, ldN, W_p, W_f, lut, dX, x_dtype == PACKR_DTYPE_F32, M, K, N, p.part, s);
    if (st != PACKR_OK) return st;
  } else if (dx) {
    gemm::Maps maps;
    if ((st = gemm::make_map(&maps.a[0], dh, N, M, ldN * 2, gemm::BM)) != PACKR_OK) return st;
    if ((st = gemm::make_map(&maps.b[0], wd_given != nullptr ? wd_given : p.wd, N, K, ldN * 2, gemm::BN_CTA)) != PACKR_OK)
      return st;
    if (wd_given == nullptr && (st = decode(W_p, W_f, lut, p.wd, K, N, s)) != PACKR_OK) return st;
    gemm::Params P{};
    P.Mg = (int)M;
    P.Ng = (int)K;
    P.Kg = (int)N;
    P.nseg = 1;
    P.out = dX;
    P.ld_out = K;
    P.out_f32 = x_dtype == PACKR_DTYPE_F32;
    const int msub = linear::plain_msub(M);
    gemm::set_split(P, p.skp, p.skf, linear::sk_pairs(), tiles_of(M, K, msub), msub);
    if ((st = gemm::launch_plain<gemm::DX>(P, maps, s)) != PACKR_OK) return st;
  }
  if (dw || dl) {
    const void* xa;
    long long ldx;
    if ((st = operand_x(x, x_dtype, M, K, p.xh, p.xl, &xa, &ldx, s)) != PACKR_OK) return st;
    // reduction segments: x.dh [+ x.dl] [+ xl.dh]
    gemm::Maps maps;
    int nseg = 0;
    auto add_seg = [&](const void* a, const void* b) -> int {
      int rc = gemm::make_map(&maps.a[nseg], a, K, M, ldx * 2, 64);
      if (rc == PACKR_OK) rc = gemm::make_map(&maps.b[nseg], b, N, M, ldN * 2, 64);
      ++nseg;
      return rc;
    };
    if ((st = add_seg(xa, dh)) != PACKR_OK) return st;
    if (p.dl != nullptr && (st = add_seg(xa, p.dl)) != PACKR_OK) return st;
    if (p.xl != nullptr && (st = add_seg(p.xl, dh)) != PACKR_OK) return st;
    if (dl && cudaMemsetAsync(p.dlut_sum, 0, 256 * 4, s) != cudaSuccess) return PACKR_ERR_CUDA;
    gemm::Params P{};
    P.Mg = (int)K;
    P.Ng = (int)N;
    P.Kg = (int)M;
    P.nseg = nseg;
    P.out = dW_f;
    P.ld_out = N;
    P.hist_idx = dl ? W_p : nullptr;
    P.dlut_sum = p.dlut_sum;
    if (!dl) {
      P.sk_flags = p.tiles;
      st = gemm::launch_dw_plain(P, maps, s);
    } else {
      st = gemm::launch<gemm::DW>(P, maps, s);
    }
    if (st != PACKR_OK) return st;
  }
  if (dl) {
    const int32_t* counts = lut_counts;
    if (counts == nullptr) {
      if ((st = prep::bincount256(W_p, K * N, p.counts, s)) != PACKR_OK) return st;
      counts = p.counts;
    }
    return prep::finalize(dlut, p.dlut_sum, counts, nullptr, nullptr, 0, s);
  }
  return PACKR_OK;
}
}  // namespace linear_act
}  // namespace packr

extern "C" int packr_linear_act_backward(const void* dout, const void* z, int out_dtype, int activation, const void* x,
                                         int x_dtype, const uint8_t* W_p, const uint16_t* W_f, const float* lut,
                                         const int32_t* lut_counts, void* dX, uint16_t* dW_f, float* dlut, void* dbias,
                                         int dbias_dtype, int64_t M, int64_t K, int64_t N, int flags, void* workspace,
                                         size_t workspace_bytes, void* stream) {
  return linear_act::backward_impl(dout, z, out_dtype, activation, x, x_dtype, W_p, W_f, lut, nullptr, lut_counts, dX,
                                   dW_f, dlut, dbias, dbias_dtype, M, K, N, flags, workspace, workspace_bytes, stream);
}

extern "C" size_t packr_linear_act_backward_decoded_workspace_bytes(int64_t M, int64_t K, int64_t N, int x_dtype,
                                                                    int flags, const uint8_t* W_p,
                                                                    const uint16_t* W_f) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  linear::Carve c{nullptr};
  linear_act::Bwd p;
  const bool skinny = linear::skinny_dx_eligible(M, N) && gemm::wtma_ok(W_p, W_f, N);
  return linear_act::plan_backward(c, p, M, K, N, x_dtype, flags, false, skinny, true, true, true, true, false, true);
}

extern "C" int packr_linear_act_backward_decoded(const void* dout, const void* z, int out_dtype, int activation,
                                                 const void* x, int x_dtype, const uint8_t* W_p, const uint16_t* W_f,
                                                 const float* lut, const uint16_t* Wd, const int32_t* lut_counts,
                                                 void* dX, uint16_t* dW_f, float* dlut, void* dbias, int dbias_dtype,
                                                 int64_t M, int64_t K, int64_t N, int flags, void* workspace,
                                                 size_t workspace_bytes, void* stream) {
  if ((N & 7) != 0 && N > 0) return PACKR_ERR_SHAPE;
  if (Wd == nullptr) return PACKR_ERR_INVALID_ARGUMENT;
  if (!aligned(Wd, 16)) return PACKR_ERR_ALIGNMENT;
  return linear_act::backward_impl(dout, z, out_dtype, activation, x, x_dtype, W_p, W_f, lut, Wd, lut_counts, dX, dW_f,
                                   dlut, dbias, dbias_dtype, M, K, N, flags, workspace, workspace_bytes, stream);
}
