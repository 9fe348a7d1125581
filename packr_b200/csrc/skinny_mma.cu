// The fused linear layer's forward for up to 16 rows, where streaming W once is
// the bound (3 bytes a weight):
//   out^T[n, m] = sum over k of W[k, n] x[m, k]
// TMA brings 64 x 128 tiles of W_f and W_p (and the 64-column tile of x) into a
// ring, 16 warps read what they need of a stage into registers, hand the stage
// back at once, decode there and feed mma.sync m16n8k16 with the weights as its
// 16-row operand.  In the tcgen05 variant for these row counts (skinny.cu) a
// stage stays taken from its TMA over the decode, which writes it back to shared
// memory, to the end of its MMAs, three latencies in turn, and six stages cover
// only half of HBM's rate; here a stage turns over with its TMA, and the tensor
// rate of mma.sync is far from the bound.  16 x 11008 -> 4096 (135 MB of W): 29.3
// us with the reduction, 4.6 TB/s, against 40.2 us.  An SM streams at 5.7 TB/s'
// share while its CTA lives (23.6 us); the rest is the start, the sums' last adds
// and the reduction (1 row: 27.2 us).
//
// Lane (g, t) = (lane / 4, lane % 4) of a warp takes, of 16 rows and 64 columns of
// a stage, rows 2t, 2t + 1, 2t + 8, 2t + 9 (the MMA's k order) and columns 8g ..
// 8g + 7 (16 bytes of W_f, 8 of W_p a row).  Which of the MMA's 16 rows is which
// column is free, so MMA i gets columns 8g + 2i (row g) and 8g + 2i + 1 (row g +
// 8): the operand is a pair-wise permute of what the lane read, plus the lut pair
// (add.rn.bf16x2, the same bits as every other route).  All shared-memory reads
// are free of bank conflicts: both W tiles and x are 128-byte swizzled by the
// TMA, the lut has a copy per lane.
//
// Work split: the (128-column tile, k-block) space is cut into equal contiguous
// ranges, one per SM.  A CTA adds its warps' sums in order at the end of each
// tile it touches and leaves them in its own partial slot; the reduction adds a
// tile's slots in CTA order, then bias and epilogue.  Nothing depends on timing.
#include "activation.cuh"
#include "common.cuh"

namespace packr {
namespace gemm {

constexpr int kSmCols = 128;                       // columns of a tile
constexpr int kSmWarps = 16, kSmThreads = 32 * (kSmWarps + 1);
constexpr int kSmRedWarps = 4;                     // warps whose sums are added at a time

template <int MT>  // groups of 8 token rows
struct SmCfg {
  static constexpr int kWBytes = BK * kSmCols * 2, kPBytes = BK * kSmCols, kXBytes = MT * 8 * BK * 2;
  static constexpr int kStageBytes = kWBytes + kPBytes + kXBytes;
  // even: a stage then always belongs to the same half of the warps, which see
  // every phase of its barrier
  static constexpr int kStages = 6;
  static constexpr int kPitch = MT * 8 + 1;  // floats per column of a warp's sums
  static constexpr int kRedBytes = kSmRedWarps * 64 * kPitch * 4;
  static constexpr int kLutOff = kStages * kStageBytes, kRedOff = kLutOff + LUT_BYTES;
  static constexpr int kBarOff = (kRedOff + kRedBytes + 15) / 16 * 16;
  static constexpr int kSmemBytes = kBarOff + 256 + 1024;
};
struct SmBars {
  uint64_t full[6];   // tiles landed                                   (count 1 + tx)
  uint64_t empty[6];  // read by the eight warps that use the stage     (count 8)
  int abort;
};

// The (tile, k-block) units in order, cut into `ctas` ranges: the first `extra`
// have per + 1 units, the others per.
struct SmPlan {
  int units, k_blocks, ctas, per, extra, slots;  // slots: tiles that one range can touch
};
__device__ __forceinline__ int sm_start(const SmPlan& p, int c) { return c * p.per + min(c, p.extra); }
__device__ __forceinline__ int sm_owner(const SmPlan& p, int u) {  // the range that has unit u
  const int head = p.extra * (p.per + 1);
  return u < head ? u / (p.per + 1) : p.extra + (u - head) / p.per;
}
// units: at most K * N / 8192, far below 2^31 for any W that fits the memory
inline SmPlan sm_plan(long long K, long long N) {
  SmPlan p{};
  p.k_blocks = (int)((K + BK - 1) / BK);
  p.units = (int)((N + kSmCols - 1) / kSmCols * p.k_blocks);
  p.ctas = p.units < sm_count() ? p.units : sm_count();
  p.per = p.units / p.ctas;
  p.extra = p.units % p.ctas;
  p.slots = (p.per + (p.extra > 0) + p.k_blocks - 2) / p.k_blocks + 1;
  return p;
}
inline int sm_groups(long long M) { return M <= 8 ? 1 : 2; }
inline size_t sm_partial_bytes(long long M, long long K, long long N) {
  const SmPlan p = sm_plan(K, N);
  return (size_t)p.ctas * p.slots * sm_groups(M) * 8 * kSmCols * sizeof(float);
}

struct SmMaps {
  CUtensorMap wf, wp, x;
};

__device__ __forceinline__ void mma_bf16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int MT>
__global__ void __launch_bounds__(kSmThreads, 1)
    skinny_mma_kernel(const __grid_constant__ SmMaps maps, const float* __restrict__ lut, float* __restrict__ partial,
                      int K, const SmPlan plan) {
  using C = SmCfg<MT>;
  constexpr int S = C::kStages, kPitch = C::kPitch;
  static_assert(C::kSmemBytes <= 227 * 1024, "shared memory per CTA");
  static_assert(S % 2 == 0 && S <= 6 && sizeof(SmBars) <= 256, "barrier block");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* const lut_b = smem + C::kLutOff;
  float* const red = reinterpret_cast<float*>(smem + C::kRedOff);
  SmBars* const bars = reinterpret_cast<SmBars*>(smem + C::kBarOff);
  volatile int* const abort_flag = &bars->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int u0 = sm_start(plan, blockIdx.x), count = sm_start(plan, blockIdx.x + 1) - u0, k_blocks = plan.k_blocks;
  int tile = u0 / k_blocks, kb = u0 % k_blocks;
  const bool producer = threadIdx.x == kSmWarps * 32;
  int it = 0;  // (producer) next stage to fill
  auto fill = [&] {
    const int s = it % S;
    uint8_t* const st = smem + s * C::kStageBytes;
    mbar_arrive_expect_tx(&bars->full[s], C::kStageBytes);
    tma_load_2d(st, &maps.wf, &bars->full[s], tile * kSmCols, kb * BK);
    tma_load_2d(st + 8192, &maps.wf, &bars->full[s], tile * kSmCols + 64, kb * BK);
    tma_load_2d(st + C::kWBytes, &maps.wp, &bars->full[s], tile * kSmCols, kb * BK);
    tma_load_2d(st + C::kWBytes + C::kPBytes, &maps.x, &bars->full[s], kb * BK, 0);
    if (++kb == k_blocks) {
      kb = 0;
      ++tile;
    }
  };
  if (producer) {
    prefetch_tmap(&maps.wf);
    prefetch_tmap(&maps.wp);
    prefetch_tmap(&maps.x);
    for (int s = 0; s < S; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], kSmWarps / 2);
    }
    bars->abort = 0;
    fence_barrier_init();
  }
  // this kernel may start before the one in front of it ends, and lets the
  // reduction start; every read of global memory comes after the wait, by
  // coherent loads (launch_overlapped)
  wait_previous_kernel();
  let_next_kernel_start();
  if (producer)  // the ring's first round, under the lut's set-up
    for (; it < count && it < S; ++it) fill();
  if (warp < 8) {  // entry e of lane l at e * 128 + l * 4, rotated stores
    const int e = threadIdx.x;
    const uint32_t v = f32_to_bf16_rne(__ldcg(lut + e));
#pragma unroll 8
    for (int l = 0; l < 32; ++l) *reinterpret_cast<uint32_t*>(lut_b + e * 128 + ((l + lane) & 31) * 4) = v;
  }
  __syncthreads();

  if (warp == kSmWarps) {
    // ------------------------------------------------ TMA producer
    if (producer) {
      bool ok = true;
      for (; it < count; ++it) {
        if (!(ok = mbar_wait(&bars->empty[it % S], ((uint32_t)(it / S) & 1u) ^ 1u, abort_flag))) break;
        fill();
      }
      if (!ok) {  // gave up: the copies in flight still land before the CTA ends
        volatile int none = 0;
        for (int j = it > S ? it - S : 0; j < it; ++j) mbar_wait(&bars->full[j % S], (uint32_t)(j / S) & 1u, &none);
      }
    }
  } else {
    // ------------------------------------------------ consumers
    // warp: 64-column half, 16-row slice of the stage's k, every other stage
    const int cg = warp & 1, q = (warp >> 1) & 3, odd = warp >> 3;
    const int g = lane >> 2, t = lane & 3;
    const uint32_t lane4 = (uint32_t)lane * 4u;
    // row r's key of the 128-byte swizzle: (2t, 2t + 1, 2t + 8, 2t + 9) & 7
    const int row0 = q * 16 + 2 * t;
    const uint32_t wf_off = (uint32_t)(cg * 8192 + row0 * 128);
    const uint32_t wp_off = (uint32_t)(C::kWBytes + row0 * 128 + (g & 1) * 8);
    const uint32_t x_off = (uint32_t)(C::kWBytes + C::kPBytes + g * 128 + 4 * t);
    const uint32_t smem0 = smem_u32(smem), lut0 = smem_u32(lut_b);
    bool ok = true;
    for (int slot = 0; it < count; ++slot, ++tile, kb = 0) {
      const int end = min(count, it + k_blocks - kb);  // of this tile's stages
      float acc[4][MT][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.0f;
      for (int i0 = it; i0 < end; ++i0) {
        if ((i0 & 1) != odd) continue;
        const int s = i0 % S;
        ok = ok && mbar_wait_warp(&bars->full[s], (uint32_t)(i0 / S) & 1u, abort_flag);
        if (!ok) continue;
        const uint32_t st = smem0 + (uint32_t)(s * C::kStageBytes);
        uint32_t f[4][4], p[4][2], b[MT][2];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t off = (uint32_t)((r & 1) + (r >> 1) * 8) * 128u;
          const uint32_t key = (uint32_t)(2 * t + (r & 1));
          asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                       : "=r"(p[r][0]), "=r"(p[r][1])
                       : "r"(st + wp_off + off + (((uint32_t)(cg * 4 + (g >> 1)) ^ key) << 4))
                       : "memory");
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(f[r][0]), "=r"(f[r][1]), "=r"(f[r][2]), "=r"(f[r][3])
                       : "r"(st + wf_off + off + (((uint32_t)g ^ key) << 4))
                       : "memory");
        }
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            asm volatile("ld.shared.b32 %0, [%1];"
                         : "=r"(b[j][h])
                         : "r"(st + x_off + j * 1024 + (((uint32_t)(2 * q + h) ^ (uint32_t)g) << 4))
                         : "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->empty[s]);
        const int k_left = K - (kb + i0 - it) * BK;  // rows of W from the stage's first on
        auto step = [&](auto tail) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // k pairs (2t, 2t + 1) and (2t + 8, 2t + 9)
              const uint32_t w0 = p[2 * h][i >> 1], w1 = p[2 * h + 1][i >> 1];
              auto entry = [&](uint32_t w, int byte) {  // 128 bytes per entry, 4 per lane
                const int sh = 8 * byte - 7;
                const uint32_t o = ((sh < 0 ? w << 7 : w >> (sh < 0 ? 0 : sh)) & 0x7F80u) | lane4;
                uint32_t v;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(lut0 + o));
                return v;
              };
              const int c = 2 * (i & 1);
              const uint32_t le = prmt(entry(w0, c), entry(w1, c), 0x5410u);
              const uint32_t lo = prmt(entry(w0, c + 1), entry(w1, c + 1), 0x5410u);
              a[2 * h] = bf16x2_add(prmt(f[2 * h][i], f[2 * h + 1][i], 0x5410u), le);      // column 8g + 2i
              a[2 * h + 1] = bf16x2_add(prmt(f[2 * h][i], f[2 * h + 1][i], 0x7632u), lo);  // column 8g + 2i + 1
              if (tail) {  // rows past W: zero, not the lut's entry 0
                const int n = k_left - row0 - 8 * h;
                const uint32_t keep = n >= 2 ? 0xFFFFFFFFu : n == 1 ? 0xFFFFu : 0u;
                a[2 * h] &= keep;
                a[2 * h + 1] &= keep;
              }
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) mma_bf16(acc[i][j], a, b[j][0], b[j][1]);
          }
        };
        if (k_left >= BK) step(std::false_type());
        else step(std::true_type());
      }
      kb = 0;
      it = end;
      // the warps' sums, added in order, kSmRedWarps of each column half at a
      // time: D rows g / g + 8 are columns 8g + 2i / + 1
      constexpr int kEach = MT * 8 * kSmCols / (kSmWarps * 32);
      float sum[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e) sum[e] = 0.0f;
#pragma unroll 1
      for (int turn = 0; turn < kSmWarps / kSmRedWarps; ++turn) {
        if ((warp >> 1) / (kSmRedWarps / 2) == turn) {  // two k-slices of both halves
          float* const mine = red + (((warp >> 1) % (kSmRedWarps / 2)) * 2 + cg) * 64 * kPitch;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
              for (int c = 0; c < 4; ++c)
                mine[(8 * g + 2 * i + (c >> 1)) * kPitch + 8 * j + 2 * t + (c & 1)] = acc[i][j][c];
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kSmWarps * 32) : "memory");
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int at = e * (kSmWarps * 32) + (int)threadIdx.x;  // [token][column]
          const float* r = red + (at % kSmCols) * kPitch + at / kSmCols;
#pragma unroll
          for (int w = 0; w < kSmRedWarps / 2; ++w) sum[e] = __fadd_rn(sum[e], r[w * 2 * 64 * kPitch]);
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kSmWarps * 32) : "memory");
      }
      float* const out = partial + ((long long)blockIdx.x * plan.slots + slot) * (MT * 8 * kSmCols);
#pragma unroll
      for (int e = 0; e < kEach; ++e) __stcg(out + e * (kSmWarps * 32) + threadIdx.x, sum[e]);
    }
  }
  __syncthreads();  // no copy in flight, no barrier in use past this point
}

// Adds a tile's slots in CTA order, then bias and epilogue: one thread per 4
// consecutive columns of one row (N % 16 == 0 on this route).
__global__ void __launch_bounds__(128) skinny_mma_reduce_kernel(const float* __restrict__ partial, int M, int N,
                                                                int slot_floats, const SmPlan plan,
                                                                const void* __restrict__ bias, int bias_f32,
                                                                const Epilogue epi) {
  const int qpr = N / 4;
  const long long q = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (q >= (long long)M * qpr) return;
  const int m = (int)(q / qpr), n = (int)(q - (long long)m * qpr) * 4;
  const long long o = (long long)m * N + n;
  float r[4] = {0.0f, 0.0f, 0.0f, 0.0f}, b[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (epi.residual != nullptr) r[j] = load_io_late(epi.residual, o + j, epi.io_f32);
    if (bias != nullptr) b[j] = load_io_late(bias, n + j, bias_f32);
  }
  const int tile = n / kSmCols, first = tile * plan.k_blocks, last = first + plan.k_blocks - 1;
  const int c0 = sm_owner(plan, first), c1 = sm_owner(plan, last);
  const float* const p = partial + m * kSmCols + n % kSmCols;
  // the first range may have begun in an earlier tile; the others begin in this one
  const int slot0 = tile - sm_start(plan, c0) / plan.k_blocks;
  wait_previous_kernel();
  let_next_kernel_start();
  constexpr int kAhead = 8;  // slots in flight
  for (int c = c0; c <= c1; c += kAhead) {
    float4 v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (c + i <= c1)
        v[i] = __ldcg(reinterpret_cast<const float4*>(
            p + ((long long)(c + i) * plan.slots + (c + i == c0 ? slot0 : 0)) * slot_floats));
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (c + i > c1) break;
      s[0] = __fadd_rn(s[0], v[i].x);
      s[1] = __fadd_rn(s[1], v[i].y);
      s[2] = __fadd_rn(s[2], v[i].z);
      s[3] = __fadd_rn(s[3], v[i].w);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    s[j] = __fadd_rn(s[j], b[j]);
    if (epi.z != nullptr) store_io(epi.z, o + j, epi.io_f32, s[j]);
  }
  act::apply_all<4>(epi.act, s);
#pragma unroll
  for (int j = 0; j < 4; ++j) store_io(epi.out, o + j, epi.io_f32, __fadd_rn(s[j], r[j]));
}

template <int MT>
int sm_launch(const SmMaps& maps, const float* lut, const void* bias, int bias_f32, const Epilogue& epi, long long M,
              long long K, long long N, float* partial, cudaStream_t st) {
  using C = SmCfg<MT>;
  static std::atomic<int> done[64];  // relaxed: concurrent first calls set the same attribute
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done[dev & 63].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(skinny_mma_kernel<MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes) !=
        cudaSuccess) {
      cudaGetLastError();
      return PACKR_ERR_CUDA;
    }
    done[dev & 63].store(1, std::memory_order_relaxed);
  }
  const SmPlan p = sm_plan(K, N);
  const int rc = launch_overlapped(skinny_mma_kernel<MT>, dim3((unsigned)p.ctas), dim3(kSmThreads), C::kSmemBytes, st, maps,
                                   lut, partial, (int)K, p);
  if (rc != PACKR_OK) return rc;
  return launch_overlapped(skinny_mma_reduce_kernel, dim3((unsigned)((M * (N / 4) + 127) / 128)), dim3(128), 0, st, partial,
                           (int)M, (int)N, MT * 8 * kSmCols, p, bias, bias_f32, epi);
}

// x_bf16: [M, ldx] with ldx % 8 == 0, 16-byte aligned; W as for the TMA-staged
// decode (wtma_ok); partial: sm_partial_bytes(M, K, N).  M <= 16.
int skinny_mma_forward(const uint16_t* x_bf16, long long ldx, const uint8_t* W_p, const uint16_t* W_f, const float* lut,
                       const void* bias, int bias_f32, const Epilogue& epi, long long M, long long K, long long N,
                       float* partial, cudaStream_t st) {
  SmMaps maps;
  const int groups = sm_groups(M);
  int rc = make_map(&maps.wf, W_f, N, K, N * 2, BK);
  if (rc == PACKR_OK) rc = make_map_u8(&maps.wp, W_p, N, K, N, kSmCols, BK, /*swizzle=*/true);
  if (rc == PACKR_OK) rc = make_map(&maps.x, x_bf16, K, M, ldx * 2, groups * 8);
  if (rc != PACKR_OK) return rc;
  return groups == 1 ? sm_launch<1>(maps, lut, bias, bias_f32, epi, M, K, N, partial, st)
                     : sm_launch<2>(maps, lut, bias, bias_f32, epi, M, K, N, partial, st);
}

}  // namespace gemm
}  // namespace packr
