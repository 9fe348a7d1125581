// The layer norm's launch rule: which kernel instance a width gets, with how many
// threads, rows and CTAs.  Host arithmetic only (no CUDA), so that it can be swept
// over every width by a plain C++ compiler.
#pragma once

#include <stddef.h>

namespace packr {
namespace norm {

constexpr int kMaxRowThreads = 1024;
constexpr long long kMaxRegN = 16LL * kMaxRowThreads;  // widest row held in registers
constexpr int kMaxGroups = 8;                          // rows in flight per CTA (named barriers 1..8)
constexpr int kMaxSmem = 220 * 1024;                   // dynamic shared memory a CTA may ask for

// CTAs of TMAX threads per SM that the register bounds are set for: 80 registers
// a thread, 128 where more values are held, 64 with 1024 threads.  Two or three
// small CTAs hide one another's reductions.
constexpr int ctas_per_sm(bool bwd, int e, int tmax) {
  return tmax > 256 ? 1 : e == 8 || (e == 16 && !bwd) ? 3 : 2;
}

struct Shape {
  int e, nt, groups, grid, stages;
  int tmax;     // threads that the instance's launch bounds allow
  bool ragged;  // rows are not whole 16-byte chunks
  size_t smem;
};

// Elements per thread: 8 up to 1024 columns, 16 beyond (fewer threads to reduce
// over), in the forward 32 beyond 4096 (CTAs of at most 512 threads).  A ragged
// row covers up to `vw` - 1 elements more than it has, and it is what it covers
// that has to fit the 256 threads of a 16-element instance.  The
// backward's column sums leave registers for 16 elements only: beyond 4096
// columns it has one CTA of up to 1024 threads per SM, and beyond 8192 the sums
// move to shared memory.  Rows per CTA: about 256 threads.  Grid: as many CTAs
// as registers and shared memory of `sms` SMs hold, a whole number of phases when
// rows are not whole chunks.  Ring: up to 3 stages, what fits.
inline Shape shape(long long M, long long N, int esize, int tensors, bool bwd, int sms) {
  Shape s{};
  const int vw = 16 / esize;
  s.ragged = N % vw != 0;
  const long long span = s.ragged ? N + vw - 1 : N;
  s.e = N <= 1024 ? 8 : span <= 4096 || bwd ? 16 : 32;
  s.nt = (int)((span + 32LL * s.e - 1) / (32LL * s.e) * 32);
  s.tmax = s.nt <= 256 ? 256 : s.nt <= 512 ? 512 : kMaxRowThreads;
  s.groups = 256 / s.nt;
  s.groups = s.groups < 1 ? 1 : s.groups > kMaxGroups ? kMaxGroups : s.groups;
  if (s.groups > M) s.groups = (int)M;
  const int threads = s.nt * s.groups;
  // column sums: 1024-thread CTAs keep them here, several groups add them here
  const size_t acc = !bwd ? 0 : s.nt > 512 ? (size_t)2 * s.e * s.nt * 4 : s.groups > 1 ? (size_t)2 * N * 4 : 0;
  const size_t stage = (size_t)tensors * s.e * esize * threads;  // at most 128 KB, with a ring
  s.stages = bwd && s.nt > 512 ? 0 : (int)((kMaxSmem - acc) / stage);
  if (s.stages > 3) s.stages = 3;
  s.smem = acc + stage * s.stages;
  const int regs = ctas_per_sm(bwd, s.e, 256) == 3 ? 80 : threads > 512 ? 64 : 128;
  int per_sm = 65536 / (regs * threads);
  if (per_sm > 4) per_sm = 4;
  if (s.smem > 0 && per_sm > (int)(kMaxSmem / s.smem)) per_sm = (int)(kMaxSmem / s.smem);
  if (per_sm < 1) per_sm = 1;
  const long long want = (M + s.groups - 1) / s.groups;
  long long cap = (long long)sms * per_sm;
  if (s.ragged && want > cap) cap = cap / vw * vw;
  s.grid = (int)(want < cap ? want : cap);
  return s;
}

// Rows this wide have no register path (a ragged row spans up to 7 more columns).
inline bool wide(long long N) { return N > kMaxRegN || (N > kMaxRegN - 8 && N % 8 != 0); }

}  // namespace norm
}  // namespace packr
