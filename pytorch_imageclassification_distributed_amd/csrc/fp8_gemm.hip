// C[M][N] = act(sum_kb 2^(ea[m][kb] + eb[n][kb]) * (A[m][kb] . B[n][kb]) + bias[n]), e4m3 operands, kb = blocks of 128.
//
// One k-step is one scale block: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 128 columns and applies both rows'
// E8M0 bytes itself, so a block scale costs no vector instruction.  (An arbitrary fp32 scale would cost an FMA an
// accumulator and k-step beside the matrix pipe; e4m3 is a floating format, so a power of two loses no significand.)
// The instruction aligns its 128 products to the largest before it adds them: sums come out within 2^-16 of the exact
// ones (1.5e-5 of the result's norm on normal data, whatever K; the bf16 instruction gives 9e-8), which a bf16 or fp16
// output does not show.
#include "conv_common.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Fp8Gemm {
  const uint8_t* A; const uint8_t* As; const uint8_t* B; const uint8_t* Bs;
  void* C; const float* bias;
  int M, N, nk;      // nk = blocks of 128 columns
  long lda, ldb;     // bytes a row
  int ldsa, ldsb;    // scale bytes a scale row (multiples of 4)
  int bshift;        // log2 of the B rows that share a scale row: 0 or 7
  long ldc;
  int act, ctype;    // ctype: 0 bf16, 1 fp16, 2 fp32
};

DEVI void store_c(const Fp8Gemm& p, long i, float v) {
  if (p.ctype == 0) ((bf16_t*)p.C)[i] = f2bf(v);
  else if (p.ctype == 1) ((_Float16*)p.C)[i] = (_Float16)v;
  else ((float*)p.C)[i] = v;
}

// BM x BN tile on WM x WN waves, two LDS stages of one k-step each filled by LDS-DMA.  Rows past M or N read the last
// row again (their results are not stored).
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void fp8_gemm_kernel(const Fp8Gemm p) {
  constexpr int NW = WM * WN;
  constexpr int WTM = BM / WM, WTN = BN / WN, RM = WTM / 16, RN = WTN / 16;
  constexpr int AL = BM / 8 / NW, BL = BN / 8 / NW;
  constexpr int STAGE = (BM + BN) * 128;
  static_assert(AL * 8 * NW == BM && BL * 8 * NW == BN, "loader mapping");
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid / WN, wn = wid % WN;
  const int gm = (p.M + BM - 1) / BM, gn = (p.N + BN - 1) / BN;
  const int lin = xcd_remap(blockIdx.x, gm * gn);
  const int bm = lin / gn, bn = lin - bm * gn;
  const int m0 = bm * BM, n0 = bn * BN;

  const int lrow = lane >> 3, pch = lane & 7;
  const uint8_t* srca[AL];
  const uint8_t* srcb[BL];
#pragma unroll
  for (int i = 0; i < AL; ++i) {
    const int row = wid * (BM / NW) + i * 8 + lrow;
    srca[i] = p.A + (long)min(m0 + row, p.M - 1) * p.lda + (pch ^ ((row >> 1) & 7)) * 16;
  }
#pragma unroll
  for (int i = 0; i < BL; ++i) {
    const int row = wid * (BN / NW) + i * 8 + lrow;
    srcb[i] = p.B + (long)min(n0 + row, p.N - 1) * p.ldb + (pch ^ ((row >> 1) & 7)) * 16;
  }
  auto issue = [&](int kt, int buf) {
    char* sa = smem + buf * STAGE;
    char* sb = sa + BM * 128;
#pragma unroll
    for (int i = 0; i < AL; ++i) glds16(srca[i] + (long)kt * 128, sa + (wid * (BM / NW) + i * 8) * 128);
#pragma unroll
    for (int i = 0; i < BL; ++i) glds16(srcb[i] + (long)kt * 128, sb + (wid * (BN / NW) + i * 8) * 128);
  };

  const int fr = lane & 15, fq = lane >> 4;
  // a lane's scale rows; four k-steps' bytes come in one word, the next word is loaded four steps ahead
  const uint32_t* ssa[RM];
  const uint32_t* ssb[RN];
  uint32_t sx[RM], sw[RN], nx[RM], nw[RN];
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    ssa[i] = (const uint32_t*)(p.As + (long)min(m0 + wm * WTM + i * 16 + fr, p.M - 1) * p.ldsa);
    nx[i] = ssa[i][0];
  }
#pragma unroll
  for (int j = 0; j < RN; ++j) {
    ssb[j] = (const uint32_t*)(p.Bs + (long)(min(n0 + wn * WTN + j * 16 + fr, p.N - 1) >> p.bshift) * p.ldsb);
    nw[j] = ssb[j][0];
  }

  f32x4 acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  issue(0, 0);
  for (int kt = 0; kt < p.nk; ++kt) {
    wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    if (kt + 1 < p.nk) issue(kt + 1, (kt + 1) & 1);
    if ((kt & 3) == 0) {
      const int nxt = min((kt >> 2) + 1, (p.nk - 1) >> 2);
#pragma unroll
      for (int i = 0; i < RM; ++i) { sx[i] = nx[i]; nx[i] = ssa[i][nxt]; }
#pragma unroll
      for (int j = 0; j < RN; ++j) { sw[j] = nw[j]; nw[j] = ssb[j][nxt]; }
    }
    const char* sa = smem + (kt & 1) * STAGE;
    const char* sb = sa + BM * 128;
    i32x8 xa[RM], wb[RN];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const int row = wm * WTM + i * 16 + fr;
      const int4 lo = *(const int4*)(sa + swz(row, fq));
      const int4 hi = *(const int4*)(sa + swz(row, fq + 4));
      xa[i] = (i32x8){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    }
#pragma unroll
    for (int j = 0; j < RN; ++j) {
      const int row = wn * WTN + j * 16 + fr;
      const int4 lo = *(const int4*)(sb + swz(row, fq));
      const int4 hi = *(const int4*)(sb + swz(row, fq + 4));
      wb[j] = (i32x8){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    }
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int j = 0; j < RN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wb[j], xa[i], acc[i][j], 0, 0, 0, (int)sw[j], 0,
                                                                     (int)sx[i]);
#pragma unroll
    for (int i = 0; i < RM; ++i) sx[i] >>= 8;
#pragma unroll
    for (int j = 0; j < RN; ++j) sw[j] >>= 8;
  }
  // acc[i][j][r]: row wm * WTM + 16 i + fr, column wn * WTN + 16 j + 4 fq + r of the tile
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int m = m0 + wm * WTM + i * 16 + fr;
    if (m >= p.M) continue;
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = n0 + wn * WTN + j * 16 + fq * 4 + r;
        if (n < p.N) store_c(p, (long)m * p.ldc + n, apply_act(acc[i][j][r] + (p.bias ? p.bias[n] : 0.f), p.act));
      }
  }
}

template <int BM, int BN, int WM, int WN>
void launch(const Fp8Gemm& p, hipStream_t s) {
  hipLaunchKernelGGL((fp8_gemm_kernel<BM, BN, WM, WN>), dim3(cdiv(p.M, BM) * cdiv(p.N, BN)), dim3(64 * WM * WN), 0, s, p);
}

}  // namespace

int fp8_gemm_launch(const uint8_t* A, const uint8_t* As, const uint8_t* B, const uint8_t* Bs, void* C,
                    const float* bias, int M, int N, int nk, long lda, long ldb, int ldsa, int ldsb, int bshift,
                    long ldc, int act, int ctype, hipStream_t s) {
  if (M <= 0 || N <= 0 || nk <= 0) return 0;
  const Fp8Gemm p{A, As, B, Bs, C, bias, M, N, nk, lda, ldb, ldsa, ldsb, bshift, ldc, act, ctype};
  launch<128, 128, 2, 2>(p, s);
  HIP_CHECK_LAUNCH();
  return 0;
}
