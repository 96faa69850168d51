// C[M][N] = act(sum_kb 2^(ea[m][kb] + eb[n][kb]) * (A[m][kb] . B[n][kb]) + bias[n]), e4m3 operands, kb = blocks of 128.
//
// One k-step is one scale block: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 128 columns and applies both rows'
// E8M0 bytes itself, so a block scale costs no vector instruction.  (An arbitrary fp32 scale would cost an FMA an
// accumulator and k-step beside the matrix pipe; e4m3 is a floating format, so a power of two loses no significand.)
// The instruction aligns its 128 products to the largest before it adds them: sums come out within 2^-16 of the exact
// ones (1.5e-5 of the result's norm on normal data, whatever K; the bf16 instruction gives 9e-8), which a bf16 or fp16
// output does not show.
#include <type_traits>

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
};

// output types (compile-time, as the activation is: a branch an element tripled the epilogue's code)
enum { C_BF16 = 0, C_F16 = 1, C_F32 = 2 };

template <int CT>
DEVI void store_c(const Fp8Gemm& p, long i, float v) {
  if constexpr (CT == C_BF16) ((bf16_t*)p.C)[i] = f2bf(v);
  else if constexpr (CT == C_F16) ((_Float16*)p.C)[i] = (_Float16)v;
  else ((float*)p.C)[i] = v;
}
template <int CT>
DEVI uint32_t pack_c(float a, float b) {
  if constexpr (CT == C_BF16) return pack2(a, b);
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
}

DEVI void dma16(__amdgpu_buffer_rsrc_t r, unsigned voff, int soff, char* lds_wave_base) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds_wave_base, 16, voff, soff, 0, 0);
}

DEVI i32x8 frag8(const char* lo, const char* hi) {
  const int4 l = *(const int4*)lo, h = *(const int4*)hi;
  return (i32x8){l.x, l.y, l.z, l.w, h.x, h.y, h.z, h.w};
}

// four consecutive outputs of one row
template <int ACT, int CT>
DEVI void store4(const Fp8Gemm& p, int m, int n, const f32x4& v, const float* bias) {
  if (m >= p.M || n >= p.N) return;
  float o[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) o[r] = apply_act(v[r] + bias[r], ACT);
  const long i = (long)m * p.ldc + n;
  if ((p.ldc & 3) == 0 && n + 4 <= p.N) {
    if constexpr (CT == C_F32) *(float4*)((float*)p.C + i) = make_float4(o[0], o[1], o[2], o[3]);
    else *(uint2*)((uint16_t*)p.C + i) = make_uint2(pack_c<CT>(o[0], o[1]), pack_c<CT>(o[2], o[3]));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < p.N) store_c<CT>(p, i + r, o[r]);
  }
}

DEVI void bias4(const Fp8Gemm& p, int n, float* b) {
#pragma unroll
  for (int r = 0; r < 4; ++r) b[r] = p.bias != nullptr && n + r < p.N ? p.bias[n + r] : 0.f;
}

// BM x BN tile on WM x WN waves, a ring of S LDS stages of one k-step each filled by LDS-DMA, S - 1 tiles in flight.
// Rows past the end read zeros (past the buffer resource).  Each stage is an array of its own: hipcc makes an LDS read
// wait for every LDS-DMA that may write what it reads, and tells them apart by the array alone.
template <int BM, int BN, int WM, int WN, int S, int ACT, int CT>
__global__ __launch_bounds__(64 * WM * WN) void fp8_gemm_kernel(const Fp8Gemm p) {
  constexpr int NW = WM * WN;
  constexpr int WTM = BM / WM, WTN = BN / WN, RM = WTM / 16, RN = WTN / 16;
  constexpr int AL = BM / 8 / NW, BL = BN / 8 / NW, LPS = AL + BL;
  constexpr int STAGE = (BM + BN) * 128;
  static_assert(AL * 8 * NW == BM && BL * 8 * NW == BN, "loader mapping");
  static_assert(S == 2 || S == 4, "ring depth");
  __shared__ __attribute__((aligned(16))) char s0[STAGE];
  __shared__ __attribute__((aligned(16))) char s1[STAGE];
  __shared__ __attribute__((aligned(16))) char s2[S == 4 ? STAGE : 16];
  __shared__ __attribute__((aligned(16))) char s3[S == 4 ? STAGE : 16];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid / WN, wn = wid % WN;
  const int gm = (p.M + BM - 1) / BM, gn = (p.N + BN - 1) / BN;
  const int lin = xcd_remap(blockIdx.x, gm * gn);
  const int m0 = __builtin_amdgcn_readfirstlane(lin / gn * BM), n0 = __builtin_amdgcn_readfirstlane(lin % gn * BN);

  const int lrow = lane >> 3, pch = lane & 7;
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.A + (long)m0 * p.lda, (long)(p.M - m0) * p.lda);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.B + (long)n0 * p.ldb, (long)(p.N - n0) * p.ldb);
  const __amdgpu_buffer_rsrc_t rz = make_rsrc(p.A, 0);
  unsigned va[AL], vb[BL];
#pragma unroll
  for (int i = 0; i < AL; ++i) {
    const int row = wid * (BM / NW) + i * 8 + lrow;
    va[i] = (unsigned)(row * (int)p.lda + (pch ^ ((row >> 1) & 7)) * 16);
  }
#pragma unroll
  for (int i = 0; i < BL; ++i) {
    const int row = wid * (BN / NW) + i * 8 + lrow;
    vb[i] = (unsigned)(row * (int)p.ldb + (pch ^ ((row >> 1) & 7)) * 16);
  }
  const int nk = p.nk;
  // every step issues its pieces (past the last tile from an empty resource), so the counted waits are constant
  auto issue = [&](int kt, char* buf) __attribute__((always_inline)) {
    const bool live = kt < nk;
#pragma unroll
    for (int i = 0; i < AL; ++i) dma16(live ? ra : rz, va[i], kt * 128, buf + (wid * (BM / NW) + i * 8) * 128);
#pragma unroll
    for (int i = 0; i < BL; ++i) dma16(live ? rb : rz, vb[i], kt * 128, buf + BM * 128 + (wid * (BN / NW) + i * 8) * 128);
  };
  auto stage = [&](auto c) __attribute__((always_inline)) -> char* {
    constexpr int U = decltype(c)::value % S;
    if constexpr (U == 0) return s0;
    else if constexpr (U == 1) return s1;
    else if constexpr (U == 2) return s2;
    else return s3;
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

  // step kt = S n + U: tile kt has landed (S - 2 younger ones are in flight), every wave has left step kt - 1, whose
  // stage takes tile kt + S - 1
  auto step = [&](auto c, int kt) __attribute__((always_inline)) {
    constexpr int U = decltype(c)::value;
    wait_vmcnt<(S - 2) * LPS>();
    __builtin_amdgcn_s_barrier();
    issue(kt + S - 1, stage(std::integral_constant<int, U + S - 1>{}));
    if ((kt & 3) == 0) {
      const int nxt = min((kt >> 2) + 1, (nk - 1) >> 2);
#pragma unroll
      for (int i = 0; i < RM; ++i) { sx[i] = nx[i]; nx[i] = ssa[i][nxt]; }
#pragma unroll
      for (int j = 0; j < RN; ++j) { sw[j] = nw[j]; nw[j] = ssb[j][nxt]; }
    }
    const char* sa = stage(c);
    const char* sb = sa + BM * 128;
    i32x8 xa[RM], wb[RN];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const int row = wm * WTM + i * 16 + fr;
      xa[i] = frag8(sa + swz(row, fq), sa + swz(row, fq + 4));
    }
#pragma unroll
    for (int j = 0; j < RN; ++j) {
      const int row = wn * WTN + j * 16 + fr;
      wb[j] = frag8(sb + swz(row, fq), sb + swz(row, fq + 4));
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
  };
  issue(0, s0);
  if constexpr (S == 4) {
    issue(1, s1);
    issue(2, s2);
  }
  for (int kt = 0;;) {
    step(std::integral_constant<int, 0>{}, kt);
    if (++kt >= nk) break;
    step(std::integral_constant<int, 1>{}, kt);
    if (++kt >= nk) break;
    if constexpr (S == 4) {
      step(std::integral_constant<int, 2>{}, kt);
      if (++kt >= nk) break;
      step(std::integral_constant<int, 3>{}, kt);
      if (++kt >= nk) break;
    }
  }
  wait_vmcnt<0>();
  // acc[i][j][r]: row wm * WTM + 16 i + fr, column wn * WTN + 16 j + 4 fq + r of the tile
#pragma unroll
  for (int j = 0; j < RN; ++j) {
    const int n = n0 + wn * WTN + j * 16 + fq * 4;
    float bias[4];
    bias4(p, n, bias);
#pragma unroll
    for (int i = 0; i < RM; ++i) store4<ACT, CT>(p, m0 + wm * WTM + i * 16 + fr, n, acc[i][j], bias);
  }
}

// ---- few rows ----
// 16 RM rows x 16 columns a block, its 8 waves each a share of the k-steps, their partial sums joined through LDS in a
// fixed order.  The weights' bytes bound it, so they go from memory straight into the fragments (16 rows x 128 whole
// bytes a wave and k-step; no LDS, no barrier before the join), and a launch has N / 16 x 8 waves to keep them coming.
template <int RM, int ACT, int CT>
__global__ __launch_bounds__(512) void fp8_gemm_few_kernel(const Fp8Gemm p) {
  constexpr int W = 8;
  __shared__ f32x4 part[W][RM][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * RM;
  const int nk = p.nk, k0 = wid * nk / W, k1 = (wid + 1) * nk / W;
  const uint8_t* B = p.B + (long)min(n0 + fr, p.N - 1) * p.ldb + fq * 16;
  const uint8_t* Bs = p.Bs + (long)(min(n0 + fr, p.N - 1) >> p.bshift) * p.ldsb;
  const uint8_t* A[RM];
  const uint8_t* As[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const long m = min(m0 + i * 16 + fr, p.M - 1);
    A[i] = p.A + m * p.lda + fq * 16;
    As[i] = p.As + m * p.ldsa;
  }
  f32x4 acc[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) acc[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int kt = k0; kt < k1; ++kt) {
    const uint8_t* b = B + (long)kt * 128;
    const i32x8 wb = frag8((const char*)b, (const char*)b + 64);
    const int sw = Bs[kt];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const uint8_t* a = A[i] + (long)kt * 128;
      const i32x8 xa = frag8((const char*)a, (const char*)a + 64);
      acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wb, xa, acc[i], 0, 0, 0, sw, 0, (int)As[i][kt]);
    }
  }
#pragma unroll
  for (int i = 0; i < RM; ++i) part[wid][i][lane] = acc[i];
  __syncthreads();
  if (tid >= RM * 64) return;
  const int i = wid;  // wave i joins fragment i
  f32x4 s = part[0][i][lane];
#pragma unroll
  for (int w = 1; w < W; ++w) s += part[w][i][lane];
  float bias[4];
  bias4(p, n0 + fq * 4, bias);
  store4<ACT, CT>(p, m0 + i * 16 + fr, n0 + fq * 4, s, bias);
}

// ---- the large tile ----
// 256 x 256 on 4 waves of 128 x 128, one block a CU.  A k-step of a wave is 64 MFMAs fed by 32 ds_read_b128: (128 + 128)
// rows x 128 B x 4 waves + the 64 KB that LDS-DMA writes are 192 KB a step through the LDS port, against 256 KB for
// 8 waves of 128 x 64 (where the port, not the matrix pipe, would set the pace).  The 256 accumulators of a lane live in
// AGPRs, the fragments of one k-step in 128 VGPRs; the step runs in two halves of four B fragments each (all eight A
// fragments in both), so that every register is refilled where its last MFMA has been issued:
//   first half of step kt (B 0-3):   B 4-7 of kt are read;
//   middle: tile kt + 1 has landed, this buffer's reads have ended in every wave: the step's one barrier;
//   second half (B 4-7):             the 16 LDS-DMA pieces of tile kt + 2 go into this buffer, and B 0-3 and, row by
//                                    row, A of kt + 1 are read from the other one.
// One memory instruction or two stand between two MFMAs; a tile has a whole step (64 x 32 cycles) to arrive.
// The MFMAs are asm statements (accumulators pinned to AGPRs, order kept); each carries the two wait states between a
// VALU write and a matrix read.
template <int R>
DEVI void mma_step(f32x4& acc, const i32x8& b, const i32x8& a, uint32_t sb, uint32_t sa) {
  static_assert(R >= 0 && R < 4, "scale byte");
  if constexpr (R == 0)
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa) : "memory");
  else if constexpr (R == 1)
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa) : "memory");
  else if constexpr (R == 2)
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[1,1,0]" : "+a"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa) : "memory");
  else
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[1,1,0]" : "+a"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa) : "memory");
}

constexpr int BIG_STAGE = 512 * 128;
constexpr int BIG_CST = 256 + 8;  // 16-bit elements a row of the staged output tile: 4 rows differ by 16 banks
constexpr int BIG_BUF = 128 * BIG_CST * 2 > BIG_STAGE ? 128 * BIG_CST * 2 : BIG_STAGE;  // half of the output tile each

template <int ACT, int CT>
__global__ __launch_bounds__(256, 1) void fp8_gemm_big_kernel(const Fp8Gemm p) {
  // two arrays, not one: hipcc makes an LDS read wait for every LDS-DMA that may write what it reads, and tells them
  // apart by the array alone
  __shared__ __attribute__((aligned(16))) char buf0[BIG_BUF];
  __shared__ __attribute__((aligned(16))) char buf1[BIG_BUF];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid >> 1, wn = wid & 1;
  const int gm = (p.M + 255) >> 8, gn = (p.N + 255) >> 8;
  const int lin = xcd_remap(blockIdx.x, gm * gn);
  // an XCD's consecutive tiles walk a band of 4 tile rows column by column: its L2 then holds 4 row panels and a few
  // column panels at a time
  const int band = lin / (4 * gn), first = band * 4, rows = min(gm - first, 4), rest = lin - band * 4 * gn;
  const int m0 = __builtin_amdgcn_readfirstlane((first + rest % rows) * 256);
  const int n0 = __builtin_amdgcn_readfirstlane((rest / rows) * 256);

  // LDS-DMA sources: piece q of a wave is rows [64 wid + 8 q, + 8) of its 256; lane l brings 16-B chunk (l & 7) of row
  // l >> 3, from source chunk (l & 7) ^ ((row >> 1) & 7), which takes two values over q.  Rows past the end are past
  // the buffer resource: zeros.
  const int lrow = lane >> 3, pch = lane & 7;
  const long abytes = (long)(p.M - m0) * p.lda, bbytes = (long)(p.N - n0) * p.ldb;
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.A + (long)m0 * p.lda, abytes), rb = make_rsrc(p.B + (long)n0 * p.ldb, bbytes);
  const __amdgpu_buffer_rsrc_t za = make_rsrc(p.A, 0);
  const int lda = (int)p.lda, ldb = (int)p.ldb;
  unsigned va[2], vb[2];
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const int ch = (pch ^ ((lrow >> 1) + 4 * o)) * 16;
    va[o] = (unsigned)((wid * 64 + lrow) * lda + ch);
    vb[o] = (unsigned)((wid * 64 + lrow) * ldb + ch);
  }
  auto piece = [&](int kt, char* buf, int q, bool live) __attribute__((always_inline)) {
    char* dst = buf + (wid * 64 + (q & 7) * 8) * 128;
    if (q < 8) dma16(live ? ra : za, va[q & 1], kt * 128 + q * 8 * lda, dst);
    else dma16(live ? rb : za, vb[q & 1], kt * 128 + (q - 8) * 8 * ldb, dst + 256 * 128);
  };

  const int fr = lane & 15, fq = lane >> 4;
  // fragment i of a buffer: row 16 i + fr of the wave's 128, chunks fq and fq + 4 (the swizzle depends on fr alone)
  const int oa = swz(wm * 128 + fr, fq), oah = swz(wm * 128 + fr, fq + 4);
  const int ob = 256 * 128 + swz(wn * 128 + fr, fq), obh = 256 * 128 + swz(wn * 128 + fr, fq + 4);

  // scales: a word holds four k-steps' bytes; a pair of steps takes bytes 0 and 1, then the words are shifted.  The next
  // words are loaded four steps ahead.  An odd number of steps runs one more on zeros (the DMA pieces past the end come
  // from an empty resource); its scale byte is cleared, so that padding cannot hold a NaN scale.
  const int nk = p.nk;
  const __amdgpu_buffer_rsrc_t rsa = make_rsrc(p.As + (long)m0 * p.ldsa, (long)(p.M - m0) * p.ldsa);
  const int vsa = (wm * 128 + fr) * p.ldsa;
  const uint32_t* wsb = (const uint32_t*)(p.Bs + (long)(min(n0 + wn * 128, p.N - 1) >> 7) * p.ldsb);
  const int words = (nk + 3) >> 2;
  const uint32_t last = (nk & 3) ? (1u << (8 * (nk & 3))) - 1 : ~0u;
  uint32_t sx[8], nx[8], sw, nw;
  auto scales = [&](int word) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) nx[i] = __builtin_amdgcn_raw_buffer_load_b32(rsa, vsa, word * 4 + i * 16 * p.ldsa, 0);
    nw = wsb[word];
  };

  f32x4 acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  asm volatile("s_nop 7");

  i32x8 a[8], b[8];
#pragma unroll
  for (int q = 0; q < 16; ++q) piece(0, buf0, q, true);
#pragma unroll
  for (int q = 0; q < 16; ++q) piece(1, buf1, q, nk > 1);
  scales(0);
  wait_vmcnt<0>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = frag8(buf0 + oa + i * 2048, buf0 + oah + i * 2048);
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = frag8(buf0 + ob + j * 2048, buf0 + obh + j * 2048);

  auto step = [&](auto rc, int kt) __attribute__((always_inline)) {
    constexpr int P = decltype(rc)::value;  // kt & 1
    auto cur = [&]() __attribute__((always_inline)) { if constexpr (P == 0) return (char*)buf0; else return (char*)buf1; };
    auto nxt = [&]() __attribute__((always_inline)) { if constexpr (P == 0) return (char*)buf1; else return (char*)buf0; };
#pragma unroll
    for (int t = 0; t < 32; ++t) {
      const int i = t >> 2, j = t & 3;
      mma_step<P>(acc[i][j], b[j], a[i], sw, sx[i]);
      if ((t & 3) == 1 && t < 16) b[4 + (t >> 2)] = frag8(cur() + ob + (4 + (t >> 2)) * 2048, cur() + obh + (4 + (t >> 2)) * 2048);
    }
    wait_vmcnt<0>();
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    const bool live = kt + 2 < nk;
#pragma unroll
    for (int t = 0; t < 32; ++t) {
      const int i = t >> 2, j = 4 + (t & 3);
      mma_step<P>(acc[i][j], b[j], a[i], sw, sx[i]);
      if (t < 16) piece(kt + 2, cur(), t, live);
      if ((t & 3) == 2 && t < 16) b[t >> 2] = frag8(nxt() + ob + (t >> 2) * 2048, nxt() + obh + (t >> 2) * 2048);
      if (j == 7) a[i] = frag8(nxt() + oa + i * 2048, nxt() + oah + i * 2048);
    }
  };
  for (int kt = 0; kt < nk; kt += 2) {
    if ((kt & 2) == 0) {
      const uint32_t m = (kt >> 2) == words - 1 ? last : ~0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) sx[i] = nx[i] & m;
      sw = nw & m;
      scales(min((kt >> 2) + 1, words - 1));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) sx[i] >>= 16;
      sw >>= 16;
    }
    step(std::integral_constant<int, 0>{}, kt);
    step(std::integral_constant<int, 1>{}, kt + 1);
  }
  wait_vmcnt<0>();
  // the last MFMAs' results before the first read of an accumulator: waits that every accumulator depends on
#pragma unroll
  for (int i = 0; i < 8; ++i)
    asm volatile("s_nop 15\n\ts_nop 15" : "+a"(acc[i][0]), "+a"(acc[i][1]), "+a"(acc[i][2]), "+a"(acc[i][3]), "+a"(acc[i][4]), "+a"(acc[i][5]), "+a"(acc[i][6]), "+a"(acc[i][7]));
  __syncthreads();
  float bias[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + wn * 128 + j * 16 + fq * 4 + r;
      bias[j][r] = p.bias != nullptr && n < p.N ? p.bias[n] : 0.f;
    }
  if constexpr (CT == C_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = m0 + wm * 128 + i * 16 + fr;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int n = n0 + wn * 128 + j * 16 + fq * 4 + r;
          if (m < p.M && n < p.N) store_c<CT>(p, (long)m * p.ldc + n, apply_act(acc[i][j][r] + bias[j][r], ACT));
        }
      __builtin_amdgcn_sched_barrier(0);
    }
    return;
  }
  // 16-bit outputs go through LDS, so that rows leave in whole 16-B chunks of 512 contiguous bytes
  uint16_t* ct = (uint16_t*)(wm == 0 ? buf0 : buf1);  // rows 0-127 and 128-255 of the tile
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = apply_act(acc[i][j][r] + bias[j][r], ACT);
      *(uint2*)(ct + (i * 16 + fr) * BIG_CST + wn * 128 + j * 16 + fq * 4) = make_uint2(pack_c<CT>(v[0], v[1]), pack_c<CT>(v[2], v[3]));
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  uint16_t* C = (uint16_t*)p.C;
  const int cc = (tid & 31) * 8;
  const int nv = min(8, p.N - n0 - cc);
  const bool vec = (p.ldc & 7) == 0;
  for (int r = tid >> 5; r < 256 && m0 + r < p.M; r += 8) {
    const uint4 v = *(const uint4*)((const uint16_t*)(r < 128 ? buf0 : buf1) + (r & 127) * BIG_CST + cc);
    uint16_t* o = C + (long)(m0 + r) * p.ldc + n0 + cc;
    if (vec && nv == 8) *(uint4*)o = v;
    else {
      const uint16_t* e = (const uint16_t*)&v;
      for (int k = 0; k < nv; ++k) o[k] = e[k];
    }
  }
}

template <int BM, int BN, int S, int ACT, int CT>
void launch_tile(const Fp8Gemm& p, hipStream_t s) {
  hipLaunchKernelGGL((fp8_gemm_kernel<BM, BN, 2, 2, S, ACT, CT>), dim3(cdiv(p.M, BM) * cdiv(p.N, BN)), dim3(256), 0, s, p);
}

template <int RM, int ACT, int CT>
void launch_few(const Fp8Gemm& p, hipStream_t s) {
  hipLaunchKernelGGL((fp8_gemm_few_kernel<RM, ACT, CT>), dim3(cdiv(p.N, 16), cdiv(p.M, 16 * RM)), dim3(512), 0, s, p);
}

int g_force = -1;  // tests and measurements: run this kernel whatever the sizes (fp8_gemm_force)

template <int ACT, int CT>
void launch(const Fp8Gemm& p, hipStream_t s) {
  const long t256 = (long)cdiv(p.M, 256) * cdiv(p.N, 256), t128 = (long)cdiv(p.M, 128) * cdiv(p.N, 128);
  // (the tiled kernels keep 32-bit offsets inside a tile: 256 rows of at most 2^22 bytes)
  const bool narrow = p.lda <= (1 << 22) && p.ldb <= (1 << 22);
  int pick = 0;
  if (!narrow || p.M <= 64) pick = p.M <= 16 ? 0 : p.M <= 32 ? 1 : 2;
  else if (p.bshift == 7 && t256 >= 128) pick = 5;
  else if (t128 >= 128) pick = 4;
  else pick = 3;
  if (g_force >= 0 && (g_force < 3 || narrow) && (g_force != 5 || p.bshift == 7)) pick = g_force;
  switch (pick) {
    case 0: launch_few<1, ACT, CT>(p, s); break;
    case 1: launch_few<2, ACT, CT>(p, s); break;
    case 2: launch_few<4, ACT, CT>(p, s); break;
    case 3: launch_tile<64, 64, 4, ACT, CT>(p, s); break;
    case 4: launch_tile<128, 128, 2, ACT, CT>(p, s); break;
    default: hipLaunchKernelGGL((fp8_gemm_big_kernel<ACT, CT>), dim3((unsigned)t256), dim3(256), 0, s, p);
  }
}

template <int ACT>
void launch_act(const Fp8Gemm& p, int ctype, hipStream_t s) {
  if (ctype == C_BF16) launch<ACT, C_BF16>(p, s);
  else if (ctype == C_F16) launch<ACT, C_F16>(p, s);
  else launch<ACT, C_F32>(p, s);
}

}  // namespace

void fp8_gemm_force(int k) { g_force = k; }

int fp8_gemm_launch(const uint8_t* A, const uint8_t* As, const uint8_t* B, const uint8_t* Bs, void* C,
                    const float* bias, int M, int N, int nk, long lda, long ldb, int ldsa, int ldsb, int bshift,
                    long ldc, int act, int ctype, hipStream_t s) {
  if (M <= 0 || N <= 0 || nk <= 0) return 0;
  const Fp8Gemm p{A, As, B, Bs, C, bias, M, N, nk, lda, ldb, ldsa, ldsb, bshift, ldc};
  if (lda > (1 << 22) && cdiv(M, 64) > 65535) return (int)hipErrorInvalidValue;  // (grid of the few-row kernel)
  if (act == ACT_NONE) launch_act<ACT_NONE>(p, ctype, s);
  else if (act == ACT_RELU) launch_act<ACT_RELU>(p, ctype, s);
  else launch_act<ACT_SILU>(p, ctype, s);
  HIP_CHECK_LAUNCH();
  return 0;
}
