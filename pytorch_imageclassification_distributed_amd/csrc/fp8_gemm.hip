// C[M][N] = act(sum_kb 2^(ea[m][kb] + eb[n][kb]) * (A[m][kb] . B[n][kb]) + bias[n]), e4m3 operands, kb = blocks of 128.
//
// One k-step is one scale block: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 128 columns and applies both rows'
// E8M0 bytes itself, so a block scale costs no vector instruction.  (An arbitrary fp32 scale would cost an FMA an
// accumulator and k-step beside the matrix pipe; e4m3 is a floating format, so a power of two loses no significand.)
// The instruction adds the products of 8 neighbouring columns at a time, and cuts each at 2^-13 of the power of two of
// the largest (the sum of the two operands' exponents; a subnormal counts with its format's least, -6); the groups' sums
// keep float32's bits.  So an output is off by at most 7 x 2^-13 of the groups' largest such powers added up: 2^-10.2 of
// sum |a||b| where the largest products are of normal values, more where they are not.  That takes one large product
// beside seven just below the cut; measured are 2^-12.0 of sum |a||b| at most on random bytes (K 128; 2^-14.5 at 1024), and
// 1.5e-5 of the result's norm on normal data, whatever K (the bf16 instruction: 9e-8).  Nothing bounds it relative to a
// result whose terms cancel.
#include <type_traits>

#include "conv_common.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Fp8Gemm {
  const uint8_t* A; const uint8_t* As; const uint8_t* B; const uint8_t* Bs;
  void* C; const float* bias;
  int M, N, nk;      // nk = blocks of 128 columns
  int tail;          // columns of the last block where it is not whole and the bytes behind them may be anything; else 0
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

// a NaN stays one through a ReLU (fmaxf would make it 0)
template <int ACT>
DEVI float act_of(float v) {
  if constexpr (ACT == ACT_RELU) return v < 0.f ? 0.f : v;
  else return apply_act(v, ACT);
}

// four consecutive outputs of one row
template <int ACT, int CT>
DEVI void store4(const Fp8Gemm& p, int m, int n, const f32x4& v, const float* bias) {
  if (m >= p.M || n >= p.N) return;
  float o[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) o[r] = act_of<ACT>(v[r] + bias[r]);
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

// Bytes behind the last column count as zeros, whatever they are (times another operand's zero a NaN byte would still
// make the sum NaN).  bytes[4 i, 4 i + 4) of a piece whose first `keep` bytes are inside:
DEVI uint32_t inside(int keep, int i) {
  const int b = keep - 4 * i;
  return b >= 4 ? ~0u : b <= 0 ? 0u : (1u << (8 * b)) - 1;
}
// A stage of LDS, ROWS x 128 B: every wave sees the last block's tile landed when it calls this, and cleared when it
// returns.  (In LDS, between a barrier and the fragments' reads: once a launch, and nothing added to the other steps.)
template <int ROWS, int NT>
DEVI void clear_tail(char* stage, int tail) {
  const int part = tail >> 4, keep = tail & 15;  // chunk `part` of a row is the first that is not whole
  for (int row = threadIdx.x; row < ROWS; row += NT) {
    uint4* const at = (uint4*)(stage + swz(row, part));
    uint4 v = *at;
    v.x &= inside(keep, 0); v.y &= inside(keep, 1); v.z &= inside(keep, 2); v.w &= inside(keep, 3);
    *at = v;
#pragma unroll
    for (int ch = 1; ch < 8; ++ch)
      if (ch > part) *(uint4*)(stage + swz(row, ch)) = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
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
  const int nk = p.nk, tail_step = p.tail ? nk - 1 : -1;
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
  auto step = [&](auto c, int kt, auto last) __attribute__((always_inline)) {
    constexpr int U = decltype(c)::value;
    wait_vmcnt_lds<(S - 2) * LPS>();
    __builtin_amdgcn_s_barrier();
    if constexpr (decltype(last)::value)
      if (kt == tail_step) clear_tail<BM + BN, 64 * NW>(stage(c), p.tail);
    issue(kt + S - 1, stage(std::integral_constant<int, U + S - 1>{}));
    if (S == 4 ? U == 0 : (kt & 3) == 0) {
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
  // (whole rounds of the ring, then the rest, a cut last step always in it: with exits inside the loop hipcc joins their
  // states at its head, and waits for every load there; a branch there costs it half its registers again)
  const int whole = nk - (p.tail ? 1 : 0);
  constexpr std::false_type N{};
  constexpr std::true_type Y{};
  int kt = 0;
  for (; kt + S <= whole; kt += S) {
    step(std::integral_constant<int, 0>{}, kt, N);
    step(std::integral_constant<int, 1>{}, kt + 1, N);
    if constexpr (S == 4) {
      step(std::integral_constant<int, 2>{}, kt + 2, N);
      step(std::integral_constant<int, 3>{}, kt + 3, N);
    }
  }
  if (kt < nk) {
    step(std::integral_constant<int, 0>{}, kt, Y);
    if (kt + 1 < nk) {
      step(std::integral_constant<int, 1>{}, kt + 1, Y);
      if constexpr (S == 4)
        if (kt + 2 < nk) {
          step(std::integral_constant<int, 2>{}, kt + 2, Y);
          if (kt + 3 < nk) step(std::integral_constant<int, 3>{}, kt + 3, Y);
        }
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
// CUT: the last block is not whole (as a test of p.tail it cost the other case 3 %, and 1 % in the large tile)
template <int RM, bool CUT, int ACT, int CT>
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
  const bool cut = CUT && wid == W - 1;  // this wave has the last block
#pragma unroll 4
  for (int kt = k0; kt < k1 - (cut ? 1 : 0); ++kt) {
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
  if (cut) {
    const long at = (long)(nk - 1) * 128;
    i32x8 tb = frag8((const char*)B + at, (const char*)B + at + 64), ta[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) ta[i] = frag8((const char*)A[i] + at, (const char*)A[i] + at + 64);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const int m = (int)inside(p.tail - fq * 16 - (d >> 2) * 64, d & 3);
      tb[d] &= m;
#pragma unroll
      for (int i = 0; i < RM; ++i) ta[i][d] &= m;
    }
#pragma unroll
    for (int i = 0; i < RM; ++i)
      acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(tb, ta[i], acc[i], 0, 0, 0, (int)Bs[nk - 1], 0, (int)As[i][nk - 1]);
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
// 256 x 256 on 4 waves of 128 x 128, one block a CU.  A k-step of a wave is 32 MFMAs of 32 x 32 x 64 fed by 32
// ds_read_b128: (128 + 128) rows x 128 B x 4 waves + the 64 KB that LDS-DMA writes are 192 KB a step through the LDS
// port, against 256 KB for 8 waves of 128 x 64 (where the port, not the matrix pipe, would set the pace).  The 256
// accumulators of a lane live in AGPRs, the fragments of one k-step in 128 VGPRs; the step runs in two halves of two B
// blocks each (all four A blocks in both), so that every register is refilled where its last MFMA has been issued:
//   first half of step kt (B 0, 1):  B 2, 3 of kt are read;
//   middle: tile kt + 1 has landed, this buffer's reads have ended in every wave: the step's one barrier;
//   second half (B 2, 3):            the 16 LDS-DMA pieces of tile kt + 2 go into this buffer, one an MFMA (two an MFMA
//                                    stall at the 64 B a cycle of the load path: 206 us against 186), and B 0, 1 and,
//                                    block by block, A of kt + 1 are read from the other one.
// 256 x 256 with the ring kernel's schedule, same size: 8 waves of 64 x 128 313 us, of 128 x 64 342, 4 of 128 x 128 482 (it
// spills there: the builtin's accumulators and the fragments share the file), 128 x 128 tiles 405; this schedule needs the
// registers that only a lone wave of a SIMD has.
// 8192 x 8192 x 4096: 211 to 226 us by operands and clock (2.4 to 2.6 PFLOP/s), 186 of 211 the main loop; with loads that always hit L2, or a prefetch into
// L2, no faster; without any load 170 (the clock under full load), so the matrix pipe bounds it.  The rest is the
// epilogue and a block's first loads; persistent blocks that issue the next tile's loads before the outputs were slower
// (249 us: their registers spill).
// The MFMAs are asm statements (accumulators pinned to AGPRs, order kept).  hipcc knows nothing of their hazards: their
// operands come from LDS (its waits see asm operands), a VALU result (the scales) passes a wait of its own, an
// accumulator is used again two MFMAs (128 cycles) later, and the epilogue reads them behind a wait that depends on all of them.
typedef float f32x16_t __attribute__((ext_vector_type(16)));

template <int R>
DEVI void mma32(f32x16_t& acc, const i32x8& b, const i32x8& a, uint32_t sb, uint32_t sa) {
  static_assert(R == 0 || R == 1, "scale byte");
  if constexpr (R == 0)
    asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa) : "memory");
  else
    asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa) : "memory");
}

constexpr int BIG_STAGE = 512 * 128;
constexpr int BIG_BAND = 4;     // tile rows of a band

template <bool CUT, int ACT, int CT>
__global__ __launch_bounds__(256, 1) void fp8_gemm_big_kernel(const Fp8Gemm p) {
  // separate arrays, not one: hipcc makes an LDS read wait for every LDS-DMA that may write what it reads, and tells
  // them apart by the array alone
  __shared__ __attribute__((aligned(16))) char buf0[BIG_STAGE];
  __shared__ __attribute__((aligned(16))) char buf1[BIG_STAGE];
  __shared__ __attribute__((aligned(16))) char out[4][32 * 256];  // a wave's 32 x 128 16-bit outputs
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid >> 1, wn = wid & 1;
  const int gm = (p.M + 255) >> 8, gn = (p.N + 255) >> 8;
  const int lda = (int)p.lda, ldb = (int)p.ldb, nk = p.nk;

  // LDS-DMA sources: piece q of a wave is rows [64 wid + 8 q, + 8) of its 256; lane l brings 16-B chunk (l & 7) of row
  // l >> 3, from source chunk (l & 7) ^ ((row >> 1) & 7), which takes two values over q.  Rows past the end are past
  // the buffer resource: zeros.
  const int lrow = lane >> 3, pch = lane & 7;
  unsigned va[2], vb[2];
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const int ch = (pch ^ ((lrow >> 1) + 4 * o)) * 16;
    va[o] = (unsigned)((wid * 64 + lrow) * lda + ch);
    vb[o] = (unsigned)((wid * 64 + lrow) * ldb + ch);
  }
  const int fr = lane & 31, fh = lane >> 5;
  // fragment (block i, half s) of a buffer: row 32 i + fr of the wave's 128, chunks 4 s + fh and 4 s + fh + 2 (the
  // swizzle depends on fr alone)
  int oa[4], ob[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    oa[c] = swz(wm * 128 + fr, 2 * c + fh);  // chunk 2 c + fh
    ob[c] = 256 * 128 + swz(wn * 128 + fr, 2 * c + fh);
  }
  auto frag = [&](const char* buf, const int* o, int i, int s) __attribute__((always_inline)) {
    return frag8(buf + o[2 * s] + i * 4096, buf + o[2 * s + 1] + i * 4096);
  };

  // an XCD's consecutive tiles walk a band of tile rows column by column, so that its L2 holds four row panels and a few
  // column panels at a time
  const int lin = xcd_remap(blockIdx.x, gm * gn);
  const int band = lin / (BIG_BAND * gn), first = band * BIG_BAND, rows = min(gm - first, BIG_BAND);
  const int rest = lin - band * BIG_BAND * gn;
  const int m0 = __builtin_amdgcn_readfirstlane((first + rest % rows) * 256);
  const int n0 = __builtin_amdgcn_readfirstlane(rest / rows * 256);
  const __amdgpu_buffer_rsrc_t za = make_rsrc(p.A, 0);
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.A + (long)m0 * p.lda, (long)(p.M - m0) * p.lda);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.B + (long)n0 * p.ldb, (long)(p.N - n0) * p.ldb);
  const __amdgpu_buffer_rsrc_t rsa = make_rsrc(p.As + (long)m0 * p.ldsa, (long)(p.M - m0) * p.ldsa);
  const uint32_t* wsb = (const uint32_t*)(p.Bs + (long)(min(n0 + wn * 128, p.N - 1) >> 7) * p.ldsb);
  auto piece = [&](int kt, char* buf, int q, bool live) __attribute__((always_inline)) {
    char* dst = buf + (wid * 64 + (q & 7) * 8) * 128;
    if (q < 8) dma16(live ? ra : za, va[q & 1], kt * 128 + q * 8 * lda, dst);
    else dma16(live ? rb : za, vb[q & 1], kt * 128 + (q - 8) * 8 * ldb, dst + 256 * 128);
  };
  // scales: a word holds four k-steps' bytes; a pair of steps takes bytes 0 and 1, then the words are shifted.  The next
  // words are loaded four steps ahead.  An odd number of steps runs one more on zeros (the DMA pieces past the end come
  // from an empty resource); its scale byte is cleared, so that padding cannot hold a NaN scale.
  const int vsa = (wm * 128 + fr) * p.ldsa;
  const int words = (nk + 3) >> 2;
  const uint32_t last = (nk & 3) ? (1u << (8 * (nk & 3))) - 1 : ~0u;
  uint32_t sx[4], nx[4], sw, nw;
  auto scales = [&](int word) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) nx[i] = __builtin_amdgcn_raw_buffer_load_b32(rsa, vsa, word * 4 + i * 32 * p.ldsa, 0);
    nw = wsb[word];
  };
  // the words have arrived (called behind a wait that covers them): without this hipcc waits again, for everything, where
  // they are used
  auto scales_here = [&]() __attribute__((always_inline)) {
    asm volatile("" : "+v"(nx[0]), "+v"(nx[1]), "+v"(nx[2]), "+v"(nx[3]), "+v"(nw));
  };

  f32x16_t acc[4][4];
  i32x8 a[4][2], b[4][2];
  auto step = [&](auto rc, int kt) __attribute__((always_inline)) {
    constexpr int P = decltype(rc)::value;  // kt & 1
    auto cur = [&]() __attribute__((always_inline)) { if constexpr (P == 0) return (char*)buf0; else return (char*)buf1; };
    auto nxt = [&]() __attribute__((always_inline)) { if constexpr (P == 0) return (char*)buf1; else return (char*)buf0; };
    // MFMA t of a half: A block t / 4, k-half (t >> 1) & 1, B block t & 1 of the half's two
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const int i = t >> 2, s = (t >> 1) & 1, j = t & 1;
      mma32<P>(acc[i][j], b[j][s], a[i][s], sw, sx[i]);
      if (t < 8 && (t & 1) == 0) b[2 + (t >> 2)][(t >> 1) & 1] = frag(cur(), ob, 2 + (t >> 2), (t >> 1) & 1);
    }
    wait_vmcnt<0>();
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    if constexpr (CUT)
      if (kt + 2 == nk) clear_tail<512, 256>(nxt(), p.tail);
    if constexpr (P == 0) {
      if ((kt & 2) == 0) scales(min((kt >> 2) + 1, words - 1));
    } else {
      scales_here();
    }
    const bool live = kt + 2 < nk;
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const int i = t >> 2, s = (t >> 1) & 1, j = 2 + (t & 1);
      mma32<P>(acc[i][j], b[j][s], a[i][s], sw, sx[i]);
      piece(kt + 2, cur(), t, live);
      if (t >= 2 && t < 10 && (t & 1) == 0) b[(t - 2) >> 2][((t - 2) >> 1) & 1] = frag(nxt(), ob, (t - 2) >> 2, ((t - 2) >> 1) & 1);
      if ((t & 3) == 1) a[i][0] = frag(nxt(), oa, i, 0);
      if ((t & 3) == 3) a[i][1] = frag(nxt(), oa, i, 1);
    }
  };

  // the first two k-steps
#pragma unroll
  for (int q = 0; q < 16; ++q) piece(0, buf0, q, true);
#pragma unroll
  for (int q = 0; q < 16; ++q) piece(1, buf1, q, nk > 1);
  scales(0);
  wait_vmcnt<0>();
  __builtin_amdgcn_s_barrier();
  if constexpr (CUT)
    if (nk == 1) clear_tail<512, 256>(buf0, p.tail);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x16_t{};
  acc_ready(acc);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i][0] = frag(buf0, oa, i, 0);
    a[i][1] = frag(buf0, oa, i, 1);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    b[j][0] = frag(buf0, ob, j, 0);
    b[j][1] = frag(buf0, ob, j, 1);
  }
  scales_here();
  int kt = 0;
  do {
    if ((kt & 2) == 0) {
      const uint32_t m = (kt >> 2) == words - 1 ? last : ~0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) sx[i] = nx[i] & m;
      sw = nw & m;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) sx[i] >>= 16;
      sw >>= 16;
    }
    asm volatile("s_nop 1" : "+v"(sx[0]), "+v"(sx[1]), "+v"(sx[2]), "+v"(sx[3]), "+v"(sw));  // VALU result -> MFMA
    step(std::integral_constant<int, 0>{}, kt);
    step(std::integral_constant<int, 1>{}, kt + 1);
    kt += 2;
  } while (kt < nk);
  acc_done(acc);
  wait_vmcnt<0>();  // (LDS-DMA must not outlive the block)
  const int cm = m0 + wm * 128, cn = n0 + wn * 128;
  const bool vec = (p.ldc & 7) == 0;  // then a lane's 8 columns are all inside or all outside
  // bias: past N (and without one) the resource gives zeros
  const __amdgpu_buffer_rsrc_t rbias = make_rsrc(p.bias, p.bias != nullptr ? (long)p.N * 4 : 0);
  float bias[4][4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        bias[j][g][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rbias, (cn + fh * 4) * 4, (j * 32 + g * 8 + r) * 4, 0));
  // acc[i][j][4 g + r]: row 32 i + fr, column 32 j + 8 g + 4 fh + r of the wave's 128 x 128
  if constexpr (CT == C_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          store4<ACT, CT>(p, cm + i * 32 + fr, cn + j * 32 + g * 8 + fh * 4,
                          (f32x4){acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]},
                          bias[j][g]);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    // 16-bit outputs pass through the wave's own LDS, 32 rows at a time, and leave in 16-B chunks, 256 contiguous bytes
    // a row.  16-B chunk c of row r sits at c ^ (r & 15): neither side meets a bank conflict.
    char* st = out[wid];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float v[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = act_of<ACT>(acc[i][j][4 * g + r] + bias[j][g][r]);
          *(uint2*)(st + fr * 256 + (((j * 4 + g) ^ (fr & 15)) << 4) + fh * 8) = make_uint2(pack_c<CT>(v[0], v[1]), pack_c<CT>(v[2], v[3]));
          if (g == 3) __builtin_amdgcn_sched_barrier(0);
        }
      const int c = lane & 15, r0 = lane >> 4;
      uint16_t* C = (uint16_t*)p.C + (long)(cm + i * 32 + r0) * p.ldc + cn + c * 8;
      if (vec) {
        const int left = cn + c * 8 < p.N ? p.M - cm - i * 32 - r0 : 0;  // rows of this lane still inside
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const uint4 v = *(const uint4*)(st + (q * 4 + r0) * 256 + ((c ^ ((q * 4 + r0) & 15)) << 4));
          if (q * 4 < left) *(uint4*)(C + (long)q * 4 * p.ldc) = v;
        }
      } else {  // one column a lane, so that a row still leaves in one piece
        uint16_t* o = (uint16_t*)p.C + (long)(cm + i * 32) * p.ldc + cn + lane;
        const int left = p.M - cm - i * 32;
#pragma unroll 4
        for (int r = 0; r < 32; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = h * 64 + lane;
            const uint16_t v = *(const uint16_t*)(st + r * 256 + (((col >> 3) ^ (r & 15)) << 4) + (col & 7) * 2);
            if (r < left && cn + col < p.N) o[(long)r * p.ldc + h * 64] = v;
          }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

template <int BM, int BN, int S, int ACT, int CT>
void launch_tile(const Fp8Gemm& p, hipStream_t s) {
  hipLaunchKernelGGL((fp8_gemm_kernel<BM, BN, 2, 2, S, ACT, CT>), dim3(cdiv(p.M, BM) * cdiv(p.N, BN)), dim3(256), 0, s, p);
}

template <int RM, int ACT, int CT>
void launch_few(const Fp8Gemm& p, hipStream_t s) {
  const dim3 grid(cdiv(p.N, 16), cdiv(p.M, 16 * RM));
  if (p.tail) hipLaunchKernelGGL((fp8_gemm_few_kernel<RM, true, ACT, CT>), grid, dim3(512), 0, s, p);
  else hipLaunchKernelGGL((fp8_gemm_few_kernel<RM, false, ACT, CT>), grid, dim3(512), 0, s, p);
}

thread_local int g_force = -1;  // tests and measurements: this thread's calls run this kernel where it fits (fp8_gemm_force)

// Which kernel: the one whose time this estimates lowest, in us, from what each measured on 256 CUs - a round of blocks
// costs so much a k-step, plus its first loads and its outputs.  Measured (K 4096 unless given; kernel: us):
//   16 x 4096        few16 7.5   64x64 9.9    128x64 12.6  128x128(4) 19.5  128x128(2) 25   256 38
//   32 x 4096        few32 10.2  64x64 10.4
//   64 x 4096        few32 17.3  64x64 11.3
//   512 x 4096                   64x64 23.2   128x64 18.4  128x128(4) 23.9  128x128(2) 33   256 42
//   1024 x 4096                  64x64 42.2   128x64 34.5  128x128(4) 27.5  128x128(2) 35   256 42
//   2048 x 4096                  64x64 79.6   128x64 64.7  128x128(4) 52.4  128x128(2) 48   256 44
//   4096 x 4096                  64x64 161    128x64 136   128x128(4) 107   128x128(2) 97   256 58
//   8192 x 8192                  64x64 623    128x64 533   128x128(4) 432   128x128(2) 456  256 226
//   8192 x 2048, K 512           64x64 31.8   128x64 36.5  128x128(4) 30.6  128x128(2) 24   256 18
// The constants come from launches that leave part of the chip idle; under full load its clock is lower, and the estimate
// 15 to 25 % short for the two widest tiles (8192 x 8192: 178 of 226; 4096 x 4096: 45 of 58).  That changes the choice
// where they lie within that of each other: 2048 x 4096 takes 128x128(2), 7 % above the best.
enum { K_FEW16, K_FEW32, K_64, K_128x64, K_128_4, K_128_2, K_256, K_COUNT };

double estimate(int k, const Fp8Gemm& p) {
  auto rounds = [&](int bm, int bn, int slots) { return (double)(((long)cdiv(p.M, bm) * cdiv(p.N, bn) + slots - 1) / slots); };
  const long t64 = (long)cdiv(p.M, 64) * cdiv(p.N, 64);
  switch (k) {
    case K_FEW16: return 2.5 + 0.0005 * cdiv(p.N, 16) * cdiv(p.M, 16) * p.nk;
    case K_FEW32: return 2.5 + 0.00077 * cdiv(p.N, 16) * cdiv(p.M, 32) * p.nk;
    case K_64: return rounds(64, 64, 512) * ((t64 <= 256 ? 0.40 : 0.66) * p.nk + 2);  // two blocks a CU
    case K_128x64: return rounds(128, 64, 256) * (0.50 * p.nk + 2.5);
    case K_128_4: return rounds(128, 128, 256) * (0.74 * p.nk + 4);
    case K_128_2: return rounds(128, 128, 512) * (1.05 * p.nk + 7);  // two blocks a CU
    default: return rounds(256, 256, 256) * (1.05 * p.nk + 11);
  }
}

template <int ACT, int CT>
void launch_big(const Fp8Gemm& p, hipStream_t s) {
  const dim3 grid((unsigned)(cdiv(p.M, 256) * cdiv(p.N, 256)));
  if (p.tail) hipLaunchKernelGGL((fp8_gemm_big_kernel<true, ACT, CT>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((fp8_gemm_big_kernel<false, ACT, CT>), grid, dim3(256), 0, s, p);
}

// the kernel of a launch; -1: none takes these sizes
int pick_kernel(const Fp8Gemm& p) {
  // (a grid holds fewer than 2^32 threads a dimension, and 65535 blocks in its second)
  auto tiles = [&](long m, long n) { return ((p.M + m - 1) / m) * ((p.N + n - 1) / n); };
  auto fits = [&](int k) {
    if (k <= K_FEW32) return tiles(1L << 40, 16) < (1L << 23) && (p.M + 15L) / 16 <= 65535;  // 512 threads a block
    const int bm = k == K_64 ? 64 : k == K_256 ? 256 : 128, bn = k <= K_128x64 ? 64 : k == K_256 ? 256 : 128;
    if (tiles(bm, bn) >= (1L << 24)) return false;                // 256
    if (p.lda > (1 << 22) || p.ldb > (1 << 22)) return false;     // 32-bit offsets inside a tile of 256 rows
    return k != K_256 || p.bshift == 7;                           // it takes one scale for its 128 columns
  };
  if (g_force >= 0 && g_force < K_COUNT && fits(g_force)) return g_force;
  int pick = -1;
  double best = 1e30;
  for (int k = 0; k < K_COUNT; ++k)
    if (fits(k) && estimate(k, p) < best) best = estimate(pick = k, p);
  return pick;
}

template <int ACT, int CT>
int launch(const Fp8Gemm& p, hipStream_t s) {
  switch (pick_kernel(p)) {
    case K_FEW16: launch_few<1, ACT, CT>(p, s); break;
    case K_FEW32: launch_few<2, ACT, CT>(p, s); break;
    case K_64: launch_tile<64, 64, 4, ACT, CT>(p, s); break;
    case K_128x64: launch_tile<128, 64, 4, ACT, CT>(p, s); break;
    case K_128_4: launch_tile<128, 128, 4, ACT, CT>(p, s); break;
    case K_128_2: launch_tile<128, 128, 2, ACT, CT>(p, s); break;
    case K_256: launch_big<ACT, CT>(p, s); break;
    default: return (int)hipErrorInvalidValue;
  }
  HIP_CHECK_LAUNCH();
  return 0;
}

template <int ACT>
int launch_act(const Fp8Gemm& p, int ctype, hipStream_t s) {
  if (ctype == C_BF16) return launch<ACT, C_BF16>(p, s);
  if (ctype == C_F16) return launch<ACT, C_F16>(p, s);
  return launch<ACT, C_F32>(p, s);
}

}  // namespace

void fp8_gemm_force(int k) { g_force = k; }

// the kernel that a call of these sizes would run in this thread
int fp8_gemm_plan(int M, int N, int nk, int bshift) {
  Fp8Gemm p{};
  p.M = M; p.N = N; p.nk = nk; p.bshift = bshift;
  p.lda = p.ldb = (long)nk * 128;
  return pick_kernel(p);
}

int fp8_gemm_launch(const uint8_t* A, const uint8_t* As, const uint8_t* B, const uint8_t* Bs, void* C,
                    const float* bias, int M, int N, int nk, int tail, long lda, long ldb, int ldsa, int ldsb, int bshift,
                    long ldc, int act, int ctype, hipStream_t s) {
  if (M <= 0 || N <= 0 || nk <= 0) return 0;
  const Fp8Gemm p{A, As, B, Bs, C, bias, M, N, nk, tail, lda, ldb, ldsa, ldsb, bshift, ldc};
  if (act == ACT_NONE) return launch_act<ACT_NONE>(p, ctype, s);
  if (act == ACT_RELU) return launch_act<ACT_RELU>(p, ctype, s);
  return launch_act<ACT_SILU>(p, ctype, s);
}
