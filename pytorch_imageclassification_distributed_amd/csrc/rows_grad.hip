// dW[N][K] = sum over M rows of dY[m][n] X[m][k]: the weight gradient of a linear layer, bf16 operands, float32 sums.
//
// Both operands are row-major with the contracted index outermost, so their MFMA fragments are read from LDS images
// [64 rows][256 columns] by transposing reads.  256 x 256 outputs on 4 waves of 128 x 128, one block a CU, 32 x 32 x 16
// instructions; a stage of 64 rows is 64 MFMAs of 32 cycles a wave, fed by 64 ds_read_b64_tr_b16 and 16 LDS-DMA pieces:
// the bytes and cycles of the 8-bit product's large tile, and its schedule - one barrier a stage, fragments refilled in
// the registers whose last MFMA has been issued, memory instructions one by one between the MFMAs:
//   first half of a stage (B blocks 0, 1):  B 2, 3 are read;
//   middle: the next stage has landed, this buffer's reads have ended in every wave: the barrier;
//   second half (B 2, 3): the stage after next goes into this buffer; B 0, 1 and, block by block, A of the next stage are
//                         read from the other one.
// Bound by the matrix pipe at the clock that it can hold: 8192 x 8192 x 4096 in 420 us (1.3 PFLOP/s), 65536 rows of
// 512 x 512 in 50 us, 1024 x 1000 x 2048 in 25 us (few output tiles: the rows are split, and the slabs added in order).
#include <type_traits>

#include "conv_common.h"

namespace {

typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct RowsGrad {
  const bf16_t* Y; const bf16_t* X;
  float* C;         // [splits][N][K]
  int M, N, K;
  int ldy, ldx;     // elements a row, multiples of 8
  int rows;         // rows a split, a multiple of 64
};

DEVI void mma(f32x16_t& acc, const bf16x8& b, const bf16x8& a) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a) : "memory");
}

DEVI void dma16(__amdgpu_buffer_rsrc_t r, unsigned voff, int soff, char* lds_wave_base) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds_wave_base, 16, voff, soff, 0, 0);
}

constexpr int STAGE_ROWS = 64, ROW_BYTES = 512, IMAGE = STAGE_ROWS * ROW_BYTES;
constexpr int BAND = 4;

__global__ __launch_bounds__(256, 1) void rows_grad_kernel(const RowsGrad p) {
  // separate arrays, not one: hipcc makes an LDS read wait for every LDS-DMA that may write what it reads, and tells
  // them apart by the array alone
  __shared__ __attribute__((aligned(16))) char buf0[2 * IMAGE];
  __shared__ __attribute__((aligned(16))) char buf1[2 * IMAGE];
  __shared__ __attribute__((aligned(16))) char out[4][32 * 256];  // a wave's 32 x 64 outputs
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid >> 1, wn = wid & 1;
  const int gm = (p.N + 255) >> 8, gn = (p.K + 255) >> 8, tiles = gm * gn;
  // an XCD's consecutive tiles walk a band of tile rows column by column; splits are outermost
  const int all = xcd_remap(blockIdx.x, gridDim.x), split = all / tiles, lin = all - split * tiles;
  const int band = lin / (BAND * gn), first = band * BAND, brows = min(gm - first, BAND), rest = lin - band * BAND * gn;
  const int n0 = __builtin_amdgcn_readfirstlane((first + rest % brows) * 256);
  const int k0 = __builtin_amdgcn_readfirstlane(rest / brows * 256);
  const int m0 = __builtin_amdgcn_readfirstlane(split * p.rows), nrows = min(p.M - m0, p.rows);
  const int stages = (nrows + STAGE_ROWS - 1) / STAGE_ROWS;

  // rows past this split's end are past the resource: zeros in both operands.  Columns past N or K hold other values (or
  // zeros), which reach no output that is stored.
  const __amdgpu_buffer_rsrc_t ry = make_rsrc(p.Y + (long)m0 * p.ldy + n0, 2 * ((long)nrows * p.ldy - n0));
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.X + (long)m0 * p.ldx + k0, 2 * ((long)nrows * p.ldx - k0));
  // piece q of a wave: rows 16 wid + 2 q, + 1 of an image; lane l brings 16-B chunk l & 31 of row l >> 5.  The 32-B block
  // b of row r sits at b ^ 2 (r & 3), so that the four rows of a transposing read meet different banks.
  unsigned vy[2], vx[2];
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const int r = lane >> 5, ch = lane & 31;
    const int src = (((ch >> 1) ^ ((2 * o + r) << 1)) << 5) + ((ch & 1) << 4);
    vy[o] = (unsigned)((wid * 16 + r) * p.ldy * 2 + src);
    vx[o] = (unsigned)((wid * 16 + r) * p.ldx * 2 + src);
  }
  const int sy = 2 * p.ldy, sx = 2 * p.ldx;
  auto piece = [&](int st, char* buf, int q) __attribute__((always_inline)) {
    char* dst = buf + (wid * 16 + (q & 7) * 2) * ROW_BYTES;
    if (q < 8) dma16(ry, vy[q & 1], (st * STAGE_ROWS + q * 2) * sy, dst);
    else dma16(rx, vx[q & 1], (st * STAGE_ROWS + (q - 8) * 2) * sx, dst + IMAGE);
  };

  // fragment (block i of 32 columns, quarter s of 16 rows): lane l holds column l & 31, rows 8 (l >> 5) + 0 .. 7 of the
  // quarter, four rows a transposing read: 16 lanes read 4 rows x 16 columns, lane (tq, tp) 8 bytes of row tq, and
  // receive a column each
  const int fr = lane & 31, fh = lane >> 5;
  const int tq = (lane & 15) >> 2, tp = lane & 3, half16 = (lane >> 4) & 1;
  const int row0 = 8 * fh + tq;  // + 16 s + 4 e: the swizzle depends on tq alone
  int oa[4], ob[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    oa[i] = row0 * ROW_BYTES + (((wm * 8 + i * 2 + half16) ^ (tq << 1)) << 5) + tp * 8;
    ob[i] = IMAGE + row0 * ROW_BYTES + (((wn * 8 + i * 2 + half16) ^ (tq << 1)) << 5) + tp * 8;
  }
  auto frag = [&](char* buf, int o, int s) __attribute__((always_inline)) {
    const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4_t*)(buf + o + s * 16 * ROW_BYTES));
    const bf16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4_t*)(buf + o + (s * 16 + 4) * ROW_BYTES));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  f32x16_t acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x16_t{};
  asm volatile("s_nop 7");

  bf16x8 a[4][4], b[4][4];
#pragma unroll
  for (int q = 0; q < 16; ++q) piece(0, buf0, q);
#pragma unroll
  for (int q = 0; q < 16; ++q) piece(1, buf1, q);
  wait_vmcnt<0>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      a[i][s] = frag(buf0, oa[i], s);
      if (i < 2) b[i][s] = frag(buf0, ob[i], s);
    }

  auto stage = [&](auto rc, int st) __attribute__((always_inline)) {
    constexpr int P = decltype(rc)::value;  // st & 1
    auto cur = [&]() __attribute__((always_inline)) { if constexpr (P == 0) return (char*)buf0; else return (char*)buf1; };
    auto nxt = [&]() __attribute__((always_inline)) { if constexpr (P == 0) return (char*)buf1; else return (char*)buf0; };
    // MFMA t of a half: A block t / 8, quarter (t >> 1) & 3, B block t & 1 of the half's two
#pragma unroll
    for (int t = 0; t < 32; ++t) {
      const int i = t >> 3, s = (t >> 1) & 3, j = t & 1;
      mma(acc[i][j], b[j][s], a[i][s]);
      if (t < 16 && (t & 1) == 0) b[2 + (t >> 3)][(t >> 1) & 3] = frag(cur(), ob[2 + (t >> 3)], (t >> 1) & 3);
    }
    wait_vmcnt<0>();
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int t = 0; t < 32; ++t) {
      const int i = t >> 3, s = (t >> 1) & 3, j = 2 + (t & 1);
      mma(acc[i][j], b[j][s], a[i][s]);
      if ((t & 1) == 0) piece(st + 2, cur(), t >> 1);
      if (t >= 4 && t < 20 && (t & 1) == 0) b[(t - 4) >> 3][((t - 4) >> 1) & 3] = frag(nxt(), ob[(t - 4) >> 3], ((t - 4) >> 1) & 3);
      if (t & 1) a[i][s] = frag(nxt(), oa[i], s);
    }
  };
  int st = 0;
  do {  // an odd number of stages runs one more on zeros
    stage(std::integral_constant<int, 0>{}, st);
    stage(std::integral_constant<int, 1>{}, st + 1);
    st += 2;
  } while (st < stages);
  // the last MFMAs' results before the first read of an accumulator: waits that every accumulator depends on
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm volatile("s_nop 15\n\ts_nop 15" : "+a"(acc[i][0]), "+a"(acc[i][1]), "+a"(acc[i][2]), "+a"(acc[i][3]));
  wait_vmcnt<0>();  // (LDS-DMA must not outlive the block)

  // acc[i][j][4 g + r]: row 32 i + fr, column 32 j + 8 g + 4 fh + r of the wave's 128 x 128.  Through the wave's own LDS,
  // 32 rows x 64 columns at a time, so that a row leaves in 256 contiguous bytes; 16-B chunk c of row r sits at
  // c ^ (r & 15).
  const int cn = n0 + wm * 128, ck = k0 + wn * 128;
  const bool vec = (p.K & 3) == 0;  // then a lane's 4 columns are all inside or all outside
  float* C = p.C + (long)split * p.N * p.K;
  char* so = out[wid];
  const int c = lane & 15, r0 = lane >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x16_t& v = acc[i][jj * 2 + j];
          *(float4*)(so + fr * 256 + (((j * 8 + g * 2 + fh) ^ (fr & 15)) << 4)) =
              make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        }
      float* o = C + (long)(cn + i * 32 + r0) * p.K + ck + jj * 64 + c * 4;
      if (vec) {
        const int left = ck + jj * 64 + c * 4 < p.K ? p.N - cn - i * 32 - r0 : 0;  // rows of this lane still inside
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float4 v = *(const float4*)(so + (q * 4 + r0) * 256 + ((c ^ ((q * 4 + r0) & 15)) << 4));
          if (q * 4 < left) *(float4*)(o + (long)q * 4 * p.K) = v;
        }
      } else {  // one column a lane, so that a row still leaves in one piece
        float* o1 = C + (long)(cn + i * 32) * p.K + ck + jj * 64 + lane;
        const int left = p.N - cn - i * 32;
#pragma unroll 4
        for (int r = 0; r < 32; ++r) {
          const float v = *(const float*)(so + r * 256 + (((lane >> 2) ^ (r & 15)) << 4) + (lane & 3) * 4);
          if (r < left && ck + jj * 64 + lane < p.K) o1[(long)r * p.K] = v;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
}

// out = the sum of the slabs, in order
__global__ __launch_bounds__(256) void slab_sum_kernel(const float* __restrict__ slabs, float* __restrict__ out, long n,
                                                       int count) {
  const long i = (blockIdx.x * 256L + threadIdx.x) * 4;
  if (i + 4 <= n && (n & 3) == 0) {
    float4 s = *(const float4*)(slabs + i);
#pragma unroll 8
    for (int k = 1; k < count; ++k) {
      const float4 v = *(const float4*)(slabs + (long)k * n + i);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    *(float4*)(out + i) = s;
    return;
  }
  for (long e = i; e < i + 4 && e < n; ++e) {
    float s = slabs[e];
    for (int k = 1; k < count; ++k) s += slabs[(long)k * n + e];
    out[e] = s;
  }
}

__global__ __launch_bounds__(256) void zero_kernel(float* __restrict__ p, long n) {
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += (long)gridDim.x * 256) p[i] = 0.f;
}

int stages_of(int M) { return (M + STAGE_ROWS - 1) / STAGE_ROWS; }

}  // namespace

// Row splits: few tiles over many rows leave CUs idle, slabs cost their bytes twice.  Estimated time in us: a round of
// 256 blocks takes 1.05 a stage and 12 for first loads and outputs; the slabs' sum 4 TB/s.  At least as many as keep the
// byte offsets inside a split (and the three stages past its end) in 32 bits.
int rows_grad_splits(int M, int N, int K, int ld) {
  const long tiles = (long)cdiv(N, 256) * cdiv(K, 256);
  const int stages = stages_of(M);
  if (stages == 0) return 1;
  const long most = ((1L << 31) - 1) / (2L * STAGE_ROWS * ld) - 4;  // stages a split can hold
  if (most < 1) return 0;
  const int fewest = (int)((stages + most - 1) / most);
  int best = fewest;
  double least = 1e30;
  for (int s = fewest; s <= (fewest > 64 ? fewest : 64) && s <= stages; ++s) {
    const double t = (double)((tiles * s + 255) / 256) * (1.05 * ((stages + s - 1) / s) + 12) +
                     (s > 1 ? (s + 1) * 4e-6 * N * (double)K / 4 + 3 : 0);
    if (t < least) { least = t; best = s; }
  }
  const int per = (stages + best - 1) / best;  // no empty split
  return (stages + per - 1) / per;
}

// slabs: float32 [splits][N][K], used where splits > 1
int rows_grad_launch(const bf16_t* Y, const bf16_t* X, float* C, float* slabs, int M, int N, int K, int ldy, int ldx,
                     int splits, hipStream_t s) {
  if (N <= 0 || K <= 0) return 0;
  const long n = (long)N * K;
  if (M <= 0) {
    hipLaunchKernelGGL(zero_kernel, dim3((unsigned)((n + 255) / 256 < 4096 ? (n + 255) / 256 : 4096)), dim3(256), 0, s, C, n);
    HIP_CHECK_LAUNCH();
    return 0;
  }
  const int stages = stages_of(M), per = (stages + splits - 1) / splits;
  const long tiles = (long)cdiv(N, 256) * cdiv(K, 256);
  if ((per + 4L) * STAGE_ROWS * 2 * (ldy > ldx ? ldy : ldx) >= (1L << 31) || (splits - 1L) * per >= stages ||
      tiles * splits >= (1L << 31) || (splits > 1 && slabs == nullptr))
    return (int)hipErrorInvalidValue;
  const RowsGrad p{Y, X, splits > 1 ? slabs : C, M, N, K, ldy, ldx, per * STAGE_ROWS};
  hipLaunchKernelGGL(rows_grad_kernel, dim3((unsigned)(tiles * splits)), dim3(256), 0, s, p);
  HIP_CHECK_LAUNCH();
  if (splits > 1) {
    hipLaunchKernelGGL(slab_sum_kernel, dim3((unsigned)((n / 4 + 256) / 256)), dim3(256), 0, s, slabs, C, n, splits);
    HIP_CHECK_LAUNCH();
  }
  return 0;
}
