// dW[N][K] = sum over M rows of dY[m][n] X[m][k]: the weight gradient of a linear layer, bf16 operands, float32 sums.
//
// Both operands are row-major with the contracted index outermost, so their MFMA fragments are read from LDS images
// [64 rows][256 columns] by transposing reads.  256 x 256 outputs on 4 waves of 128 x 128, one block a CU, 32 x 32 x 16
// instructions; a stage of 64 rows is 64 MFMAs of 32 cycles a wave, fed by 64 ds_read_b64_tr_b16 and 16 LDS-DMA pieces:
// the bytes and cycles of the 8-bit product's large tile (128 KB read and 64 KB written through the LDS port in the 2048
// cycles of a stage's MFMAs; waves of 128 x 64 would read 192 KB), and its schedule - one barrier a stage, fragments refilled in
// the registers whose last MFMA has been issued, memory instructions one by one between the MFMAs:
//   first half of a stage (B blocks 0, 1):  B 2, 3 are read;
//   middle: the next stage has landed, this buffer's reads have ended in every wave: the barrier;
//   second half (B 2, 3): the stage after next goes into this buffer; B 0, 1 and, block by block, A of the next stage are
//                         read from the other one.
// Bound by the matrix pipe at the clock that it can hold: 8192 x 8192 x 4096 in 420 us (1.3 PFLOP/s), 65536 rows of
// 512 x 512 in 50 us (few output tiles: the rows are split, and the slabs added in order).
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

// a fragment's 8 rows of a column: two transposing reads of four rows each, `next` bytes apart
DEVI bf16x8 tr_frag(char* at, int next) {
  const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4_t*)at);
  const bf16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4_t*)(at + next));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// 32 x 64 outputs at (row, col): v0 the left 32 columns, v1 the right; v[4 g + r] is row fr, column 8 g + 4 fh + r.  They
// pass through 8 KB of the wave's own LDS, so that a row leaves in 256 contiguous bytes; 16-B chunk c of row r sits at
// c ^ (r & 15).
DEVI void put_32x64(char* so, const f32x16_t& v0, const f32x16_t& v1, float* C, int N, int K, int row, int col, int lane) {
  const int fr = lane & 31, fh = lane >> 5, c = lane & 15, r0 = lane >> 4;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    *(float4*)(so + fr * 256 + (((g * 2 + fh) ^ (fr & 15)) << 4)) = make_float4(v0[4 * g], v0[4 * g + 1], v0[4 * g + 2], v0[4 * g + 3]);
    *(float4*)(so + fr * 256 + (((8 + g * 2 + fh) ^ (fr & 15)) << 4)) = make_float4(v1[4 * g], v1[4 * g + 1], v1[4 * g + 2], v1[4 * g + 3]);
  }
  if ((K & 3) == 0) {  // then a lane's 4 columns are all inside or all outside
    float* o = C + (long)(row + r0) * K + col + c * 4;
    const int left = col + c * 4 < K ? N - row - r0 : 0;  // rows of this lane still inside
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float4 v = *(const float4*)(so + (q * 4 + r0) * 256 + ((c ^ ((q * 4 + r0) & 15)) << 4));
      if (q * 4 < left) *(float4*)(o + (long)q * 4 * K) = v;
    }
  } else {  // one column a lane, so that a row still leaves in one piece
    float* o = C + (long)row * K + col + lane;
    const int left = N - row;
#pragma unroll 4
    for (int r = 0; r < 32; ++r) {
      const float v = *(const float*)(so + r * 256 + (((lane >> 2) ^ (r & 15)) << 4) + (lane & 3) * 4);
      if (r < left && col + lane < K) o[(long)r * K] = v;
    }
  }
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
  const int fh = lane >> 5;
  const int tq = (lane & 15) >> 2, tp = lane & 3, half16 = (lane >> 4) & 1;
  const int row0 = 8 * fh + tq;  // + 16 s + 4 e: the swizzle depends on tq alone
  int oa[4], ob[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    oa[i] = row0 * ROW_BYTES + (((wm * 8 + i * 2 + half16) ^ (tq << 1)) << 5) + tp * 8;
    ob[i] = IMAGE + row0 * ROW_BYTES + (((wn * 8 + i * 2 + half16) ^ (tq << 1)) << 5) + tp * 8;
  }
  auto frag = [&](char* buf, int o, int s) __attribute__((always_inline)) {
    return tr_frag(buf + o + s * 16 * ROW_BYTES, 4 * ROW_BYTES);
  };

  f32x16_t acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x16_t{};
  acc_ready(acc);

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
  acc_done(acc);
  wait_vmcnt<0>();  // (LDS-DMA must not outlive the block)

  const int cn = n0 + wm * 128, ck = k0 + wn * 128;
  float* C = p.C + (long)split * p.N * p.K;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      put_32x64(out[wid], acc[i][jj * 2], acc[i][jj * 2 + 1], C, p.N, p.K, cn + i * 32, ck + jj * 64, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
}

// ---- the small tile ----
// 128 x 128 outputs on 4 waves of 64 x 64, for gradients of few outputs over few rows: four times the blocks of the large
// tile.  A ring of four 32 KB stages of 64 rows, three in flight, since a wave's 16 MFMAs a stage (512 cycles) are
// shorter than the way to memory.  Bound by the LDS port (a stage is 32 KB in and 64 KB out, 96 KB at 128 B a cycle = 770
// cycles) and, for few stages, by the first loads and the outputs.  small / large tile: 1024 x 1000 x 2048 13.2 / 24.6 us,
// 2048 x 2048 x 2048 23.8 / 36.6, 65536 x 512 x 512 42 / 50, 4096 x 4096 x 4096 162 / 105.
__global__ __launch_bounds__(256, 1) void rows_grad_small_kernel(const RowsGrad p) {
  constexpr int PITCH = 256, IMG = STAGE_ROWS * PITCH, PIECES = 8;
  __shared__ __attribute__((aligned(16))) char s0[2 * IMG];  // (separate arrays: as above)
  __shared__ __attribute__((aligned(16))) char s1[2 * IMG];
  __shared__ __attribute__((aligned(16))) char s2[2 * IMG];
  __shared__ __attribute__((aligned(16))) char s3[2 * IMG];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid >> 1, wn = wid & 1;
  const int gm = (p.N + 127) >> 7, gn = (p.K + 127) >> 7, tiles = gm * gn;
  const int all = xcd_remap(blockIdx.x, gridDim.x), split = all / tiles, lin = all - split * tiles;
  const int n0 = __builtin_amdgcn_readfirstlane(lin / gn * 128), k0 = __builtin_amdgcn_readfirstlane(lin % gn * 128);
  const int m0 = __builtin_amdgcn_readfirstlane(split * p.rows), nrows = min(p.M - m0, p.rows);
  const int stages = (nrows + STAGE_ROWS - 1) / STAGE_ROWS;

  // rows past this split's end are past the resource: zeros, also for the stages behind the last
  const __amdgpu_buffer_rsrc_t ry = make_rsrc(p.Y + (long)m0 * p.ldy + n0, 2 * ((long)nrows * p.ldy - n0));
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.X + (long)m0 * p.ldx + k0, 2 * ((long)nrows * p.ldx - k0));
  // piece q of a wave: rows 16 wid + 4 q .. + 3 of an image, lane l chunk l & 15 of row l >> 4; swizzle as above
  const int pr = lane >> 4, ch = lane & 15;
  const int src = (((ch >> 1) ^ (pr << 1)) << 5) + ((ch & 1) << 4);
  const int sy = 2 * p.ldy, sx = 2 * p.ldx;
  const unsigned vy = (unsigned)((wid * 16 + pr) * sy + src), vx = (unsigned)((wid * 16 + pr) * sx + src);
  auto issue = [&](int st, char* buf) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) dma16(ry, vy, (st * STAGE_ROWS + q * 4) * sy, buf + (wid * 16 + q * 4) * PITCH);
#pragma unroll
    for (int q = 0; q < 4; ++q) dma16(rx, vx, (st * STAGE_ROWS + q * 4) * sx, buf + IMG + (wid * 16 + q * 4) * PITCH);
  };
  auto ring = [&](auto c) __attribute__((always_inline)) -> char* {
    constexpr int U = decltype(c)::value % 4;
    if constexpr (U == 0) return s0;
    else if constexpr (U == 1) return s1;
    else if constexpr (U == 2) return s2;
    else return s3;
  };

  const int fh = lane >> 5, tq = (lane & 15) >> 2, tp = lane & 3, half16 = (lane >> 4) & 1;
  int oa[2], ob[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    oa[i] = (8 * fh + tq) * PITCH + (((wm * 4 + i * 2 + half16) ^ (tq << 1)) << 5) + tp * 8;
    ob[i] = IMG + (8 * fh + tq) * PITCH + (((wn * 4 + i * 2 + half16) ^ (tq << 1)) << 5) + tp * 8;
  }
  f32x16_t acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x16_t{};

  // stage st = 4 n + U: it has landed (two younger ones are in flight), every wave has left stage st - 1, whose buffer
  // takes stage st + 3
  auto step = [&](auto c, int st) __attribute__((always_inline)) {
    constexpr int U = decltype(c)::value;
    wait_vmcnt_lds<2 * PIECES>();
    __builtin_amdgcn_s_barrier();
    issue(st + 3, ring(std::integral_constant<int, U + 3>{}));
    char* buf = ring(c);
    bf16x8 a[2][4], b[2][4];
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[i][s] = tr_frag(buf + oa[i] + s * 16 * PITCH, 4 * PITCH);
        b[i][s] = tr_frag(buf + ob[i] + s * 16 * PITCH, 4 * PITCH);
      }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[j][s], a[i][s], acc[i][j], 0, 0, 0);
  };
  issue(0, s0);
  issue(1, s1);
  issue(2, s2);
  // (whole rounds of the ring, then the rest: with exits inside the loop hipcc joins their states at its head, and waits
  // for every load there)
  int st = 0;
  for (; st + 4 <= stages; st += 4) {
    step(std::integral_constant<int, 0>{}, st);
    step(std::integral_constant<int, 1>{}, st + 1);
    step(std::integral_constant<int, 2>{}, st + 2);
    step(std::integral_constant<int, 3>{}, st + 3);
  }
  if (st < stages) {
    step(std::integral_constant<int, 0>{}, st);
    if (st + 1 < stages) {
      step(std::integral_constant<int, 1>{}, st + 1);
      if (st + 2 < stages) step(std::integral_constant<int, 2>{}, st + 2);
    }
  }
  wait_vmcnt<0>();
  __syncthreads();  // s0 holds outputs now
  float* C = p.C + (long)split * p.N * p.K;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    put_32x64(s0 + wid * 8192, acc[i][0], acc[i][1], C, p.N, p.K, n0 + wm * 64 + i * 32, k0 + wn * 64, lane);
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

// tests: the tile of the weight gradients of this thread's forward calls, whatever the sizes (0: by estimate).  The
// backward pass runs in a thread of its own: a call's node takes the value along.
static thread_local int g_force = 0;
void rows_grad_force(int tile) { g_force = tile; }
int rows_grad_forced() { return g_force; }

// The tile's width and the row splits: few tiles over few rows leave CUs idle, slabs cost their bytes twice.  Estimated
// time in us: a round of 256 blocks takes 1.45 a stage and 14 for first loads and outputs, with the small tile 0.5 and 7
// (4096 x 4096 x 4096: 105 and 162 us; 300 x 4096 x 4096: 22 and 31; 4096 x 2048 x 2048: 50 and 38); the slabs' sum
// 4 TB/s.  At least as many splits as keep the byte offsets inside one (and the three stages past its end) in 32 bits; 0
// where even the shortest split is too long.
int rows_grad_plan(int M, int N, int K, int ld, int force, int* tile) {
  const int stages = stages_of(M);
  *tile = 256;
  if (stages == 0) return 1;
  const long most = ((1L << 31) - 1) / (2L * STAGE_ROWS * ld) - 4;  // stages a split can hold
  if (most < 1) return 0;
  const int fewest = (int)((stages + most - 1) / most);
  int best = fewest;
  double least = 1e30;
  for (int t = 128; t <= 256; t += 128) {
    if (force && force != t) continue;
    const long tiles = (long)cdiv(N, t) * cdiv(K, t);
    for (int s = fewest; s <= (fewest > 64 ? fewest : 64) && s <= stages; ++s) {
      const double rounds = (double)((tiles * s + 255) / 256), per = (stages + s - 1) / s;
      const double us = rounds * (t == 256 ? 1.45 * per + 14 : 0.5 * per + 7) +
                        (s > 1 ? (s + 1) * 4e-6 * N * (double)K / 4 + 3 : 0);
      if (us < least) { least = us; best = s; *tile = t; }
    }
  }
  const int per = (stages + best - 1) / best;  // no empty split
  return (stages + per - 1) / per;
}

// slabs: float32 [splits][N][K], used where splits > 1
int rows_grad_launch(const bf16_t* Y, const bf16_t* X, float* C, float* slabs, int M, int N, int K, int ldy, int ldx,
                     int tile, int splits, hipStream_t s) {
  if (N <= 0 || K <= 0) return 0;
  const long n = (long)N * K;
  if (M <= 0) {
    hipLaunchKernelGGL(zero_kernel, dim3((unsigned)((n + 255) / 256 < 4096 ? (n + 255) / 256 : 4096)), dim3(256), 0, s, C, n);
    HIP_CHECK_LAUNCH();
    return 0;
  }
  const int stages = stages_of(M), per = (stages + splits - 1) / splits;
  const long tiles = (long)cdiv(N, tile) * cdiv(K, tile);
  if ((tile != 128 && tile != 256) || (per + 4L) * STAGE_ROWS * 2 * (ldy > ldx ? ldy : ldx) >= (1L << 31) || (splits - 1L) * per >= stages ||
      tiles * splits >= (1L << 31) || (splits > 1 && slabs == nullptr))
    return (int)hipErrorInvalidValue;
  const RowsGrad p{Y, X, splits > 1 ? slabs : C, M, N, K, ldy, ldx, per * STAGE_ROWS};
  if (tile == 256) hipLaunchKernelGGL(rows_grad_kernel, dim3((unsigned)(tiles * splits)), dim3(256), 0, s, p);
  else hipLaunchKernelGGL(rows_grad_small_kernel, dim3((unsigned)(tiles * splits)), dim3(256), 0, s, p);
  HIP_CHECK_LAUNCH();
  if (splits > 1) {
    hipLaunchKernelGGL(slab_sum_kernel, dim3((unsigned)((n / 4 + 256) / 256)), dim3(256), 0, s, slabs, C, n, splits);
    HIP_CHECK_LAUNCH();
  }
  return 0;
}
