// Row operators of the pre-norm 8-bit linear block: counter-based dropout, root-mean-square norm with the
// residual's addition, and quantisation to e4m3 with a power-of-two scale per block of 128.
//
// All of them stream rows once; a lane owns 8 consecutive elements (16 B of bf16), which is also what one Philox
// call covers (8 x 16 random bits) and a sixteenth of a quantisation block (16 lanes = 128 columns).
#include "common.h"

#include <type_traits>

namespace {

typedef unsigned long long u64;

// ---- element types ----
template <typename T> DEVI float to_f(T v);
template <> DEVI float to_f<bf16_t>(bf16_t v) { return bf2f(v); }
template <> DEVI float to_f<_Float16>(_Float16 v) { return (float)v; }
template <> DEVI float to_f<float>(float v) { return v; }
template <typename T> DEVI T from_f(float v);
template <> DEVI bf16_t from_f<bf16_t>(float v) { return f2bf(v); }
template <> DEVI _Float16 from_f<_Float16>(float v) { return (_Float16)v; }
template <> DEVI float from_f<float>(float v) { return v; }

template <typename T>
struct alignas(16) Pack8 {
  T e[8];
};

// 8 elements as loaded (half the registers of their float values in a 16-bit type)
template <typename T>
struct Raw8 {
  static constexpr int W = (int)sizeof(T) * 2;
  uint32_t w[W];
  DEVI float get(int k) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[k]);
    else if constexpr (std::is_same<T, bf16_t>::value) return __uint_as_float(k & 1 ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[k >> 1] >> (16 * (k & 1))));
  }
  // forget that the float values are known: they are made again where they are used next, not kept in registers
  DEVI void launder() {
#pragma unroll
    for (int i = 0; i < W; ++i) asm volatile("" : "+v"(w[i]));
  }
};

// The same at any address that a T may have: one access as well (the hardware splits it where it must).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Loose8 {
  T e[8];
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 8 consecutive elements of a row from column c on, `valid` of them inside it, as they come from memory.  VEC: rows of
// whole aligned vectors (valid is 0 or 8).  Otherwise a row may begin at any element (by elements alone, 16384 x 4095 took
// four times as long as 16384 x 4096), and its last vector is cut.  In a 16-bit type that vector is the 8 elements that end
// with the row, and settle8 shifts it down, zeros behind (a row shorter than 8 is read by elements): guarded loads of one
// element follow each other, and a wait stands between each (16384 x 4095 bf16 norm, forward + backward: 144 + 220 us
// against 112 + 124).  In float32 the shift costs more than they do (264 + 197 us against 239 + 165).
template <typename T, bool VEC>
DEVI Raw8<T> raw8(const T* p, long c, int valid) {
  Raw8<T> v;
#pragma unroll
  for (int i = 0; i < Raw8<T>::W; ++i) v.w[i] = 0u;
  if constexpr (VEC) {
    if (valid > 0) {
#pragma unroll
      for (int i = 0; i < Raw8<T>::W; i += 4) {
        const uint4 u = ((const uint4*)p)[i >> 2];
        v.w[i] = u.x; v.w[i + 1] = u.y; v.w[i + 2] = u.z; v.w[i + 3] = u.w;
      }
    }
  } else if (valid == 8 || (sizeof(T) == 2 && valid > 0 && c > 0)) {
    const Loose8<T> l = *(const Loose8<T>*)(p + (valid - 8));
    __builtin_memcpy(v.w, l.e, sizeof(l));
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 7; ++k) v.w[k] = k < valid ? __float_as_uint(p[k]) : 0u;
  } else if (valid > 0) {
#pragma unroll
    for (int k = 1; k < 8; ++k)  // place k holds element k + valid - 8, as in the vector that ends with a longer row
      if (k + valid >= 8) v.w[k >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, p[k + valid - 8]) << (16 * (k & 1));
  }
  return v;
}

template <typename T, bool VEC>
DEVI void settle8(Raw8<T>& r, int valid) {
  if constexpr (!VEC && sizeof(T) == 2) {
    const int d = (8 - valid) & 7;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    u32x4 a = {r.w[0], r.w[1], r.w[2], r.w[3]};
    a = d & 4 ? __builtin_shufflevector(a, zero, 2, 3, 4, 5) : a;
    a = d & 2 ? __builtin_shufflevector(a, zero, 1, 2, 3, 4) : a;
    const unsigned sh = (unsigned)(d & 1) * 16;
    r.w[0] = __builtin_amdgcn_alignbit(a[1], a[0], sh);
    r.w[1] = __builtin_amdgcn_alignbit(a[2], a[1], sh);
    r.w[2] = __builtin_amdgcn_alignbit(a[3], a[2], sh);
    r.w[3] = __builtin_amdgcn_alignbit(0u, a[3], sh);
  }
}

template <typename T, bool VEC>
DEVI void load8(const T* p, long c, int valid, float* f) {
  if (valid > 0 || (!VEC && sizeof(T) == 4)) {  // (guarded loads need no branch around them)
    Raw8<T> v = raw8<T, VEC>(p, c, valid);
    settle8<T, VEC>(v, valid);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = v.get(k);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 0.f;
  }
}

template <typename T, bool VEC>
DEVI void store8(T* p, int valid, const float* f) {
  if constexpr (VEC) {
    if (valid > 0) {
      Pack8<T> v;
#pragma unroll
      for (int k = 0; k < 8; ++k) v.e[k] = from_f<T>(f[k]);
      *(Pack8<T>*)p = v;
    }
  } else {
    if (valid == 8) {
      Loose8<T> v;
#pragma unroll
      for (int k = 0; k < 8; ++k) v.e[k] = from_f<T>(f[k]);
      *(Loose8<T>*)p = v;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < valid) p[k] = from_f<T>(f[k]);
    }
  }
}

// ---- dropout ----
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): the counter
// is (element / 8, offset), the key the seed, so element n's number depends on nothing but (n, seed, offset) and the
// backward pass makes the mask again.  16 bits an element: the multiplications, not the bytes, would bound a
// 32-bit-an-element form (two 32 x 32 -> 64 products a round); the drop probability is a multiple of 2^-16 and the
// scale is that of the probability in force, so the expectation is exact.
struct Drop {
  const long long* state;  // [seed, offset] in device memory, or null: the values below
  u64 seed, offset;
  unsigned t;   // dropped where the 16-bit number < t
  float scale;  // 65536 / (65536 - t); 0 where everything is dropped
};

DEVI void philox(u64 g, u64 offset, u64 seed, uint32_t* c) {
  c[0] = (uint32_t)g; c[1] = (uint32_t)(g >> 32); c[2] = (uint32_t)offset; c[3] = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const u64 p0 = (u64)c[0] * 0xD2511F53u, p1 = (u64)c[2] * 0xCD9E8D57u;
    c[0] = (uint32_t)(p1 >> 32) ^ c[1] ^ k0;
    c[1] = (uint32_t)p1;
    c[2] = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
    c[3] = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// bit k: element 8 g + k is kept
DEVI unsigned keep8(u64 g, u64 offset, u64 seed, unsigned t) {
  uint32_t c[4];
  philox(g, offset, seed, c);
  unsigned m = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    m |= ((c[k] & 0xffffu) >= t ? 1u : 0u) << (2 * k);
    m |= ((c[k] >> 16) >= t ? 1u : 0u) << (2 * k + 1);
  }
  return m;
}

// f[k] -> kept ? f[k] * scale : 0 for the elements [first, first + 8).  A select, not a product with 0: an infinity
// in a dropped place leaves 0.  Rows of a width that is no multiple of 8 straddle two Philox blocks.
template <bool VEC>
DEVI void drop8(const Drop& d, u64 seed, u64 offset, long first, float* f) {
  unsigned m = keep8((u64)first >> 3, offset, seed, d.t);
  if constexpr (!VEC) {
    const int sh = (int)(first & 7);
    if (sh) m = ((m | (keep8(((u64)first >> 3) + 1, offset, seed, d.t) << 8)) >> sh);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = (m >> k) & 1 ? f[k] * d.scale : 0.f;
}

DEVI void drop_state(const Drop& d, u64& seed, u64& offset) {
  seed = d.state ? (u64)d.state[0] : d.seed;
  offset = d.state ? (u64)d.state[1] : d.offset;
}

// y = (res +) keep * scale * x over n elements, summed in fp32 and rounded once
template <typename T, bool RES>
__global__ __launch_bounds__(256) void dropout_counter_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                              T* __restrict__ y, long n, Drop d) {
  u64 seed, offset;
  drop_state(d, seed, offset);
  const long groups = (n + 7) >> 3;
  for (long g = blockIdx.x * 256L + threadIdx.x; g < groups; g += (long)gridDim.x * 256) {
    const long i = g * 8;
    const int valid = n - i < 8 ? (int)(n - i) : 8;
    float f[8], r[8];
    if (valid == 8) {
      load8<T, true>(x + i, i, 8, f);
      if constexpr (RES) load8<T, true>(res + i, i, 8, r);
    } else {
      load8<T, false>(x + i, i, valid, f);
      if constexpr (RES) load8<T, false>(res + i, i, valid, r);
    }
    if (d.t != 0) drop8<true>(d, seed, offset, i, f);  // (0: evaluation, the residual's addition alone)
    if constexpr (RES)
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] += r[k];
    if (valid == 8) store8<T, true>(y + i, 8, f);
    else store8<T, false>(y + i, valid, f);
  }
}

// ---- e4m3 blocks ----
constexpr float F32_MAX = 3.4028234663852886e38f;
DEVI float finite_abs(float v) { return fabsf(v) <= F32_MAX ? fabsf(v) : 0.f; }

// the smallest e with amax <= 448 * 2^e = 1.75 * 2^(e + 8), read off the bits of amax; 0 for a block of zeros
DEVI int block_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  if (b == 0) return 0;
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -127 ? -127 : e;  // at most 120 for a finite amax
}

// block b's byte of a scale row; the last block also writes 2^0 into the padding up to a multiple of 4 bytes
DEVI void put_scale(uint8_t* row, int b, int nblocks, int ldsc, int e) {
  row[b] = (uint8_t)(e + 127);
  if (b == nblocks - 1)
    for (int i = nblocks; i < ldsc; ++i) row[i] = 127;
}

// 8 values * 2^-e as e4m3 (round to nearest even).  |v| <= 448 * 2^e, so nothing saturates; an infinity or NaN is
// stored as NaN (e4m3 has no infinity) and does not enter the block's maximum.
DEVI uint2 to_e4m3x8(const float* v, int e) {
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  float s[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) s[k] = fabsf(v[k]) <= F32_MAX ? v[k] * inv : __uint_as_float(0x7fc00000u);
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(s[4], s[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(s[6], s[7], hi, true);
  return make_uint2((unsigned)lo, (unsigned)hi);
}

// maximum over the 16 lanes that hold one 128-column block
DEVI float block_max(const float* f) {
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_abs(f[k]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  return m;
}

// ---- root-mean-square norm ----
// sum over the TPR threads of a row
template <int TPR>
DEVI float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (TPR > 64) {
    const int w = threadIdx.x >> 6;
    __syncthreads();  // the previous row's sums have been read
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += red[i];
  }
  return v;
}

constexpr int nthreads(int tpr) { return tpr == 64 ? 256 : tpr; }  // one row a block where a row needs several waves

// h = res + drop(x), rounded to T (what backward reads); y = h * rsqrt(mean h^2 + eps) * w.  A row stays in registers
// between the two (V vectors a lane), so x, res are read and h, y written once.
template <typename T, int TPR, int V, bool VEC, bool DROP, bool FP8>
__global__ __launch_bounds__(nthreads(TPR)) void rms_fwd_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                                const float* __restrict__ w, T* __restrict__ h,
                                                                T* __restrict__ y, uint8_t* __restrict__ q,
                                                                uint8_t* __restrict__ sc, float* __restrict__ rstd,
                                                                long rows, int N, long ldq, int ldsc, float eps,
                                                                Drop d) {
  __shared__ float red[16];
  constexpr int RPB = nthreads(TPR) / TPR;
  const int t = threadIdx.x % TPR;
  u64 seed = 0, offset = 0;
  if constexpr (DROP) drop_state(d, seed, offset);
  // (a block of several rows holds a wave a row and meets no barrier; otherwise the whole block takes the same rows)
  for (long row = (long)blockIdx.x * RPB + threadIdx.x / TPR; row < rows; row += (long)gridDim.x * RPB) {
    const long base = row * N;
    float f[V][8];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * TPR + t) * 8, valid = N - c < 8 ? (N - c < 0 ? 0 : N - c) : 8;
      load8<T, VEC>(x + base + c, c, valid, f[j]);
      if constexpr (DROP)
        if (valid > 0) drop8<VEC>(d, seed, offset, base + c, f[j]);
      if (res != nullptr) {
        float r[8];
        load8<T, VEC>(res + base + c, c, valid, r);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[j][k] += r[k];
      }
      if (DROP || res != nullptr) {  // what is normalised is h in its own type, stored or not
#pragma unroll
        for (int k = 0; k < 8; ++k) f[j][k] = to_f<T>(from_f<T>(f[j][k]));
        if (h != nullptr) store8<T, VEC>(h + base + c, valid, f[j]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) s += f[j][k] * f[j][k];
    }
    s = row_sum<TPR>(s, red);
    const float inv = 1.f / sqrtf(s / (float)N + eps);
    if (rstd != nullptr && t == 0) rstd[row] = inv;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * TPR + t) * 8, valid = N - c < 8 ? (N - c < 0 ? 0 : N - c) : 8;
      if (w != nullptr) {
        float g[8];
        load8<float, VEC>(w + c, c, valid, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[j][k] *= inv * g[k];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[j][k] *= inv;
      }
      if constexpr (FP8) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k >= valid) f[j][k] = 0.f;  // columns up to the next multiple of 128 are stored as zeros
        const int e = block_exponent(block_max(f[j]));
        if (c < ldq) {
          *(uint2*)(q + row * ldq + c) = to_e4m3x8(f[j], e);
          if ((t & 15) == 0) put_scale(sc + row * ldsc, c >> 7, (int)(ldq >> 7), ldsc, e);
        }
      } else {
        store8<T, VEC>(y + base + c, valid, f[j]);
      }
    }
  }
}

// dh = r (dy w - h r^2 mean(dy w h)) (+ dh_out); dx = drop(dh); a block walks rows and keeps its part of
// dw = sum_rows dy h r in registers: part[block][N], added up by rows_sum_kernel in a fixed order.  A row's three
// inputs are all asked for before the first is used, and stay in their own type until then.
template <typename T, int TPR, int V, bool VEC, bool DROP>
__global__ __launch_bounds__(nthreads(TPR)) void rms_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ h,
                                                                const T* __restrict__ dh_out,
                                                                const float* __restrict__ w,
                                                                const float* __restrict__ rstd, T* __restrict__ dx,
                                                                T* __restrict__ dres, float* __restrict__ part,
                                                                long rows, int N, Drop d) {
  constexpr int RPB = nthreads(TPR) / TPR;
  __shared__ float red[16];
  __shared__ float comb[RPB > 1 ? RPB * TPR * V * 8 : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  u64 seed = 0, offset = 0;
  if constexpr (DROP) drop_state(d, seed, offset);
  float dw[V][8];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[j][k] = 0.f;
  constexpr bool GREG = TPR < 1024;  // the weights stay in registers over the rows where there is room for them
  float gw[GREG ? V : 1][8];
  auto weights = [&](int j, float* g) {
    const int c = (j * TPR + t) * 8, valid = N - c < 8 ? (N - c < 0 ? 0 : N - c) : 8;
    if (w != nullptr) load8<float, VEC>(w + c, c, valid, g);
    else
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = 1.f;
  };
  if constexpr (GREG)
#pragma unroll
    for (int j = 0; j < V; ++j) weights(j, gw[j]);
  for (long row = (long)blockIdx.x * RPB + sub; row < rows; row += (long)gridDim.x * RPB) {
    const long base = row * N;
    Raw8<T> ra[V], rb[V], rc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * TPR + t) * 8, valid = N - c < 8 ? (N - c < 0 ? 0 : N - c) : 8;
      ra[j] = raw8<T, VEC>(dy + base + c, c, valid);
      rb[j] = raw8<T, VEC>(h + base + c, c, valid);
    }
    if (dh_out != nullptr) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (j * TPR + t) * 8, valid = N - c < 8 ? (N - c < 0 ? 0 : N - c) : 8;
        rc[j] = raw8<T, VEC>(dh_out + base + c, c, valid);
      }
    }
    const float inv = rstd[row];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int valid = min(max(N - (j * TPR + t) * 8, 0), 8);
      settle8<T, VEC>(ra[j], valid);
      settle8<T, VEC>(rb[j], valid);
      if constexpr (!GREG) weights(j, gw[0]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float p = ra[j].get(k) * rb[j].get(k);
        dw[j][k] += p * inv;
        s += p * gw[GREG ? j : 0][k];
      }
      ra[j].launder();
      rb[j].launder();
    }
    s = row_sum<TPR>(s, red);
    const float m = s * inv * inv / (float)N;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * TPR + t) * 8, valid = N - c < 8 ? (N - c < 0 ? 0 : N - c) : 8;
      float o[8];
      if (dh_out != nullptr) settle8<T, VEC>(rc[j], valid);
      if constexpr (!GREG) weights(j, gw[0]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        o[k] = inv * (ra[j].get(k) * gw[GREG ? j : 0][k] - rb[j].get(k) * m);
        if (dh_out != nullptr) o[k] += rc[j].get(k);
      }
      if (dres != nullptr) store8<T, VEC>(dres + base + c, valid, o);
      if constexpr (DROP)
        if (valid > 0) drop8<VEC>(d, seed, offset, base + c, o);
      if (dx != nullptr) store8<T, VEC>(dx + base + c, valid, o);
    }
  }
  if (part == nullptr) return;
  float* out = part + (long)blockIdx.x * N;
  if constexpr (RPB > 1) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) comb[(sub * V + j) * TPR * 8 + t * 8 + k] = dw[j][k];
    __syncthreads();
    for (int c = threadIdx.x; c < N; c += nthreads(TPR)) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < RPB; ++i) s += comb[i * V * TPR * 8 + c];
      out[c] = s;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * TPR + t) * 8, valid = N - c < 8 ? (N - c < 0 ? 0 : N - c) : 8;
      store8<float, VEC>(out + c, valid, dw[j]);
    }
  }
}

// out[c] = sum_i part[i][c] in a fixed order.  A block owns 64 columns: 16 lanes of 4 columns x 64 row lanes, so that
// the few hundred partial rows of a column are read in a handful of loads in flight at once (a block of 4 row lanes
// took 75 us for 1024 x 2048 partials: one load after the other).
template <bool VEC>
__global__ __launch_bounds__(1024) void rows_sum_kernel(const float* __restrict__ part, float* __restrict__ out, int G,
                                                        int N) {
  __shared__ float red[64][65];
  __shared__ float fin[4][64];
  const int lc = threadIdx.x & 15, lr = threadIdx.x >> 4;
  const int c = blockIdx.x * 64 + lc * 4;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = lr; i < G; i += 64) {
    if constexpr (VEC) {
      if (c < N) {
        const float4 v = *(const float4*)(part + (long)i * N + c);
        s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += c + k < N ? part[(long)i * N + c + k] : 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) red[lr][lc * 4 + k] = s[k];
  __syncthreads();
  if (threadIdx.x < 256) {
    const int col = threadIdx.x & 63, q = threadIdx.x >> 6;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += red[q * 16 + i][col];
    fin[q][col] = v;
  }
  __syncthreads();
  const int cc = blockIdx.x * 64 + threadIdx.x;
  if (threadIdx.x < 64 && cc < N) out[cc] = (fin[0][threadIdx.x] + fin[1][threadIdx.x]) + (fin[2][threadIdx.x] + fin[3][threadIdx.x]);
}

// ---- quantisation ----
// rows [M][N] of T -> e4m3 [M][ldq] + E8M0 [M][ldsc], 1 x 128 blocks.  256 threads: 16 rows x 128 columns a step,
// down `chunk` rows, so the column sums (a bias gradient) come along.  MASK: where ymask <= 0 the value counts as 0
// (the gradient of a ReLU's input; a NaN there passes it on).  COPY: also a bf16 copy with row stride ldb (zeros behind N).
template <typename T, bool VEC, bool MASK, bool COPY>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* __restrict__ x, const T* __restrict__ ymask,
                                                         uint8_t* __restrict__ q, uint8_t* __restrict__ sc,
                                                         bf16_t* __restrict__ copy, float* __restrict__ part, long M,
                                                         int N, int chunk, long ldq, int ldsc, int ldb) {
  __shared__ float red[16][129];
  const int lc = threadIdx.x & 15, lr = threadIdx.x >> 4;
  const int c = blockIdx.x * 128 + lc * 8, valid = N - c < 8 ? (N - c < 0 ? 0 : N - c) : 8;
  const long r0 = (long)blockIdx.y * chunk, r1 = r0 + chunk < M ? r0 + chunk : M;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (long rr = r0; rr < r1; rr += 16) {
    const long r = rr + lr;
    float f[8];
    load8<T, VEC>(x + r * N + c, c, r < r1 ? valid : 0, f);
    if constexpr (MASK) {
      float y[8];
      load8<T, VEC>(ymask + r * N + c, c, r < r1 ? valid : 0, y);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = y[k] <= 0.f ? 0.f : f[k];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum[k] += f[k];
    const int e = block_exponent(block_max(f));
    if (r < r1) {
      if (q != nullptr) {
        *(uint2*)(q + r * ldq + c) = to_e4m3x8(f, e);
        if (lc == 0) put_scale(sc + r * ldsc, blockIdx.x, gridDim.x, ldsc, e);
      }
      if constexpr (COPY)
        if (c < ldb) *(uint4*)(copy + r * ldb + c) = pack8(f);
    }
  }
  if (part == nullptr) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) red[lr][lc * 8 + k] = sum[k];
  __syncthreads();
  const int cc = blockIdx.x * 128 + threadIdx.x;
  if (threadIdx.x < 128 && cc < N) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += red[i][threadIdx.x];
    part[(long)blockIdx.y * N + cc] = s;
  }
}

// weights [M][N] of T -> e4m3 [M][ldq] and (qt) its transpose [N][ldt], one E8M0 scale a 128 x 128 tile, the same for
// both: sc[tile row][tile column], sct transposed.  One tile a block, 64 values a thread kept in registers.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void quant_tiles_kernel(const T* __restrict__ w, uint8_t* __restrict__ q,
                                                          uint8_t* __restrict__ sc, uint8_t* __restrict__ qt,
                                                          uint8_t* __restrict__ sct, int M, int N, long ldq, int ldsc,
                                                          long ldt, int ldsct) {
  __shared__ float red[4];
  __shared__ uint8_t tile[128][132];  // [column][row]: 33 words a row, so the transposing byte stores spread
  const int lc = threadIdx.x & 15, lr = threadIdx.x >> 4;
  const int c = blockIdx.x * 128 + lc * 8, valid = N - c < 8 ? (N - c < 0 ? 0 : N - c) : 8;
  float f[8][8];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = blockIdx.y * 128 + i * 16 + lr;
    load8<T, VEC>(w + (long)r * N + c, c, r < M ? valid : 0, f[i]);
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_abs(f[i][k]));
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const int e = block_exponent(m);
  if (threadIdx.x == 0) {
    put_scale(sc + (long)blockIdx.y * ldsc, blockIdx.x, gridDim.x, ldsc, e);
    if (qt != nullptr) put_scale(sct + (long)blockIdx.x * ldsct, blockIdx.y, gridDim.y, ldsct, e);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 16 + lr;
    const uint2 v = to_e4m3x8(f[i], e);
    if (blockIdx.y * 128 + r < M) *(uint2*)(q + (long)(blockIdx.y * 128 + r) * ldq + c) = v;
    if (qt != nullptr) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        tile[lc * 8 + k][r] = (uint8_t)(v.x >> (8 * k));
        tile[lc * 8 + 4 + k][r] = (uint8_t)(v.y >> (8 * k));
      }
    }
  }
  if (qt == nullptr) return;
  __syncthreads();
  // 128 columns x 32 words: a wave writes two rows of the transpose a step
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int u = i * 256 + threadIdx.x, col = u >> 5, word = u & 31;
    if (blockIdx.x * 128 + col < N)
      *(uint32_t*)(qt + (long)(blockIdx.x * 128 + col) * ldt + blockIdx.y * 128 + word * 4) =
          *(const uint32_t*)&tile[col][word * 4];
  }
}

// e4m3 blocks -> T (`tile` rows share a scale)
template <typename T>
__global__ __launch_bounds__(256) void dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sc,
                                                      T* __restrict__ y, long M, int N, long ldq, int ldsc, int tile) {
  const long total = M * N;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long r = i / N;
    const int c = (int)(i - r * N);
    const float v = __builtin_amdgcn_cvt_f32_fp8((int)q[r * ldq + c], 0);
    const int s = sc[(r / tile) * ldsc + (c >> 7)];
    y[i] = from_f<T>(s == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(v, s - 127));  // (an E8M0 byte of 255 is a NaN)
  }
}

}  // namespace

// T codes: 0 bf16, 1 fp16, 2 fp32
#define BLOCK_TYPE(code, ...)                                            \
  switch (code) {                                                        \
    case 0: { using T = bf16_t; __VA_ARGS__; } break;                    \
    case 1: { using T = _Float16; __VA_ARGS__; } break;                  \
    case 2: { using T = float; __VA_ARGS__; } break;                     \
    default: return (int)hipErrorInvalidValue;                           \
  }

static Drop make_drop(const long long* state, unsigned long long seed, unsigned long long offset, int t) {
  return Drop{state, seed, offset, (unsigned)t, t >= 65536 ? 0.f : (float)(65536.0 / (65536 - t))};
}

int dropout_counter_launch(const void* x, const void* res, void* y, long n, int type, const long long* state,
                           unsigned long long seed, unsigned long long offset, int t, hipStream_t s) {
  if (n <= 0) return 0;
  const Drop d = make_drop(state, seed, offset, t);
  const long blocks = ((n + 7) / 8 + 255) / 256;
  const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
  BLOCK_TYPE(type, {
    if (res) hipLaunchKernelGGL((dropout_counter_kernel<T, true>), grid, dim3(256), 0, s, (const T*)x, (const T*)res, (T*)y, n, d);
    else hipLaunchKernelGGL((dropout_counter_kernel<T, false>), grid, dim3(256), 0, s, (const T*)x, (const T*)nullptr, (T*)y, n, d);
  })
  HIP_CHECK_LAUNCH();
  return 0;
}

// Threads a row and vectors a thread, the smallest that hold the row.  Forward: two vectors a thread, few registers
// and 8 waves a SIMD (8192 x 2048 with dropout 27.5 us against 28.7 with four vectors, 16384 x 8192 184 against 192).
// Backward: four, where a row's partial dw sits in fewer threads and a row of 2048 needs no barrier (31.3 us against
// 44.0, and 210 against 220).
#define RMS_CASE(LIMIT, T_, V_, ...) if (N <= LIMIT) { constexpr int TPR = T_, V = V_; __VA_ARGS__; }
#define RMS_FWD_SHAPE(N, ...)                      \
  RMS_CASE(512, 64, 1, __VA_ARGS__)                \
  else RMS_CASE(1024, 64, 2, __VA_ARGS__)          \
  else RMS_CASE(2048, 128, 2, __VA_ARGS__)         \
  else RMS_CASE(4096, 256, 2, __VA_ARGS__)         \
  else RMS_CASE(8192, 512, 2, __VA_ARGS__)         \
  else RMS_CASE(16384, 1024, 2, __VA_ARGS__)       \
  else RMS_CASE(32768, 1024, 4, __VA_ARGS__)       \
  else return (int)hipErrorInvalidValue;
#define RMS_BWD_SHAPE(N, ...)                      \
  RMS_CASE(512, 64, 1, __VA_ARGS__)                \
  else RMS_CASE(1024, 64, 2, __VA_ARGS__)          \
  else RMS_CASE(2048, 64, 4, __VA_ARGS__)          \
  else RMS_CASE(4096, 256, 2, __VA_ARGS__)         \
  else RMS_CASE(8192, 256, 4, __VA_ARGS__)         \
  else RMS_CASE(16384, 1024, 2, __VA_ARGS__)       \
  else RMS_CASE(32768, 1024, 4, __VA_ARGS__)       \
  else return (int)hipErrorInvalidValue;

int rms_max_cols() { return 32768; }

int rms_fwd_launch(const void* x, const void* res, const float* w, void* h, void* y, uint8_t* q, uint8_t* sc,
                   float* rstd, long rows, int N, long ldq, int ldsc, float eps, int type, const long long* state,
                   unsigned long long seed, unsigned long long offset, int t, hipStream_t s) {
  if (rows <= 0) return 0;
  const Drop d = make_drop(state, seed, offset, t);
  BLOCK_TYPE(type, {
    RMS_FWD_SHAPE(N, {
      constexpr int NT = nthreads(TPR);
      const long need = (rows + NT / TPR - 1) / (NT / TPR);
      const dim3 grid((unsigned)(need < (1L << 21) ? need : (1L << 21)));
      auto go = [&](auto vec, auto drop, auto fp8) {
        hipLaunchKernelGGL((rms_fwd_kernel<T, TPR, V, decltype(vec)::value, decltype(drop)::value, decltype(fp8)::value>),
                           grid, dim3(NT), 0, s, (const T*)x, (const T*)res, w, (T*)h, (T*)y, q, sc, rstd, rows, N, ldq,
                           ldsc, eps, d);
      };
      using Y = std::true_type; using F = std::false_type;
      const bool vec = N % 8 == 0;
      if (q != nullptr) {
        if (t > 0) return (int)hipErrorInvalidValue;
        if (vec) go(Y{}, F{}, Y{}); else go(F{}, F{}, Y{});
      } else if (t > 0) {
        if (vec) go(Y{}, Y{}, F{}); else go(F{}, Y{}, F{});
      } else {
        if (vec) go(Y{}, F{}, F{}); else go(F{}, F{}, F{});
      }
    })
  })
  HIP_CHECK_LAUNCH();
  return 0;
}

// blocks of a backward launch = rows of the dw partials.  512 keep the chip busy; 1024 cost 3 us more in the sum over
// the partials than they save here (8192 x 2048)
int rms_bwd_blocks(long rows, int N) {
  const long per = N <= 2048 ? 4 : 1, need = (rows + per - 1) / per;
  return (int)(need < 1 ? 1 : need < 512 ? need : 512);
}

int rms_bwd_launch(const void* dy, const void* h, const void* dh, const float* w, const float* rstd, void* dx,
                   void* dres, float* part, int blocks, long rows, int N, int type, const long long* state,
                   unsigned long long seed, unsigned long long offset, int t, hipStream_t s) {
  if (rows <= 0) return 0;
  const Drop d = make_drop(state, seed, offset, t);
  BLOCK_TYPE(type, {
    RMS_BWD_SHAPE(N, {
      constexpr int NT = nthreads(TPR);
      auto go = [&](auto vec, auto drop) {
        hipLaunchKernelGGL((rms_bwd_kernel<T, TPR, V, decltype(vec)::value, decltype(drop)::value>), dim3(blocks),
                           dim3(NT), 0, s, (const T*)dy, (const T*)h, (const T*)dh, w, rstd, (T*)dx, (T*)dres, part, rows,
                           N, d);
      };
      using Y = std::true_type; using F = std::false_type;
      const bool vec = N % 8 == 0;
      if (t > 0) { if (vec) go(Y{}, Y{}); else go(F{}, Y{}); }
      else { if (vec) go(Y{}, F{}); else go(F{}, F{}); }
    })
  })
  HIP_CHECK_LAUNCH();
  return 0;
}

int rows_sum_launch(const float* part, float* out, int G, int N, hipStream_t s) {
  if (N <= 0) return 0;
  if (N % 4 == 0) hipLaunchKernelGGL(rows_sum_kernel<true>, dim3(cdiv(N, 64)), dim3(1024), 0, s, part, out, G, N);
  else hipLaunchKernelGGL(rows_sum_kernel<false>, dim3(cdiv(N, 64)), dim3(1024), 0, s, part, out, G, N);
  HIP_CHECK_LAUNCH();
  return 0;
}

// rows a block of the quantiser walks: enough blocks to fill the chip, at most 256 rows
int quant_rows_chunk(long M, int N) {
  const long cb = (N + 127) / 128;
  int chunk = 16;
  while (chunk < 256 && cb * ((M + chunk * 2 - 1) / (chunk * 2)) >= 2048) chunk *= 2;
  while ((M + chunk - 1) / chunk > 65535) chunk *= 2;  // grid.y
  return chunk;
}

int quant_rows_launch(const void* x, const void* ymask, uint8_t* q, uint8_t* sc, bf16_t* copy, float* part, long M,
                      int N, int chunk, long ldq, int ldsc, int ldb, int type, hipStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  const dim3 grid((unsigned)((N + 127) / 128), (unsigned)((M + chunk - 1) / chunk));
  BLOCK_TYPE(type, {
    auto go = [&](auto vec, auto mask, auto cp) {
      hipLaunchKernelGGL((quant_rows_kernel<T, decltype(vec)::value, decltype(mask)::value, decltype(cp)::value>), grid,
                         dim3(256), 0, s, (const T*)x, (const T*)ymask, q, sc, copy, part, M, N, chunk, ldq, ldsc, ldb);
    };
    using Y = std::true_type; using F = std::false_type;
    const bool vec = N % 8 == 0, mask = ymask != nullptr, cp = copy != nullptr;
    if (vec) {
      if (mask) { if (cp) go(Y{}, Y{}, Y{}); else go(Y{}, Y{}, F{}); }
      else { if (cp) go(Y{}, F{}, Y{}); else go(Y{}, F{}, F{}); }
    } else {
      if (mask) { if (cp) go(F{}, Y{}, Y{}); else go(F{}, Y{}, F{}); }
      else { if (cp) go(F{}, F{}, Y{}); else go(F{}, F{}, F{}); }
    }
  })
  HIP_CHECK_LAUNCH();
  return 0;
}

int quant_tiles_launch(const void* w, uint8_t* q, uint8_t* sc, uint8_t* qt, uint8_t* sct, int M, int N, long ldq,
                       int ldsc, long ldt, int ldsct, int type, hipStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  const dim3 grid((unsigned)((N + 127) / 128), (unsigned)((M + 127) / 128));
  BLOCK_TYPE(type, {
    if (N % 8 == 0) hipLaunchKernelGGL((quant_tiles_kernel<T, true>), grid, dim3(256), 0, s, (const T*)w, q, sc, qt, sct, M, N, ldq, ldsc, ldt, ldsct);
    else hipLaunchKernelGGL((quant_tiles_kernel<T, false>), grid, dim3(256), 0, s, (const T*)w, q, sc, qt, sct, M, N, ldq, ldsc, ldt, ldsct);
  })
  HIP_CHECK_LAUNCH();
  return 0;
}

int dequant_launch(const uint8_t* q, const uint8_t* sc, void* y, long M, int N, long ldq, int ldsc, int tile, int type,
                   hipStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  const long blocks = (M * N + 255) / 256;
  const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
  BLOCK_TYPE(type, {
    hipLaunchKernelGGL((dequant_kernel<T>), grid, dim3(256), 0, s, q, sc, (T*)y, M, N, ldq, ldsc, tile);
  })
  HIP_CHECK_LAUNCH();
  return 0;
}
