// Key/value cache in 8 bits: writing rows, reading them back, preparing
// projected rows into it, and attention over it (gfx950).
//
// A block is 64 tokens of one KV head, K and V apart: 16384 e4m3 codes and one
// power of two 2^e, the smallest with amax * 2^-e <= 448 (the byte e + 127; an
// all-zero block has e = -127). A power of two costs e4m3 nothing (its relative
// step is the same at every scale but for the subnormals below amax * 2^-15), the
// multiplication is exact, and a block that a larger token joins is rescaled
// exactly but for codes that become subnormal.
//
// The codes of a block lie in the order in which the matrix instructions take
// them, 16 bytes a lane, so that an operand is one 1024-byte load of a wave with
// no transposition and no conversion:
//   K  [token / 32][d / 64][(d / 16) & 1][(d / 32) & 1][token % 32][d % 16]
//   V  [d / 32][(token / 8) & 1][(token / 4) & 1][d % 32][token / 16][token % 4]
// In V a 16-byte piece holds one d of 16 tokens: those whose scores one lane
// receives from the product with K (four consecutive tokens of every 16), so the
// probabilities it makes of them are the other operand as they stand.
//
// A bf16 has eight significant bits and is the exact sum of two e4m3 of four
// bits each (and a signed rest): x = hi + lo, hi the nearest e4m3, lo = x - hi.
// Queries and probabilities enter the 8-bit products in these two parts, a query at
// a power of two of its own, probabilities at one for each 32 keys (shift_of below), so that
// what bf16 products would take is kept (the matrix cores align the addends of an
// 8-bit product to about 2^-13 of the largest: measured rms 1e-5 of it).
#include "es_kernels.hpp"

#include <type_traits>

namespace es {
namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short i16x2 __attribute__((ext_vector_type(2)));

constexpr int kBlockBytes = kKv8Block * kHeadDim;
constexpr int kNanCode = 0x7f;
constexpr float kNone = -3.0e38f;  // running maximum before the first key

// e of a block (or row) whose largest finite magnitude is m: m = f * 2^x with
// f in [0.5, 1), and 448 = 0.875 * 2^9.
__device__ __forceinline__ int scale_exponent(float m, int least) {
  if (m == 0.0f) return least;
  const int e = __builtin_amdgcn_frexp_expf(m) - (__builtin_amdgcn_frexp_mantf(m) <= 0.875f ? 9 : 8);
  return e < least ? least : e;
}
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u; }

// Four values -> four codes (nearest even; the values are at most 448 or NaN).
__device__ __forceinline__ int pack_e4m3(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// The same of four values times 2^-e; scale: 2^e.
__device__ __forceinline__ int pack_e4m3(float scale, float a, float b, float c, float d) {
  i16x2 r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(i16x2{0, 0}, a, b, scale, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
  return __builtin_bit_cast(int, r);
}
// Four codes of a block whose power of two rises by 2^shift; those of a NaN row stay.
__device__ __forceinline__ int rescale_e4m3(int codes, int shift) {
  if (codes == 0x01010101 * kNanCode) return codes;
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
  return pack_e4m3(ldexpf(a[0], -shift), ldexpf(a[1], -shift), ldexpf(b[0], -shift), ldexpf(b[1], -shift));
}

// Byte of K's piece (16 dims from 16 c) of token t, and of V's piece of dim d
// with the tokens of t's slot, within a block.
__device__ __forceinline__ int k_piece(int t, int c) {
  return (((t >> 5) * 4 + (c >> 2)) * 2 + (c & 1)) * 1024 + ((c >> 1) & 1) * 512 + (t & 31) * 16;
}
__device__ __forceinline__ int v_piece(int t, int d) {
  return (d >> 5) * 2048 + ((t >> 3) & 1) * 1024 + ((t >> 2) & 1) * 512 + (d & 31) * 16;
}

__device__ __forceinline__ void unpack16(const u32x4 a, const u32x4 b, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf_lo(a[i]);
    x[2 * i + 1] = bf_hi(a[i]);
    x[8 + 2 * i] = bf_lo(b[i]);
    x[8 + 2 * i + 1] = bf_hi(b[i]);
  }
}
__device__ __forceinline__ void load16(const uint16_t* p, float* x) {
  const u32x4* v = reinterpret_cast<const u32x4*>(p);
  unpack16(v[0], v[1], x);
}

// RMS norm of a 256-wide head in 32 bits, 16 dims in each lane of a row of 16. Where
// the sum of squares passes their range the head is taken times 2^-70, which leaves nothing of the epsilon.
__device__ __forceinline__ void norm16(float* x, const float* gain) {
  auto mean = [&]() {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
    return tree16(ss) * (1.0f / 256.0f);
  };
  float ms = mean() + 1e-6f;
  if (__any(!finite(ms))) {
    const float down = finite(ms) ? 1.0f : 0x1p-70f;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] *= down;
    ms = mean() + 1e-6f * down * down;
  }
  const float inv = 1.0f / sqrtf(ms);
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = x[i] * inv * gain[i];
}
// Rotation of dims d and d + 32 (d < 32) of a head: lanes 0, 1 of a row of 16
// hold the first of each pair, lanes 2, 3 the second. cs: 32 (cos, sin) of the
// token. Every lane of the row runs it.
__device__ __forceinline__ void rotate16(float* x, const float2* cs, int c) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float other = dpp_xor2(x[i]);
    const float2 t = cs[(c & 1) * 16 + i];
    x[i] = c < 2 ? fmaf(x[i], t.x, -(other * t.y)) : c < 4 ? fmaf(other, t.y, x[i] * t.x) : x[i];
  }
}
// (cos, sin) of position * inv: the product in double (at position 131071 one
// rounded to 24 bits is off by up to 0.004).
__device__ __forceinline__ float2 angle_cs(int position, float inv) {
  float s, c;
  es_sincos_angle((double)position * (double)inv, &s, &c);
  return make_float2(c, s);
}

// The same of a row of K, in 64 bits up to its e4m3: a code is decided by the last
// bits of a value at a boundary between two (one in four million is within 32 bits'
// rounding of one). The sum of squares, the root by one Newton step, a dim times its gain
// (which 32 bits do not always hold), the angles.
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const i32x2 w = __builtin_bit_cast(i32x2, v);
  return __builtin_bit_cast(double, i32x2{__builtin_amdgcn_update_dpp(0, w[0], CTRL, 0xf, 0xf, false),
                                          __builtin_amdgcn_update_dpp(0, w[1], CTRL, 0xf, 0xf, false)});
}
// To 32 bits, an inexact value to the neighbour with an odd last bit: the
// rounding to e4m3 that follows is that of the value itself.
__device__ __forceinline__ float to_odd(double v) {
  const float f = (float)v;
  const double back = (double)f;
  const uint32_t bits = __float_as_uint(f), down = bits - (fabs(back) > fabs(v));
  return back == v || !finite(f) ? f : __uint_as_float(down | 1);
}
__device__ __forceinline__ double2 angle_cs64(int position, float inv) {
  const double x = (double)position * (double)inv, k = rint(x * 0.63661977236758134308);
  double r = fma(-k, 1.5707963267948966192, x);
  r = fma(-k, 6.123233995736766036e-17, r);
  const double z = r * r;
  double sp = -1.0 / 1307674368000.0, cp = 1.0 / 20922789888000.0;  // Taylor's, |r| <= pi / 4
  const double st[] = {1.0 / 6227020800.0, -1.0 / 39916800.0, 1.0 / 362880.0, -1.0 / 5040.0, 1.0 / 120.0, -1.0 / 6.0};
  const double ct[] = {-1.0 / 87178291200.0, 1.0 / 479001600.0, -1.0 / 3628800.0, 1.0 / 40320.0, -1.0 / 720.0, 1.0 / 24.0, -0.5};
#pragma unroll
  for (int i = 0; i < 6; ++i) sp = fma(sp, z, st[i]);
#pragma unroll
  for (int i = 0; i < 7; ++i) cp = fma(cp, z, ct[i]);
  const double sn = fma(sp * z, r, r), cs = fma(cp, z, 1.0);
  const int q = (int)((long long)k & 3);
  return make_double2(q == 0 ? cs : q == 1 ? -sn : q == 2 ? -cs : sn, q == 0 ? sn : q == 1 ? cs : q == 2 ? -sn : -cs);
}
// cs: 32 (cos, sin) of the token, then somewhere 16 of angle 0 for the lanes that hold no pair.
__device__ __forceinline__ void prepare_key(float* x, const float* gain, const double2* cs, const double2* none, int c) {
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = fma((double)x[i], (double)x[i], ss);
  ss += dpp64<0xB1>(ss);  // xor 1, xor 2, mirrors of 8 and 16 lanes
  ss += dpp64<0x4E>(ss);
  ss += dpp64<0x141>(ss);
  ss += dpp64<0x140>(ss);
  ss = fma(ss, 1.0 / 256.0, 1e-6);
  double inv = __builtin_amdgcn_rsq(ss);
  inv = fma(0.5 * inv, fma(-ss * inv, inv, 1.0), inv);
  const double2* t = c < 4 ? cs + (c & 1) * 16 : none;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const double y = (double)x[i] * (double)gain[i] * inv, other = dpp64<0x4E>(y);
    x[i] = to_odd(fma(y, t[i].x, (c < 2 ? -other : other) * t[i].y));
  }
}
// One (row, query head): 16 lanes, 16 dims in each.
__device__ __forceinline__ void prepare_query(const Kv8Prep& p, size_t at, const float* gain, const float2* cs, int chunk) {
  float x[16];
  load16(p.q_proj + at * 512 + chunk * 16, x);
  norm16(x, gain);
  rotate16(x, cs, chunk);
  u32x4 o[2];
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j >> 2][j & 3] = pack_bf2(x[2 * j], x[2 * j + 1]);
  u32x4* q = reinterpret_cast<u32x4*>(p.query + at * 256 + chunk * 16);
  q[0] = o[0];
  q[1] = o[1];
}

// ---- writing ----
// Block of 64 tokens x one KV head: half of its waves K, half V. A thread holds 16
// dims of T tokens; the block's largest magnitudes meet in LDS, then K goes out in
// pieces as it is held (a wave's four tokens make 64-byte lines) and V through LDS,
// where its tokens and dims change places (padded: 16 bytes every 16 pieces). A
// piece whose tokens are not all written is read, merged and written back; no
// other byte changes. Prepare (PREP) makes the K rows from projections by norm and
// rotation, two tokens a thread so that their 64-bit work spreads over more waves, and
// further blocks make the queries, eight rows each.
// Memory bounds it: 131072 rows of 2 heads, 403 MB, take 77 us (5.2 TB/s, what a
// large copy reaches). Prepare of 4096 rows, 8 query and 2 KV heads: 46 MB in
// 15 us (alone the queries 10.4, the keys with their 64-bit arithmetic on half of the
// CUs 12, when their product with the gain was in 32 bits).
constexpr int kVPad = kBlockBytes + (kBlockBytes / 256) * 16;
__device__ __forceinline__ int v_lds(int byte) { return byte + (byte >> 8) * 16; }

template <bool PREP, int T = PREP ? 2 : 4>
__global__ __launch_bounds__(2048 / T) void k_kv8_write(Kv8 c, Kv8Rows r, Kv8Prep p) {
  constexpr int kHalf = 1024 / T, kWaves = kHalf / 64;  // threads and waves of K (of V)
  __shared__ __attribute__((aligned(16))) uint8_t vt[kVPad];
  __shared__ double2 cs[PREP ? 64 : 1][32], none[PREP ? 16 : 1];
  __shared__ float top[2 * kWaves];       // the waves' largest magnitudes
  __shared__ uint64_t bad[2 * kWaves][T];  // and their lanes with a NaN or infinity, of their T tokens each
  const int tid = threadIdx.x, chunk = tid & 15;
  const int first = r.position / kKv8Block, nblk = (r.position + r.rows - 1) / kKv8Block - first + 1;
  if (PREP && (int)blockIdx.x >= nblk * c.heads) {
    // queries: 32 (row, head) pairs at a time, 16 lanes each
    const int row0 = ((int)blockIdx.x - nblk * c.heads) * 8, rows = min(8, r.rows - row0);
    float2(*qcs)[32] = reinterpret_cast<float2(*)[32]>(cs);
    if (tid < rows * 32) qcs[tid >> 5][tid & 31] = angle_cs(r.position + row0 + (tid >> 5), p.inv_freq[tid & 31]);
    float gain[16];
    load16(p.q_gain + chunk * 16, gain);
    __syncthreads();
    for (int i = tid >> 4; i < rows * p.q_heads; i += 2 * kHalf / 16)
      prepare_query(p, (size_t)row0 * p.q_heads + i, gain, qcs[i / p.q_heads], chunk);
    return;
  }
  const int blk = first + (int)blockIdx.x % nblk, head = (int)blockIdx.x / nblk;
  const int base = blk * kKv8Block;
  const int lo = max(r.position - base, 0), hi = min(r.position + r.rows - base, kKv8Block);
  const bool is_v = tid >= kHalf;
  const int g = (tid % kHalf) >> 4;
  const size_t store = (size_t)head * c.blocks + blk;
  uint8_t* codes = (is_v ? c.v : c.k) + store * kBlockBytes;
  uint8_t* scale = (is_v ? c.v_scale : c.k_scale) + store;
  // All that is read is on its way before any of it is used. K: tokens g,
  // g + 64 / T, ..: V: tokens T g .. T g + T - 1. Pieces that keep other tokens' codes:
  // K's of tokens before the first (if the power of two rises), any of V.
  u32x4 row[T][2], old[T];
#pragma unroll
  for (int i = 0; i < T; ++i) {
    const int t = min(max(is_v ? T * g + i : 64 / T * i + g, lo), hi - 1);
    const u32x4* from = reinterpret_cast<const u32x4*>((is_v ? r.v : r.k) + (int64_t)(base + t - r.position) * r.row_stride +
                                                       (int64_t)head * r.head_stride + chunk * 16);
    row[i][0] = __builtin_nontemporal_load(from);  // read once
    row[i][1] = __builtin_nontemporal_load(from + 1);
  }
  const bool whole = lo == 0 && hi == kKv8Block;
  int before = 255;  // 255: the block holds none
  if (!whole) {
#pragma unroll
    for (int i = 0; i < T; ++i)
      old[i] = *reinterpret_cast<const u32x4*>(codes + (is_v ? (tid % kHalf + kHalf * i) * 16 : k_piece(64 / T * i + g, chunk)));
    if (lo > 0) before = (int)*scale;
  }
  issue_fence();
  if (PREP) {
    for (int i = tid; i < (hi - lo) * 32; i += 2 * kHalf)
      cs[lo + (i >> 5)][i & 31] = angle_cs64(base + lo + (i >> 5), p.inv_freq[i & 31]);
    if (tid < 16) none[tid] = make_double2(1.0, 0.0);
    __syncthreads();
  }
  // The rows stay as bf16 (84 registers and three blocks a CU instead of 107 and two: 77 us
  // instead of 85 for the 131072 above), prepared ones become fp32.
  float x[PREP ? T : 1][16];
  auto value = [&](int i, int j) {
    if constexpr (PREP) return x[i][j];
    const uint32_t u = row[i][j >> 3][(j >> 1) & 3];
    return j & 1 ? bf_hi(u) : bf_lo(u);
  };
  float largest = 0.0f;
  float gain[16];
  uint64_t own_bad[T];
  if (PREP && !is_v) load16(p.k_gain + chunk * 16, gain);
#pragma unroll
  for (int i = 0; i < T; ++i) {
    const int t = is_v ? T * g + i : 64 / T * i + g;
    const bool in = t >= lo && t < hi;
    if (PREP) unpack16(row[i][0], row[i][1], x[PREP ? i : 0]);
    if (PREP && !is_v) prepare_key(x[PREP ? i : 0], gain, cs[min(max(t, lo), hi - 1)], none, chunk);
    // magnitudes compare as integers, a NaN or infinity above every number
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) most = max(most, __float_as_uint(value(i, j)) & 0x7fffffffu);
    most = in ? most : 0;
    own_bad[i] = __ballot(most >= 0x7f800000u);
    if (own_bad[i]) {
      most = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (!finite(value(i, j))) {
          if constexpr (PREP)
            x[i][j] = 0.0f;
          else
            row[i][j >> 3][(j >> 1) & 3] &= j & 1 ? 0xffffu : 0xffff0000u;
        }
        most = max(most, __float_as_uint(value(i, j)) & 0x7fffffffu);
      }
      most = in ? most : 0;
    }
    largest = fmaxf(largest, __uint_as_float(most));
  }
  largest = wave_max(largest);
  const int wave = tid >> 6;
  if ((tid & 63) == 0) {
    top[wave] = largest;
#pragma unroll
    for (int i = 0; i < T; ++i) bad[wave][i] = own_bad[i];
  }
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) largest = fmaxf(largest, top[kWaves * is_v + i]);
  int e = scale_exponent(largest, -127), shift = 0;
  if (before != 255) {  // earlier rows of the block stay: its power of two only rises
    e = max(e, before - 127);
    shift = e + 127 - before;
  }
  const float power = __uint_as_float((uint32_t)(e + 127) << 23);
  if (is_v) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {  // piece of dim 16 chunk + j, dword token / 16
      uint8_t* const to = &vt[v_lds(v_piece(T * g, chunk * 16 + j)) + (T * g >> 4) * 4];
      const int w = pack_e4m3(power, value(0, j), value(1, j), value(T - 2, j), value(T - 1, j));
      if constexpr (T == 4)
        *reinterpret_cast<int*>(to) = w;
      else
        reinterpret_cast<uint16_t*>(to)[g & 1] = (uint16_t)w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const int t = 64 / T * i + g;
      u32x4* at = reinterpret_cast<u32x4*>(codes + k_piece(t, chunk));
      u32x4 o;
      if (t >= lo && t < hi) {
        const uint64_t lanes = (own_bad[i] >> ((g & 3) * 16)) | (bad[kWaves + t / (4 * T)][t % T] >> (t / T % 4 * 16));
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = lanes & 0xffff ? 0x01010101u * kNanCode
                                : (uint32_t)pack_e4m3(power, value(i, 4 * j), value(i, 4 * j + 1), value(i, 4 * j + 2), value(i, 4 * j + 3));
        *at = o;
      } else if (t < lo && shift > 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = (uint32_t)rescale_e4m3((int)old[i][j], shift);
        *at = o;
      }
    }
  }
  __syncthreads();
  if (!is_v) {
    if (tid == 0) *scale = (uint8_t)(e + 127);
    return;
  }
  if (tid == kHalf) *scale = (uint8_t)(e + 127);
#pragma unroll
  for (int n = 0; n < T; ++n) {
    const int piece = tid % kHalf + kHalf * n;
    const int t0 = ((piece >> 6) & 1) * 8 + ((piece >> 5) & 1) * 4;  // its tokens: 16 s + t0 .. + 3, s = 0..3
    u32x4* at = reinterpret_cast<u32x4*>(codes + piece * 16);
    const u32x4 fresh = *reinterpret_cast<const u32x4*>(&vt[v_lds(piece * 16)]);
    if (whole) {
      *at = fresh;
      continue;
    }
    uint32_t take[4], keep[4], any = 0;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      take[s] = keep[s] = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int t = 16 * s + t0 + b;
        if (t >= lo && t < hi) take[s] |= 0xffu << (8 * b);
        if (t < lo && shift > 0) keep[s] |= 0xffu << (8 * b);
      }
      any |= take[s] | keep[s];
    }
    if (!any) continue;
    u32x4 o = old[n];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t moved = keep[s] ? (uint32_t)rescale_e4m3((int)o[s], shift) : 0;
      o[s] = (o[s] & ~(take[s] | keep[s])) | (fresh[s] & take[s]) | (moved & keep[s]);
    }
    *at = o;
  }
}

// One row: a block per head. Every wave holds the whole row (K 16 dims in each of 16
// lanes, V four a lane) and so both powers of two; the first one writes it, and
// where a power of two has risen all of them rescale the rows before it. What bounds it is one
// trip to memory and the fetch of its code: 2.6 us, where the kernel above takes 6.4
// (prepare: 3.9 and more than 10).
template <bool PREP>
__global__ __launch_bounds__(512) void k_kv8_write_one(Kv8 c, Kv8Rows r, Kv8Prep p) {
  __shared__ double2 cs[PREP ? 32 : 1], none[PREP ? 16 : 1];
  const int tid = threadIdx.x, lane = tid & 63, chunk = tid & 15, head = blockIdx.x;
  float gain[16];
  if (PREP && head >= c.heads) {
    const int at = (head - c.heads) * 32 + (tid >> 4);
    float2* qcs = reinterpret_cast<float2*>(cs);
    if (tid < 32) qcs[tid] = angle_cs(r.position, p.inv_freq[tid]);
    load16(p.q_gain + chunk * 16, gain);
    __syncthreads();
    if (at < p.q_heads) prepare_query(p, at, gain, qcs, chunk);
    return;
  }
  const int t = r.position % kKv8Block;
  const size_t store = (size_t)head * c.blocks + r.position / kKv8Block;
  uint8_t *kcodes = c.k + store * kBlockBytes, *vcodes = c.v + store * kBlockBytes;
  const u32x4* k = reinterpret_cast<const u32x4*>(r.k + (int64_t)head * r.head_stride + chunk * 16);
  const u32x4 k0 = k[0], k1 = k[1];
  const uint2 v = *reinterpret_cast<const uint2*>(r.v + (int64_t)head * r.head_stride + lane * 4);
  int kbefore = 255, vbefore = 255;  // 255: the block holds none
  if (t > 0) {
    kbefore = c.k_scale[store];
    vbefore = c.v_scale[store];
  }
  if (PREP) load16(p.k_gain + chunk * 16, gain);
  if (PREP && tid < 32) cs[tid] = angle_cs64(r.position, p.inv_freq[tid]);
  if (PREP && tid < 16) none[tid] = make_double2(1.0, 0.0);
  issue_fence();
  __syncthreads();  // all have read the powers of two (and the angles are there)
  float x[16], y[4] = {bf_lo(v.x), bf_hi(v.x), bf_lo(v.y), bf_hi(v.y)};
  unpack16(k0, k1, x);
  if (PREP) prepare_key(x, gain, cs, none, chunk);
  bool bad = false;
  float kmost = 0.0f, vmost = 0.0f;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    bad |= !finite(x[j]);
    x[j] = finite(x[j]) ? x[j] : 0.0f;
    kmost = fmaxf(kmost, fabsf(x[j]));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bad |= !finite(y[j]);
    y[j] = finite(y[j]) ? y[j] : 0.0f;
    vmost = fmaxf(vmost, fabsf(y[j]));
  }
  bad = __any(bad);
  int ke = scale_exponent(row16_max(kmost), -127), ve = scale_exponent(wave_max(vmost), -127);
  const int kshift = kbefore == 255 ? 0 : max(ke + 127 - kbefore, 0), vshift = vbefore == 255 ? 0 : max(ve + 127 - vbefore, 0);
  if (kbefore != 255) ke = max(ke, kbefore - 127);
  if (vbefore != 255) ve = max(ve, vbefore - 127);
  if (kshift > 0) {
    for (int n = 0; n < 2; ++n) {
      const int token = (tid >> 4) + 32 * n;
      if (token >= t) break;
      u32x4* at = reinterpret_cast<u32x4*>(kcodes + k_piece(token, chunk));
      u32x4 o = *at;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = (uint32_t)rescale_e4m3((int)o[j], kshift);
      *at = o;
    }
  }
  if (vshift > 0) {
    for (int n = 0; n < 2; ++n) {
      const int piece = tid + 512 * n, first = ((piece >> 6) & 1) * 8 + ((piece >> 5) & 1) * 4;
      uint32_t* at = reinterpret_cast<uint32_t*>(vcodes + piece * 16);
      const u32x4 w = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int left = t - first - 16 * s;  // tokens of these four before the row's
        const uint32_t o = (uint32_t)rescale_e4m3((int)w[s], vshift);
        if (left >= 4)
          at[s] = o;
        else
          for (int b = 0; b < left; ++b) reinterpret_cast<uint8_t*>(at + s)[b] = (uint8_t)(o >> (8 * b));
      }
    }
  }
  if (tid >= 64) return;
  if (lane < 16) {
    const float power = __uint_as_float((uint32_t)(ke + 127) << 23);
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = bad ? 0x01010101u * kNanCode : (uint32_t)pack_e4m3(power, x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
    *reinterpret_cast<u32x4*>(kcodes + k_piece(t, chunk)) = o;
  }
  const uint32_t o = (uint32_t)pack_e4m3(__uint_as_float((uint32_t)(ve + 127) << 23), y[0], y[1], y[2], y[3]);
  uint8_t* at = vcodes + v_piece(t, lane * 4) + (t >> 4) * 4 + (t & 3);
#pragma unroll
  for (int j = 0; j < 4; ++j) at[16 * j] = (uint8_t)(o >> (8 * j));
  if (lane == 0) {
    c.k_scale[store] = (uint8_t)(ke + 127);
    c.v_scale[store] = (uint8_t)(ve + 127);
  }
}

// ---- reading ----
// Block of 256 threads = 64 tokens x one head x K or V; V through LDS as above.
__global__ __launch_bounds__(256) void k_kv8_read(Kv8 c, int position, int rows, uint16_t* k, uint16_t* v,
                                                  int64_t row_stride, int64_t head_stride) {
  __shared__ __attribute__((aligned(16))) uint8_t vt[kVPad];
  const int tid = threadIdx.x, chunk = tid & 15, g = tid >> 4;
  const int first = position / kKv8Block, nblk = (position + rows - 1) / kKv8Block - first + 1;
  const int blk = first + (int)blockIdx.x % nblk, head = (int)blockIdx.x / nblk;
  const bool is_v = blockIdx.y;
  const int base = blk * kKv8Block;
  const int lo = max(position - base, 0), hi = min(position + rows - base, kKv8Block);
  const size_t store = (size_t)head * c.blocks + blk;
  const uint8_t* codes = (is_v ? c.v : c.k) + store * kBlockBytes;
  const int e = (int)(is_v ? c.v_scale : c.k_scale)[store] - 127;
  int w[4][4];  // codes of 16 dims of four tokens
  bool nan[4];
  if (is_v) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int piece = tid + 256 * n;
      *reinterpret_cast<u32x4*>(&vt[v_lds(piece * 16)]) = *reinterpret_cast<const u32x4*>(codes + piece * 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      nan[i] = (c.k[store * kBlockBytes + k_piece(4 * g + i, 0)] & 0x7f) == kNanCode;
    __syncthreads();
    uint32_t d[16];
#pragma unroll
    for (int j = 0; j < 16; ++j)
      d[j] = *reinterpret_cast<const uint32_t*>(&vt[v_lds(v_piece(4 * g, chunk * 16 + j)) + (g >> 2) * 4]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[i][j] = (int)(((d[4 * j] >> (8 * i)) & 255) | (((d[4 * j + 1] >> (8 * i)) & 255) << 8) |
                        (((d[4 * j + 2] >> (8 * i)) & 255) << 16) | (((d[4 * j + 3] >> (8 * i)) & 255) << 24));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const i32x4 a = *reinterpret_cast<const i32x4*>(codes + k_piece(16 * i + g, chunk));
#pragma unroll
      for (int j = 0; j < 4; ++j) w[i][j] = a[j];
      nan[i] = false;  // its codes say so themselves
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = is_v ? 4 * g + i : 16 * i + g;
    if (t < lo || t >= hi) continue;
    u32x4 o[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w[i][j], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w[i][j], true);
      o[j >> 1][(j & 1) * 2] = nan[i] ? 0x7fc07fc0u : pack_bf2(ldexpf(a[0], e), ldexpf(a[1], e));
      o[j >> 1][(j & 1) * 2 + 1] = nan[i] ? 0x7fc07fc0u : pack_bf2(ldexpf(b[0], e), ldexpf(b[1], e));
    }
    u32x4* at = reinterpret_cast<u32x4*>((is_v ? v : k) + (int64_t)(base + t - position) * row_stride +
                                         (int64_t)head * head_stride + chunk * 16);
    at[0] = o[0];
    at[1] = o[1];
  }
}

// ---- attention ----
constexpr float kLog2e = 1.44269504088896341f;
// Four values (at most 448, of eight significant bits) in two parts: the nearest
// codes, and the codes of 16 times the rest (which below 2^-6 rounds by 2^-14 at most).
__device__ __forceinline__ int2 split_e4m3(float a, float b, float c, float d) {
  const int h = pack_e4m3(a, b, c, d);
  const f32x2 u = __builtin_amdgcn_cvt_pk_f32_fp8(h, false), v = __builtin_amdgcn_cvt_pk_f32_fp8(h, true);
  return make_int2(h, pack_e4m3((a - u[0]) * 16.0f, (b - u[1]) * 16.0f, (c - v[0]) * 16.0f, (d - v[1]) * 16.0f));
}
// A float's magnitude as bits that compare as integers, zero for a NaN or infinity.
__device__ __forceinline__ uint32_t finite_bits(uint32_t x) {
  x &= 0x7fffffffu;
  return x < 0x7f800000u ? x : 0;
}

// The reference m of a query's exponents lies kShift below the largest score at which
// it was set, and moves when a score passes m + kShift by more than kSlack (base 2).
constexpr float kSlack = 4.0f, kShift = 4.0f;
constexpr int kOne = 127, kLo = 127 - 4, kProb = 127 - 4;  // scale operands, 2^(byte - 127)

// A probability enters its product as the sum of two e4m3, the lower one 2^5 times
// too large, at a power of two that 32 keys of a query share: a lane's scale operand covers
// 16 bytes of several lanes, which are of a block the tokens 16 j + 0 .. 7, or 16 j + 8 .. 15. The
// largest of the 32 is brought to 2^7 .. 2^8. So each has eight significant bits down to 2^-13 of
// that one, and an error of 2^-15, 2^-22 of it, below; a long flat rest keeps its weight
// however far it lies below a single key elsewhere. (At one power for all keys, and the lower part
// at the upper's, 131072 keys 10 nats below a first one lost 0.8 %, 16384 of 128 heads half.)
// For the rest of those 32 themselves: where their largest outweighs the other three of its four
// eights by 2^kAlone, what is at most the largest of these takes a product of its
// own, at a power of two by that one. (For every block with a key 2^18 below its largest a
// prompt chunk took 4 % longer at scores of unit deviation and 24 % at a deviation of two, so 2 and 3.)
constexpr float kRest = 0.03125f, kMostShift = kProb - 5, kNoShift = -2.0f, kMostRef = 0x1p18f, kAlone = 13.0f;
constexpr int kRestScale = -5, kNever = 500;
// Exponent of a power of two by the logarithm, less m, of what comes to 2^7 .. 2^8: the most where there
// is no key (-inf), or far below m. A reference too large to take it off exactly keeps all at one power.
__device__ __forceinline__ float shift_of(float x, float m) {
  return fminf(floorf(8.0f - x), fabsf(m) < kMostRef ? kMostShift : kNoShift);
}
// Four probabilities in two parts.
__device__ __forceinline__ int2 split_probabilities(const float* y) {
  const int h = pack_e4m3(y[0], y[1], y[2], y[3]);
  const f32x2 u = __builtin_amdgcn_cvt_pk_f32_fp8(h, false), w = __builtin_amdgcn_cvt_pk_f32_fp8(h, true);
  return make_int2(h, pack_e4m3(kRest, y[0] - u[0], y[1] - u[1], y[2] - w[0], y[3] - w[1]));
}
// Moves those of y that times 2^up are at most 2^8 (as rounded) to z, so multiplied; kNever: none.
__device__ __forceinline__ void take_small(float* y, float* z, int up) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = ldexpf(y[i], up);
    const bool is = x <= 257.0f;
    z[i] = is ? x : 0.0f;
    y[i] = is ? 0.0f : y[i];
  }
}

// the hardware's reciprocal, within 1 ulp
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }
// Numbers 0 .. 2^22 by a small divisor: (int)(n * inv) is off by one at most.
__device__ __forceinline__ int2 divide(int n, int by, float inv) {
  int q = (int)((float)n * inv), r = n - q * by;
  if (r < 0) q -= 1, r += by;
  if (r >= by) q += 1, r -= by;
  return make_int2(q, r);
}

// Barrier that publishes LDS writes but leaves DMA on its way.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Few queries: 16 NT (row, query head) pairs of one KV head against a range of
// keys. Four waves share a 64-token block of it; a block of threads is one to
// four such groups, which take the range's blocks in turn.
//   S[token, query] = K Q^T, 16x16x128: wave w takes tokens 16 w .. 16 w + 15; lane
//   (n = lane % 16, g = lane / 16) gives K bytes of token n and Q bytes of query n
//   and receives tokens 4 g .. 4 g + 3 of query n;
//   O^T[d, query] += V^T P^T: wave w takes dims 64 w .. 64 w + 63; the 128 places along
//   tokens hold the upper parts of the 64 probabilities and their lower parts,
//   against V twice.
// So each byte of K and V enters one wave's registers once, straight from memory,
// and the largest scores and the probabilities alone pass between waves, through LDS with one
// barrier a block: it publishes a block's largest scores, from which every wave takes the
// powers of two of 32 keys and the reference, and the block before's probabilities. What bounds a
// short context is how many bytes each CU must fetch (measured 20 a cycle), a long one memory
// (131072 tokens, 2 heads: 134 MB in 25 us, 5.3 TB/s), many queries the products and
// exponentials of four waves on a SIMD. (Probabilities before the barrier, at one power of
// two for all keys, with 8 query and 2 KV heads: 1000 rows alone 14.2 us and 15.8 so, 128 behind 28672
// 44.2 and 48.8, one behind 131071 28.4 and 28.9.)
// The next block's K is fetched as soon as this one's products have read it, its V
// likewise: 32 KB of a group on their way.
// The bound of 1024 threads holds for every G: it keeps the compiler to the 128
// vector registers of 16 waves a CU and off the accumulator registers.
template <int NT, int G>
__global__ __launch_bounds__(1024) void k_kv8_attn_few(Kv8 c, Kv8Attn a) {
  // bytes: the queries' parts; a group's two buffers of probabilities, and of those with a power of two of their own
  constexpr int kQueryBytes = NT * 8192, kProbBytes = NT * 4096, kLowBytes = NT * 4608;
  constexpr int kSumRow = 260, kSum = NT * 16 * kSumRow;  // floats: a query's row of sums; a group's sums
  // the queries and probabilities; at the end, in their place, the groups' sums
  constexpr int kLow = kQueryBytes + G * kProbBytes, kTops = kLow + G * kLowBytes, kTopBytes = NT * 16 * 32;  // largest scores: of a group, one buffer
  constexpr int kIn = kTops + 2 * G * kTopBytes, kOut = G > 1 ? G * kSum * 4 : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kIn > kOut ? kIn : kOut];
  __shared__ __attribute__((aligned(16))) float sums[G][NT * 16][4];
  __shared__ float most[G][NT * 16];
  __shared__ struct {
    float power;  // the query's power of two / 16, for base 2
    int last;     // its last key
  } of_query[NT * 16];
  const int tid = threadIdx.x, lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 3), group = __builtin_amdgcn_readfirstlane(tid >> 8);
  int split = blockIdx.x, tile = blockIdx.y, head = blockIdx.z;
  if (gridDim.y < (uint32_t)a.tiles) {  // all tiles of a range on one XCD: they share its keys in the L2
    const int local = split >> 3, range = local / a.tiles * 8 + (split & 7);
    tile = local % a.tiles;
    head = range / a.splits;
    split = range % a.splits;
    if (head >= c.heads) return;
  }
  const int pairs = a.rows * a.group, end = a.position + a.rows;  // keys that exist
  const int pair0 = tile * 16 * NT;
  const int tile_last = a.position + divide(min(pair0 + 16 * NT - 1, pairs - 1), a.group, a.inv_group).x;
  const int nblk = tile_last / kKv8Block + 1;
  const int b0 = split * a.per, b1 = min(b0 + a.per, nblk), turns = max(0, (b1 - b0 + G - 1) / G);
  const size_t store = (size_t)head * c.blocks;
  // the wave's part of the block and the lane's of that
  const uint8_t* kp = c.k + store * kBlockBytes + (wave >> 1) * 8192 + (wave & 1) * 256 + 2048;  // all its offsets fit a load's
  const uint8_t* vp = c.v + store * kBlockBytes + wave * 4096;
  const uint32_t klane = (g >> 1) * 2048 + (g & 1) * 512 + n * 16, vlane = (g >> 1) * 1024 + (g & 1) * 512 + n * 16;
  i32x4 kr[4], vr[4];
  int ke = 0, ve = 0;
  auto fetch_k = [&](int b) {
    const uint8_t* at = kp + (size_t)b * kBlockBytes;
    ke = c.k_scale[store + b];
#pragma unroll
    for (int i = 0; i < 4; ++i) kr[i] = *reinterpret_cast<const i32x4*>(at + ((i >> 1) * 4096 + (i & 1) * 1024 - 2048) + klane);
  };
  auto fetch_v = [&](int b) {
    const uint8_t* at = vp + (size_t)b * kBlockBytes;
    ve = c.v_scale[store + b];
#pragma unroll
    for (int i = 0; i < 4; ++i) vr[i] = *reinterpret_cast<const i32x4*>(at + (i >> 1) * 2048 + (i & 1) * 256 + vlane);
  };
  if (tid < 16 * NT) of_query[tid].last = a.position + divide(min(pair0 + tid, pairs - 1), a.group, a.inv_group).x;
  // queries: 16 lanes a query, 16 dims a lane; their loads go out before the first
  // keys' (loads return in order), which are on their way during the conversion
  {
    const int chunk = tid & 15;
    u32x4 x[2];
    const int at = min(tid >> 4, 16 * NT - 1);
    const int2 rq = divide(min(pair0 + at, pairs - 1), a.group, a.inv_group);
    const u32x4* qp = reinterpret_cast<const u32x4*>(
        a.query + ((size_t)rq.x * a.q_heads + head * a.group + rq.y) * 256 + chunk * 16);
    x[0] = qp[0];
    x[1] = qp[1];
    issue_fence();
    const int first = b0 < b1 ? min(b0 + group, b1 - 1) : nblk - 1;
    fetch_k(first);
    fetch_v(first);
    issue_fence();
    // 256 threads convert 16 queries at a time
    for (int q = tid >> 4; q < 16 * NT; q += G * 16) {
      if (q != at) {
        const int2 next = divide(min(pair0 + q, pairs - 1), a.group, a.inv_group);
        qp = reinterpret_cast<const u32x4*>(a.query + ((size_t)next.x * a.q_heads + head * a.group + next.y) * 256 + chunk * 16);
        x[0] = qp[0];
        x[1] = qp[1];
      }
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        top = max(top, max(finite_bits(x[i >> 2][i & 3] << 16), finite_bits(x[i >> 2][i & 3] & 0xffff0000u)));
      const int e = scale_exponent(row16_max(__uint_as_float(top)), -100);
      if (chunk == 0) of_query[q].power = ldexpf(kLog2e / 16.0f, e);
      i32x4 hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = x[i >> 1][(i & 1) * 2], w = x[i >> 1][(i & 1) * 2 + 1];
        const int2 p = split_e4m3(ldexpf(bf_lo(u), -e), ldexpf(bf_hi(u), -e), ldexpf(bf_lo(w), -e), ldexpf(bf_hi(w), -e));
        hi[i] = p.x;
        lo[i] = p.y;
      }
      // [tile][part][128 dims][16 of 32 dims][lane of the product]
      uint8_t* to = lds + (q >> 4) * 8192 + (chunk >> 3) * 2048 + (chunk & 1) * 1024 + ((chunk >> 1) & 3) * 256 + (q & 15) * 16;
      *reinterpret_cast<i32x4*>(to) = hi;
      *reinterpret_cast<i32x4*>(to + 4096) = lo;
    }
  }
  lds_barrier();
  f32x4 o[NT][4];
  float m[NT], l[NT];  // the reference, less kShift; the lane's part of the sum, times 2^kShift
#pragma unroll
  for (int q = 0; q < NT; ++q) {
    m[q] = kNone;
    l[q] = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[q][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // of a turn's buffer and a tile: upper parts, lower parts
  auto prob_of = [&](int turn, int q) {
    return reinterpret_cast<int*>(lds + kQueryBytes + group * kProbBytes) + ((turn & 1) * NT + q) * 512;
  };
  // the same of those with a power of two of their own, then the lanes' scale operands
  auto low_of = [&](int turn, int q) { return reinterpret_cast<int*>(lds + kLow + group * kLowBytes) + ((turn & 1) * NT + q) * 576; };
  // hi of dims 0 .. 127 and 128 .. 255, lo of both
  auto queries = [&](int q, i32x8* w, int from) {
    const i32x4* at = reinterpret_cast<const i32x4*>(lds + q * 8192) + lane;
#pragma unroll
    for (int i = from; i < 4; ++i) w[i] = __builtin_shufflevector(at[i * 128], at[i * 128 + 64], 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // One tile's upper parts stay in registers, which have no room for the lower ones too (40 rows behind
  // 20000 18.4 us, 19.1 with none).
  i32x8 w[4];
  if constexpr (NT == 1) queries(0, w, 0);
  // largest scores of a query in a block: [first or second 8 of every 16 tokens][wave]
  auto top_of = [&](int turn, int q) {
    return reinterpret_cast<float*>(lds + kTops + ((turn & 1) * G + group) * kTopBytes) + (q * 16 + n) * 8;
  };
  f32x4 s[NT];
  int scales = 0;  // operands of the lane's parts of the probabilities, a byte each
  auto scores = [&](int turn, auto more) {
    const int mine = b0 + group + turn * G, b = min(mine, b1 - 1);
    {
      i32x8 k[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) k[h] = __builtin_shufflevector(kr[2 * h], kr[2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        queries(q, w, NT == 1 ? 2 : 0);
        const f32x4 zero = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        s[q] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k[0], w[0], zero, 0, 0, 0, kOne, 0, kOne);
        f32x4 rest = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k[0], w[2], zero, 0, 0, 0, kOne, 0, kLo);
        s[q] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k[1], w[1], s[q], 0, 0, 0, kOne, 0, kOne);
        rest = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k[1], w[3], rest, 0, 0, 0, kOne, 0, kLo);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[q][i] += rest[i];
      }
    }
#pragma unroll
    for (int q = 0; q < NT; ++q) asm volatile("" : "+v"(s[q]));  // the keys' registers are free
    const float power = ldexpf(1.0f, ke - 127);
    issue_fence();
    if constexpr (decltype(more)::value) fetch_k(min(mine + G, b1 - 1));
    issue_fence();
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      const auto own = of_query[16 * q + n];
      const float cs = fmaxf(own.power * power, 1e-37f);
      const int left = (mine < b1 ? own.last : -1) - (b * 64 + 16 * wave + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[q][i] = i <= left ? s[q][i] * cs : -__builtin_inff();
      const float2 top = rows_xor16(fmaxf(fmaxf(s[q][0], s[q][1]), fmaxf(s[q][2], s[q][3])));
      top_of(turn, q)[2 * (g & 2) + wave] = fmaxf(top.x, top.y);  // of two lanes each
    }
  };
  // A lane's own tokens are of the first or second kind by g / 2; its operand covers by g the upper parts of the
  // first ones, of the second ones, the lower parts of the first ones, of the second ones.
  auto operand = [&](float shift) {
    const float2 both = rows_xor32(shift);
    return (g & 2 ? kProb + kRestScale : kProb) - (int)(g & 1 ? both.y : both.x);
  };
  float limit = kMostShift;
  bool low = false;  // whether the turn's have some with a power of two of their own
  auto put = [&](const float* y, int* to) {
    const int2 p = split_probabilities(y);
    to[lane * 4 + wave] = p.x;
    to[256 + lane * 4 + wave] = p.y;
  };
  auto probabilities = [&](int turn) {
    float top[NT];
    auto is_alone = [](float top, float next) { return top - next > kAlone && next > kNone; };
    auto tops = [&](int q) { return *reinterpret_cast<const f32x4*>(top_of(turn, q) + 2 * (g & 2)); };  // of four eights
    auto second = [](f32x4 t) {
      return fmaxf(fminf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fminf(t[0], t[1]), fminf(t[2], t[3])));
    };
    bool pass = false, alone = false;
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      const f32x4 t = tops(q);
      top[q] = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      pass |= top[q] - m[q] > kShift + kSlack;
      alone |= is_alone(top[q], second(t));
    }
    if (__any(pass)) {  // in all four waves or in none
      bool large = false;
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        const float2 both = rows_xor32(top[q]);
        const float mn = fmaxf(m[q], fmaxf(both.x, both.y) - kShift), f = __builtin_amdgcn_exp2f(m[q] - mn);
        m[q] = mn;
        l[q] *= f;
        large |= mn != kNone && fabsf(mn) >= kMostRef;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[q][i][k] *= f;
      }
      limit = __any(large) ? kNoShift : kMostShift;
    }
    low = __any(alone);
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      const float shift = fminf(floorf(8.0f - (top[q] - m[q])), limit);
      scales = q == 0 ? operand(shift) : scales | operand(shift) << 8;
      const float from = m[q] - shift;
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_exp2f(s[q][i] - from);
      l[q] += ldexpf((y[0] + y[1]) + (y[2] + y[3]), -(int)shift);
      if (low) {
        const float next = second(tops(q)), own = fminf(floorf(8.0f - (next - m[q])), limit);
        float z[4];
        take_small(y, z, is_alone(top[q], next) ? (int)(own - shift) : kNever);
        put(z, low_of(turn, q));
        low_of(turn, q)[512 + lane] = operand(own);  // the same in all four waves
      }
      put(y, prob_of(turn, q));
    }
  };
  auto values = [&](int turn, auto more) {
    const int b = min(b0 + group + turn * G, b1 - 1);
    if (b * 64 + 64 > end) {  // bytes behind the last key may be anything
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int left = end - (b * 64 + 16 * t + 4 * g);
        const int mask = left >= 4 ? -1 : left <= 0 ? 0 : (1 << (8 * left)) - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) vr[i][t] &= mask;
      }
    }
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      const i32x4* at = reinterpret_cast<const i32x4*>(prob_of(turn, q)) + lane;
      const i32x8 p = __builtin_shufflevector(at[0], at[64], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const i32x8 v = __builtin_shufflevector(vr[i], vr[i], 0, 1, 2, 3, 0, 1, 2, 3);
        o[q][i] = q == 0 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(v, p, o[q][i], 0, 0, 0, ve, 0, scales)
                         : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(v, p, o[q][i], 0, 0, 0, ve, 1, scales);
      }
    }
    if (low) {
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        const i32x4* at = reinterpret_cast<const i32x4*>(low_of(turn, q)) + lane;
        const i32x8 p = __builtin_shufflevector(at[0], at[64], 0, 1, 2, 3, 4, 5, 6, 7);
        const int own = low_of(turn, q)[512 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const i32x8 v = __builtin_shufflevector(vr[i], vr[i], 0, 1, 2, 3, 0, 1, 2, 3);
          o[q][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(v, p, o[q][i], 0, 0, 0, ve, 0, own);
        }
      }
    }
    issue_fence();
    if constexpr (decltype(more)::value) fetch_v(min(b0 + group + (turn + 1) * G, b1 - 1));
    issue_fence();
  };
  // A turn's barrier publishes its largest scores and the probabilities of the turn before. The last
  // one apart, so that the waits for loads count what is on its way in each.
  for (int turn = 0; turn + 1 < turns; ++turn) {
    scores(turn, std::true_type{});
    lds_barrier();
    if (turn > 0) values(turn - 1, std::true_type{});
    probabilities(turn);
  }
  if (turns > 0) {
    scores(turns - 1, std::false_type{});
    lds_barrier();
    if (turns > 1) values(turns - 2, std::true_type{});
    probabilities(turns - 1);
    lds_barrier();
    values(turns - 1, std::false_type{});
  }
  // the lane again, so that nothing of it takes registers in the loop
  const int lane2 = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), n2 = lane2 & 15, g2 = lane2 >> 4;
  // the lanes and waves of a query hold its tokens' parts of the sum
  __syncthreads();
#pragma unroll
  for (int q = 0; q < NT; ++q) {
    const float2 x = rows_xor16(l[q]);
    const float2 y = rows_xor32(x.x + x.y);
    if (g2 == 0) {
      sums[group][q * 16 + n2][wave] = (y.x + y.y) * (1.0f / 16.0f);
      if (wave == 0) most[group][q * 16 + n2] = m[q];
    }
  }
  if constexpr (G > 1) {
    float* sum = reinterpret_cast<float*>(lds) + group * kSum;
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(sum + (q * 16 + n2) * kSumRow + wave * 64 + i * 16 + g2 * 4) = o[q][i];
  }
  __syncthreads();
  // group k finishes tiles k, k + G, ..
#pragma unroll
  for (int q = 0; q < NT; ++q) {
    const int pair = pair0 + 16 * q + n2, at = q * 16 + n2;
    if (q % G != group || pair >= pairs) continue;
    float ref = kNone, f[G], total = 0.0f;
#pragma unroll
    for (int k = 0; k < G; ++k) ref = fmaxf(ref, most[k][at]);
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(sums[k][at]);
      f[k] = __builtin_amdgcn_exp2f(most[k][at] - ref);
      total = fmaf((t[0] + t[1]) + (t[2] + t[3]), f[k], total);
    }
    const int2 to = divide(pair, a.group, a.inv_group);
    const size_t row = (size_t)to.x * a.q_heads + head * a.group + to.y;
    const int d = wave * 64 + g2 * 4;
    float* part = a.part + (row * a.splits + split) * kKv8PartFloats;
    const float inv = 1.0f / total;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 x = o[q][i];
      if constexpr (G > 1) {
        x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(lds) + k * kSum +
                                                          at * kSumRow + d + 16 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = fmaf(y[j], f[k], x[j]);
        }
      }
      if (a.splits > 1) {
        *reinterpret_cast<f32x4*>(part + d + 16 * i) = x;
        if (i == 0 && wave == 0 && g2 == 0) *reinterpret_cast<float2*>(part + 256) = make_float2(ref, total);
        continue;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] *= inv;
      if (a.gate) {
        const uint2 gate = *reinterpret_cast<const uint2*>(a.gate + row * 512 + 256 + d + 16 * i);
        x[0] *= sigmoid(bf_lo(gate.x));
        x[1] *= sigmoid(bf_hi(gate.x));
        x[2] *= sigmoid(bf_lo(gate.y));
        x[3] *= sigmoid(bf_hi(gate.y));
      }
      *reinterpret_cast<uint2*>(a.out + row * 256 + d + 16 * i) = make_uint2(pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]));
    }
  }
}

// Joins the ranges of keys of one (row, query head), 64 dims a block: thread t
// holds range t's maximum and sum, and four dims of ranges t / 16 + 16 i, all
// fetched at once.
__global__ __launch_bounds__(256) void k_kv8_attn_join(Kv8Attn a) {
  __shared__ __attribute__((aligned(16))) float sum[16][64];
  __shared__ float weight[256], wmax[4], wden[4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, slot = t >> 4;
  const size_t at = blockIdx.x >> 2;
  const int d0 = (blockIdx.x & 3) * 64;
  const float* part = a.part + at * a.splits * kKv8PartFloats;
  const float2 md = t < a.splits ? *reinterpret_cast<const float2*>(part + (size_t)t * kKv8PartFloats + 256)
                                 : make_float2(kNone, 0.0f);
  const float* mine = part + (size_t)slot * kKv8PartFloats + d0 + (t & 15) * 4;
  f32x4 x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (slot + 16 * i < a.splits) x[i] = *reinterpret_cast<const f32x4*>(mine + (size_t)i * 16 * kKv8PartFloats);
  const float wm = wave_max(md.x);
  if (lane == 0) wmax[wave] = wm;
  __syncthreads();
  const float top = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
  const float f = __builtin_amdgcn_exp2f(md.x - top);
  weight[t] = f;
  const float den = tree64(md.y * f);
  if (lane == 0) wden[wave] = den;
  __syncthreads();
  f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (slot + 16 * i >= a.splits) break;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = fmaf(x[i][k], weight[slot + 16 * i], o[k]);
  }
  for (int s = slot + 128; s < a.splits; s += 16) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(mine + (size_t)(s - slot) * kKv8PartFloats);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = fmaf(y[k], weight[s], o[k]);
  }
  *reinterpret_cast<f32x4*>(&sum[slot][(t & 15) * 4]) = o;
  __syncthreads();
  if (t >= 64) return;
  const float total = (wden[0] + wden[1]) + (wden[2] + wden[3]);
  float y = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) y += sum[i][t];
  y = y / total;
  if (a.gate) y *= sigmoid(bf2f(a.gate[at * 512 + 256 + d0 + t]));
  a.out[at * 256 + d0 + t] = (uint16_t)f2bf(y);
}

// The same of many: a wave each, four dims a lane.
__global__ __launch_bounds__(256) void k_kv8_attn_join_rows(Kv8Attn a) {
  const int lane = threadIdx.x & 63;
  const size_t at = (size_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (at >= (size_t)a.rows * a.q_heads) return;
  const float* part = a.part + at * a.splits * kKv8PartFloats;
  const float2 md = lane < a.splits ? *reinterpret_cast<const float2*>(part + (size_t)lane * kKv8PartFloats + 256)
                                    : make_float2(kNone, 0.0f);
  const float f = __builtin_amdgcn_exp2f(md.x - wave_max(md.x)), total = tree64(md.y * f);
  f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < a.splits; s += 4) {
    f32x4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = *reinterpret_cast<const f32x4*>(part + (size_t)min(s + i, a.splits - 1) * kKv8PartFloats + lane * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s + i >= a.splits) break;
      const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s + i));
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = fmaf(x[i][k], w, o[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) o[k] /= total;
  if (a.gate) {
    const uint2 gate = *reinterpret_cast<const uint2*>(a.gate + at * 512 + 256 + lane * 4);
    o[0] *= sigmoid(bf_lo(gate.x));
    o[1] *= sigmoid(bf_hi(gate.x));
    o[2] *= sigmoid(bf_lo(gate.y));
    o[3] *= sigmoid(bf_hi(gate.y));
  }
  *reinterpret_cast<uint2*>(a.out + at * 256 + lane * 4) = make_uint2(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]));
}

// DMA into LDS: 16 bytes a lane from `uniform` + `lane` of a buffer, piece I of
// 1024 bytes behind each other, to LDS `to`; or one byte of a buffer to each dword of
// the 64 at `to`. In assembly, so that the compiler's waits before it reads LDS do
// not count these (the kernel's own do); a buffer spans all 32-bit offsets: what is
// in range is the caller's affair.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
__device__ __forceinline__ u32x4 buffer_of(const uint8_t* base) {
  return u32x4{(uint32_t)(uintptr_t)base, (uint32_t)((uintptr_t)base >> 32), 0xffffffffu, 0x00020000u};
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved, and clobbered here
template <int I>
__device__ __forceinline__ void dma16(u32x4 from, uint32_t lane, uint32_t uniform, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen offset:%4 lds"
               :
               : "s"(to), "v"(lane), "s"(from), "s"(uniform), "n"(I * 1024)
               : "memory", "m0");
}
__device__ __forceinline__ void dma1(u32x4 from, uint32_t uniform, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_ubyte off, %1, %2 lds"
               :
               : "s"(to), "s"(from), "s"(uniform)
               : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// Many queries: 128 (row, query head) pairs of one KV head, eight waves, two a SIMD.
// Wave w holds the 32 pairs 32 (w % 4) ..; the lower four waves take the even blocks
// of keys, the upper four the odd ones, and both halves are joined at the end.
//   S^T[token, query] = K Q^T and O^T[d, query] += V^T P^T on 32x32x64, each query
//   (probability) as the sum of two e4m3 numbers, the lower one 16 (32) times too large
//   and with a power of two of its own. Lane (r = lane % 32, h = lane / 32) gives K's
//   bytes of token r (V's of dim r) and those of query r, and receives tokens (dims)
//   8 i + 4 h .. + 3 of query r: the tokens whose probabilities it has to give next.
// In phase p the waves of block p make its scores, those of block p - 1 its
// probabilities and their products, so that of a SIMD's two waves one uses the
// matrix core while the other works on its softmax. K and V reach LDS by DMA, in the
// order of the operands, two to three phases ahead; the queries' lower part stays in
// LDS, as registers are full: 128 of sums, 24 of queries, 32 of scores, operands.
// Measured: 4096 rows behind 28672, 8 query and 2 KV heads, 803 to 870 us by the card (1.0e12
// operations, 1.2e15 a second; 2 % less with one power of two for all keys). A phase takes 3100
// cycles, 2048 of them of the matrix core, and with all 256 CUs at it the clock falls from 2.4 to
// 1.9 GHz. Four waves with 32 queries and
// all keys each, the same steps interleaved within a wave, took 3530 cycles; eight
// with 16 queries, both parts as columns of one product, 3560.
typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int kRowPairs = 128, kRowDma = 3;      // DMA instructions of a wave for a block's K (or V)
constexpr int kKStages = 3, kVStages = 4;
// LDS: the queries' lower parts, 64 dims of their upper ones, K, V
constexpr int kRowLast = kRowPairs * 256, kRowStages = kRowLast + kRowPairs * 64;
constexpr int kRowBytes = kRowStages + (kKStages + kVStages) * kBlockBytes;
__global__ __launch_bounds__(512, 1) void k_kv8_attn_rows(Kv8 c, Kv8Attn a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[kRowBytes];
  __shared__ int exponent[kKStages + kVStages][64];  // each 64 times
  __shared__ float scaled[kRowPairs], most[2][kRowPairs], sums[2][kRowPairs];
  const int tid = threadIdx.x, lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), r = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), upper = wave >> 2, mine = (wave & 3) * 32 + r;
  // heads in turn, then ranges of keys, so that an XCD's blocks share keys where
  // heads and ranges divide the XCDs; the tiles with most keys first
  const int head = (int)blockIdx.x % c.heads, rest = (int)blockIdx.x / c.heads;
  const int split = rest % a.splits, tile = a.tiles - 1 - rest / a.splits;
  const int pairs = a.rows * a.group, end = a.position + a.rows, pair0 = tile * kRowPairs;
  const int all = (a.position + divide(min(pair0 + kRowPairs - 1, pairs - 1), a.group, a.inv_group).x) / kKv8Block + 1;
  const int b0 = split * all / a.splits, nblk = (split + 1) * all / a.splits - b0;  // the block's own: b0 + 0 .. nblk - 1
  const size_t store = (size_t)head * c.blocks;
  const auto kbuf = buffer_of(c.k + store * kBlockBytes), vbuf = buffer_of(c.v + store * kBlockBytes);
  const auto kscale = buffer_of(c.k_scale + store), vscale = buffer_of(c.v_scale + store);
  const uint32_t part = wave * 2048;
  auto kstage = [](int b) { return (uint32_t)b % kKStages; };
  auto vstage = [](int b) { return kKStages + (uint32_t)b % kVStages; };
  // K and V of block b. One behind the last is fetched as the last, into the stage of
  // a block that is done with, so that every phase's wait counts the same instructions.
  auto issue = [&](int b) {
    const uint32_t at = b0 + min(b, nblk - 1), k = kstage(b), v = vstage(b), to = lds_address(lds) + kRowStages + part;
    dma16<0>(kbuf, part + lane * 16, at * kBlockBytes, to + k * kBlockBytes);
    dma16<1>(kbuf, part + lane * 16, at * kBlockBytes, to + k * kBlockBytes);
    dma1(kscale, at, lds_address(exponent) + k * 256);
    dma16<0>(vbuf, part + lane * 16, at * kBlockBytes, to + v * kBlockBytes);
    dma16<1>(vbuf, part + lane * 16, at * kBlockBytes, to + v * kBlockBytes);
    dma1(vscale, at, lds_address(exponent) + v * 256);
  };
  auto read = [&](uint32_t at) {  // 32 bytes a lane of 2048
    const i32x4* from = reinterpret_cast<const i32x4*>(lds + at) + lane;
    return __builtin_shufflevector(from[0], from[64], 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // queries: 16 lanes a query, 16 dims a lane; the upper parts through V's last stages
  i32x8 qhi[3];
  {
    const int chunk = tid & 15;
    u32x4 x[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int2 rq = divide(min(pair0 + 32 * i + (tid >> 4), pairs - 1), a.group, a.inv_group);
      const u32x4* qp = reinterpret_cast<const u32x4*>(
          a.query + ((size_t)rq.x * a.q_heads + head * a.group + rq.y) * 256 + chunk * 16);
      x[i][0] = qp[0];
      x[i][1] = qp[1];
    }
    issue_fence();
    issue(0);
    issue(1);
    issue_fence();
    const int upper_parts = kRowStages + vstage(2) * kBlockBytes;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        top = max(top, max(finite_bits(x[i][j >> 2][j & 3] << 16), finite_bits(x[i][j >> 2][j & 3] & 0xffff0000u)));
      const int e = scale_exponent(row16_max(__uint_as_float(top)), -100);
      scaled[32 * i + (tid >> 4)] = ldexpf(kLog2e / 16.0f, e);
      i32x4 hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u = x[i][j >> 1][(j & 1) * 2], w = x[i][j >> 1][(j & 1) * 2 + 1];
        const int2 p = split_e4m3(ldexpf(bf_lo(u), -e), ldexpf(bf_hi(u), -e), ldexpf(bf_lo(w), -e), ldexpf(bf_hi(w), -e));
        hi[j] = p.x;
        lo[j] = p.y;
      }
      // [32 queries][64 dims][16 of 32 dims][lane of the product]
      const int to = i * 8192 + (chunk >> 2) * 2048 + (chunk & 1) * 1024 + ((chunk >> 1) & 1) * 512 + (tid >> 4) * 16;
      *reinterpret_cast<i32x4*>(lds + (chunk < 12 ? upper_parts + to : kRowLast + to - i * 6144 - 6144)) = hi;
      *reinterpret_cast<i32x4*>(lds + to) = lo;
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 3; ++i) qhi[i] = read(upper_parts + (wave & 3) * 8192 + i * 2048);
  }
  const float cq = scaled[mine];
  const int last = a.position + divide(min(pair0 + mine, pairs - 1), a.group, a.inv_group).x;  // last key of the lane's query
  f32x16 o[8], s[2];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int k = 0; k < 16; ++k) o[i][k] = 0.0f;
  float m = kNone, l = 0.0f, cs = 0.0f;  // reference less kShift; the lane's part of the sum, times 2^kShift
  float top32 = 0.0f, next32 = 0.0f;     // the largest of 32 scores, and of the other three eights of them
  auto scores = [&](int b) {
    const uint32_t from = kRowStages + kstage(b) * kBlockBytes, lower = (wave & 3) * 8192;
    const int ke = exponent[kstage(b)][lane];
    auto key = [&](int t) { return read(from + (t & 1) * 8192 + (t >> 1) * 2048); };
    i32x8 k[8], ql[4], qh[4] = {qhi[0], qhi[1], qhi[2]};
    k[0] = key(0);
    k[1] = key(1);
    ql[0] = read(lower);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[0][i] = s[1][i] = 0.0f;
#pragma unroll
    for (int t = 0; t < 9; ++t) {  // 64 dims t / 2 by 32 tokens t % 2, the lower parts a step later
      issue_fence();
      if (t < 8) s[t & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k[t], qh[t / 2], s[t & 1], 0, 0, 0, kOne, 0, kOne);
      if (t > 0) {
        const int u = t - 1;
        s[u & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k[u], ql[u / 2], s[u & 1], 0, 0, 0, kOne, 0, kLo);
      }
      issue_fence();
      if (t < 6) k[t + 2] = key(t + 2);
      if (t == 4) qh[3] = read(kRowLast + (wave & 3) * 2048);
      if (t % 2 == 0 && t > 0 && t < 8) ql[t / 2] = read(lower + t * 1024);
    }
    if ((b0 + b) * 64 + 63 > a.position) {  // the causal border
      const int left = last - (b0 + b) * 64 - 4 * h;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) s[i][k] = 32 * i + 8 * (k >> 2) + (k & 3) <= left ? s[i][k] : -__builtin_inff();
    }
    float tops[4];  // of the lane's tokens 16 j + 0 .. 7 and 16 j + 8 .. 15, in either half of the block
#pragma unroll
    for (int k = 0; k < 4; ++k) tops[k] = s[k >> 1][4 * (k & 1)];
#pragma unroll
    for (int k = 1; k < 8; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)  // the larger; fmaxf would first quiet what a product gave
        tops[i] = __builtin_amdgcn_fmed3f(tops[i], s[i >> 1][4 * (i & 1) + (k & 3) + 8 * (k >> 2)], __builtin_inff());
    const float front = fmaxf(tops[0], tops[2]), back = fmaxf(tops[1], tops[3]);
    // of the query's four eights of the first kind in the lower lanes, of the second in the upper: the two largest
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(front), __float_as_uint(back), false, false);
    const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(fminf(tops[0], tops[2])), __float_as_uint(fminf(tops[1], tops[3])),
                                                    false, false);
    top32 = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    next32 = fmaxf(fminf(__uint_as_float(a[0]), __uint_as_float(a[1])), fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1])));
    cs = fmaxf(ldexpf(cq, ke - 127), 1e-37f);
    const float top = fmaxf(front, back) * cs - kShift;
    if (__any(top > m + kSlack)) {
      const float2 u = rows_xor32(top);
      const float next = fmaxf(m, fmaxf(u.x, u.y)), f = __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) o[i][k] *= f;
    }
  };
  auto values = [&](int b) {
    const uint32_t from = kRowStages + vstage(b) * kBlockBytes;
    const int ve = exponent[vstage(b)][lane];
    i32x8 v[8], phi, plo;
    // sums 0 .. 3 are of the wave's own half of the dims, 4 .. 7 of the other's
    auto fetch = [&](int t) { v[t] = read(t < 4 ? from + upper * 8192 + t * 2048 : from - upper * 8192 + t * 2048); };
    const float x = fmaf(top32, cs, -m), xnext = fmaf(next32, cs, -m);
    const float shift = shift_of(x, m);
    const float2 shifts = rows_xor32(shift);  // of the tokens 16 j + 0 .. 7, of the others
    const float from_m[2] = {m - shifts.x, m - shifts.y};
    const int scale = kProb - (int)shift;
    int low_scale = 0;
    float sum[2] = {0.0f, 0.0f};
    auto probabilities = [&](int i, float* y) {
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][4 * (i & 3) + k], cs, -from_m[i & 1]));
      sum[i & 1] += (y[0] + y[1]) + (y[2] + y[3]);
    };
    auto parts = [&](int i, const float* y, i32x8& upper, i32x8& lower) {
      const int2 p = split_probabilities(y);
      upper[(i & 1) * 4 + (i >> 1)] = p.x;
      lower[(i & 1) * 4 + (i >> 1)] = p.y;
    };
    i32x8 low[2];  // the parts of those with a power of two of their own
    const bool alone = x - xnext > kAlone && xnext > kNone;
    const int lows = __any(alone) ? 2 : 0;
    if (lows) {
      const float own = shift_of(xnext, m);
      const float2 ups = rows_xor32(alone ? own - shift : (float)kNever);
      low_scale = kProb - (int)own;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float y[4], z[4];
        probabilities(i, y);
        take_small(y, z, (int)(i & 1 ? ups.y : ups.x));
        parts(i, y, phi, plo);
        parts(i, z, low[0], low[1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float y[4];
        probabilities(i, y);
        parts(i, y, phi, plo);
      }
    }
    l += ldexpf(sum[0], -(int)shifts.x) + ldexpf(sum[1], -(int)shifts.y);
    fetch(0);
    fetch(1);
#pragma unroll
    for (int t = 0; t < 9; ++t) {
      issue_fence();
      if (t < 8) o[t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v[t], phi, o[t], 0, 0, 0, ve, 0, scale);
      if (t < 6) fetch(t + 2);
      if (t > 0) {
        o[t - 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v[t - 1], plo, o[t - 1], 0, 0, 0, ve, 0, scale + kRestScale);
#pragma unroll 1
        for (int i = 0; i < lows; ++i)
          o[t - 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v[t - 1], i ? low[1] : low[0], o[t - 1], 0, 0, 0, ve, 0,
                                                                     low_scale + i * kRestScale);
      }
    }
  };
  // K of the phase and V of the one before have arrived once all but the last three
  // groups have; every wave is past what the next ones replace.
  auto phase = [&](int p) {
    wait_vmcnt<3 * kRowDma>();
    lds_barrier();
    issue(p + 2);
    issue_fence();
    if (p == nblk - 1 && (b0 + nblk) * 64 > end) {  // bytes behind the last key may be anything
      wait_vmcnt<4 * kRowDma>();             // V of the phase's block: each wave clears what it fetched
      int own = lane;
      asm volatile("" : "+v"(own));  // masks are no registers of the loop's
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        i32x4* at = reinterpret_cast<i32x4*>(lds + kRowStages + vstage(p) * kBlockBytes + part) + i * 64 + own;
        i32x4 w = *at;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int left = end - (b0 + p) * 64 - (16 * k + 8 * i + 4 * (own >> 5));
          w[k] &= (int)((1ull << (8 * min(max(left, 0), 4))) - 1);
        }
        *at = w;
      }
    }
  };
  if (upper) phase(0);
  for (int b = upper; b < nblk; b += 2) {
    phase(b);
    scores(b);
    phase(b + 1);
    values(b);
  }
  if ((nblk & 1) == upper) {  // the half without the last block: its part of that block's V, which the other half reads
    wait_vmcnt<3 * kRowDma>();
    lds_barrier();
  }
  wait_vmcnt<0>();  // no DMA outlives this
  // Both halves: each wave finishes half of the dims. The lane again, so that nothing of it takes registers in the loop.
  int lane2 = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
  asm("" : "+v"(lane2));
  const int h2 = lane2 >> 5, mine2 = (wave & 3) * 32 + (lane2 & 31);
  const int2 rq = divide(min(pair0 + mine2, pairs - 1), a.group, a.inv_group);
  const float2 t = rows_xor32(l);
  if (h2 == 0) {
    most[upper][mine2] = m;
    sums[upper][mine2] = t.x + t.y;
  }
  lds_barrier();
  f32x4* const swap = reinterpret_cast<f32x4*>(lds) + lane2;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f32x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = o[4 + i][4 * k + j];
      swap[wave * 1024 + (4 * i + k) * 64] = x;
    }
  lds_barrier();
  const float other = most[1 - upper][mine2], ref = fmaxf(m, other);
  float f = __builtin_amdgcn_exp2f(m - ref), fo = __builtin_amdgcn_exp2f(other - ref);
  const float total = fmaf(sums[0][mine2], upper ? fo : f, sums[1][mine2] * (upper ? f : fo)) * 0.0625f;  // 2^-kShift
  const float inv = a.splits > 1 ? 1.0f : 1.0f / total;
  f *= inv;
  fo *= inv;
  const size_t row = (size_t)rq.x * a.q_heads + head * a.group + rq.y;
  // a lane without a pair stores behind the end of the buffer, which drops it
  const auto out = __builtin_amdgcn_make_buffer_rsrc((void*)a.out, 0, (int)((uint32_t)a.rows * a.q_heads * 512u), 0x00020000);
  const uint32_t to = pair0 + mine2 < pairs ? (uint32_t)row * 512u + upper * 256 + h2 * 16 : 0xfffff000u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // 16 dims: lower lanes end with 0 .. 7, upper with 8 .. 15
      float z[8], y[8];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const f32x4 x = swap[(wave ^ 4) * 1024 + (4 * i + 2 * j + k) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          z[4 * k + e] = fmaf(o[i][8 * j + 4 * k + e], f, x[e] * fo);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(z[k]), __float_as_uint(z[4 + k]), false, false);
        y[k] = __uint_as_float(w[0]);
        y[4 + k] = __uint_as_float(w[1]);
      }
      if (a.splits > 1) {
        float* part = a.part + (row * a.splits + split) * kKv8PartFloats;
        if (pair0 + mine2 < pairs) {
          *reinterpret_cast<f32x4*>(part + upper * 128 + 32 * i + 16 * j + 8 * h2) = f32x4{y[0], y[1], y[2], y[3]};
          *reinterpret_cast<f32x4*>(part + upper * 128 + 32 * i + 16 * j + 8 * h2 + 4) = f32x4{y[4], y[5], y[6], y[7]};
          if (i + j + h2 + upper == 0) *reinterpret_cast<float2*>(part + 256) = make_float2(ref, total);
        }
        continue;
      }
      if (a.gate) {
        const u32x4 gate = *reinterpret_cast<const u32x4*>(a.gate + row * 512 + 256 + upper * 128 + 32 * i + 16 * j + 8 * h2);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          y[2 * k] *= sigmoid(bf_lo(gate[k]));
          y[2 * k + 1] *= sigmoid(bf_hi(gate[k]));
        }
      }
      const u32x4 packed{pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]), pack_bf2(y[4], y[5]), pack_bf2(y[6], y[7])};
      __builtin_amdgcn_raw_buffer_store_b128(packed, out, to + (32 * i + 16 * j) * 2, 0, 0);
    }
}

int few_tiles(int nt, int pairs) { return (pairs + 16 * nt - 1) / (16 * nt); }  // nt: 16-pair tiles of a block
// Whether the tiles of a range of keys go to one XCD (whose L2 then fetches them
// once): while groups of that many fill most of its 32 CUs.
bool few_grouped(int tiles) { return tiles > 1 && tiles <= 10; }
// Ranges of keys of one call: enough blocks for the chip's 256 CUs.
int few_ranges(int heads, int tiles) { return max(1, few_grouped(tiles) ? 32 / tiles * 8 / heads : 256 / (heads * tiles)); }

// 128-pair blocks of a head; and of all heads' the ranges of keys that fill `rounds`
// rounds of blocks on the chip's 256 CUs, 1 if they end no sooner than whole rounds do.
int row_tiles(int pairs) { return (pairs + kRowPairs - 1) / kRowPairs; }
constexpr int kRowRounds = 4;
int row_ranges(int tiles, int rounds) {
  const int ranges = min(256, 256 * rounds / tiles);
  return ranges > 1 && (tiles * ranges + 255) / 256 < (tiles + 255) / 256 * ranges ? ranges : 1;
}
constexpr int kRowLeast = 96;  // pairs of a head from which on 128-pair blocks come into question

// Estimates in us by which a call takes one form or another, fitted to calls of 5 to
// 8192 rows at 0 to 70000, 1 to 8 KV heads:
//   few: for 64 keys of 16 pairs 0.42, of 32 together 0.6; for each round of blocks 8 and 13
//   rows: 1.28 for 64 keys of 128 pairs with a CU of its own, up to 1.6 when all CUs are
//     at it (the clock falls), 10 a round; with ranges 6, and writing and joining them
// Measured, 8 query and 2 KV heads where not said otherwise: 500 rows alone 8 us with 16 pairs
// a block and 14 with 32; 1000 alone 19 and 16; 32 rows behind 70000 40 and 34, rows 47
// with 128 ranges; 128 behind 28672 49, 48 and rows 57 with 32; 512 behind 28672 few 146,
// rows 119 with eight; 2048 behind 30000 few 568, rows 663 with one, 435 with two; 4200
// behind 28672 few 1273, rows 1304 with one and 1010 with three; 700 behind 20000, 32 and
// 8 heads, 557, 444 with one; 4096 alone 111 and 107.
float few_us(int nt, int heads, int pairs, float keys) {
  const float tiles = (float)few_tiles(nt, pairs) * heads;
  return tiles * keys / 256 * (nt == 1 ? 0.42f : 0.6f) + (nt == 1 ? 8 : 13) * ceilf(tiles / 256);
}
// most and least: blocks of keys of the last tile and the first
float rows_us(int tiles, int ranges, int least, int most) {
  const int n = tiles * ranges, rounds = (n + 255) / 256;
  const float unit = 1.28f + 0.32f * fminf(1.0f, n / 256.0f);
  const float mean = 0.5f * (least + most);
  if (ranges > 1) return rounds * (ceilf((rounds == 1 ? most : mean) / ranges) * unit + 6) + 4 + n * 0.054f;
  // with two rounds, as the longest come first, two of the length in the middle follow each other
  const float keys = rounds == 1 ? most : rounds == 2 ? fmaxf(most, 2 * (most - (most - least) * 256.0f / n))
                                                      : fmaxf(most, mean * n / 256 * (1 + 0.5f / rounds));
  return keys * unit + 10 * rounds;
}

// After a launch with ranges of keys. A wave for each output fills the chip from about
// 1024 on (with 1600 outputs a call takes 21.0 us and 23.0 with blocks, with 800 17.9 and
// 17.4, with 320 18.6 and 13.8); it holds the weights of 64 ranges.
hipError_t join(const Kv8Attn& a, hipStream_t s) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int outputs = a.rows * a.q_heads;
  if (outputs >= 1024 && a.splits <= 64)
    hipLaunchKernelGGL(k_kv8_attn_join_rows, dim3((outputs + 3) / 4), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(k_kv8_attn_join, dim3(outputs * 4), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace

size_t kv8_attn_scratch_bytes(int q_heads, int kv_heads, int rows) {
  const int pairs = rows * (q_heads / kv_heads);
  const int few = max(few_ranges(kv_heads, few_tiles(1, pairs)), few_ranges(kv_heads, few_tiles(2, pairs)));
  int most = few;
  for (int rounds = 1; rounds <= kRowRounds && pairs >= kRowLeast; ++rounds)
    most = max(most, row_ranges(row_tiles(pairs) * kv_heads, rounds));
  return most < 2 ? 0 : (size_t)rows * q_heads * most * kKv8PartFloats * sizeof(float);
}

hipError_t launch_kv8_write(const Kv8& c, const Kv8Rows& r, hipStream_t s) {
  const int nblk = (r.position + r.rows - 1) / kKv8Block - r.position / kKv8Block + 1;
  if (r.rows == 1) {
    hipLaunchKernelGGL(k_kv8_write_one<false>, dim3(c.heads), dim3(512), 0, s, c, r, Kv8Prep{});
    return hipGetLastError();
  }
  hipLaunchKernelGGL(k_kv8_write<false>, dim3(nblk * c.heads), dim3(512), 0, s, c, r, Kv8Prep{});
  return hipGetLastError();
}

hipError_t launch_kv8_prepare(const Kv8& c, const Kv8Rows& r, const Kv8Prep& p, hipStream_t s) {
  const int nblk = (r.position + r.rows - 1) / kKv8Block - r.position / kKv8Block + 1;
  if (r.rows == 1) {
    hipLaunchKernelGGL(k_kv8_write_one<true>, dim3(c.heads + (p.q_heads + 31) / 32), dim3(512), 0, s, c, r, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(k_kv8_write<true>, dim3(nblk * c.heads + (r.rows + 7) / 8), dim3(1024), 0, s, c, r, p);
  return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8& c, int position, int rows, uint16_t* k, uint16_t* v, int64_t row_stride,
                           int64_t head_stride, hipStream_t s) {
  const int nblk = (position + rows - 1) / kKv8Block - position / kKv8Block + 1;
  hipLaunchKernelGGL(k_kv8_read, dim3(nblk * c.heads, 2), dim3(256), 0, s, c, position, rows, k, v, row_stride,
                     head_stride);
  return hipGetLastError();
}

hipError_t launch_kv8_attn(const Kv8& c, Kv8Attn a, hipStream_t s) {
  a.inv_group = 1.0f / (float)a.group;
  const int pairs = a.rows * a.group, all = row_tiles(pairs) * c.heads;
  const int least = a.position / kKv8Block + 1, most = (a.position + a.rows - 1) / kKv8Block + 1;
  const float one = few_us(1, c.heads, pairs, 0.5f * (least + most)), two = few_us(2, c.heads, pairs, 0.5f * (least + most));
  const int nt = one <= two ? 1 : 2;
  float best = fminf(one, two);
  a.splits = 0;
  for (int rounds = 0; rounds <= kRowRounds && pairs >= kRowLeast; ++rounds) {
    const int ranges = rounds == 0 ? 1 : min(row_ranges(all, rounds), least);  // none of no keys
    const float us = rows_us(all, ranges, least, most);
    if (us < best) {
      best = us;
      a.splits = ranges;
    }
  }
  if (a.splits) {
    a.tiles = row_tiles(pairs);
    hipLaunchKernelGGL(k_kv8_attn_rows, dim3(all * a.splits), dim3(512), 0, s, c, a);
    return join(a, s);
  }
  const int tiles = few_tiles(nt, pairs), ranges = few_ranges(c.heads, tiles);
  a.tiles = tiles;
  // Up to 12 blocks of keys one range: the second launch costs more than it saves (one
  // token behind 100, 500, 750: 6.6, 7.6, 8.7 us, and 9.4 with a block to a range).
  a.per = most <= 12 ? most : (most + ranges - 1) / ranges;
  a.splits = (most + a.per - 1) / a.per;
  // Groups of four waves a block. Where one tile of 16 pairs reads its keys alone memory sets the time
  // and one group fetches as fast as four, with nothing to join; more pairs of a range, or the
  // one range of a short context, have work for all 16 waves, two tiles only where a range is
  // long. (4 and 2 groups, 8 query and 2 KV heads: 8 rows behind 40000, two tiles of 16 pairs with ranges of
  // 10 blocks of keys, 13.9 and 13.2 us; of 32 and 8 heads, with 20, 20.4 and 21.8; 16 rows behind 70000, four tiles,
  // 21.7 and 25.1; 32 behind 70000, four tiles of 32, 34.2 and 41.0.) Tiles of 32 leave no registers to one group.
  const int sixteens = tiles * nt;
  const int most_groups = a.splits == 1 || sixteens > 2 ? 4 : sixteens == 1 ? 1 : a.per >= 20 ? 4 : 2;
  const int g = min(most_groups, a.per >= 4 ? 4 : a.per >= 2 || nt == 2 ? 2 : 1);
  const auto few = nt == 1
                       ? (g == 4 ? k_kv8_attn_few<1, 4> : g == 2 ? k_kv8_attn_few<1, 2> : k_kv8_attn_few<1, 1>)
                       : (g == 4 ? k_kv8_attn_few<2, 4> : k_kv8_attn_few<2, 2>);
  const dim3 grid = few_grouped(tiles) ? dim3((a.splits * c.heads + 7) / 8 * 8 * tiles) : dim3(a.splits, tiles, c.heads);
  hipLaunchKernelGGL(few, grid, dim3(256 * g), 0, s, c, a);
  return join(a, s);
}

}  // namespace es
