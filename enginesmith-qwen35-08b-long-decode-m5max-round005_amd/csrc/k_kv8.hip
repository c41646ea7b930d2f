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
// Queries and probabilities enter the 8-bit products in these two parts, which
// loses nothing against bf16 products (the matrix cores align the addends of an
// 8-bit product to about 2^-13 of the largest: measured rms 1e-5 of it).
#include "es_kernels.hpp"

namespace es {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

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

// RMS norm of a 256-wide head in 32 bits, 16 dims in each lane of a row of 16.
__device__ __forceinline__ void norm16(float* x, const float* gain) {
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
  const float inv = 1.0f / sqrtf(tree16(ss) * (1.0f / 256.0f) + 1e-6f);
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

// ---- writing ----
// Block of 512 threads = 64 tokens x one KV head: waves 0..3 K, 4..7 V. A
// thread holds 64 values; the block's largest magnitudes meet in LDS, then K
// goes out in pieces as it is held (a wave's four tokens make 64-byte lines) and V
// through LDS, where its tokens and dims change places (padded: 16 bytes
// every 16 pieces). A piece whose tokens are not all written is read,
// merged and written back; no other byte changes. Prepare (PREP) makes the K
// rows from projections by norm and rotation, and further blocks make the
// queries, eight rows each.
constexpr int kVPad = kBlockBytes + (kBlockBytes / 256) * 16;
__device__ __forceinline__ int v_lds(int byte) { return byte + (byte >> 8) * 16; }

template <bool PREP>
__global__ __launch_bounds__(512) void k_kv8_write(Kv8 c, Kv8Rows r, Kv8Prep p) {
  __shared__ __attribute__((aligned(16))) uint8_t vt[kVPad];
  __shared__ float2 cs[PREP ? 64 : 1][32];
  __shared__ uint32_t top[2];
  __shared__ int bad[64];
  const int tid = threadIdx.x, chunk = tid & 15;
  const int first = r.position / kKv8Block, nblk = (r.position + r.rows - 1) / kKv8Block - first + 1;
  if (PREP && (int)blockIdx.x >= nblk * c.heads) {
    // queries: 32 (row, head) pairs at a time, 16 lanes each
    const int row0 = ((int)blockIdx.x - nblk * c.heads) * 8, rows = min(8, r.rows - row0);
    if (tid < rows * 32) cs[tid >> 5][tid & 31] = angle_cs(r.position + row0 + (tid >> 5), p.inv_freq[tid & 31]);
    float gain[16];
    load16(p.q_gain + chunk * 16, gain);
    __syncthreads();
    for (int i = tid >> 4; i < rows * p.q_heads; i += 32) {
      const int row = i / p.q_heads;
      const size_t at = (size_t)row0 * p.q_heads + i;
      float x[16];
      load16(p.q_proj + at * 512 + chunk * 16, x);
      norm16(x, gain);
      rotate16(x, cs[row], chunk);
      u32x4 o[2];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j >> 2][j & 3] = pack_bf2(x[2 * j], x[2 * j + 1]);
      u32x4* q = reinterpret_cast<u32x4*>(p.query + at * 256 + chunk * 16);
      q[0] = o[0];
      q[1] = o[1];
    }
    return;
  }
  const int blk = first + (int)blockIdx.x % nblk, head = (int)blockIdx.x / nblk;
  const int base = blk * kKv8Block;
  const int lo = max(r.position - base, 0), hi = min(r.position + r.rows - base, kKv8Block);
  const bool is_v = tid >= 256;
  const int g = (tid & 255) >> 4;
  if (tid < 2) top[tid] = 0;
  if (tid < 64) bad[tid] = 0;
  if (PREP) {
    for (int i = tid; i < (hi - lo) * 32; i += 512)
      cs[lo + (i >> 5)][i & 31] = angle_cs(base + lo + (i >> 5), p.inv_freq[i & 31]);
  }
  __syncthreads();
  const size_t store = (size_t)head * c.blocks + blk;
  uint8_t* codes = (is_v ? c.v : c.k) + store * kBlockBytes;
  uint8_t* scale = (is_v ? c.v_scale : c.k_scale) + store;
  // K: tokens g, g + 16, ..: V: tokens 4 g .. 4 g + 3
  float x[4][16];
  float largest = 0.0f;
  float gain[16];
  if (PREP && !is_v) load16(p.k_gain + chunk * 16, gain);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = is_v ? 4 * g + i : 16 * i + g;
    const bool in = t >= lo && t < hi;
#pragma unroll
    for (int j = 0; j < 16; ++j) x[i][j] = 0.0f;
    if (in) {
      const int64_t at = (int64_t)(base + t - r.position) * r.row_stride + (int64_t)head * r.head_stride + chunk * 16;
      load16((is_v ? r.v : r.k) + at, x[i]);
    }
    if (PREP && !is_v) {
      norm16(x[i], gain);
      rotate16(x[i], cs[t], chunk);
    }
    // magnitudes compare as integers, a NaN or infinity above every number
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) most = max(most, __float_as_uint(x[i][j]) & 0x7fffffffu);
    if (most >= 0x7f800000u) {
      most = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        x[i][j] = finite(x[i][j]) ? x[i][j] : 0.0f;
        most = max(most, __float_as_uint(x[i][j]) & 0x7fffffffu);
      }
      if (in) bad[t] = 1;
    }
    largest = fmaxf(largest, __uint_as_float(most));
  }
  largest = wave_max(largest);
  if ((tid & 63) == 0) atomicMax(&top[is_v], __float_as_uint(largest));  // not negative: ordered as integers
  __syncthreads();
  int e = scale_exponent(__uint_as_float(top[is_v]), -127), shift = 0;
  if (lo > 0) {  // earlier rows of the block stay: its power of two only rises
    const int before = (int)*scale;
    if (before != 255) {  // 255: the block holds none
      e = max(e, before - 127);
      shift = e + 127 - before;
    }
  }
  if (is_v) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = ldexpf(x[i][j], -e);
      // piece of dim 16 chunk + j, dword token / 16
      *reinterpret_cast<int*>(&vt[v_lds(v_piece(4 * g, chunk * 16 + j)) + (g >> 2) * 4]) =
          pack_e4m3(y[0], y[1], y[2], y[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 16 * i + g;
      if (t >= lo && t < hi) {
        u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = bad[t] ? 0x01010101u * kNanCode
                        : (uint32_t)pack_e4m3(ldexpf(x[i][4 * j], -e), ldexpf(x[i][4 * j + 1], -e),
                                              ldexpf(x[i][4 * j + 2], -e), ldexpf(x[i][4 * j + 3], -e));
        *reinterpret_cast<u32x4*>(codes + k_piece(t, chunk)) = o;
      } else if (t < lo && shift > 0) {
        u32x4* at = reinterpret_cast<u32x4*>(codes + k_piece(t, chunk));
        u32x4 o = *at;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = (uint32_t)rescale_e4m3((int)o[j], shift);
        *at = o;
      }
    }
  }
  __syncthreads();
  if (!is_v) {
    if (tid == 0) *scale = (uint8_t)(e + 127);
    return;
  }
  if (tid == 256) *scale = (uint8_t)(e + 127);
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int piece = (tid & 255) + 256 * n;
    const int t0 = ((piece >> 6) & 1) * 8 + ((piece >> 5) & 1) * 4;  // its tokens: 16 s + t0 .. + 3, s = 0..3
    u32x4* at = reinterpret_cast<u32x4*>(codes + piece * 16);
    const u32x4 fresh = *reinterpret_cast<const u32x4*>(&vt[v_lds(piece * 16)]);
    if (lo == 0 && hi == kKv8Block) {
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
    u32x4 o = *at;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t moved = keep[s] ? (uint32_t)rescale_e4m3((int)o[s], shift) : 0;
      o[s] = (o[s] & ~(take[s] | keep[s])) | (fresh[s] & take[s]) | (moved & keep[s]);
    }
    *at = o;
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
// Scale operands of the matrix instructions (2^(byte - 127), one byte used).
constexpr int kOne = 127, kLo = 127 - 4, kProb = 127 - 8;

__device__ __forceinline__ float gated(float o, const uint16_t* gate) {
  return o / (1.0f + __expf(-bf2f(*gate)));
}

// Few queries: 16 (row, query head) pairs of one KV head a block, four waves
// that take every fourth 64-token block of the block's range of keys, operands
// straight from memory to registers, a softmax state for each wave.
//   S[token, query] = K Q^T, 16x16x128: lane (n = lane % 16, g = lane / 16) gives
//   K bytes of token n and Q bytes of query n, receives tokens 4 g .. 4 g + 3
//   of query n;
//   O^T[d, query] += V^T P^T: the 128 places along tokens hold the hi parts of
//   the 64 probabilities and their lo parts, against V twice.
__global__ __launch_bounds__(256, 1) void k_kv8_attn_few(Kv8 c, Kv8Attn a) {
  __shared__ __attribute__((aligned(16))) float sum[4][16][260];
  __shared__ float mx[4][16], den[4][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const int split = (int)blockIdx.x % a.splits, unit = (int)blockIdx.x / a.splits;
  const int head = unit / a.tiles, tile = unit % a.tiles;
  const int pairs = a.rows * a.group;
  const int pair = min(tile * 16 + n, pairs - 1);
  const int row = pair / a.group, qh = head * a.group + pair % a.group;
  // queries: bytes d = 128 s + 32 g .. + 31
  i32x8 qhi[2], qlo[2];
  float cq;
  {
    const uint16_t* q = a.query + ((size_t)row * a.q_heads + qh) * 256 + g * 32;
    float x[4][16];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      load16(q + (i >> 1) * 128 + (i & 1) * 16, x[i]);
#pragma unroll
      for (int j = 0; j < 16; ++j) top = finite(x[i][j]) ? fmaxf(top, fabsf(x[i][j])) : top;
    }
    float2 t = rows_xor16(top);
    t = rows_xor32(fmaxf(t.x, t.y));
    const int e = scale_exponent(fmaxf(t.x, t.y), -100);
    cq = ldexpf(kLog2e / 16.0f, e);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) y[b] = ldexpf(x[i][4 * j + b], -e);
        const int h = pack_e4m3(y[0], y[1], y[2], y[3]);
        const f32x2 u = __builtin_amdgcn_cvt_pk_f32_fp8(h, false), v = __builtin_amdgcn_cvt_pk_f32_fp8(h, true);
        qhi[i >> 1][(i & 1) * 4 + j] = h;
        qlo[i >> 1][(i & 1) * 4 + j] = pack_e4m3((y[0] - u[0]) * 16.0f, (y[1] - u[1]) * 16.0f, (y[2] - v[0]) * 16.0f,
                                                 (y[3] - v[1]) * 16.0f);
      }
  }
  const int last = a.position + row, end = a.position + a.rows;  // last key of the query; keys that exist
  const int tile_end = a.position + min(tile * 16 + 15, pairs - 1) / a.group + 1;
  const int nblk = (tile_end + kKv8Block - 1) / kKv8Block;
  const int b0 = (int)((int64_t)nblk * split / a.splits), b1 = (int)((int64_t)nblk * (split + 1) / a.splits);
  const size_t store = (size_t)head * c.blocks;
  const uint8_t* kp = c.k + store * kBlockBytes + (g >> 1) * 2048 + (g & 1) * 512 + n * 16;
  const uint8_t* vp = c.v + store * kBlockBytes + (g >> 1) * 1024 + (g & 1) * 512 + n * 16;
  f32x4 o[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kNone, l = 0.0f;
  for (int b = b0 + wave; b < b1; b += 4) {
    const uint8_t* kb = kp + (size_t)b * kBlockBytes;
    const uint8_t* vb = vp + (size_t)b * kBlockBytes;
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* at = kb + (t >> 1) * 8192 + (t & 1) * 256 + h * 4096;
        const i32x4 x = *reinterpret_cast<const i32x4*>(at), y = *reinterpret_cast<const i32x4*>(at + 1024);
        const i32x8 k = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        s[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, qhi[h], s[t], 0, 0, 0, kOne, 0, kOne);
        s[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, qlo[h], s[t], 0, 0, 0, kOne, 0, kLo);
      }
    }
    const float cs = ldexpf(cq, (int)c.k_scale[store + b] - 127);
    float top = kNone;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = s[t][i] * cs;
        if (b * 64 + 63 > a.position) x = b * 64 + 16 * t + 4 * g + i <= last ? x : -__builtin_inff();
        s[t][i] = x;
        top = fmaxf(top, x);
      }
    float2 u = rows_xor16(top);
    u = rows_xor32(fmaxf(u.x, u.y));
    const float mn = fmaxf(m, fmaxf(u.x, u.y));
    const float f = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= f;
    i32x8 p;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = __builtin_amdgcn_exp2f(s[t][i] - mn + 8.0f);
        l += y[i];
      }
      const int h = pack_e4m3(y[0], y[1], y[2], y[3]);
      const f32x2 v = __builtin_amdgcn_cvt_pk_f32_fp8(h, false), w = __builtin_amdgcn_cvt_pk_f32_fp8(h, true);
      p[t] = h;
      p[4 + t] = pack_e4m3(y[0] - v[0], y[1] - v[1], y[2] - w[0], y[3] - w[1]);
    }
    const int vs = c.v_scale[store + b];
#pragma unroll
    for (int d = 0; d < 16; ++d) {
      i32x4 x = *reinterpret_cast<const i32x4*>(vb + (d >> 1) * 2048 + (d & 1) * 256);
      if (b * 64 + 64 > end) {  // bytes behind the last key may be anything
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int left = end - (b * 64 + 16 * t + 4 * g);
          x[t] = left >= 4 ? x[t] : left <= 0 ? 0 : x[t] & ((1 << (8 * left)) - 1);
        }
      }
      const i32x8 v = __builtin_shufflevector(x, x, 0, 1, 2, 3, 0, 1, 2, 3);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[d][i] *= f;
      o[d] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(v, p, o[d], 0, 0, 0, vs, 0, kProb);
    }
  }
  // l counts p * 2^8; the lanes of a query hold its tokens' parts
  float2 t = rows_xor16(l);
  t = rows_xor32(t.x + t.y);
  if (lane < 16) {
    mx[wave][n] = m;
    den[wave][n] = (t.x + t.y) * (1.0f / 256.0f);
  }
#pragma unroll
  for (int d = 0; d < 16; ++d) *reinterpret_cast<f32x4*>(&sum[wave][n][d * 16 + g * 4]) = o[d];
  __syncthreads();
  const int qi = tid >> 4, dd = (tid & 15) * 4;
  if (tile * 16 + qi >= pairs) return;
  float top = kNone;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, mx[w][qi]);
  float f[4], total = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = __builtin_amdgcn_exp2f(mx[w][qi] - top);
    total = fmaf(den[w][qi], f[w], total);
  }
  const int i = tile * 16 + qi, r = i / a.group, hq = head * a.group + i % a.group;
  const size_t at = (size_t)r * a.q_heads + hq;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f32x4 x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(&sum[w][qi][dd + 64 * j]);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = fmaf(y[k], f[w], x[k]);
    }
    if (a.splits > 1) {
      float* part = a.part + (at * a.splits + split) * kKv8PartFloats;
      *reinterpret_cast<f32x4*>(part + dd + 64 * j) = x;
      if (tid % 16 == 0 && j == 0) {
        part[256] = top;
        part[257] = total;
      }
      continue;
    }
    const uint16_t* gp = a.gate ? a.gate + at * 512 + 256 + dd + 64 * j : nullptr;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = x[k] / total;
      if (gp) x[k] = gated(x[k], gp + k);
    }
    *reinterpret_cast<uint2*>(a.out + at * 256 + dd + 64 * j) = make_uint2(pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]));
  }
}

// Joins the ranges of keys of one (row, query head): four waves take every
// fourth range, lane = four dims.
__global__ __launch_bounds__(256) void k_kv8_attn_join(Kv8Attn a) {
  __shared__ __attribute__((aligned(16))) float sum[4][256];
  __shared__ float mx[4], den[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const size_t at = blockIdx.x;
  const float* part = a.part + at * a.splits * kKv8PartFloats;
  float m = kNone, l = 0.0f;
  f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = wave; s < a.splits; s += 4) {
    const float* p = part + (size_t)s * kKv8PartFloats;
    const f32x4 x = *reinterpret_cast<const f32x4*>(p + lane * 4);
    const float mn = fmaxf(m, p[256]), f = __builtin_amdgcn_exp2f(m - mn), fx = __builtin_amdgcn_exp2f(p[256] - mn);
    l = fmaf(p[257], fx, l * f);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = fmaf(x[k], fx, o[k] * f);
    m = mn;
  }
  if (lane == 0) {
    mx[wave] = m;
    den[wave] = l;
  }
  *reinterpret_cast<f32x4*>(&sum[wave][lane * 4]) = o;
  __syncthreads();
  const int d = threadIdx.x;
  const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
  float x = 0.0f, total = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = __builtin_amdgcn_exp2f(mx[w] - top);
    x = fmaf(sum[w][d], f, x);
    total = fmaf(den[w], f, total);
  }
  x = x / total;
  if (a.gate) x = gated(x, a.gate + at * 512 + 256 + d);
  a.out[at * 256 + d] = (uint16_t)f2bf(x);
}

int few_tiles(int rows, int group) { return (rows * group + 15) / 16; }
// Ranges of keys of one call: enough blocks for the chip's 256 CUs, none without work for its four waves.
int few_splits(int heads, int tiles, int position, int rows) {
  const int nblk = (position + rows + kKv8Block - 1) / kKv8Block;
  const int most = 256 / (heads * tiles), want = (nblk + 3) / 4;
  return most < 2 || want < 2 ? 1 : most < want ? most : want;
}

}  // namespace

size_t kv8_attn_scratch_bytes(int q_heads, int kv_heads, int rows) {
  const int tiles = few_tiles(rows, q_heads / kv_heads);
  const int most = 256 / (kv_heads * tiles);
  return most < 2 ? 0 : (size_t)rows * q_heads * most * kKv8PartFloats * sizeof(float);
}

hipError_t launch_kv8_write(const Kv8& c, const Kv8Rows& r, hipStream_t s) {
  const int nblk = (r.position + r.rows - 1) / kKv8Block - r.position / kKv8Block + 1;
  hipLaunchKernelGGL(k_kv8_write<false>, dim3(nblk * c.heads), dim3(512), 0, s, c, r, Kv8Prep{});
  return hipGetLastError();
}

hipError_t launch_kv8_prepare(const Kv8& c, const Kv8Rows& r, const Kv8Prep& p, hipStream_t s) {
  const int nblk = (r.position + r.rows - 1) / kKv8Block - r.position / kKv8Block + 1;
  hipLaunchKernelGGL(k_kv8_write<true>, dim3(nblk * c.heads + (r.rows + 7) / 8), dim3(512), 0, s, c, r, p);
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
  a.tiles = few_tiles(a.rows, a.group);
  a.splits = few_splits(c.heads, a.tiles, a.position, a.rows);
  hipLaunchKernelGGL(k_kv8_attn_few, dim3(a.splits * c.heads * a.tiles), dim3(256), 0, s, c, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL(k_kv8_attn_join, dim3(a.rows * a.q_heads), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace es
