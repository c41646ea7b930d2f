// Attention of a tree of drafted tokens over the bf16 cache, and the keys and
// values of an accepted path into the cache.
//
// Node i is a query at position `position` + the number of its ancestors. It
// attends to the whole context and to its path:
//   o_i = sum over keys j of p_ij v_j / sum of p_ij, p_ij = exp(q_i . k_j / 16),
// out = o_i * sigmoid(gate_i). All nodes read the context once together: a block
// takes a KV head, a tile of 128 queries (node and query head in the group) and a
// range of keys, keeps maximum, sum and output sums of each query for it in 32
// bits, and leaves them to the kernel that joins the ranges. The nodes' own keys
// are one more range, the only one with a mask.
#include <algorithm>
#include <type_traits>

#include "es_kernels.hpp"

namespace es {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTileQ = 128;   // queries of a block: four tiles of 32, each on two waves
constexpr int kKeys = 32;     // keys of a stage
constexpr int kStages = 4;
constexpr int kRow = 256;     // bf16 elements between rows in LDS
constexpr int kStage = 2 * kKeys * kRow;  // K rows, then V rows
constexpr int kHalf = 64 * 128;  // output sums that a wave leaves for the other of its tile

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// ---- queries and keys of the nodes ----
// One wave a (node, head): the q heads, then the k heads. RMS norm with the
// squares in 64 bits (they pass 32 bits' range before the head does), rotation with
// angles in 64 bits, one rounding. A node left out gets zeros.
__global__ __launch_bounds__(256) void k_tree_prepare(TreeAttn a) {
  const int lane = threadIdx.x & 63, heads = a.q_heads + a.kv_heads;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= a.rows * heads) return;
  const int row = i / heads, head = i - row * heads;
  const bool of_q = head < a.q_heads;
  const size_t at = of_q ? (size_t)row * a.q_heads + head : (size_t)row * a.kv_heads + head - a.q_heads;
  const uint16_t* const from = of_q ? a.q_proj + at * 512 : a.k_proj + at * 256;
  const uint2 xv = *reinterpret_cast<const uint2*>(from + 4 * lane);
  const uint2 gv = *reinterpret_cast<const uint2*>((of_q ? a.q_gain : a.k_gain) + 4 * lane);
  const uint64_t path = tree_path(a.paths[row], row);
  float sn, cs;
  es_sincos_angle((double)(a.position + __popcll(path) - 1) * (double)a.inv_freq[lane & 31], &sn, &cs);
  const float x[4] = {bf_lo(xv.x), bf_hi(xv.x), bf_lo(xv.y), bf_hi(xv.y)};
  const float gain[4] = {bf_lo(gv.x), bf_hi(gv.x), bf_lo(gv.y), bf_hi(gv.y)};
  double ss = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) ss = fma((double)x[e], (double)x[e], ss);
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) ss += __shfl_xor(ss, k);
  const double inv = 1.0 / sqrt(ss * (1.0 / 256.0) + 1e-6);
  float r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float y = (float)((double)x[e] * inv * (double)gain[e]);
    const int f = ((lane * 4) & 31) + e;
    const float s1 = __shfl(sn, f), c1 = __shfl(cs, f), p1 = dpp_row_ror8(y);  // dim d ^ 32 is in lane ^ 8
    r[e] = lane < 8 ? fmaf(y, c1, -(p1 * s1)) : lane < 16 ? fmaf(p1, s1, y * c1) : y;
  }
  const uint2 packed = path ? make_uint2(pack_bf2(r[0], r[1]), pack_bf2(r[2], r[3])) : make_uint2(0, 0);
  *reinterpret_cast<uint2*>((of_q ? a.query : a.k_tree) + at * 256 + 4 * lane) = packed;
}

// ---- attention ----
// Chunk c (16 bytes) of a row lies at slot c ^ (row & 15) of K and c ^ 4 (row & 3) of
// V, so that the 16 rows of a fragment's read, and the four rows x 64 bytes of a
// transposing read, cover all banks once.
//
// V^T fragments by transposing reads: keys 0..3 and 4..7 of the lane's eight for the
// four 32-dim tiles whose addresses are a[0..3], OFF bytes on. All complete before
// the statement ends.
template <int OFF>
__device__ __forceinline__ void read_v(const uint32_t (&a)[4], u32x4 (&v)[4]) {
  uint64_t x0, x1, x2, x3, y0, y1, y2, y3;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %1, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
      "ds_read_b64_tr_b16 %2, %10 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %10 offset:%13\n\t"
      "ds_read_b64_tr_b16 %3, %11 offset:%12\n\t"
      "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x0), "=&v"(x1), "=&v"(x2), "=&v"(x3), "=&v"(y0), "=&v"(y1), "=&v"(y2), "=&v"(y3)
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(OFF), "n"(OFF + 2 * 4 * kRow)
      : "memory");
  const uint64_t x[4] = {x0, x1, x2, x3}, y[4] = {y0, y1, y2, y3};
#pragma unroll
  for (int t = 0; t < 4; ++t)
    v[t] = u32x4{(uint32_t)x[t], (uint32_t)(x[t] >> 32), (uint32_t)y[t], (uint32_t)(y[t] >> 32)};
}

// K fragments: the four 16-byte chunks at a[0..3], OFF bytes on. As the V reads in
// assembly with their own wait: the compiler takes a read of LDS as dependent on
// every DMA in flight and would wait for the next stages' too.
template <int OFF>
__device__ __forceinline__ void read_k(const uint32_t (&a)[4], u32x4 (&k)[4]) {
  asm volatile(
      "ds_read_b128 %0, %4 offset:%8\n\t"
      "ds_read_b128 %1, %5 offset:%8\n\t"
      "ds_read_b128 %2, %6 offset:%8\n\t"
      "ds_read_b128 %3, %7 offset:%8\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(OFF)
      : "memory");
}
// Barrier for what the waves have waited for themselves (their DMA, counted) and LDS.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Block = (range, KV head, tile of 128 queries), eight waves: wave w has the 32
// queries of tile w & 3 and the keys 16 (w >> 2) .. + 15 of every 32, with a
// softmax state of its own; the two halves meet at the end. Scores S^T = K Q^T on
// 16x16x32 products, a row swap leaves lane l with query l % 32 and eight keys,
// whose exponentials, rounded to bf16, are the operand of O^T += V^T P^T on
// 32x32x16 products. The sum is taken over the rounded ones, so a key that outweighs
// all others leaves its value as it is.
__global__ __launch_bounds__(512, 1) void k_tree_attn(TreeAttn a) {
  __shared__ __attribute__((aligned(16))) uint16_t kv[kStages][kStage];
  __shared__ float half_ref[4][64], half_sum[4][64];
  __shared__ uint64_t path[kTree];
  __shared__ uint32_t odd_rows[2];  // nodes whose V holds an infinity or a NaN
  static_assert(sizeof(kv) >= 4 * kHalf * sizeof(float), "the halves fit the staging memory");
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  // the tiles that read the same keys on one XCD (block b on XCD b % 8)
  const int unit = (blockIdx.x >> 3) / a.tiles * 8 + (blockIdx.x & 7), tile = (blockIdx.x >> 3) % a.tiles;
  if (unit >= (a.ranges + 1) * a.kv_heads) return;
  const int range = unit / a.kv_heads, kvh = unit % a.kv_heads;
  const bool tree = range == a.ranges;
  const int n = tree ? a.rows : a.position;  // keys
  const int blocks = (n + kKeys - 1) / kKeys;
  // A range is every `ranges`-th block of 32 keys, so that at any time all blocks read
  // one window of the cache: contiguous ranges read 256 streams at equal distances, at
  // 3.9 TB/s against 4.4, and 5.0 with loads that pass the caches by (1 node at 131008,
  // whole calls of 69, 60 and 54 us).
  const int first = tree ? 0 : range, every = tree ? 1 : a.ranges;
  const int steps = (blocks - first + every - 1) / every;
  const int qi = lane & 15, g = lane >> 4, kh = wave >> 2;
  const int q0 = tile * kTileQ + 32 * (wave & 3);  // the wave's queries
  const bool busy = q0 < a.queries;
  const int mine = min(q0 + (lane & 31), a.queries - 1);  // the lane's query once the scores are swapped
  bf16x8 qf[2][8];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int q = min(q0 + 16 * u + qi, a.queries - 1), row = q / a.group;
    const uint16_t* const from = a.query + ((size_t)row * a.q_heads + kvh * a.group + q - row * a.group) * 256 + 8 * g;
#pragma unroll
    for (int s = 0; s < 8; ++s) qf[u][s] = *reinterpret_cast<const bf16x8*>(from + 32 * s);
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int s = 0; s < 8; ++s) asm volatile("" : "+v"(qf[u][s]));
  // DMA of 32 keys: wave w rows 4 w .. 4 w + 3 of K and of V, two rows (1 KB) an
  // instruction, lane l slot l % 32 of row l / 32 of the two. Rows past the last one
  // repeat it: their products are masked.
  const uint16_t* const kbase = tree ? a.k_tree + kvh * 256 : a.kcache + (size_t)kvh * a.capacity * 256;
  const uint16_t* const vbase = tree ? a.v_proj + kvh * 256 : a.vcache + (size_t)kvh * a.capacity * 256;
  const uint32_t stride = tree ? (uint32_t)a.kv_heads * 512u : 512u;
  const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc((void*)kbase, 0, -1, 0x00020000);
  const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc((void*)vbase, 0, -1, 0x00020000);
  uint32_t kchunk[2], vchunk[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 4 * wave + 2 * i + (lane >> 5);
    kchunk[i] = (uint32_t)(((lane & 31) ^ (r & 15)) * 16);
    vchunk[i] = (uint32_t)(((lane & 31) ^ 4 * (r & 3)) * 16);
  }
  auto issue = [&](int kb, int st) {
    uint16_t* const stage = kv[st];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 4 * wave + 2 * i;
      uint32_t at = (uint32_t)(kb * kKeys + r) * stride, more = (uint32_t)(lane >> 5) * stride;
      if (kb * kKeys + kKeys > n) {
        at = 0;
        more = (uint32_t)min(kb * kKeys + r + (lane >> 5), n - 1) * stride;
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(krs, (__attribute__((address_space(3))) void*)(stage + r * kRow), 16,
                                               kchunk[i] + more, at, 0, kLoadNonTemporal);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vrs, (__attribute__((address_space(3))) void*)(stage + (kKeys + r) * kRow), 16,
                                               vchunk[i] + more, at, 0, kLoadNonTemporal);
    }
  };
  for (int i = 0; i < min(kStages - 1, steps); ++i) issue(first + i * every, i);
  f32x16 ot[8];  // O^T: dims 32 i + 8 (r / 4) + 4 (l / 32) + r % 4 of query l % 32
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) ot[i][r] = 0.0f;
  // The reference starts below every score but finite: a half may have no key.
  float ref = -3.0e38f, sum = 0.0f;
  const float c = 0.0625f * 1.4426950408889634f;  // log2(e) / 16
  const uint32_t kv_base = (uint32_t)(uintptr_t)((const __attribute__((address_space(3))) uint16_t*)(&kv[0][0]));
  uint32_t k_at[4], v_at[4];  // LDS bytes: dims 32 s + 8 g of key qi, s % 4 = i; dims 32 t + 16 (g & 1), t % 4 = i
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    k_at[i] = kv_base + (uint32_t)(2 * ((16 * kh + qi) * kRow + ((4 * i + g) ^ qi) * 8));
    const int r = 16 * kh + 8 * (g >> 1) + (qi >> 2);
    v_at[i] = kv_base + (uint32_t)(2 * ((kKeys + r) * kRow + 32 * (i ^ (r & 3)) + 16 * (g & 1) + 4 * (qi & 3)));
  }
  uint64_t seen = 0;
  if (tree) {
    if (t < kTree) path[t] = t < a.rows ? tree_path(a.paths[t], t) : 0;
    if (t < 2) odd_rows[t] = 0;
    __syncthreads();
    seen = path[mine / a.group];
  }
  int st = kStages - 1;
  for (int i = 0, kb = first; i < steps; ++i, kb += every) {
    st = (st + 1) % kStages;
    const int ahead = min(kStages - 2, steps - 1 - i);
    if (ahead >= 2)
      wait_vmcnt<8>();
    else if (ahead == 1)
      wait_vmcnt<4>();
    else
      wait_vmcnt<0>();
    stage_barrier();  // block kb is there, and every wave is past block kb - 1
    if (i + kStages - 1 < steps) issue(kb + (kStages - 1) * every, (st + kStages - 1) % kStages);
    if (tree) {
      // A masked key's value counts 0 times: infinities and NaN leave the products and join at the end.
      uint32_t* const v = reinterpret_cast<uint32_t*>(kv[st] + (kKeys + (t >> 4)) * kRow + (t & 15) * 16);
      bool odd = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t w = v[e];
        const bool lo = (w & 0x7f80u) == 0x7f80u, hi = (w & 0x7f800000u) == 0x7f800000u;
        if (lo) w &= 0xffff0000u;
        if (hi) w &= 0xffffu;
        if (lo || hi) v[e] = w;
        odd |= lo || hi;
      }
      const int key = kb * kKeys + (t >> 4);
      if (odd && key < n) atomicOr(&odd_rows[key >> 5], 1u << (key & 31));
      __syncthreads();
    }
    if (!busy) continue;
    uint32_t ka[4], va[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ka[i] = k_at[i] + (uint32_t)(2 * kStage) * st;
      va[i] = v_at[i] + (uint32_t)(2 * kStage) * st;
    }
    f32x4 sc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int s4 = 0; s4 < 2; ++s4) {
      u32x4 kf[4];
      if (s4 == 0)
        read_k<0>(ka, kf);
      else
        read_k<256>(ka, kf);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf[i]), qf[u][4 * s4 + i], sc[u], 0, 0, 0);
    }
    // keys 4 g + r of query l % 16 of both groups -> keys 8 (l / 32) + e of query l % 32
    float x[8];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(sc[0][r]), __float_as_uint(sc[1][r]), false, false);
      x[r] = __uint_as_float(p[0]);
      x[4 + r] = __uint_as_float(p[1]);
    }
    const int key0 = kb * kKeys + 16 * kh + 8 * (lane >> 5);
    if (tree) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = seen >> (key0 + e) & 1 ? x[e] : -INFINITY;
    } else if (kb * kKeys + kKeys > n) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = key0 + e < n ? x[e] : -INFINITY;
    }
    float mloc = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mloc = fmaxf(mloc, x[e]);
    const float2 m2 = rows_xor32(mloc);
    // the reference moves only where the maximum passes it by more than 8
    const float mblk = fmaxf(m2.x, m2.y) * c, mnew = mblk > ref + 8.0f ? mblk : ref;
    const float factor = __builtin_amdgcn_exp2f(ref - mnew);
    u32x4 pb;
    float psum = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      pb[e] = pack_bf2(__builtin_amdgcn_exp2f(fmaf(x[2 * e], c, -mnew)), __builtin_amdgcn_exp2f(fmaf(x[2 * e + 1], c, -mnew)));
      psum += bf_lo(pb[e]) + bf_hi(pb[e]);
    }
    const float2 s2 = rows_xor32(psum);
    sum = sum * factor + (s2.x + s2.y);
    if (__any(mnew > ref)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) ot[i][r] *= factor;
    }
    ref = mnew;
    const bf16x8 pf = __builtin_bit_cast(bf16x8, pb);
#pragma unroll
    for (int d4 = 0; d4 < 2; ++d4) {
      u32x4 vf[4];
      if (d4 == 0)
        read_v<0>(va, vf);
      else
        read_v<256>(va, vf);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        ot[4 * d4 + i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vf[i]), pf, ot[4 * d4 + i], 0, 0, 0);
    }
  }
  stage_barrier();  // the staging memory is free
  float* const half = reinterpret_cast<float*>(&kv[0][0]) + (wave & 3) * kHalf;
  if (kh && busy) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<float4*>(half + ((4 * i + r) * 64 + lane) * 4) =
            make_float4(ot[i][4 * r], ot[i][4 * r + 1], ot[i][4 * r + 2], ot[i][4 * r + 3]);
    half_ref[wave & 3][lane] = ref;
    half_sum[wave & 3][lane] = sum;
  }
  __syncthreads();
  if (kh || !busy) return;
  const float ref1 = half_ref[wave][lane], sum1 = half_sum[wave][lane], top = fmaxf(ref, ref1);
  const float f0 = __builtin_amdgcn_exp2f(ref - top), f1 = __builtin_amdgcn_exp2f(ref1 - top);
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float4 o = *reinterpret_cast<const float4*>(half + ((4 * i + r) * 64 + lane) * 4);
      ot[i][4 * r] = fmaf(o.x, f1, ot[i][4 * r] * f0);
      ot[i][4 * r + 1] = fmaf(o.y, f1, ot[i][4 * r + 1] * f0);
      ot[i][4 * r + 2] = fmaf(o.z, f1, ot[i][4 * r + 2] * f0);
      ot[i][4 * r + 3] = fmaf(o.w, f1, ot[i][4 * r + 3] * f0);
    }
  if (tree) {
    const uint64_t odd = (uint64_t)odd_rows[1] << 32 | odd_rows[0];
#pragma unroll 1
    for (uint64_t left = odd; left; left &= left - 1) {
      const int j = __builtin_ctzll(left);
      const uint16_t* const v = vbase + (size_t)j * a.kv_heads * 256 + 4 * (lane >> 5);
      const bool on = seen >> j & 1;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint2 w = *reinterpret_cast<const uint2*>(v + 32 * i + 8 * r);
          const float y[4] = {bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y)};
#pragma unroll
          for (int e = 0; e < 4; ++e) ot[i][4 * r + e] += on && !(fabsf(y[e]) < INFINITY) ? y[e] : 0.0f;
        }
    }
  }
  const int q = q0 + (lane & 31);
  if (q >= a.queries) return;
  float* const part = a.part + ((size_t)unit * a.queries + q) * kTreePartFloats;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<float4*>(part + 32 * i + 8 * r + 4 * (lane >> 5)) =
          make_float4(ot[i][4 * r], ot[i][4 * r + 1], ot[i][4 * r + 2], ot[i][4 * r + 3]);
  if (lane < 32) *reinterpret_cast<float2*>(part + 256) = make_float2(top, fmaf(sum1, f1, sum * f0));
}

// Joins the ranges of a node's head: block = (node, head), wave w takes ranges w,
// w + 4, ..., a lane four dims; then the output gate.
__global__ __launch_bounds__(256) void k_tree_join(TreeAttn a) {
  __shared__ float4 part_o[4][64];
  __shared__ float2 part_s[4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int row = blockIdx.x / a.q_heads, head = blockIdx.x % a.q_heads;
  const int kvh = head / a.group, q = row * a.group + head % a.group;
  float ref = -3.0e38f, sum = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto join = [&](float r1, float s1, float4 o1) {
    const float top = fmaxf(ref, r1), f0 = __builtin_amdgcn_exp2f(ref - top), f1 = __builtin_amdgcn_exp2f(r1 - top);
    o.x = fmaf(o1.x, f1, o.x * f0);
    o.y = fmaf(o1.y, f1, o.y * f0);
    o.z = fmaf(o1.z, f1, o.z * f0);
    o.w = fmaf(o1.w, f1, o.w * f0);
    sum = fmaf(s1, f1, sum * f0);
    ref = top;
  };
#pragma unroll 4
  for (int i = wave; i <= a.ranges; i += 4) {
    const float* const part = a.part + ((size_t)(i * a.kv_heads + kvh) * a.queries + q) * kTreePartFloats;
    const float4 o1 = *reinterpret_cast<const float4*>(part + 4 * lane);
    const float2 s1 = *reinterpret_cast<const float2*>(part + 256);
    join(s1.x, s1.y, o1);
  }
  part_o[wave][lane] = o;
  if (lane == 0) part_s[wave] = make_float2(ref, sum);
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < 4; ++w) join(part_s[w].x, part_s[w].y, part_o[w][lane]);
  const size_t at = (size_t)row * a.q_heads + head;
  const uint2 gate = *reinterpret_cast<const uint2*>(a.q_proj + at * 512 + 256 + 4 * lane);
  auto gated = [&](float x, float z) { return x / sum / (1.0f + __builtin_amdgcn_exp2f(-z * 1.44269504088896341f)); };
  uint2 out = make_uint2(pack_bf2(gated(o.x, bf_lo(gate.x)), gated(o.y, bf_hi(gate.x))),
                         pack_bf2(gated(o.z, bf_lo(gate.y)), gated(o.w, bf_hi(gate.y))));
  if (!tree_path(a.paths[row], row)) out = make_uint2(0, 0);
  *reinterpret_cast<uint2*>(a.gated + at * 256 + 4 * lane) = out;
}

// ---- an accepted path into the cache ----
// 32 lanes a row of 256: block (8 places of the path, KV head, K or V).
__global__ __launch_bounds__(256) void k_tree_keep_kv(TreeKeepKv a) {
  const int place = blockIdx.x * 8 + (threadIdx.x >> 5), kvh = blockIdx.y, c = 8 * (threadIdx.x & 31);
  uint64_t path = tree_path(a.paths[a.node], a.node);
  const int64_t position = (int64_t)a.position + place;
  if (place >= __popcll(path) || position >= a.capacity) return;
  for (int k = 0; k < place; ++k) path &= path - 1;
  const size_t from = ((size_t)__builtin_ctzll(path) * a.kv_heads + kvh) * 256 + c;
  const size_t to = ((size_t)kvh * a.capacity + position) * 256 + c;
  if (blockIdx.z)
    *reinterpret_cast<u32x4*>(a.vcache + to) = *reinterpret_cast<const u32x4*>(a.v_proj + from);
  else
    *reinterpret_cast<u32x4*>(a.kcache + to) = *reinterpret_cast<const u32x4*>(a.k_tree + from);
}

// Ranges of the context: with the nodes' own, as many blocks as CUs.
int most_ranges(int kv_heads, int tiles) { return std::max(1, 256 / (kv_heads * tiles) - 1); }

}  // namespace

size_t tree_attn_scratch_bytes(int q_heads, int kv_heads, int rows) {
  const int queries = rows * (q_heads / kv_heads), tiles = (queries + kTileQ - 1) / kTileQ;
  return (size_t)rows * q_heads * 512 +
         (size_t)(most_ranges(kv_heads, tiles) + 1) * kv_heads * queries * kTreePartFloats * sizeof(float);
}

hipError_t launch_tree_attn(TreeAttn a, hipStream_t s) {
  a.group = a.q_heads / a.kv_heads;
  a.queries = a.rows * a.group;
  a.tiles = (a.queries + kTileQ - 1) / kTileQ;
  const int blocks = (a.position + kKeys - 1) / kKeys;
  a.ranges = std::min(most_ranges(a.kv_heads, a.tiles), (blocks + 1) / 2);
  a.query = static_cast<uint16_t*>(a.scratch);
  a.part = reinterpret_cast<float*>(a.query + (size_t)a.rows * a.q_heads * 256);
  const int heads = a.rows * (a.q_heads + a.kv_heads), units = (a.ranges + 1) * a.kv_heads;
  k_tree_prepare<<<(heads + 3) / 4, 256, 0, s>>>(a);
  k_tree_attn<<<(units + 7) / 8 * 8 * a.tiles, 512, 0, s>>>(a);
  k_tree_join<<<a.rows * a.q_heads, 256, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_tree_keep_kv(const TreeKeepKv& a, hipStream_t s) {
  k_tree_keep_kv<<<dim3((a.node + 8) / 8, a.kv_heads, 2), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace es
