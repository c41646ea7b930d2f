// A Gated DeltaNet layer over a tree of drafted tokens, and the layer's state
// behind an accepted path.
//
// With S0 the state before the draft, i a node, j an ancestor of it (or itself),
// G_i the product of the gates on i's path and G_i / G_j that of the gates behind j:
//   u_i = beta_i (v_i - G_i S0 k_i - sum over ancestors j of (G_i / G_j) (k_j . k_i) u_j)
//   y_i = G_i S0 q_i + sum over ancestors j and i of (G_i / G_j) (k_j . q_i) u_j
//   S_i = G_i S0 + sum over ancestors j and i of (G_i / G_j) u_j k_j^T
// so no node's state is formed: the draft reads S0 once, and only an accepted path
// writes a state. The products of gates are exponentials of differences of sums of
// log gates (in 64 bits), which never overflow and need no division.
#include "es_kernels.hpp"

namespace es {
namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kSlice = 16;               // value rows of a block
constexpr int kStaged = 256 + kSlice;    // channels of a head that a block takes: q, k, its part of v
constexpr int kStagedRow = kStaged + 8;  // bf16 elements between staged rows
constexpr int kQk = 132;                 // floats between rows of q and of k
constexpr int kPair = 65;                // floats between rows of the pair matrices

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __builtin_amdgcn_exp2f(-x * kLog2e)); }
// Log gates count from here down as gates of 0.
__device__ __forceinline__ double bounded(float log_g) { return log_g < -1e30f ? -1e30 : (double)log_g; }

// Block = (16 value rows, head), four waves; 128 blocks.
__global__ __launch_bounds__(256) void k_gdn_tree(TreeGdn a) {
  __shared__ float qs[kTree][kQk], ks[kTree][kQk];
  __shared__ __attribute__((aligned(16))) union {
    uint16_t staged[4 + kTree][kStagedRow];  // the ring's rows, then the nodes'
    struct {
      float low[kTree][kPair], pair[kTree][kPair];
    } m;
  } un;
  __shared__ float b[kTree][kSlice + 1], y0[kTree][kSlice + 1];
  __shared__ uint64_t path[kTree];
  __shared__ double total[kTree];
  __shared__ float log_gate[kTree], beta[kTree];
  __shared__ uint8_t tap[kTree][4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, n16 = lane & 15, g = lane >> 4;
  const int h = blockIdx.x >> 3, v0 = (blockIdx.x & 7) * kSlice;
  const int rows = a.rows, tiles = (rows + 15) >> 4;
  // the slice of the state: lane holds S[v0 + n16][16 s + 4 g .. + 3]
  f32x4 st[8];
#pragma unroll
  for (int s = 0; s < 8; ++s)
    st[s] = *reinterpret_cast<const f32x4*>(a.state + ((size_t)h * 128 + v0 + n16) * 128 + 16 * s + 4 * g);
  for (int i = t; i < (4 + rows) * (kStaged / 8); i += 256) {
    const int r = i / (kStaged / 8), c = i % (kStaged / 8);
    const int channel = c < 16 ? h * 128 + 8 * c : c < 32 ? 2048 + h * 128 + 8 * (c - 16) : 4096 + h * 128 + v0 + 8 * (c - 32);
    const uint16_t* const from = r < 4 ? a.ring + r * kConv : a.raw + (size_t)(r - 4) * kConv;
    *reinterpret_cast<u32x4*>(&un.staged[r][8 * c]) = *reinterpret_cast<const u32x4*>(from + channel);
  }
  if (t < kTree) {
    const uint64_t p = t < rows ? tree_path(a.paths[t], t) : 0;
    path[t] = p;
    // rows of the convolution's taps, oldest first: the ring's slot or the ancestor's row
    const int depth = __popcll(p) - 1;
    uint64_t up = p;
    for (int k = 3; k >= 0; --k) {
      const int back = 3 - k;
      if (back <= depth) {
        const int j = 63 - __clzll(up);
        tap[t][k] = (uint8_t)(4 + j);
        up &= ~(1ull << j);
      } else {
        tap[t][k] = (uint8_t)((a.position + depth - back) & 3);
      }
    }
    float log_g = 0.0f, be = 0.0f;
    if (p) {
      const float x = bf2f(a.a_proj[t * 16 + h]) + bf2f(a.dt_bias[h]);
      log_g = -expf(a.a_log[h]) * (fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))));
      be = sigmoid(bf2f(a.b_proj[t * 16 + h]));
    }
    log_gate[t] = log_g;
    beta[t] = be;
    if (v0 == 0 && t < rows) a.log_decay[t * 16 + h] = log_g;
  }
  __syncthreads();
  if (t < kTree) {
    double sum = 0.0;
    for (uint64_t p = path[t]; p; p &= p - 1) sum += bounded(log_gate[__builtin_ctzll(p)]);
    total[t] = sum;
  }
  // convolution and SiLU: a thread one channel of q or k, then 16 channels of v
  auto conv = [&](int r, int c, uint2 w) {
    float x = bf2f(un.staged[tap[r][0]][c]) * bf_lo(w.x);
    x = fmaf(bf2f(un.staged[tap[r][1]][c]), bf_hi(w.x), x);
    x = fmaf(bf2f(un.staged[tap[r][2]][c]), bf_lo(w.y), x);
    x = fmaf(bf2f(un.staged[tap[r][3]][c]), bf_hi(w.y), x);
    return x / (1.0f + __builtin_amdgcn_exp2f(-x * kLog2e));
  };
  {
    const int channel = (t >> 7) * 2048 + h * 128 + (t & 127);
    const uint2 w = *reinterpret_cast<const uint2*>(a.conv_w + channel * 4);
    float* const out = t < 128 ? &qs[0][t] : &ks[0][t - 128];
    for (int r = 0; r < 16 * tiles; ++r) out[r * kQk] = path[r] ? conv(r, t, w) : 0.0f;
    const uint2 wv = *reinterpret_cast<const uint2*>(a.conv_w + (4096 + h * 128 + v0 + (t & 15)) * 4);
    for (int r = t >> 4; r < 16 * tiles; r += 16) b[r][t & 15] = path[r] ? conv(r, 256 + (t & 15), wv) : 0.0f;
  }
  __syncthreads();
  // norms: 16 lanes a row, its squares in 64 bits (they pass 32 bits' range before the row does)
  for (int i = t >> 4; i < 32 * tiles; i += 16) {
    float* const x = (i & 1 ? ks[i >> 1] : qs[i >> 1]) + 8 * n16;
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = fma((double)x[k], (double)x[k], ss);
#pragma unroll
    for (int k = 1; k < 16; k <<= 1) ss += __shfl_xor(ss, k);
    const double inv = (i & 1 ? 1.0 : 0.08838834764831844055) / sqrt(ss + 1e-6);  // q by 128^-1/2 too
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = (float)((double)x[k] * inv);
  }
  __syncthreads();
  if (v0 == 0)
    for (int i = t; i < rows * 32; i += 256)
      *reinterpret_cast<float4*>(a.keys + ((size_t)(i >> 5) * 16 + h) * 128 + 4 * (i & 31)) =
          *reinterpret_cast<const float4*>(&ks[i >> 5][4 * (i & 31)]);
  // 16 x 16 tiles of k S0^T and q S0^T, then of k k^T and q k^T on and below the diagonal
  const int lower = tiles * (tiles + 1) / 2, all = 2 * tiles + 2 * lower;
  for (int i = wave; i < all; i += 4) {
    const bool with_state = i < 2 * tiles;
    const int k = with_state ? i : i - 2 * tiles;
    const bool of_q = with_state ? k >= tiles : k >= lower;
    int ti = with_state ? k % tiles : k % lower, tj = 0;
    if (!with_state)
      for (tj = ti, ti = 0; tj > ti; ++ti) tj -= ti + 1;
    const float* const left = (of_q ? qs[0] : ks[0]) + (16 * ti + n16) * kQk + 4 * g;
    const float* const right = ks[16 * tj + n16] + 4 * g;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(left + 16 * s);
      const f32x4 y = with_state ? st[s] : *reinterpret_cast<const f32x4*>(right + 16 * s);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 16 * ti + 4 * g + e;
      if (with_state) {
        const float decay = expf((float)total[r]);
        if (of_q)
          y0[r][n16] = path[r] ? decay * acc[e] : 0.0f;
        else
          b[r][n16] = path[r] ? beta[r] * (b[r][n16] - decay * acc[e]) : 0.0f;
      } else {
        const int c = 16 * tj + n16;
        const bool on = path[r] >> c & 1;
        const float x = on ? acc[e] * expf((float)(total[r] - total[c])) : 0.0f;
        if (of_q)
          un.m.pair[r][c] = x;
        else
          un.m.low[r][c] = c < r ? beta[r] * x : 0.0f;
      }
    }
  }
  __syncthreads();
  // Substitution, a node a lane and four value rows a wave: node i's u is final
  // once its ancestors' have left the sum; its descendants take it from theirs.
  // What is not on a path is selected away, so a NaN stays on its own.
  const uint64_t mine = path[lane];
  float u[4], y[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    u[k] = lane < 16 * tiles ? b[lane][4 * wave + k] : 0.0f;
    y[k] = lane < 16 * tiles ? y0[lane][4 * wave + k] : 0.0f;
  }
  for (int c = 0; c < tiles; ++c) {
    float low[16], pair[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool in = lane >= 16 * c && lane < 16 * tiles;
      low[e] = in ? un.m.low[lane][16 * c + e] : 0.0f;
      pair[e] = in ? un.m.pair[lane][16 * c + e] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int i = 16 * c + e;
      const bool on = mine >> i & 1;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float ui = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(u[k]), i));
        u[k] = on && lane != i ? fmaf(-low[e], ui, u[k]) : u[k];
        y[k] = on ? fmaf(pair[e], ui, y[k]) : y[k];
      }
    }
  }
  if (lane < rows) {
    const size_t at = ((size_t)lane * 16 + h) * 128 + v0 + 4 * wave;
    *reinterpret_cast<float4*>(a.updates + at) = make_float4(u[0], u[1], u[2], u[3]);
    *reinterpret_cast<uint2*>(a.y + at) = make_uint2(pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]));
  }
}

// The state behind a path: blocks 0 .. 255 (8 value rows of a head each) four
// elements a thread; blocks 256 .. 258 the ring, whose slots take the raw rows of
// the path's last four nodes.
__global__ __launch_bounds__(256) void k_gdn_tree_keep(TreeKeepGdn a) {
  const int t = threadIdx.x;
  const uint64_t path = tree_path(a.paths[a.node], a.node);
  if (blockIdx.x >= 256) {
    const int c = 8 * ((blockIdx.x - 256) * 256 + t);
    uint64_t p = path;
    for (int place = __popcll(p) - 1, k = 0; k < 4 && p; ++k, --place) {
      const int j = 63 - __clzll(p);
      p &= ~(1ull << j);
      *reinterpret_cast<u32x4*>(a.ring + ((a.position + place) & 3) * kConv + c) =
          *reinterpret_cast<const u32x4*>(a.raw + (size_t)j * kConv + c);
    }
    return;
  }
  const int h = blockIdx.x >> 4, v = (blockIdx.x & 15) * 8 + (t >> 5), k = 4 * (t & 31);
  const size_t at = ((size_t)h * 128 + v) * 128 + k;
  f32x4 s = *reinterpret_cast<const f32x4*>(a.state + at);
  double behind = 0.0;  // log of the gates behind the node at hand
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint64_t p = path; p;) {
    const int j = 63 - __clzll(p);
    p &= ~(1ull << j);
    const size_t row = (size_t)j * 16 + h;
    const float w = expf((float)behind) * a.updates[row * 128 + v];
    const f32x4 key = *reinterpret_cast<const f32x4*>(a.keys + row * 128 + k);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = fmaf(w, key[e], sum[e]);
    behind += bounded(a.log_decay[row]);
  }
  const float decay = expf((float)behind);
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = path ? fmaf(decay, s[e], sum[e]) : s[e];
  *reinterpret_cast<f32x4*>(a.state_out + at) = s;
}

}  // namespace

hipError_t launch_tree_gdn(const TreeGdn& a, hipStream_t s) {
  k_gdn_tree<<<128, 256, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_tree_keep_gdn(const TreeKeepGdn& a, hipStream_t s) {
  k_gdn_tree_keep<<<256 + kConv / 2048, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace es
