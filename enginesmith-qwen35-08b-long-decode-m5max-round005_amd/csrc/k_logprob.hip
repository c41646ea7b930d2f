// Scores of rows of bf16 logits: log probability of a given token, entropy,
// log sum and the `top` largest with their log probabilities.
//
// With m the row's largest logit, R = sum of exp(x - m) over all elements but one
// that equals m, D = the same sum of exp(x - m) (x - m), and A = log1p(R):
//   log sum = m + A,  log p(x) = (x - m) - A,  entropy = A - D / (1 + R).
// The 1 of the largest element never joins a 32-bit sum, so a nearly certain token
// keeps the digits of its log probability and of the entropy.
//
// One read of the row. A block walks a range of it in segments, 16 bytes a
// thread and load, with the maximum so far as the reference of its sums; the
// segment after the one at hand is on its way. The top list is kept in LDS as
// 64-bit keys (the value's bits made monotone, then the complement of the index:
// of equal values the lowest index ranks first), and a segment is looked at for it
// only if its maximum passes the list's last value. Rows too few to fill the card
// are cut in ranges, which a second kernel joins.
#include <algorithm>

#include "es_kernels.hpp"

namespace es {
namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kCand = 1024;  // candidates a selection ranks at once: kLogprobTop lists or threads of 32
static_assert(kLogprobTop == 32, "kCand holds 32 elements of 32 threads, or 32 lists of 32");

struct RangeStats {
  float m;       // largest logit (NaN if there is one)
  float pad;
  double r, d;   // R and D (in units of log 2) of the range
};

__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Monotone 64-bit key of a logit: value first (-0 as +0, NaN below -inf), then the lower index.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  const uint32_t b = __float_as_uint(x + 0.0f) >> 16;
  const uint32_t o = x != x ? 0u : b & 0x8000u ? b ^ 0xffffu : b | 0x8000u;
  return (uint64_t)o << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0 ? __builtin_nanf("") : bf2f(o & 0x8000u ? o ^ 0x8000u : o ^ 0xffffu);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return ~(uint32_t)key; }

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, s);
    v = v > o ? v : o;
  }
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) v += __shfl_xor(v, s);
  return v;
}

struct Shared {
  uint64_t list[2][kLogprobTop];  // the largest keys so far, in order; one of the two at a time
  uint64_t cand[kCand];
  float lane_max[256];
  uint64_t wave_key[2][4];
  float wave_max[2][4];
  double sum[2][4];
  float t0;
  int count;
};

// Joins the n candidates to the nl keys of list `at`: the `top` largest of both,
// in order, into the other one. A key's place is the number of larger ones.
__device__ __forceinline__ void rank_into(Shared& sh, int at, int nl, int n, int top) {
  const int all = nl + n;
  for (int i = threadIdx.x; i < all; i += 256) {
    const uint64_t mine = i < nl ? sh.list[at][i] : sh.cand[i - nl];
    int place = 0;
    for (int j = 0; j < nl; ++j) place += sh.list[at][j] > mine;
    for (int j = 0; j < n; ++j) place += sh.cand[j] > mine;
    if (place < top) sh.list[at ^ 1][place] = mine;
  }
  __syncthreads();
}

// A row's outputs from its largest logit, R, D and the list (called by the whole block).
__device__ __forceinline__ void finish_row(const LogprobArgs& a, int row, float m, double r, double d,
                                           const uint64_t* list) {
  const bool finite = fabsf(m) < __builtin_inff();
  const double log_sum = finite ? log1p(r) : (double)__builtin_nanf("");
  if (threadIdx.x == 0) {
    if (a.logprob) {
      const uint32_t token = a.tokens[row];
      float x = __builtin_nanf("");
      if (token < (uint32_t)a.vocab) x = bf2f(a.logits[(int64_t)row * a.stride + token]);
      a.logprob[row] = (float)(((double)x - (double)m) - log_sum);
    }
    if (a.entropy) a.entropy[row] = (float)(log_sum - d * 0.69314718055994530942 / (1.0 + r));
    if (a.lse) a.lse[row] = finite ? (float)((double)m + log_sum) : m;
  }
  const int i = threadIdx.x;
  if (i < a.top) {
    const uint64_t key = list[i];
    a.top_ids[(size_t)row * a.top + i] = key_index(key);
    a.top_logprobs[(size_t)row * a.top + i] = (float)(((double)key_value(key) - (double)m) - log_sum);
  }
}

// V: 16-byte vectors of a thread in a segment.
template <int V>
__global__ __launch_bounds__(256) void k_logprob(LogprobArgs a) {
  __shared__ Shared sh;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int row = blockIdx.x / a.ranges, range = blockIdx.x % a.ranges;
  // Vectors lie on the 16-byte grid of memory: vector j holds elements 8 j - off .. + 7 of the row.
  const uint16_t* const x0 = a.logits + (int64_t)row * a.stride;
  const int off = (int)((uintptr_t)x0 >> 1 & 7);
  const u32x4* const grid = reinterpret_cast<const u32x4*>(x0 - off);
  const int j0 = range * a.per, j1 = min(j0 + a.per, (a.vocab + off + 7) >> 3);
  const int whole0 = off ? 1 : 0, whole1 = (a.vocab + off) >> 3;  // vectors within the row
  auto load = [&](int first, u32x4 (&x)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int j = first + v * 256 + t;
      x[v] = u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};  // -inf outside the row
      if (j >= whole0 && j < min(whole1, j1)) {
        x[v] = grid[j];
      } else if (j < j1) {
        uint64_t lo = 0, hi = 0;
#pragma unroll 1
        for (int e = 7; e >= 0; --e) {
          const int i = 8 * j + e - off;
          hi = hi << 16 | lo >> 48;
          lo = lo << 16 | (i >= 0 && i < a.vocab ? x0[i] : 0xff80u);
        }
        x[v] = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
      }
    }
  };
  // f(element, index) of the thread's elements of the row, in a rolled loop: for what few segments need
  auto each = [&](const u32x4 (&x)[V], int seg, auto f) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      uint64_t lo = x[v][0] | (uint64_t)x[v][1] << 32, hi = x[v][2] | (uint64_t)x[v][3] << 32;
      const int j = seg + v * 256 + t;
      if (j >= j1) continue;
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        const int i = 8 * j + e - off;
        if (i >= 0 && i < a.vocab) f(bf2f((uint32_t)lo & 0xffffu), (uint32_t)i);
        lo = lo >> 16 | hi << 48;
        hi >>= 16;
      }
    }
  };
  auto value = [](const u32x4 (&x)[V], int v, int e) { return e & 1 ? bf_hi(x[v][e >> 1]) : bf_lo(x[v][e >> 1]); };
  float m = -__builtin_inff(), last = -__builtin_inff();  // largest so far; the list's last value once it is full
  float r = 0.0f, d = 0.0f;                               // the thread's part of R and D
  int at = 0, nl = 0, buf = 0;
  u32x4 next[V];
  load(j0, next);
  for (int seg = j0; seg < j1; seg += 256 * V) {
    u32x4 x[V];
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = next[v];
    if (seg + 256 * V < j1) load(seg + 256 * V, next);
    float tm = -__builtin_inff();
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) tm = maximum(tm, value(x, v, e));
    float wm = tm;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) wm = maximum(wm, __shfl_xor(wm, s));
    if (lane == 0) sh.wave_max[buf][wave] = wm;
    __syncthreads();
    const float* const w = sh.wave_max[buf];
    const float ms = maximum(maximum(w[0], w[1]), maximum(w[2], w[3]));
    const int first_wave = w[0] == ms ? 0 : w[1] == ms ? 1 : w[2] == ms ? 2 : 3;
    buf ^= 1;
    if (a.top && !(nl == a.top && ms <= last)) {
      // Candidates pass the list's last value, or, while the list is not full, reach
      // the top-th largest of the threads' maxima, which as many elements at least do.
      const int top = a.top;
      const bool nan = ms != ms || last != last;
      bool strict = nl == top, done = false;
      auto threshold = [&] {
        sh.lane_max[t] = tm;
        __syncthreads();
        int gt = 0, ge = 0;
        for (int i = 0; i < 256; ++i) {
          const float o = sh.lane_max[i];
          gt += o > tm;
          ge += o >= tm;
        }
        if (gt < top && ge >= top) sh.t0 = tm;
        __syncthreads();
        return sh.t0;
      };
      float thr = last;
      int n = 0;
      if (!nan) {
        if (!strict) thr = threshold();
        for (int attempt = 0; attempt < 2; ++attempt) {
          if (t == 0) sh.count = 0;
          __syncthreads();
          if (strict ? tm > thr : tm >= thr)
            each(x, seg, [&](float y, uint32_t i) {
              if (strict ? y > thr : y >= thr) {
                const int p = atomicAdd(&sh.count, 1);
                if (p < kCand) sh.cand[p] = key_of(y, i);
              }
            });
          __syncthreads();
          n = sh.count;
          __syncthreads();
          done = n <= kCand;
          if (done || !strict) break;
          // over kCand elements pass `last`, so more threads than the list is long do: their top-th maximum passes it too
          thr = threshold();
          strict = false;
        }
      }
      if (done) {
        rank_into(sh, at, nl, n, top);
        nl = min(top, nl + n);
      } else {
        // Too many equals, or a NaN: the largest key below the one before, `top` times.
        uint64_t below = ~0ull;
        int got = 0;
        for (; got < top; ++got) {
          uint64_t best = 0;
          if (t < nl && sh.list[at][t] < below) best = sh.list[at][t];
          each(x, seg, [&](float y, uint32_t i) {
            const uint64_t k = key_of(y, i);
            if (k < below && k > best) best = k;
          });
          best = wave_max_u64(best);
          if (lane == 0) sh.wave_key[got & 1][wave] = best;
          __syncthreads();
          const uint64_t* const k4 = sh.wave_key[got & 1];
          for (int i = 0; i < 4; ++i) best = k4[i] > best ? k4[i] : best;
          if (best == 0) break;
          if (t == 0) sh.list[at ^ 1][got] = best;
          below = best;
        }
        nl = got;
        __syncthreads();
      }
      at ^= 1;
      last = nl == top ? key_value(sh.list[at][top - 1]) : -__builtin_inff();
    }
    if (!(fabsf(ms) < __builtin_inff())) {  // only -inf, or an infinity or a NaN, which stays
      m = maximum(m, ms);
      continue;
    }
    if (ms > m) {
      if (m > -__builtin_inff()) {  // the sums to the new reference; what was the largest joins them
        const float delta = (m - ms) * kLog2e, f = __builtin_amdgcn_exp2f(delta);
        d = f > 0.0f ? f * fmaf(delta, r, d) : 0.0f;
        r *= f;
        if (t == 0 && f > 0.0f) {
          r += f;
          d = fmaf(f, delta, d);
        }
      }
      m = ms;
      if (wave == first_wave && lane == __ffsll(__ballot(tm == ms)) - 1) {  // one copy of it leaves
        bool gone = false;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool hit = !gone && value(x, v, e) == ms;
            if (hit) x[v][e >> 1] = e & 1 ? (x[v][e >> 1] & 0xffffu) | 0xff800000u : (x[v][e >> 1] & 0xffff0000u) | 0xff80u;
            gone |= hit;
          }
      }
    }
    if (!(fabsf(m) < __builtin_inff())) continue;
    // x log2(e) - c in one rounding, c = m log2(e) rounded; delta takes the sums to m itself
    const bool small = fabsf(m) < 1e30f;
    const float c = m * kLog2e, delta = fmaf(m, kLog2e, -c);
    float pr = 0.0f, pd = 0.0f;
    if (small) {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = fmaf(value(x, v, e), kLog2e, -c), p = __builtin_amdgcn_exp2f(z);
          pr += p;
          pd = fmaf(p, z, pd);
        }
    }
    if (!small || __any(pd != pd)) {  // an excluded element (0 times -inf), or magnitudes that the product would pass
      pr = pd = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = small ? fmaf(value(x, v, e), kLog2e, -c) : (value(x, v, e) - m) * kLog2e;
          const float p = __builtin_amdgcn_exp2f(z);
          pr += p;
          pd = fmaf(p, fmaxf(z, -3e38f), pd);
        }
    }
    const float f = small ? __builtin_amdgcn_exp2f(-delta) : 1.0f;
    d = fmaf(f, small ? fmaf(-delta, pr, pd) : pd, d);
    r = fmaf(f, pr, r);
  }
  const double wr = wave_sum((double)r), wd = wave_sum((double)d);
  if (lane == 0) {
    sh.sum[0][wave] = wr;
    sh.sum[1][wave] = wd;
  }
  __syncthreads();
  const double sr = sh.sum[0][0] + sh.sum[0][1] + sh.sum[0][2] + sh.sum[0][3];
  const double sd = sh.sum[1][0] + sh.sum[1][1] + sh.sum[1][2] + sh.sum[1][3];
  if (a.ranges == 1) {
    finish_row(a, row, m, sr, sd, sh.list[at]);
    return;
  }
  RangeStats* const stats = static_cast<RangeStats*>(a.scratch);
  uint64_t* const keys = reinterpret_cast<uint64_t*>(stats + (size_t)a.rows * a.ranges);
  if (t == 0) stats[blockIdx.x] = RangeStats{m, 0.0f, sr, sd};
  if (t < a.top) keys[(size_t)blockIdx.x * a.top + t] = t < nl ? sh.list[at][t] : 0;
}

// Joins a row's ranges (at most 256): a thread each for the sums, then the top
// list from the ranges' lists: those whose first key is among the `top` largest
// first keys hold all of it.
__global__ __launch_bounds__(256) void k_logprob_join(LogprobArgs a) {
  __shared__ Shared sh;
  __shared__ uint64_t heads[256];
  __shared__ uint64_t t0;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, row = blockIdx.x, top = a.top, n = a.ranges;
  const RangeStats* const stats = static_cast<const RangeStats*>(a.scratch) + (size_t)row * n;
  const uint64_t* const keys =
      reinterpret_cast<const uint64_t*>(static_cast<const RangeStats*>(a.scratch) + (size_t)a.rows * n) + (size_t)row * n * top;
  RangeStats s = {-__builtin_inff(), 0.0f, 0.0, 0.0};
  if (t < n) s = stats[t];
  float m = s.m;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) m = maximum(m, __shfl_xor(m, k));
  if (lane == 0) sh.wave_max[0][wave] = m;
  if (top) heads[t] = t < n ? keys[(size_t)t * top] : 0;
  if (t == 0) {
    sh.count = 0;
    t0 = 0;
  }
  __syncthreads();
  const float* const w = sh.wave_max[0];
  m = maximum(maximum(w[0], w[1]), maximum(w[2], w[3]));
  const int first_wave = w[0] == m ? 0 : w[1] == m ? 1 : w[2] == m ? 2 : 3;
  double r = 0.0, d = 0.0;
  if (fabsf(m) < __builtin_inff() && s.m > -__builtin_inff()) {
    const double delta = ((double)s.m - (double)m) * 1.4426950408889634074, f = exp2(delta);
    const bool owner = wave == first_wave && lane == __ffsll(__ballot(s.m == m)) - 1;
    r = s.r + (owner ? 0.0 : 1.0);
    d = f > 0.0 ? f * (s.d + delta * r) : 0.0;
    r *= f;
  }
  r = wave_sum(r);
  d = wave_sum(d);
  if (lane == 0) {
    sh.sum[0][wave] = r;
    sh.sum[1][wave] = d;
  }
  if (top) {
    if (n >= top && t < n) {
      int place = 0;
      for (int i = 0; i < n; ++i) place += heads[i] > heads[t];
      if (place == top - 1) t0 = heads[t];
    }
    __syncthreads();
    if (t < n && heads[t] >= t0) {
      for (int i = 0; i < top; ++i) {
        const uint64_t key = keys[(size_t)t * top + i];
        if (key < t0 || key == 0) break;
        sh.cand[atomicAdd(&sh.count, 1)] = key;  // at most top lists of top keys: kCand
      }
    }
    __syncthreads();
    rank_into(sh, 0, 0, sh.count, top);
  } else {
    __syncthreads();
  }
  finish_row(a, row, m, sh.sum[0][0] + sh.sum[0][1] + sh.sum[0][2] + sh.sum[0][3],
             sh.sum[1][0] + sh.sum[1][1] + sh.sum[1][2] + sh.sum[1][3], sh.list[1]);
}

// Ranges of a row and vectors of each.
int ranges_of(int rows, int vocab, int* per) {
  const int vectors = (vocab + 14) / 8;  // on the 16-byte grid, wherever the row starts
  int n = rows >= 1024 ? 1 : (1024 + rows - 1) / rows;
  n = std::min(std::min(n, 256), (vectors + 255) / 256);
  *per = (vectors + n - 1) / n;
  return (vectors + *per - 1) / *per;
}

}  // namespace

size_t logprob_scratch_bytes(int rows, int vocab, int top) {
  int per;
  const int n = ranges_of(rows, vocab, &per);
  return n == 1 ? 0 : (size_t)rows * n * (sizeof(RangeStats) + 8 * (size_t)top);
}

hipError_t launch_logprob(LogprobArgs a, hipStream_t s) {
  a.ranges = ranges_of(a.rows, a.vocab, &a.per);
  const dim3 grid((unsigned)a.rows * a.ranges);
  if (a.per >= 1024)
    k_logprob<4><<<grid, 256, 0, s>>>(a);
  else
    k_logprob<1><<<grid, 256, 0, s>>>(a);
  if (a.ranges > 1) k_logprob_join<<<a.rows, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace es
