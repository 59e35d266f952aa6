// verify.cu -- verification of drafted tokens against the model's
// distributions, from given uniform random numbers.
//
// riallm decodes greedily, one token per forward (src/model.rs:1223-1270).
// A drafted step runs the model once over the last token and n drafted ones;
// position i of its n + 1 rows of logits gives p_i, the distribution of the
// token after it. Draft x_i, drawn from q_i, is accepted when
// u_i q_i(x_i) < p_i(x_i). After the accepted drafts one more token is taken
// by inverse CDF: from max(0, p_i - q_i) where draft i was rejected, from
// p_i where there was none. The tokens are then distributed as if each had
// been drawn from p_i alone (Leviathan, Kalman and Matias, 2023).
//
// p_i = softmax(logits_i / temperature) in 64 bits: a sample falls between
// two borders of a cumulative sum over the vocabulary, and float32 sums over
// 1e5 tokens would move those borders by more than a rare token's share.
// Temperature 0 (and a row whose softmax is undefined: a NaN, +inf, or -inf
// throughout) puts all of p_i on the first maximum.
//
// Three or four launches:
//   stats_kernel : every row's maximum and sum of exponentials in float32, a
//                  slice of a row per CTA; bound by the exponential unit and
//                  by reading the logits once;
//   judge        : finds a sequence's first rejection (a comparison that
//                  float32 sums leave within 1e-4 of equality is made again
//                  with 64-bit ones), in judge_kernel or, for small calls, in
//                  every CTA of weigh_kernel;
//   weigh_kernel : goes over the one row that the token comes from, in 64
//                  bits, a chunk of the vocabulary per CTA; bound by its
//                  instructions, 30 a token at 67 % of the issue slots;
//   pick_kernel  : the chunks' weights after the draft's distribution is taken
//                  off; a sequence's last CTA finds the token. 36 instructions
//                  a token or more, 49 % of the slots: bound by the latency of
//                  its start (a sum over all parts) and of 64-bit arithmetic
//                  as well.
// 128 sequences of 5 drafts over 128001 tokens (bf16 logits and float32 draft
// probabilities, 262 MB): 100 us, 2.6 TB/s, of which the four take about 35,
// 7, 22 and 37 %; one sequence: 16 us with the host's part. A cluster of CTAs
// per sequence in place of the last three takes 218 us (8 CTAs) or 352 (16):
// its fixed cost, 10 us, comes 8 times over.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBatch = 8;  // loads of an array that a thread has in flight
constexpr int kStep = 4;   // tokens of a thread where the last part is searched
constexpr int kChunk = kThreads * kStep * kWarps;  // largest chunk: its parts are searched in one go
constexpr int kTable = 256;
static_assert(kTable == kThreads, "a thread fills an entry");

using rl::ex2;

__device__ __forceinline__ float load_logit(const void* x, bool bf16, int64_t i) {
  return bf16 ? __uint_as_float((uint32_t)static_cast<const uint16_t*>(x)[i] << 16) : static_cast<const float*>(x)[i];
}

struct VerifyArgs {
  const void* logits;
  int bf16;
  const int* drafts;
  const float* probs;
  const float* temperature;
  const float* accept_u;
  const float* sample_u;
  int n, V;
  int* tokens;
  int* accepted;
};

struct Stat;
// What the first rejection of a sequence comes to.
struct Verdict {
  int acc;    // accepted drafts: the token comes from row acc
  int draft;  // the rejected draft, or -1
  float m;    // the row's maximum
  int done;   // the row's p lies on one token, which has been written
};
// The workspace: statistics of the rows' slices; a table of powers and per
// sequence 256 log2(e) / temperature (see Exp64); per sequence and part (an
// eighth of a chunk, a warp's share) the sum of exponentials and of weights;
// per sequence the verdict and a count of finished chunks.
struct Space {
  Stat* stats;
  double* table;
  double* scale;
  double* z;
  double* w;
  Verdict* verdict;
  unsigned* done;
  int slices, slice, chunks, part;
};

// Of a slice of a row: its maximum (NaN left out); the sum of
// 2^((x - max) c), NaN where the softmax is undefined; at temperature 0 the
// lowest index that holds the maximum, and no sum.
struct Stat {
  float m, s;
  int top, pad;
};
// log2(e) / temperature, kept where 0 * c and inf * c are harmless: from the
// smallest number (of an infinite temperature) to the largest. That one is
// not the quotient of temperatures below kTiny: what the statistics say of
// their sums is not used.
constexpr float kTiny = 4.5e-39f;  // above log2(e) / FLT_MAX
__device__ __forceinline__ float scale_of(float t) {
  return t > 0.f ? fminf(fmaxf(1.4426950408889634f / t, 1.4e-45f), 3.402823466e38f) : 1.f;
}

// A thread's part of a slice. Its sum is relative to `base`, at most 60
// octaves below the maximum, so that a new maximum seldom costs more than
// being noted.
struct Part {
  float m = -INFINITY, base = 0.f, s0 = 0.f, s1 = 0.f;
  int top = 0x7fffffff;
  bool begun = false;
  template <int N>
  __device__ __forceinline__ void sum(float (&x)[N], float c) {
    float mx = x[0];
#pragma unroll
    for (int e = 1; e + 1 < N; e += 2) mx = rl::max3(mx, x[e], x[e + 1]);
    m = N > 1 ? rl::max3(m, mx, x[N - 1]) : fmaxf(m, mx);
    if ((m - base) * c > 60.f || !begun) {  // -inf and NaN leave base as it is
      // Sums that have not begun are 0, or NaN, relative to whatever base: the
      // power of a first maximum far below 0 is infinite, and 0 times it NaN.
      const float b = m > -INFINITY ? m : 0.f, f = begun ? ex2((base - b) * c) : 1.f;
      begun = m > -INFINITY;
      s0 *= f;
      s1 *= f;
      base = b;
    }
    if (N == 1) {
      s0 += ex2((x[0] - base) * c);
    } else {
#pragma unroll
      for (int e = 0; e + 1 < N; e += 2) {
        rl::add_f32x2(x[e], x[e + 1], -base, -base);
        rl::mul_f32x2(x[e], x[e + 1], c, c);
        rl::add_f32x2(s0, s1, ex2(x[e]), ex2(x[e + 1]));
      }
    }
  }
  template <int N>
  __device__ __forceinline__ void first(const float (&x)[N], int j) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (x[e] > m || (x[e] == m && j + e < top)) {
        m = x[e];
        top = j + e;
      }
  }
};

// 2^(i / 256) for the table of Exp64: the upper word is i << 12 below.
__device__ __forceinline__ double table_entry(int i) {
  const double p = exp2((double)i / kTable);
  return __hiloint2double(__double2hiint(p) - (i << 12), __double2loint(p));
}

// A CTA per slice of a row, row by row. 16 bytes a load where the row's place
// allows, four loads of a thread in flight and four at work.
template <bool kBf16>
__global__ void __launch_bounds__(kThreads)
    stats_kernel(const VerifyArgs a, const Space ws) {
  constexpr int N = kBf16 ? 8 : 4;
  __shared__ float sh_m[kWarps], sh_s[kWarps];
  __shared__ int sh_top[kWarps];
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const int row = blockIdx.x / ws.slices, slice = ws.slice;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = min(a.V, (int)(blockIdx.x - row * ws.slices) * slice), end = min(a.V, begin + slice);
  const float temp = a.temperature[row / (a.n + 1)], c = scale_of(temp);
  const bool greedy = !(temp > 0.f);
  if (blockIdx.x == 0) ws.table[tid] = table_entry(tid);
  const int64_t base = (int64_t)row * a.V;
  // Whole vectors of the slice: [v0, v1) as row indices, the rest one by one.
  const int skew = (int)((reinterpret_cast<uintptr_t>(a.logits) / (kBf16 ? 2 : 4) + base + begin) & (N - 1));
  const int v0 = min(end, begin + (skew ? N - skew : 0)), v1 = v0 + (end - v0) / N * N;
  const uint4* vec = reinterpret_cast<const uint4*>(static_cast<const char*>(a.logits) + (base + v0) * (kBf16 ? 2 : 4));
  const int nv = (v1 - v0) / N;
  Part part;
  uint4 next[4];
  auto fetch = [&](int i) {
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (i + y * kThreads < nv) next[y] = __ldcs(vec + i + y * kThreads);
  };
  auto vectors = [&](auto&& use) {
    fetch(tid);
    for (int i = tid; i < nv; i += 4 * kThreads) {
      uint4 w[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) w[y] = next[y];
      fetch(i + 4 * kThreads);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        if (i + y * kThreads >= nv) break;
        float x[N];
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&w[y]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (kBf16) {
            x[(2 * e) % N] = __uint_as_float(u[e] << 16);
            x[(2 * e + 1) % N] = __uint_as_float(u[e] & 0xffff0000u);
          } else {
            x[e] = __uint_as_float(u[e]);
          }
        }
        use(x, v0 + (i + y * kThreads) * N);
      }
    }
    const int ends = (v0 - begin) + (end - v1);
    for (int i = tid; i < ends; i += kThreads) {
      const int j = i < v0 - begin ? begin + i : v1 + (i - (v0 - begin));
      float x[1] = {load_logit(a.logits, kBf16, base + j)};
      use(x, j);
    }
  };
  if (greedy)
    vectors([&](auto& x, int j) { part.first(x, j); });
  else
    vectors([&](auto& x, int) { part.sum(x, c); });
  float m = part.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) sh_m[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sh_m[w]);
  const float ref = m == -INFINITY ? 0.f : m;
  // What has not begun holds 0, or NaN, and so it stays.
  float s = (part.s0 + part.s1) * (part.begun ? ex2((part.base - ref) * c) : 1.f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int top = __reduce_min_sync(0xffffffffu, part.m == m ? part.top : 0x7fffffff);
  if (lane == 0) {
    sh_s[warp] = s;
    sh_top[warp] = top;
  }
  __syncthreads();
  if (tid == 0) {
    Stat st{m, 0.f, 0x7fffffff, 0};
    for (int w = 0; w < kWarps; ++w) {
      st.s += sh_s[w];
      st.top = min(st.top, sh_top[w]);
    }
    ws.stats[blockIdx.x] = st;
    if (row * ws.slices == (int)blockIdx.x && row % (a.n + 1) == 0) {
      ws.done[row / (a.n + 1)] = 0;
      ws.scale[row / (a.n + 1)] = kTable * 1.4426950408889634 / (double)temp;
    }
  }
}

// ------------------------------------------------------------ 64 bits
//
// e^((l - m) / t): 2^(i / 256) from a table and the rest, at most 1 / 512
// octave, by the Taylor series to the 3rd power (the 4th, 1.4e-13 of the value
// at most, is the error). The table's powers lie in their upper words below
// their exponents by i << 12, so that adding i << 12 gives 2^(i / 256) for
// every i.
struct Exp64 {
  const double* table;  // in shared memory
  double k, m;          // 256 log2(e) / t
  float least;          // logits below it count as 0: 1000 octaves and more down
  __device__ __forceinline__ Exp64(const double* table_, float m_, double k_, float t)
      : table(table_), k(k_), m((double)m_) {
    const double x = m - 693.0 * (double)t;
    least = fmaxf((float)x, -3.402823466e38f);
    if ((double)least < x) least = nextafterf(least, m_);
  }
  // The value, where `some`; it is 0 otherwise.
  __device__ __forceinline__ double operator()(float l, bool& some) const {
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52
    constexpr double a = 0.6931471805599453 / kTable;
    const double d = (double)l - m;  // 0 at the maximum, whatever the temperature
    const double xf = fma(d, k, kMagic);
    const int i = __double2loint(xf);
    const double r = fma(d, k, -(xf - kMagic));
    double p = fma(r, a * a * a / 6.0, a * a / 2.0);
    p = fma(r, p, a) * r;
    const double e = table[i & (kTable - 1)], power = __hiloint2double(__double2hiint(e) + (i << 12), __double2loint(e));
    some = l >= least;
    return fma(power, p, power);
  }
  __device__ __forceinline__ double operator()(float l) const {
    bool some;
    const double p = (*this)(l, some);
    return some ? p : 0.0;
  }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ double warp_scan(double v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double u = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += u;
  }
  return v;
}

// What a row's slices say together: its sum of exponentials relative to m and
// its maximum; where all of p lies on one token, that (otherwise -1). By a
// warp, a slice a lane.
struct Row {
  double z;
  float m;
  int top;
};
constexpr int kUndefined = 0x7fffffff;  // all on the first maximum, not known yet
__device__ __forceinline__ Row row_of(const Stat* s, int slices, float t) {
  const int lane = threadIdx.x & 31;
  const float c = scale_of(t);
  Stat st{-INFINITY, 0.f, 0x7fffffff, 0};
  double z = 0.0;
#pragma unroll 4
  for (int i = lane; i < slices; i += 32) {
    const uint4 u = __ldcg(reinterpret_cast<const uint4*>(s + i));
    const float m = __uint_as_float(u.x), mn = fmaxf(st.m, m), base = mn == -INFINITY ? 0.f : mn;
    st.top = m > st.m ? (int)u.z : m < st.m ? st.top : min(st.top, (int)u.z);
    z = z * (double)(st.m == mn ? 1.f : ex2((st.m - base) * c)) +
        (double)__uint_as_float(u.y) * (double)(m == mn ? 1.f : ex2((m - base) * c));
    st.m = mn;
  }
  float M = st.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  int top = __reduce_min_sync(0xffffffffu, st.m == M ? st.top : 0x7fffffff);
  const float base = M == -INFINITY ? 0.f : M;
  z = warp_sum(z * (double)(st.m == M ? 1.f : ex2((st.m - base) * c)));
  if (t > 0.f) top = !(fabs(z) <= 1.7e308) || isinf(M) ? kUndefined : -1;
  else if (top == 0x7fffffff) top = 0;  // nothing but NaN
  return Row{z, M, top};
}

__device__ __forceinline__ double block_sum(double v, double* part) {  // of all threads, in warp order
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) v += part[w];
  return v;
}
// Sum of v[0 .. n), the same in every thread and every CTA.
__device__ __forceinline__ double sum_of(const double* v, int n, double* part) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) s += __ldcg(v + i);
  return block_sum(s, part);
}
// One row of logits.
template <bool kBf16>
struct Logits {
  const void* p;
  __device__ __forceinline__ Logits(const VerifyArgs& a, int64_t row)
      : p(static_cast<const char*>(a.logits) + row * a.V * (kBf16 ? 2 : 4)) {}
  __device__ __forceinline__ float operator()(int j) const { return load_logit(p, kBf16, j); }
};
// Calls use(j, logit j, draft probability j) for j = j0, j0 + step, ... below
// j1, kBatch loads of each array at a time (what is past j1: -inf and 0);
// ready() once, when the first of them are on their way.
template <bool kQ, typename L, typename R, typename F>
__device__ __forceinline__ void over(const L& logit, const float* q, int j0, int j1, int step, R&& ready, F&& use) {
  float l[kBatch], x[kBatch];
  auto fetch = [&](int j) {
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      const bool in = e * step < j1 - j;
      l[e] = in ? logit(j + e * step) : -INFINITY;
      x[e] = kQ && in ? __ldg(q + j + e * step) : 0.f;
    }
  };
  fetch(j0);
  ready();
  for (int j = j0; j < j1; j += kBatch * step) {
    if (j > j0) fetch(j);
#pragma unroll
    for (int e = 0; e < kBatch; ++e) use(l[e], x[e]);
  }
}

// What the CTA of sequence b finds, from the slices' statistics: how many of
// its drafts hold, and where its next token comes from. `writes`: this CTA is
// to write what is known of the result.
template <bool kBf16>
__device__ __forceinline__ Verdict judge(const VerifyArgs& a, const Space& ws, const double* table, int b, bool writes) {
  __shared__ double part[kWarps];
  __shared__ unsigned verdict[kWarps], close[kWarps];  // bits: rejected; too close to say
  __shared__ Row rows[256];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V, n = a.n;
  const float t = a.temperature[b];
  const double scale = ws.scale[b];
  const int64_t row0 = (int64_t)b * (n + 1);
  auto draft = [&](int i) {
    const int x = i < n ? a.drafts[(int64_t)b * n + i] : -1;
    return (unsigned)x < (unsigned)V ? x : -1;
  };
  for (int i = warp; i <= n; i += kWarps) {
    const Row r = row_of(ws.stats + (row0 + i) * ws.slices, ws.slices, t);
    if (lane == 0) rows[i] = r;
  }
  __syncthreads();
  if (t > 0.f) {
    for (int i = 0; i <= n; ++i) {  // a row whose softmax is undefined: look for its first maximum
      if (rows[i].top != kUndefined) continue;
      const float m = rows[i].m;
      const Logits<kBf16> logit(a, row0 + i);
      int at = kUndefined;
      for (int j = tid; j < V && at == kUndefined; j += kThreads)
        if (logit(j) == m) at = j;
      __syncthreads();  // rows[i] has been read
      if (tid == 0) rows[i].top = V;
      __syncthreads();
      at = __reduce_min_sync(0xffffffffu, at);
      if (lane == 0) atomicMin(&rows[i].top, at);
      __syncthreads();
      if (tid == 0 && rows[i].top == V) rows[i].top = 0;  // nothing but NaN
      __syncthreads();
    }
  }

  // A draft a thread (n is below 256).
  bool no = false, near = false;
  if (tid <= n) {
    const int x = draft(tid);
    no = true;
    if (x >= 0) {
      const Row r = rows[tid];
      const double q = a.probs ? (double)a.probs[((int64_t)b * n + tid) * V + x] : 1.0;
      const double lhs = (double)a.accept_u[(int64_t)b * n + tid] * q;
      if (r.top >= 0) {
        no = !(lhs < (x == r.top ? 1.0 : 0.0));
      } else {
        const double p = Exp64(table, r.m, scale, t)(Logits<kBf16>(a, row0 + tid)(x));
        near = p > 0.0 && (fabs(lhs * r.z - p) <= 1e-4 * p || t < kTiny);
        no = !(lhs * r.z < p);
      }
    }
  }
  const unsigned vno = __ballot_sync(0xffffffffu, no), vnear = __ballot_sync(0xffffffffu, near);
  if (lane == 0) {
    verdict[warp] = vno;
    close[warp] = vnear;
  }
  __syncthreads();
  int acc = 0;
  for (;; ++acc) {  // at most to n: there is no draft n
    const unsigned bit = 1u << (acc & 31);
    bool rejected = verdict[acc >> 5] & bit;
    if (close[acc >> 5] & bit) {
      // The whole CTA sums this row in 64 bits.
      const int x = draft(acc);
      const Exp64 ex(table, rows[acc].m, scale, t);
      const Logits<kBf16> logit(a, row0 + acc);
      double z = 0.0;
      over<false>(logit, nullptr, tid, V, kThreads, [] {}, [&](float l, float) { z += ex(l); });
      z = block_sum(z, part);
      const double q = a.probs ? (double)a.probs[((int64_t)b * n + acc) * V + x] : 1.0;
      rejected = !((double)a.accept_u[(int64_t)b * n + acc] * q * z < ex(logit(x)));
    }
    if (rejected) break;
  }
  const int top = rows[acc].top, x = draft(acc);
  // All of p on one token: so is what a rejected draft leaves of it.
  const Verdict v{acc, x, rows[acc].m, top >= 0};
  if (writes) {
    for (int i = tid; i <= n; i += kThreads)
      if (i != acc || top >= 0)
        a.tokens[row0 + i] = i < acc ? a.drafts[(int64_t)b * n + i] : i == acc ? top : -1;
    if (tid == 0) {
      a.accepted[b] = acc;
      ws.verdict[b] = v;
    }
  }
  return v;
}

// A CTA per sequence.
template <bool kBf16>
__global__ void __launch_bounds__(kThreads) judge_kernel(const VerifyArgs a, const Space ws) {
  __shared__ double table[kTable];
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  table[threadIdx.x] = ws.table[threadIdx.x];
  judge<kBf16>(a, ws, table, blockIdx.x, true);
}

// CTA (sequence, chunk): the sums of exponentials of the chunk's parts in the
// row that the token comes from. kJudge: every CTA of a sequence finds that
// row itself, and the first writes it down; otherwise it is known.
template <bool kBf16, bool kJudge>
__global__ void __launch_bounds__(kThreads) weigh_kernel(const VerifyArgs a, const Space ws) {
  __shared__ double table[kTable];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / ws.chunks, chunk = blockIdx.x - b * ws.chunks, V = a.V, n = a.n;
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const double entry = ws.table[tid];
  if (kJudge) table[tid] = entry;
  const Verdict v = kJudge ? judge<kBf16>(a, ws, table, b, chunk == 0) : ws.verdict[b];
  if (v.done) return;

  // A draft that was chosen outright (q = 1 there) leaves all but its own
  // token.
  const int drop = a.probs ? -1 : v.draft, p = chunk * kWarps + warp, j0 = min(V, p * ws.part), j1 = min(V, j0 + ws.part);
  const Exp64 ex(table, v.m, ws.scale[b], a.temperature[b]);
  double sum = 0.0;
  const Logits<kBf16> logit(a, (int64_t)b * (n + 1) + v.acc);
  auto add = [&](float l, float) {
    bool some;
    const double w = ex(l, some);
    if (some) sum += w;
  };
  const int cut = min(max(drop, j0), j1);  // around the dropped token, if it is here
  auto ready = [&] {
    if (kJudge) return;
    table[tid] = entry;
    __syncthreads();
  };
  over<false>(logit, nullptr, (cut == drop ? cut + 1 : cut) + lane, j1, 32, ready, add);
  over<false>(logit, nullptr, j0 + lane, cut, 32, [] {}, add);
  sum = warp_sum(sum);
  if (lane == 0) ws.z[(int64_t)b * ws.chunks * kWarps + p] = sum;
}

// CTA (sequence, chunk): what the draft's distribution leaves of the chunk's
// weights, where there is one to take off; the last CTA of a sequence to be
// done (its only one otherwise) takes the token.
template <bool kBf16>
__global__ void __launch_bounds__(kThreads) pick_kernel(const VerifyArgs a, const Space ws) {
  __shared__ double table[kTable], part[kWarps];
  __shared__ bool is_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / ws.chunks, chunk = blockIdx.x - b * ws.chunks, V = a.V, n = a.n;
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const Verdict v = ws.verdict[b];
  const double entry = ws.table[tid];
  if (v.done) return;
  const bool residual = v.draft >= 0 && a.probs;
  if (!residual && chunk != 0) return;
  const int parts = ws.chunks * kWarps;
  const int64_t row = (int64_t)b * (n + 1) + v.acc, first = (int64_t)b * parts;
  const float* q = residual ? a.probs + ((int64_t)b * n + v.acc) * V : nullptr;
  const Logits<kBf16> logit(a, row);
  const Exp64 ex(table, v.m, ws.scale[b], a.temperature[b]);
  double z;
  auto ready = [&] {
    table[tid] = entry;
    z = sum_of(ws.z + first, parts, part);  // waits for the table, too
  };
  const double* w = ws.z + first;
  bool taken_off = residual;  // weights are max(0, e - q z), or e
  auto weight = [&](float l, float x) {
    const double e = ex(l);
    return taken_off ? fma(-(double)x, z, e) : e;
  };
  double total;
  if (residual) {
    const int p = chunk * kWarps + warp, j0 = min(V, p * ws.part), j1 = min(V, j0 + ws.part);
    double sum = 0.0;
    over<true>(logit, q, j0 + lane, j1, 32, ready, [&](float l, float x) {
      const double y = weight(l, x);
      if (y > 0.0) sum += y;
    });
    sum = warp_sum(sum);
    if (lane == 0) ws.w[first + p] = sum;
    __threadfence();
    __syncthreads();
    if (tid == 0) is_last = atomicAdd(&ws.done[b], 1u) == (unsigned)ws.chunks - 1;
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    const double left = sum_of(ws.w + first, parts, part);
    if (left > 0.0) {
      w = ws.w + first;
      total = left;
    } else {
      total = z;
      taken_off = false;  // p == q: nothing is left over; p itself
    }
  } else {
    ready();
    total = z;
  }

  const int drop = a.probs ? -1 : v.draft;
  if (!(total > 0.0)) {  // all of p on the draft that was chosen outright
    if (tid == 0) a.tokens[row] = max(drop, 0);
    return;
  }
  // The first token whose cumulative weight exceeds the target lies in the
  // first part whose end does.
  const double target = (double)a.sample_u[b] * total;
  // Of a range of parts a lane takes a 32nd; the range becomes that lane's.
  int at = 0, count = parts;
  bool beyond = true;  // (false: no part's end does; it becomes the last with weight)
  double start = 0.0;
  do {
    const int each = (count + 31) / 32, i0 = lane * each, i1 = min(count, i0 + each);
    double y = 0.0;
#pragma unroll 4
    for (int i = i0; i < i1; ++i) y += __ldcg(w + at + i);
    const double upto = warp_scan(y);
    const unsigned with = __ballot_sync(0xffffffffu, y > 0.0);
    const unsigned past = __ballot_sync(0xffffffffu, beyond && start + upto > target) & with;
    beyond = past != 0;
    const int i = beyond ? __ffs(past) - 1 : max(0, 31 - __clz(with));
    const double before = __shfl_sync(0xffffffffu, upto, max(i - 1, 0));
    if (i > 0) start += before;
    at += i * each;
    count = min(each, count - i * each);
  } while (count > 1);
  // Within the part, of at most 1024 tokens, 128 a warp. No token is beyond
  // the target where the number is 1 or more, or none (NaN), or rounds up to
  // the total: then the last with weight.
  __shared__ double sums[kWarps];
  const int j0 = at * ws.part + warp * kStep * 32 + lane, j1 = min(V, (at + 1) * ws.part);
  double y[kStep], sum = 0.0;
  {
    float l[kStep], x[kStep];
#pragma unroll
    for (int e = 0; e < kStep; ++e) {
      const int i = j0 + e * 32;
      l[e] = i < j1 && i != drop ? logit(i) : -INFINITY;
      x[e] = i < j1 && taken_off ? q[i] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < kStep; ++e) {
      y[e] = fmax(0.0, weight(l[e], x[e]));
      sum += y[e];
    }
  }
  sum = warp_sum(sum);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  int in = -1, last = 0;  // the warp whose tokens reach the target, else the last with weight
  for (int i = 0; i < kWarps && in < 0; ++i) {
    if (sums[i] > 0.0) last = i;
    if (beyond && sums[i] > 0.0 && start + sums[i] > target) in = i;
    else start += sums[i];
  }
  if (warp != (in < 0 ? last : in)) return;
  int hit = -1;
  last = 0;
#pragma unroll
  for (int e = 0; e < kStep; ++e) {
    const double upto = warp_scan(y[e]);
    const unsigned with = __ballot_sync(0xffffffffu, y[e] > 0.0);
    const unsigned beyond = __ballot_sync(0xffffffffu, start + upto > target) & with;
    if (hit < 0 && in >= 0 && beyond) hit = e * 32 + __ffs(beyond) - 1;
    if (with) last = e * 32 + 31 - __clz(with);
    start += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) a.tokens[row] = j0 + (hit >= 0 ? hit : last);
}

// Slices of a row (1024 to 65536 tokens) and chunks of the row that a token
// comes from (1024 to 8192): as many as fill the GPU.
Space space_of(int num_sms, int B, int n, int V, void* base, uint64_t* bytes) {
  Space s;
  const int64_t rows = (int64_t)B * (n + 1);
  const int most = (V + 1023) / 1024;
  auto pick = [&](int64_t ctas, int64_t each, int largest) {
    const int64_t least = (V + largest - 1) / largest;
    return (int)std::max<int64_t>(least, std::min<int64_t>((ctas + each - 1) / each, most));
  };
  s.slices = pick(8ll * num_sms, rows, 65536);
  s.slice = (V + s.slices - 1) / s.slices;
  s.chunks = pick(4ll * num_sms, B, kChunk);
  s.part = (V + s.chunks * kWarps - 1) / (s.chunks * kWarps);
  uint64_t at = 0;
  auto take = [&](uint64_t size) {
    char* p = static_cast<char*>(base) + at;
    at += (size + 15) / 16 * 16;
    return p;
  };
  const uint64_t parts = (uint64_t)B * s.chunks * kWarps;
  s.stats = reinterpret_cast<Stat*>(take((uint64_t)rows * s.slices * sizeof(Stat)));
  s.table = reinterpret_cast<double*>(take(kTable * 8));
  s.scale = reinterpret_cast<double*>(take((uint64_t)B * 8));
  s.z = reinterpret_cast<double*>(take(parts * 8));
  s.w = reinterpret_cast<double*>(take(parts * 8));
  s.verdict = reinterpret_cast<Verdict*>(take((uint64_t)B * sizeof(Verdict)));
  s.done = reinterpret_cast<unsigned*>(take((uint64_t)B * 4));
  *bytes = at;
  return s;
}

template <bool kBf16>
int32_t launch_verify(riallm_ctx* ctx, const char* what, const VerifyArgs& a, int B, const Space& ws, cudaStream_t st) {
  const unsigned rows = (unsigned)B * (a.n + 1);
  if (int r = rl::launched(ctx, what, rl::launch_pdl(stats_kernel<kBf16>, dim3(rows * ws.slices), dim3(kThreads), 0, st, a, ws)))
    return r;
  // A launch costs 2 us (128 sequences, 32000 tokens, 640 CTAs: 47 us without
  // it, 51 with it); where CTAs come in more than one wave, 5 an SM, their own
  // verdicts cost more (128001 tokens, 2048 CTAs: 115 and 109 us).
  const bool apart = B * ws.chunks > 5 * ctx->num_sms;
  if (apart)
    if (int r = rl::launched(ctx, what, rl::launch_pdl(judge_kernel<kBf16>, dim3(B), dim3(kThreads), 0, st, a, ws)))
      return r;
  const auto weigh = apart ? weigh_kernel<kBf16, false> : weigh_kernel<kBf16, true>;
  if (int r = rl::launched(ctx, what, rl::launch_pdl(weigh, dim3(B * ws.chunks), dim3(kThreads), 0, st, a, ws)))
    return r;
  return rl::launched(ctx, what, rl::launch_pdl(pick_kernel<kBf16>, dim3(B * ws.chunks), dim3(kThreads), 0, st, a, ws));
}

}  // namespace

extern "C" {

uint64_t riallm_cuda_verify_draft_workspace(const riallm_ctx* ctx, int32_t B, int32_t n, int32_t V) {
  if (!ctx || B <= 0 || n < 0 || V <= 0) return 0;
  uint64_t bytes;
  space_of(ctx->num_sms, B, n, V, nullptr, &bytes);
  return bytes;
}

int32_t riallm_cuda_verify_draft(riallm_ctx* ctx, const riallm_verify_draft_args* args, void* workspace,
                                 uint64_t workspace_bytes, void* stream) {
  const char* what = "verify_draft";
  if (!args) return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "NULL argument");
  const riallm_verify_draft_args& x = *args;
  const int32_t B = x.B, n = x.n, V = x.V;
  if (B < 0 || n < 0 || n > 255 || V <= 0 || V > (1 << 30))
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "bad dimensions (at most 255 drafted tokens)");
  if (x.logits_dtype != RIALLM_DTYPE_F32 && x.logits_dtype != RIALLM_DTYPE_BF16)
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "logits must be float32 or bf16");
  if ((int64_t)B * (n + 1) * ((V + 1023) / 1024) > INT32_MAX)
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "too many logits");
  if (ctx && B == 0) return RIALLM_OK;
  if (!ctx || !x.logits || !x.temperature || !x.sample_u || !x.tokens || !x.accepted ||
      (n > 0 && (!x.draft_tokens || !x.accept_u)))
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "NULL argument");
  if (reinterpret_cast<uintptr_t>(x.logits) & (x.logits_dtype == RIALLM_DTYPE_BF16 ? 1 : 3))
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "logits must be aligned to their type");
  uint64_t bytes;
  const Space ws = space_of(ctx->num_sms, B, n, V, workspace, &bytes);
  if (!workspace || workspace_bytes < bytes || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return rl::refuse(ctx, RIALLM_ERR_MEMORY, what, "workspace missing, too small or not 16-byte aligned");
  return rl::guarded(ctx, [&]() -> int32_t {
    const VerifyArgs a{x.logits,   x.logits_dtype == RIALLM_DTYPE_BF16, x.draft_tokens, x.draft_probs, x.temperature,
                       x.accept_u, x.sample_u, n, V, x.tokens, x.accepted};
    const cudaStream_t st = (cudaStream_t)stream;
    return a.bf16 ? launch_verify<true>(ctx, what, a, B, ws, st) : launch_verify<false>(ctx, what, a, B, ws, st);
  });
}

}  // extern "C"
