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
// Two launches:
//   stats_kernel  : every row's maximum, where it is, and its sum of
//                   exponentials in float32, a slice of a row per CTA; bound
//                   by reading the logits once.
//   sample_kernel : a cluster of 8 CTAs per sequence finds the first
//                   rejection (a comparison that float32 sums leave within
//                   1e-4 of equality is made again with 64-bit ones), then
//                   goes over the one row that the token comes from, in 64
//                   bits, an eighth of the vocabulary per CTA.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kCluster = 8, kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kBatch = 8;  // loads a lane has in flight

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

// Of a slice of a row: its maximum (NaN left out), the lowest index that
// holds it, and the sum of 2^((x - max) c), NaN where the softmax is undefined.
struct Stat {
  float m, s;
  int top, pad;
};
// log2(e) / temperature, kept where 0 * c and inf * c are harmless.
__device__ __forceinline__ float scale_of(float t) {
  return t > 0.f ? fminf(fmaxf(1.4426950408889634f / t, 1e-30f), 1e30f) : 1.f;
}

// Adds N values from index j on.
template <int N>
__device__ __forceinline__ void add_stat(Stat& st, float (&x)[N], int j, float c) {
  float mx = x[0];
#pragma unroll
  for (int e = 1; e + 1 < N; e += 2) mx = rl::max3(mx, x[e], x[e + 1]);
  if (N > 1) mx = fmaxf(mx, x[N - 1]);
  if (mx > st.m) {
    int at = 0;
#pragma unroll
    for (int e = N - 1; e >= 0; --e)
      if (x[e] == mx) at = e;
    st.s *= ex2((st.m - mx) * c);
    st.m = mx;
    st.top = j + at;
  }
  const float base = st.m == -INFINITY ? 0.f : st.m;
  if (N == 1) {
    st.s += ex2((x[0] - base) * c);
    return;
  }
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int e = 0; e + 1 < N; e += 2) {
    rl::add_f32x2(x[e], x[e + 1], -base, -base);
    rl::mul_f32x2(x[e], x[e + 1], c, c);
    rl::add_f32x2(s0, s1, ex2(x[e]), ex2(x[e + 1]));
  }
  st.s += s0 + s1;
}
// The two slices' statistics together; the lower index where they tie.
__device__ __forceinline__ void merge_stat(Stat& a, const Stat& b, float c) {
  const float m = fmaxf(a.m, b.m), base = m == -INFINITY ? 0.f : m;
  a.top = a.m > b.m ? a.top : b.m > a.m ? b.top : min(a.top, b.top);
  a.s = a.s * (a.m == m ? 1.f : ex2((a.m - base) * c)) + b.s * (b.m == m ? 1.f : ex2((b.m - base) * c));
  a.m = m;
}

// A CTA per slice of a row, row by row. 16 bytes a load where the row's place allows, four loads
// in flight a thread.
template <bool kBf16>
__global__ void __launch_bounds__(kThreads) stats_kernel(const VerifyArgs a, int slices, int slice, Stat* __restrict__ stats) {
  constexpr int N = kBf16 ? 8 : 4;
  __shared__ Stat sh[kThreads / 32];
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const int row = blockIdx.x / slices;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = min(a.V, (int)(blockIdx.x - row * slices) * slice), end = min(a.V, begin + slice);
  const float c = scale_of(a.temperature[row / (a.n + 1)]);
  const int64_t base = (int64_t)row * a.V;
  // Whole vectors of the slice: [v0, v1) as row indices, the rest one by one.
  const int skew = (int)((base + begin) & (N - 1));
  const int v0 = min(end, begin + (skew ? N - skew : 0)), v1 = v0 + (end - v0) / N * N;
  Stat st{-INFINITY, 0.f, 0x7fffffff, 0};
  const uint4* vec = reinterpret_cast<const uint4*>(static_cast<const char*>(a.logits) + (base + v0) * (kBf16 ? 2 : 4));
  const int nv = (v1 - v0) / N;
  uint4 next[4];
  auto fetch = [&](int i) {
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (i + y * kThreads < nv) next[y] = __ldcs(vec + i + y * kThreads);
  };
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
      add_stat<N>(st, x, v0 + (i + y * kThreads) * N, c);
    }
  }
  const int ends = (v0 - begin) + (end - v1);
  for (int i = tid; i < ends; i += kThreads) {
    const int j = i < v0 - begin ? begin + i : v1 + (i - (v0 - begin));
    float x[1] = {load_logit(a.logits, kBf16, base + j)};
    // One thread may see a later vector before an early single value: the
    // lower index counts where they tie.
    if (x[0] == st.m) st.top = min(st.top, j);
    add_stat<1>(st, x, j, c);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    b.top = __shfl_xor_sync(0xffffffffu, st.top, o);
    // Both partners add in the same order.
    if (lane & o) {
      merge_stat(b, st, c);
      st = b;
    } else {
      merge_stat(st, b, c);
    }
  }
  if (lane == 0) sh[warp] = st;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / 32; ++w) merge_stat(st, sh[w], c);
    st.pad = 0;
    stats[blockIdx.x] = st;
  }
}

// ------------------------------------------------------------ 64 bits
//
// e^((l - m) / t): 2^(k / 64) from a table and the rest, at most 1 / 128
// octave, by the Taylor series to the 4th power (error 4e-14).
struct Exp64 {
  const double* table;  // 2^(i / 64), i < 64, in shared memory
  double m, k64;        // 64 log2(e) / t
  __device__ __forceinline__ double operator()(float l) const {
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52
    constexpr double a = 0.010830424696249145;     // ln(2) / 64
    const double t = ((double)l - m) * k64;
    if (!(t > -64000.0)) return 0.0;  // below 2^-1000; -inf
    const double kf = t + kMagic;
    const int k = __double2loint(kf);
    const double r = t - (kf - kMagic);
    double p = fma(r, a * a * a * a / 24.0, a * a * a / 6.0);
    p = fma(r, p, a * a / 2.0);
    p = fma(r, p, a);
    p = fma(r, p, 1.0);
    p *= table[k & 63];
    return __hiloint2double(__double2hiint(p) + ((k >> 6) << 20), __double2loint(p));
  }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a row's slices say together: its sum of exponentials relative to m, its
// maximum and where it is. By a warp, a slice a lane.
struct Row {
  double z;
  float m;
  int top;  // negative where all of p lies on ~top
};
__device__ __forceinline__ Row row_of(const Stat* s, int slices, float t) {
  const int lane = threadIdx.x & 31;
  const float c = scale_of(t);
  Stat st{-INFINITY, 0.f, 0x7fffffff, 0};
  double z = 0.0;
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
  if (top == 0x7fffffff) top = 0;
  const bool greedy = !(t > 0.f) || !(fabs(z) <= 1.7e308) || isinf(M);
  return Row{z, M, greedy ? ~top : top};
}

// Cluster of kCluster CTAs per sequence.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kSampleThreads)
    sample_kernel(const VerifyArgs a, int slices, const Stat* __restrict__ stats) {
  __shared__ double table[64];
  __shared__ double part[kSampleWarps];
  __shared__ double shared_sum[2];  // this CTA's sum, read by the cluster
  __shared__ int shared_last;
  __shared__ unsigned verdict[kSampleWarps];  // bits: drafts not plainly accepted
  __shared__ unsigned close[kSampleWarps];
  __shared__ Row rows[256];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster.block_rank();
  const int b = blockIdx.x / kCluster, V = a.V, n = a.n;
  if (tid < 64) table[tid] = exp2((double)tid / 64.0);
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const float t = a.temperature[b];
  const double k64 = 64.0 * 1.4426950408889634 / (double)t;
  const Stat* st = stats + (int64_t)b * (n + 1) * slices;
  const int64_t row0 = (int64_t)b * (n + 1);
  auto draft = [&](int i) {
    const int x = i < n ? a.drafts[(int64_t)b * n + i] : -1;
    return (unsigned)x < (unsigned)V ? x : -1;
  };
  for (int i = warp; i <= n; i += kSampleWarps) {
    const Row r = row_of(st + (int64_t)i * slices, slices, t);
    if (lane == 0) rows[i] = r;
  }
  __syncthreads();

  // A draft a thread (n is below 256): accepted, rejected, or too close to say.
  bool no = false, near = false;
  if (tid <= n) {
    const int x = draft(tid);
    no = true;
    if (x >= 0) {
      const Row r = rows[tid];
      const double q = a.probs ? (double)a.probs[((int64_t)b * n + tid) * V + x] : 1.0;
      const double lhs = (double)a.accept_u[(int64_t)b * n + tid] * q;
      if (r.top < 0) {
        no = !(lhs < (x == ~r.top ? 1.0 : 0.0));
      } else {
        const double p = Exp64{table, (double)r.m, k64}(load_logit(a.logits, a.bf16, (row0 + tid) * V + x));
        near = p > 0.0 && fabs(lhs * r.z - p) <= 1e-4 * p;
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
  for (;; ++acc) {  // up to n: there is no draft n
    const unsigned bit = 1u << (acc & 31);
    bool rejected = verdict[acc >> 5] & bit;
    if (close[acc >> 5] & bit) {
      // The whole CTA sums this row in 64 bits.
      const int x = draft(acc);
      const Exp64 ex{table, (double)rows[acc].m, k64};
      double z = 0.0;
#pragma unroll 4
      for (int j = tid; j < V; j += kSampleThreads) z += ex(load_logit(a.logits, a.bf16, (row0 + acc) * V + j));
      z = warp_sum(z);
      __syncthreads();
      if (lane == 0) part[warp] = z;
      __syncthreads();
      z = 0.0;
      for (int w = 0; w < kSampleWarps; ++w) z += part[w];
      const double q = a.probs ? (double)a.probs[((int64_t)b * n + acc) * V + x] : 1.0;
      rejected = !((double)a.accept_u[(int64_t)b * n + acc] * q * z <
                   ex(load_logit(a.logits, a.bf16, (row0 + acc) * V + x)));
    }
    if (rejected) break;
  }

  // The token after them: weights z * max(0, p - q) or z * p of row acc. Each
  // CTA takes an eighth of the vocabulary, each warp a sixteenth of that.
  const bool greedy = rows[acc].top < 0;
  const int top = greedy ? ~rows[acc].top : rows[acc].top;
  const Exp64 ex{table, (double)rows[acc].m, k64};
  const int x = draft(acc);
  const int64_t base = (row0 + acc) * V;
  const float* q = x >= 0 && a.probs ? a.probs + ((int64_t)b * n + acc) * V : nullptr;
  const int per_cta = (V + kCluster - 1) / kCluster, c0 = min(V, rank * per_cta), c1 = min(V, c0 + per_cta);
  const int per_warp = (per_cta + kSampleWarps - 1) / kSampleWarps;
  const int j0 = min(c1, c0 + warp * per_warp), j1 = min(c1, j0 + per_warp);
  bool residual = x >= 0;
  double z = 1.0;
  if (residual && q && !greedy) {
    double s = 0.0;
    for (int j = j0 + lane; j < j1; j += 32 * kBatch) {
      float l[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e)
        l[e] = j + 32 * e < j1 ? load_logit(a.logits, a.bf16, base + j + 32 * e) : -INFINITY;
#pragma unroll
      for (int e = 0; e < kBatch; ++e) s += ex(l[e]);
    }
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) part[warp] = s;
    __syncthreads();
    if (tid == 0) {
      s = 0.0;
      for (int w = 0; w < kSampleWarps; ++w) s += part[w];
      shared_sum[1] = s;
    }
    cluster.sync();
    z = 0.0;
    for (int c = 0; c < kCluster; ++c) z += *cluster.map_shared_rank(&shared_sum[1], c);
  }
  auto weight = [&](int j, float l, float qj) {
    const double w = greedy ? (j == top ? 1.0 : 0.0) : ex(l);
    if (!residual) return w;
    return fmax(0.0, w - (q ? (double)qj * z : j == x ? w : 0.0));
  };
  double mine, before, total;
  for (;;) {
    mine = 0.0;
    int last = -1;
    for (int j = j0 + lane; j < j1; j += 32 * kBatch) {
      float l[kBatch], qj[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const bool in = j + 32 * e < j1;
        l[e] = in ? load_logit(a.logits, a.bf16, base + j + 32 * e) : 0.f;
        qj[e] = in && q ? q[j + 32 * e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        if (j + 32 * e >= j1) break;
        const double w = weight(j + 32 * e, l[e], qj[e]);
        mine += w;
        if (w > 0.0) last = j + 32 * e;
      }
    }
    mine = warp_sum(mine);
    last = __reduce_max_sync(0xffffffffu, last);
    __syncthreads();
    if (tid == 0) shared_last = -1;
    if (lane == 0) part[warp] = mine;
    __syncthreads();
    if (lane == 0) atomicMax(&shared_last, last);
    if (tid == 0) {
      double s = 0.0;
      for (int w = 0; w < kSampleWarps; ++w) s += part[w];
      shared_sum[0] = s;
    }
    cluster.sync();
    total = before = 0.0;
    for (int c = 0; c < kCluster; ++c) {
      const double s = *cluster.map_shared_rank(&shared_sum[0], c);
      if (c < rank) before += s;
      total += s;
    }
    if (total > 0.0 || !residual) break;
    residual = false;  // p == q: nothing is left over
    cluster.sync();    // every CTA has read the sums
  }
  // The first token whose cumulative weight exceeds the target lies in the
  // first part (CTA, then warp) whose end does.
  const double target = (double)a.sample_u[b] * total;
  bool owner = shared_sum[0] > 0.0 && before + shared_sum[0] > target;
  if (owner && rank > 0) {  // no earlier one
    double c = 0.0;
    for (int i = 0; i < rank; ++i) {
      const double s = *cluster.map_shared_rank(&shared_sum[0], i);
      c += s;
      if (s > 0.0 && c > target) owner = false;
    }
  }
  if (owner) {
    double c = before;
    int w0 = -1;
    double start = 0.0;
    for (int w = 0; w < kSampleWarps; ++w) {
      if (w0 < 0 && part[w] > 0.0 && (c + part[w] > target)) {
        w0 = w;
        start = c;
      }
      c += part[w];
    }
    if (w0 < 0)  // the parts' sums round below their total: the last with weight
      for (int w = 0; w < kSampleWarps; ++w)
        if (part[w] > 0.0) w0 = w;
    if (warp == w0) {
      int hit = 0x7fffffff, last = -1;
      float l = 0.f, qj = 0.f;
      auto fetch = [&](int j) {
        if (j < j1) {
          l = load_logit(a.logits, a.bf16, base + j);
          if (q) qj = q[j];
        }
      };
      fetch(j0 + lane);
      for (int j = j0; j < j1; j += 32) {
        const double w = j + lane < j1 ? weight(j + lane, l, qj) : 0.0;
        fetch(j + 32 + lane);
        double s = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += y;
        }
        const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && start + s > target);
        const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
        if (over) {
          hit = j + __ffs(over) - 1;
          break;
        }
        if (some) last = j + 31 - __clz(some);
        start += __shfl_sync(0xffffffffu, s, 31);
      }
      if (lane == 0) a.tokens[row0 + acc] = hit != 0x7fffffff ? hit : last;
    }
  }
  // A number of 1 or more, or none (NaN): the last token with weight.
  if (rank == 0 && !(total > target)) {
    int last = -1;
    for (int c = 0; c < kCluster; ++c) last = max(last, *cluster.map_shared_rank(&shared_last, c));
    if (tid == 0) a.tokens[row0 + acc] = last < 0 ? top : last;
  }
  if (rank == 0) {
    for (int i = tid; i <= n; i += kSampleThreads)
      if (i != acc) a.tokens[row0 + i] = i < acc ? a.drafts[(int64_t)b * n + i] : -1;
    if (tid == 0) a.accepted[b] = acc;
  }
  cluster.sync();  // no CTA leaves while another reads its sums
}

// Slices of a row: as many as fill the GPU, of 1024 to 65536 tokens.
int slices_of(int num_sms, int64_t rows, int V) {
  const int most = (V + 1023) / 1024, least = (V + 65535) / 65536;
  const int64_t want = (8ll * num_sms + rows - 1) / std::max<int64_t>(rows, 1);
  return (int)std::max<int64_t>(least, std::min<int64_t>(want, most));
}

}  // namespace

extern "C" {

uint64_t riallm_cuda_verify_draft_workspace(const riallm_ctx* ctx, int32_t B, int32_t n, int32_t V) {
  if (!ctx || B <= 0 || n < 0 || V <= 0) return 0;
  const int64_t rows = (int64_t)B * (n + 1);
  return (uint64_t)rows * slices_of(ctx->num_sms, rows, V) * sizeof(Stat);
}

int32_t riallm_cuda_verify_draft(riallm_ctx* ctx, const void* logits, int32_t logits_dtype, const int32_t* draft_tokens,
                                 const float* draft_probs, const float* temperature, const float* accept_u,
                                 const float* sample_u, int32_t B, int32_t n, int32_t V, int32_t* tokens,
                                 int32_t* accepted, void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* what = "verify_draft";
  if (B < 0 || n < 0 || n > 255 || V <= 0 || V > (1 << 30))
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "bad dimensions (at most 255 drafted tokens)");
  if (logits_dtype != RIALLM_DTYPE_F32 && logits_dtype != RIALLM_DTYPE_BF16)
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "logits must be float32 or bf16");
  if ((int64_t)B * (n + 1) * ((V + 1023) / 1024) > INT32_MAX)
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "too many logits");
  if (ctx && B == 0) return RIALLM_OK;
  if (!ctx || !logits || !temperature || !sample_u || !tokens || !accepted || (n > 0 && (!draft_tokens || !accept_u)))
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "NULL argument");
  if (reinterpret_cast<uintptr_t>(logits) & 15)
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "logits must be 16-byte aligned");
  const int64_t rows = (int64_t)B * (n + 1);
  const int slices = slices_of(ctx->num_sms, rows, V);
  if (!workspace || workspace_bytes < (uint64_t)rows * slices * sizeof(Stat) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15))
    return rl::refuse(ctx, RIALLM_ERR_MEMORY, what, "workspace missing, too small or not 16-byte aligned");
  return rl::guarded(ctx, [&]() -> int32_t {
    const VerifyArgs a{logits, logits_dtype == RIALLM_DTYPE_BF16, draft_tokens, draft_probs, temperature, accept_u,
                       sample_u, n, V, tokens, accepted};
    Stat* stats = static_cast<Stat*>(workspace);
    const int slice = (V + slices - 1) / slices;
    const cudaStream_t st = (cudaStream_t)stream;
    if (int s = rl::launched(ctx, what,
                             rl::launch_pdl(a.bf16 ? stats_kernel<true> : stats_kernel<false>,
                                            dim3((unsigned)rows * slices), dim3(kThreads), 0, st, a, slices, slice,
                                            stats)))
      return s;
    return rl::launched(ctx, what,
                        rl::launch_pdl(sample_kernel, dim3(B * kCluster), dim3(kSampleThreads), 0, st, a, slices,
                                       static_cast<const Stat*>(stats)));
  });
}

}  // extern "C"
