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
#include <cfloat>

#include "common.cuh"
#include "internal.h"

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float load_logit(const void* x, bool bf16, int64_t i) {
  return bf16 ? __uint_as_float((uint32_t)static_cast<const uint16_t*>(x)[i] << 16) : static_cast<const float*>(x)[i];
}

// One row's distribution: softmax with maximum m, denominator z and 1 / t,
// or all on `top`.
struct Dist {
  double m, z, t;
  int top;
  bool greedy;
  __device__ __forceinline__ double weight(float l, int j) const {  // z * p(j)
    if (greedy) return j == top ? 1.0 : 0.0;
    return l == -INFINITY ? 0.0 : exp(((double)l - m) / t);
  }
};

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T* sh, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < kThreads / 32; ++w) v = f(v, sh[w]);
  return v;
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

// CTA per sequence.
__global__ void __launch_bounds__(kThreads) verify_draft_kernel(VerifyArgs a) {
  __shared__ double sd[kThreads / 32];
  __shared__ long long sl[kThreads / 32];
  __shared__ double scan[kThreads];
  __shared__ int found;
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const int b = blockIdx.x, tid = threadIdx.x, V = a.V;
  const float temp = a.temperature[b];
  Dist ds;
  int64_t base = 0;
  int acc = 0, x = -1;
  for (;; ++acc) {
    base = ((int64_t)b * (a.n + 1) + acc) * V;
    // Maximum with the lowest index: order key = (value, -index).
    float m = -INFINITY;
    int top = 0x7fffffff;
    int nan = 0;
    for (int j = tid; j < V; j += kThreads) {
      const float l = load_logit(a.logits, a.bf16, base + j);
      nan |= l != l;
      if (l > m) m = l, top = j;
    }
    nan = __syncthreads_or(nan);
    const double bm = block_reduce((double)m, sd, [](double p, double q) { return p > q ? p : q; });
    long long at = (double)m == bm && top != 0x7fffffff ? top : 0x7fffffffffffffffll;
    at = block_reduce(at, sl, [](long long p, long long q) { return p < q ? p : q; });
    ds.m = bm;
    ds.t = temp;
    ds.top = at == 0x7fffffffffffffffll ? 0 : (int)at;
    ds.greedy = !(temp > 0.f) || nan || bm == INFINITY || bm == -INFINITY;
    double z = 0.0;
    for (int j = tid; j < V; j += kThreads) z += ds.weight(load_logit(a.logits, a.bf16, base + j), j);
    ds.z = block_reduce(z, sd, [](double p, double q) { return p + q; });
    x = acc < a.n ? a.drafts[(int64_t)b * a.n + acc] : -1;
    if ((unsigned)x >= (unsigned)V) x = -1;
    if (x < 0) break;  // no draft here
    const int64_t qrow = ((int64_t)b * a.n + acc) * V;
    const double qx = a.probs ? (double)a.probs[qrow + x] : 1.0;
    const double px = ds.weight(load_logit(a.logits, a.bf16, base + x), x);
    if (!((double)a.accept_u[(int64_t)b * a.n + acc] * qx * ds.z < px)) break;
  }
  // The sample: weights z * max(0, p - q) after a rejection, z * p otherwise.
  const float* qrow = x >= 0 && a.probs ? a.probs + ((int64_t)b * a.n + acc) * V : nullptr;
  const int per = (V + kThreads - 1) / kThreads;
  const int j0 = min(V, tid * per), j1 = min(V, j0 + per);
  double total = 0.0, mine = 0.0;
  bool residual = x >= 0;
  auto weight = [&](int j) {
    const double w = ds.weight(load_logit(a.logits, a.bf16, base + j), j);
    if (!residual) return w;
    return fmax(0.0, w - (qrow ? (double)qrow[j] * ds.z : j == x ? ds.z : 0.0));
  };
  for (;;) {
    mine = 0.0;
    for (int j = j0; j < j1; ++j) mine += weight(j);
    __syncthreads();
    scan[tid] = mine;
    __syncthreads();
    total = 0.0;
    for (int i = 0; i < kThreads; ++i) total += scan[i];
    if (total > 0.0 || !residual) break;
    residual = false;  // p == q: nothing is left over
  }
  double before = 0.0;
  for (int i = 0; i < tid; ++i) before += scan[i];
  const double target = (double)a.sample_u[b] * total;
  // The first token whose cumulative weight exceeds the target; the last one
  // with weight where rounding leaves none.
  if (tid == 0) found = 0x7fffffff;
  __syncthreads();
  double c = before;
  int hit = 0x7fffffff, last = -1;
  for (int j = j0; j < j1; ++j) {
    const double w = weight(j);
    if (w > 0.0) {
      c += w;
      last = j;
      if (c > target && hit == 0x7fffffff) hit = j;
    }
  }
  atomicMin(&found, hit);
  const long long lastpos = block_reduce((long long)last, sl, [](long long p, long long q) { return p > q ? p : q; });
  __syncthreads();
  for (int i = tid; i <= a.n; i += kThreads)
    a.tokens[(int64_t)b * (a.n + 1) + i] = i < acc   ? a.drafts[(int64_t)b * a.n + i]
                                           : i > acc ? -1
                                           : found != 0x7fffffff ? found
                                                                 : (int)(lastpos < 0 ? ds.top : lastpos);
  if (tid == 0) a.accepted[b] = acc;
}

}  // namespace

extern "C" {

uint64_t riallm_cuda_verify_draft_workspace(const riallm_ctx* ctx, int32_t B, int32_t n, int32_t V) {
  (void)ctx, (void)B, (void)n, (void)V;
  return 0;
}

int32_t riallm_cuda_verify_draft(riallm_ctx* ctx, const void* logits, int32_t logits_dtype, const int32_t* draft_tokens,
                                 const float* draft_probs, const float* temperature, const float* accept_u,
                                 const float* sample_u, int32_t B, int32_t n, int32_t V, int32_t* tokens,
                                 int32_t* accepted, void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* what = "verify_draft";
  if (B < 0 || n < 0 || n > 255 || V <= 0)
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "bad dimensions (at most 255 drafted tokens)");
  if (logits_dtype != RIALLM_DTYPE_F32 && logits_dtype != RIALLM_DTYPE_BF16)
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "logits must be float32 or bf16");
  if (ctx && B == 0) return RIALLM_OK;
  if (!ctx || !logits || !temperature || !sample_u || !tokens || !accepted || (n > 0 && (!draft_tokens || !accept_u)))
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "NULL argument");
  (void)workspace, (void)workspace_bytes;
  return rl::guarded(ctx, [&]() -> int32_t {
    const VerifyArgs a{logits, logits_dtype == RIALLM_DTYPE_BF16, draft_tokens, draft_probs, temperature, accept_u,
                       sample_u, n, V, tokens, accepted};
    return rl::launched(ctx, what,
                        rl::launch_pdl(verify_draft_kernel, dim3(B), dim3(kThreads), 0, (cudaStream_t)stream, a));
  });
}

}  // extern "C"
