// paged.cu -- the decoder layer's attention over a paged key-value cache.
//
// The cache of one layer is a pool of pages, [num_pages, nkv, page_size, d]
// bf16 each for k and v; a page table [B, max_pages] names, for every
// sequence, the page that holds positions [i * page_size, (i+1) * page_size).
// An entry outside [0, num_pages) is a page that the sequence does not hold
// (never given, or given back behind a sliding window): its positions are
// neither written nor read. riallm keeps one contiguous cache per layer
// (KVCACHE, src/model.rs:15-38); rotary embedding and attention follow
// src/model.rs:912-1071 as the contiguous kernels in decoder.cu do.
#include <cfloat>

#include "common.cuh"
#include "internal.h"

namespace {

__device__ __forceinline__ float bf2f(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ uint16_t f2bf(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }

// The page table and the geometry of the pools.
struct Pages {
  const int* table;
  int64_t stride;  // table entries from one sequence to the next
  int max_pages;   // per sequence
  int num_pages;   // in a pool
  int nkv;
  int lg;          // log2(page_size)

  __host__ __device__ __forceinline__ int64_t cap() const { return (int64_t)max_pages << lg; }
  // Row of the pool, viewed as [num_pages * nkv * page_size, d], that holds
  // position j of sequence b for kv head kh; -1 where there is none.
  __host__ __device__ __forceinline__ int64_t row(int b, int kh, int64_t j) const {
    if (j < 0 || j >= cap()) return -1;
    const int page = table[b * stride + (j >> lg)];
    if ((unsigned)page >= (unsigned)num_pages) return -1;
    return (((int64_t)page * nkv + kh) << lg) + (j & ((1 << lg) - 1));
  }
};

// cos and sin of position * inv_freq. The product of a 31-bit and a 24-bit
// number is rounded once in 64 bits and reduced to [-pi, pi] there, so far
// positions keep float32 accuracy (a float32 product is 6e-3 off at position
// 100000), and sincosf stays on its short path.
__device__ __forceinline__ void rope_angle(int64_t p, float f, float* s, float* c) {
  const double a = (double)p * (double)f;
  const double k = rint(a * 0.15915494309189535);            // 1 / (2 pi)
  const double r = fma(-k, 2.4492935982947064e-16, fma(-k, 6.283185307179586, a));  // 2 pi = hi + lo
  sincosf((float)r, s, c);
}

// CTA (row, head): row b*T + t of qkv at position pos[b] + t.
__global__ void __launch_bounds__(64)
    rope_paged_append_kernel(const uint16_t* __restrict__ qkv, const int* __restrict__ pos, Pages pg, int T,
                             int nh, int d, const float* __restrict__ inv_freq, uint16_t* __restrict__ q_out,
                             uint16_t* __restrict__ kp, uint16_t* __restrict__ vp) {
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  const int h = blockIdx.y, half = d >> 1;
  const int b = (int)(row / T);
  const int64_t p = (int64_t)pos[b] + (row - (int64_t)b * T);
  const int nkv = pg.nkv;
  const uint16_t* src = qkv + (row * (nh + 2 * nkv) + h) * d;
  uint16_t* dst;
  if (h < nh) {
    dst = q_out + (row * nh + h) * d;
  } else {
    const int kh = (h - nh) % nkv;
    const int64_t at = pg.row(b, kh, p);
    if (at < 0) return;
    dst = (h < nh + nkv ? kp : vp) + at * d;
  }
  for (int j = threadIdx.x; j < half; j += blockDim.x) {
    if (h >= nh + nkv) {  // v is copied as it is
      dst[j] = src[j];
      dst[j + half] = src[j + half];
      continue;
    }
    const float x1 = bf2f(src[j]), x2 = bf2f(src[j + half]);
    float s, c;
    rope_angle(p, inv_freq[j], &s, &c);
    dst[j] = f2bf(fmaf(x1, c, -x2 * s));
    dst[j + half] = f2bf(fmaf(x2, c, x1 * s));
  }
}

// Which keys the row at position p sees: [0, min(p + 1, cap)), and with a
// window only the last `window` of [0, p] and the first `sinks`.
struct Window {
  int window, sinks;
  __device__ __forceinline__ int64_t first(int64_t p) const {  // first key inside the window
    return window > 0 ? max((int64_t)0, p - window + 1) : 0;
  }
};

// Warp per (row, head): keys one at a time, a lane per d / 32 dimensions,
// running maximum and sum in float32.
template <int D>
__global__ void __launch_bounds__(128)
    paged_attention_kernel(const uint16_t* __restrict__ q, const uint16_t* __restrict__ kp,
                           const uint16_t* __restrict__ vp, const int* __restrict__ pos, Pages pg, Window win,
                           int64_t pairs, int T, int nh, float scale, uint16_t* __restrict__ out) {
  constexpr int E = D / 32;
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t pair = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (pair >= pairs) return;
  const int64_t row = pair / nh;
  const int h = (int)(pair - row * nh), kh = h / (nh / pg.nkv);
  const int b = (int)(row / T);
  const int64_t p = (int64_t)pos[b] + (row - (int64_t)b * T);
  const int64_t L = max((int64_t)0, min(p + 1, pg.cap()));
  const int64_t lo = win.first(p);
  float qr[E], acc[E], m = -FLT_MAX, l = 0.f;
  bool any = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qr[e] = bf2f(q[pair * D + lane * E + e]);
    acc[e] = 0.f;
  }
  for (int64_t j = 0; j < L; ++j) {
    if (j < lo && j >= win.sinks) j = lo;
    if (j >= L) break;
    const int64_t at = pg.row(b, kh, j);
    if (at < 0) continue;
    any = true;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(qr[e], bf2f(kp[at * D + lane * E + e]), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= scale;
    const float mn = fmaxf(m, s), corr = expf(m - mn), w = expf(s - mn);
    m = mn;
    l = fmaf(l, corr, w);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(acc[e], corr, w * bf2f(vp[at * D + lane * E + e]));
  }
#pragma unroll
  for (int e = 0; e < E; ++e) out[pair * D + lane * E + e] = f2bf(any ? __fdiv_rn(acc[e], l) : 0.f);
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// What both entry points share: the checks of the cache's geometry.
int check_pages(riallm_ctx* ctx, const char* what, int32_t B, int32_t T, int32_t nh, int32_t nkv, int32_t d,
                int32_t num_pages, int32_t page_size, int32_t max_pages, int64_t table_stride) {
  auto bad = [&](const char* msg) { return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, msg); };
  if (B < 0 || T < 0 || nh <= 0 || nkv <= 0 || nh % nkv != 0)
    return bad("bad dimensions (heads must be a multiple of kv heads)");
  if (nh / nkv > 16) return bad("more than 16 heads per kv head");
  if (d != 64 && d != 128) return bad("head_dim must be 64 or 128");
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return bad("page_size must be 16, 32, 64 or 128");
  if (num_pages <= 0 || max_pages <= 0 || table_stride < max_pages) return bad("bad page table");
  if ((int64_t)num_pages * nkv * page_size > INT32_MAX || (int64_t)max_pages * page_size > INT32_MAX)
    return bad("more than 2^31 - 1 cache rows");
  if ((int64_t)B * T > INT32_MAX / 4 || (int64_t)nh + 2 * nkv > 65535) return bad("too many rows or heads");
  return RIALLM_OK;
}

Pages make_pages(const int32_t* table, int64_t stride, int32_t max_pages, int32_t num_pages, int32_t nkv,
                 int32_t page_size) {
  int lg = 4;
  while ((1 << lg) < page_size) ++lg;
  return Pages{table, stride, max_pages, num_pages, nkv, lg};
}

}  // namespace

extern "C" {

int64_t riallm_paged_row(const int32_t* page_table, int64_t table_stride, int32_t max_pages, int32_t num_pages,
                         int32_t nkv, int32_t page_size, int32_t b, int32_t kv_head, int64_t position) {
  if (!page_table) return -1;
  return make_pages(page_table, table_stride, max_pages, num_pages, nkv, page_size).row(b, kv_head, position);
}

int32_t riallm_cuda_rope_paged_append(riallm_ctx* ctx, const void* qkv, const int32_t* pos,
                                      const int32_t* page_table, int64_t table_stride, int32_t max_pages, int32_t B,
                                      int32_t T, int32_t nh, int32_t nkv, int32_t d, const float* inv_freq,
                                      void* q_out, void* k_pages, void* v_pages, int32_t num_pages,
                                      int32_t page_size, void* stream) {
  const char* what = "rope_paged_append";
  if (int s = check_pages(ctx, what, B, T, nh, nkv, d, num_pages, page_size, max_pages, table_stride)) return s;
  if (ctx && (int64_t)B * T == 0) return RIALLM_OK;
  if (!ctx || !qkv || !pos || !page_table || !inv_freq || !q_out || !k_pages || !v_pages)
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "NULL argument");
  if (!al16(qkv) || !al16(q_out) || !al16(k_pages) || !al16(v_pages) || !al16(inv_freq))
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "buffers must be 16-byte aligned");
  return rl::guarded(ctx, [&]() -> int32_t {
    const Pages pg = make_pages(page_table, table_stride, max_pages, num_pages, nkv, page_size);
    return rl::launched(ctx, what,
                        rl::launch_pdl(rope_paged_append_kernel, dim3(B * T, nh + 2 * nkv), dim3(64), 0,
                                       (cudaStream_t)stream, static_cast<const uint16_t*>(qkv), pos, pg, T, nh, d,
                                       inv_freq, static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_pages),
                                       static_cast<uint16_t*>(v_pages)));
  });
}

uint64_t riallm_cuda_paged_attention_workspace(const riallm_ctx* ctx, int32_t B, int32_t T, int32_t nh, int32_t nkv,
                                               int32_t d, int32_t max_pages, int32_t page_size) {
  (void)ctx, (void)B, (void)T, (void)nh, (void)nkv, (void)d, (void)max_pages, (void)page_size;
  return 0;
}

int32_t riallm_cuda_paged_attention(riallm_ctx* ctx, const void* q, const void* k_pages, const void* v_pages,
                                    const int32_t* pos, const int32_t* page_table, int64_t table_stride,
                                    int32_t max_pages, int32_t B, int32_t T, int32_t nh, int32_t nkv, int32_t d,
                                    int32_t num_pages, int32_t page_size, int32_t window, int32_t sinks, void* out,
                                    void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* what = "paged_attention";
  if (int s = check_pages(ctx, what, B, T, nh, nkv, d, num_pages, page_size, max_pages, table_stride)) return s;
  if (window < 0 || sinks < 0)
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "window and sinks must not be negative");
  const int64_t pairs = (int64_t)B * T * nh;
  if (ctx && pairs == 0) return RIALLM_OK;
  if (!ctx || !q || !k_pages || !v_pages || !pos || !page_table || !out)
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "NULL argument");
  if (!al16(q) || !al16(out) || !al16(k_pages) || !al16(v_pages))
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "buffers must be 16-byte aligned");
  if ((pairs + 3) / 4 > INT32_MAX) return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "too many rows");
  (void)workspace, (void)workspace_bytes;
  return rl::guarded(ctx, [&]() -> int32_t {
    const Pages pg = make_pages(page_table, table_stride, max_pages, num_pages, nkv, page_size);
    const float scale = (float)(1.0 / sqrt((double)d));
    return rl::launched(ctx, what,
                        rl::launch_pdl(d == 128 ? paged_attention_kernel<128> : paged_attention_kernel<64>,
                                       dim3((unsigned)((pairs + 3) / 4)), dim3(128), 0, (cudaStream_t)stream,
                                       static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_pages),
                                       static_cast<const uint16_t*>(v_pages), pos, pg, Window{window, sinks}, pairs, T,
                                       nh, scale, static_cast<uint16_t*>(out)));
  });
}

}  // extern "C"
