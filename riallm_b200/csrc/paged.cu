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
#include <algorithm>
#include <cmath>

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

// Which keys a row sees: j <= hi, and j >= lo or j < sinks.
struct Span {
  int lo, hi;
};
// What the attention kernels share. Row r of a (sequence, kv head) pair is
// token r / rep under query head kh * rep + r % rep: the heads of one kv head
// are rows of one matrix product with its keys.
struct AttnArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const int* pos;
  Pages pg;
  int B, T, nh, rep;
  int window, sinks;
  float scale_log2;  // log2(e) / sqrt(d): weights are powers of two
  uint16_t* out;

  __device__ __forceinline__ Span span(int64_t p) const {  // of the row at position p
    const int64_t cap = pg.cap();
    Span s;
    s.hi = (int)max((int64_t)-1, min(p, cap - 1));
    s.lo = window > 0 ? (int)max((int64_t)0, min(p - window + 1, (int64_t)INT32_MAX)) : 0;
    return s;
  }
};
__device__ __forceinline__ bool sees(Span s, int sinks, int j) { return j <= s.hi && (j >= s.lo || j < sinks); }

// The blocks of kBlock keys that some row of a sequence sees, in order: the
// first `ns` hold sinks, the others start at block `w0`.
struct Blocks {
  int ns, w0, n;
  Span all;  // what the sequence's rows see together
  __device__ __forceinline__ int index(int i) const { return i < ns ? i : w0 + i - ns; }
};
template <int kBlock>
__device__ __forceinline__ Blocks blocks_of(const AttnArgs& a, int64_t first, int64_t last) {
  Blocks r;
  r.all.hi = a.span(last).hi;
  r.all.lo = a.span(first).lo;
  r.w0 = r.all.lo / kBlock;
  const int nw = r.all.hi >= r.all.lo ? r.all.hi / kBlock - r.w0 + 1 : 0;
  const int sink_end = min(a.sinks, r.all.hi + 1);  // sinks that exist
  r.ns = a.window > 0 && sink_end > 0 ? (sink_end - 1) / kBlock + 1 : 0;
  if (nw > 0) r.ns = min(r.ns, r.w0);
  r.n = max(1, r.ns + nw);  // one block, seen by nobody, where nothing is seen
  return r;
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(rl::smem_u32(p))
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(rl::smem_u32(p))
               : "memory");
}
// d[16 x 8] += a[16 x 16] b[16 x 8], bf16 with float32 sums.
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 16 bytes, or 16 zero bytes where `bytes` is 0 (src is not read then).
__device__ __forceinline__ void cp_async_16z(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(rl::smem_u32(dst)), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool odd16(uint32_t x) {  // either bf16 of x is infinite or NaN
  return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
}

// ---------------------------------------------------------------- few rows
//
// Attention of few rows per sequence (single new tokens, drafted ones): a
// pass over the keys and values, bound by reading them. The work of a call,
// 64 keys of one (sequence, kv head, row tile) group a unit, is cut into as
// many equal contiguous shares as there are CTAs, whatever the sequences'
// lengths; a group that a share boundary cuts leaves partial results, which
// join_kernel adds up. The lengths are the device's, so a captured call
// follows them.
//
// In a CTA each of 4 warps takes 16 keys of every unit and is its own
// pipeline: cp.async into its own ring of kStages x (16 keys, 16 values),
// scores and weighted sums on m16n8k16 matrix instructions (the up to
// 16 rows against 16 keys), running maximum and sum in registers, no
// barrier with other warps until a group's end. The products are 1/40 of
// what even these instructions can do at the rate the bytes arrive, so
// nothing is gained by a 128-row tcgen05 tile of which 4 to 32 rows are
// used.
constexpr int kUnitKeys = 64, kFewWarps = 4;

template <int D>
constexpr int kFewStages = D == 128 ? 3 : 6;
template <int D>
constexpr int kFewSmem = kFewStages<D> * (kFewWarps * 2 + 1) * 16 * D * 2;

// Share of CTA c of G: units [W c / G, W (c+1) / G). The CTA of unit u.
__device__ __forceinline__ int64_t share_begin(int64_t W, int G, int c) { return W * c / G; }
__device__ __forceinline__ int share_of(int64_t W, int G, int64_t u) { return (int)(((u + 1) * G - 1) / W); }

// Finds where the first unit of share c (of the call's G shares, fewer where
// there are fewer units) lies: every thread of a block of N threads sums the
// units of its slab of sequences, and the thread whose slab holds the unit
// walks it.
struct UnitAt {
  int64_t W;      // all units of the call
  int G;          // shares, none of them empty
  int64_t u;      // the share's first unit (W where there is no such share)
  int64_t start;  // first unit of sequence b, which holds u
  int b;
  Blocks bl;
};
template <int N>
__device__ __forceinline__ UnitAt find_unit(const AttnArgs& a, int groups, int G, int c) {
  __shared__ int64_t sums[N / 32];
  __shared__ int64_t sh_start;
  __shared__ int sh_b;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (a.B + N - 1) / N;
  const int b0 = min(a.B, (int)threadIdx.x * per), b1 = min(a.B, b0 + per);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b)
    mine += (int64_t)blocks_of<kUnitKeys>(a, a.pos[b], (int64_t)a.pos[b] + a.T - 1).n * groups;
  int64_t upto = mine;  // inclusive scan
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  UnitAt at;
  at.W = 0;
  int64_t before = 0;
#pragma unroll
  for (int w = 0; w < N / 32; ++w) {
    before += w < warp ? sums[w] : 0;
    at.W += sums[w];
  }
  at.G = (int)min((int64_t)G, at.W);
  at.u = c < at.G ? share_begin(at.W, at.G, c) : at.W;
  int64_t s = before + upto - mine;
  if (at.u >= s && at.u < s + mine) {
    for (int b = b0; b < b1; ++b) {
      const int64_t n = (int64_t)blocks_of<kUnitKeys>(a, a.pos[b], (int64_t)a.pos[b] + a.T - 1).n * groups;
      if (at.u < s + n) {
        sh_b = b;
        sh_start = s;
        break;
      }
      s += n;
    }
  }
  if (at.u >= at.W) return at;
  __syncthreads();
  at.b = sh_b;
  at.start = sh_start;
  at.bl = blocks_of<kUnitKeys>(a, a.pos[at.b], (int64_t)a.pos[at.b] + a.T - 1);
  return at;
}

// Walks the units of a share.
struct Cursor {
  int b, g, i;
  int64_t p0;
  Blocks bl;
  __device__ __forceinline__ void load(const AttnArgs& a) {
    p0 = a.pos[b];
    bl = blocks_of<kUnitKeys>(a, p0, p0 + a.T - 1);
  }
  __device__ __forceinline__ void next(const AttnArgs& a, int groups) {
    if (++i < bl.n) return;
    i = 0;
    if (++g < groups) return;
    g = 0;
    if (++b < a.B) load(a);
  }
};

// A partial result: maxima, sums and accumulators of the rows of one tile.
template <int D>
constexpr int kSlotFloats = 16 * (D + 2);

template <int D>
__global__ void __launch_bounds__(kFewWarps * 32, 2)
    few_rows_kernel(const AttnArgs a, int tiles, float* __restrict__ ws) {
  constexpr int S = kFewStages<D>, C = D / 8;
  extern __shared__ __align__(128) uint16_t smem[];
  __shared__ float sm_m[kFewWarps][16], sm_l[kFewWarps][16];
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = a.pg.nkv * tiles, all_rows = a.T * a.rep;
  const UnitAt at = find_unit<kFewWarps * 32>(a, groups, gridDim.x, blockIdx.x);
  const int64_t u0 = at.u;
  if (u0 >= at.W) return;
  const int count = (int)(share_begin(at.W, at.G, blockIdx.x + 1) - u0);
  Cursor now;
  now.b = at.b;
  now.load(a);
  now.g = (int)((u0 - at.start) / now.bl.n);
  now.i = (int)((u0 - at.start) - (int64_t)now.g * now.bl.n);
  Cursor ahead = now;

  uint16_t* ring = smem + warp * (S * 2 * 16 * D);
  uint16_t* queries = smem + kFewWarps * S * 2 * 16 * D;  // S tiles of 16 query rows, for all warps

  // Loads of unit n (counted from u0) go to stage n % S, and with a group's
  // first unit its query rows, a quarter by each warp. Bit n % 32 of `held`
  // says whether this warp has anything to do in unit n.
  uint32_t held = 0;
  int issued = 0, begun = 0, page = -1;
  auto key0 = [&](const Cursor& c) { return c.bl.index(c.i) * kUnitKeys + warp * 16; };
  auto fetch_page = [&]() {  // the page of the unit that is loaded next
    page = -1;
    if (issued < count) {
      const int j = key0(ahead);
      const bool any = j <= ahead.bl.all.hi && (j + 15 >= ahead.bl.all.lo || j < a.sinks);
      if (any) page = a.pg.table[ahead.b * a.pg.stride + (j >> a.pg.lg)];
    }
  };
  auto issue = [&]() {
    if (issued < count) {
      const int kh = ahead.g / tiles;
      if (issued == 0 || ahead.i == 0) {
        const int tile = ahead.g - kh * tiles;
        uint16_t* to = queries + (begun % S) * 16 * D;
#pragma unroll
        for (int x = 0; x < 4 * C / 32; ++x) {
          const int idx = x * 32 + lane, r = warp * 4 + idx / C, c = idx % C, rr = tile * 16 + r;
          const bool in = rr < all_rows;
          const int tok = in ? rr / a.rep : 0, hd = in ? rr - tok * a.rep : 0;
          cp_async_16z(to + r * D + ((c ^ (r & 7)) * 8),
                       a.q + (((int64_t)ahead.b * a.T + tok) * a.nh + kh * a.rep + hd) * D + c * 8, in ? 16 : 0);
        }
        ++begun;
      }
      const bool ok = (unsigned)page < (unsigned)a.pg.num_pages;
      held = (held & ~(1u << (issued & 31))) | ((ok ? 1u : 0u) << (issued & 31));
      if (ok) {
        const int j = key0(ahead);
        const int64_t row = (((int64_t)page * a.pg.nkv + kh) << a.pg.lg) + (j & ((1 << a.pg.lg) - 1));
        uint16_t* ks = ring + (issued % S) * (2 * 16 * D);
        uint16_t* vs = ks + 16 * D;
#pragma unroll
        for (int x = 0; x < 16 * C / 32; ++x) {
          const int idx = x * 32 + lane, key = idx / C, c = idx % C;
          const bool in = sees(ahead.bl.all, a.sinks, j + key);
          const int64_t off = (row + (in ? key : 0)) * D + c * 8;
          const int to = key * D + ((c ^ (key & 7)) * 8);
          cp_async_16z(ks + to, a.k + off, in ? 16 : 0);
          cp_async_16z(vs + to, a.v + off, in ? 16 : 0);
        }
      }
      ++issued;
      if (issued < count) ahead.next(a, groups);
      fetch_page();
    }
    rl::cp_async_commit();
  };
  fetch_page();
#pragma unroll
  for (int s = 0; s < S - 1; ++s) issue();

  uint32_t qf[D / 16][4];
  float o[D / 8][4], m[2], l[2];
  Span sp[2];
  int tile = 0, kh = 0, first = 0, group = 0;
  for (int n = 0; n < count; ++n) {
    rl::cp_async_wait<S - 2>();
    if (n == 0 || now.i == 0) {  // a group begins
      __syncthreads();           // every warp's quarter of its query rows has arrived
      kh = now.g / tiles;
      tile = now.g - kh * tiles;
      first = n;
      const uint16_t* qs = queries + (group % S) * 16 * D;
      ++group;
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        const int r = lane & 15, c = 2 * x + (lane >> 4);
        ldmatrix_x4(qf[x], qs + r * D + ((c ^ (r & 7)) * 8));
      }
#pragma unroll
      for (int x = 0; x < D / 8; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[x][e] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = tile * 16 + h * 8 + (lane >> 2);
        m[h] = -INFINITY;
        l[h] = 0.f;
        sp[h] = r < all_rows ? a.span(now.p0 + r / a.rep) : Span{0, -1};
      }
    } else {
      __syncwarp();
    }
    uint16_t* ks = ring + (n % S) * (2 * 16 * D);
    uint16_t* vs = ks + 16 * D;
    if (held >> (n & 31) & 1) {
      const int j0 = key0(now);
      float sc[2][4];
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[y][e] = 0.f;
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        uint32_t kf[4];
        const int key = (lane & 7) + ((lane >> 4) << 3), c = 2 * x + ((lane >> 3) & 1);
        ldmatrix_x4(kf, ks + key * D + ((c ^ (key & 7)) * 8));
        mma_16816(sc[0], qf[x], kf[0], kf[1]);
        mma_16816(sc[1], qf[x], kf[2], kf[3]);
      }
      // Does any row of the sequence not see one of these keys?
      const int64_t pl = now.p0 + a.T - 1;
      const bool edge = j0 + 15 > min(now.p0, a.pg.cap() - 1) ||
                        (a.window > 0 && j0 < pl - a.window + 1 && j0 + 15 >= a.sinks);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = -INFINITY;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = sc[y][2 * h + e];
            x *= a.scale_log2;
            if (edge && !sees(sp[h], a.sinks, j0 + y * 8 + (lane & 3) * 2 + e)) x = -INFINITY;
            top = fmaxf(top, x);
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mn = fmaxf(m[h], top);
        const float base = mn == -INFINITY ? 0.f : mn;
        const float corr = ex2(m[h] - base);
        m[h] = mn;
        float sum = 0.f;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = sc[y][2 * h + e];
            x = ex2(x - base);
            sum += x;
          }
        l[h] = fmaf(l[h], corr, sum);
        if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
          for (int x = 0; x < D / 8; ++x) {
            o[x][2 * h] *= corr;
            o[x][2 * h + 1] *= corr;
          }
        }
      }
      if (edge && a.T > 1) {
        // A value that is not finite, of a key that some rows see and some
        // do not: 0 times it would reach the latter through the product.
        // It is added to the rows that see it and zeroed for the product.
        bool odd = false;
#pragma unroll
        for (int x = 0; x < 16 * C / 32; ++x) {
          const uint4 w = *reinterpret_cast<const uint4*>(vs + (x * 32 + lane) * 8);
          odd |= odd16(w.x) | odd16(w.y) | odd16(w.z) | odd16(w.w);
        }
        if (__any_sync(0xffffffffu, odd)) {
          for (int key = 0; key < 16; ++key)
#pragma unroll
            for (int x = 0; x < D / 8; ++x) {
              const uint32_t w =
                  *reinterpret_cast<const uint32_t*>(vs + key * D + ((x ^ (key & 7)) * 8) + (lane & 3) * 2);
              if (!odd16(w)) continue;
              const float lo = bf2f((uint16_t)w), hi = bf2f((uint16_t)(w >> 16));
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (sees(sp[h], a.sinks, j0 + key)) {
                  if (!isfinite(lo)) o[x][2 * h] += lo;
                  if (!isfinite(hi)) o[x][2 * h + 1] += hi;
                }
            }
          __syncwarp();
          for (int x = lane; x < 16 * D; x += 32)
            if ((vs[x] & 0x7f80u) == 0x7f80u) vs[x] = 0;
          __syncwarp();
        }
      }
      // The weights as bf16 and what that leaves, also as bf16: two products
      // keep 16 bits of each weight (one alone costs as much accuracy again
      // as the rounding of the output), and the matrix pipe is idle anyway.
      uint32_t ph[4], pr[4];
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x0 = sc[y][2 * h], x1 = sc[y][2 * h + 1];
          const uint32_t hi = rl::pack_bf16x2(x0, x1);
          ph[2 * y + h] = hi;
          pr[2 * y + h] = rl::pack_bf16x2(x0 - __uint_as_float(hi << 16), x1 - __uint_as_float(hi & 0xffff0000u));
        }
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        uint32_t vf[4];
        const int key = lane & 15, c = 2 * x + (lane >> 4);
        ldmatrix_x4_trans(vf, vs + key * D + ((c ^ (key & 7)) * 8));
        mma_16816(o[2 * x], ph, vf[0], vf[1]);
        mma_16816(o[2 * x + 1], ph, vf[2], vf[3]);
        mma_16816(o[2 * x], pr, vf[0], vf[1]);
        mma_16816(o[2 * x + 1], pr, vf[2], vf[3]);
      }
    }
    __syncwarp();
    issue();  // into the stage that was read before this one

    const bool whole_end = now.i + 1 == now.bl.n;
    if (whole_end || n + 1 == count) {
      // The group ends, or this CTA's share of it. Each warp leaves its
      // result in the stage it has just read (2 * 16 * D bf16 hold 16 * D
      // floats), columns swizzled by the row; then all add up the four.
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const int r = h * 8 + (lane >> 2);
        if ((lane & 3) == 0) {
          sm_m[warp][r] = m[h];
          sm_l[warp][r] = l[h];
        }
#pragma unroll
        for (int x = 0; x < D / 8; ++x)
          *reinterpret_cast<float2*>(reinterpret_cast<float*>(ks) + r * D + ((x * 8 + (lane & 3) * 2) ^ ((r & 3) * 8))) =
              make_float2(o[x][2 * h], o[x][2 * h + 1]);
      }
      __syncthreads();
      // Whole group here: the output. Otherwise the CTA's slot of partial
      // results, 2 per CTA: one for a group that began in an earlier share
      // or with this share, one for a group that began inside it.
      const bool whole = whole_end && now.i == n - first;
      const int rows = min(16, all_rows - tile * 16);
      float* slot = ws + (2 * (int64_t)blockIdx.x + (first == 0 ? 0 : 1)) * kSlotFloats<D>;
      const float* part = reinterpret_cast<const float*>(smem) + (n % S) * (16 * D);
      for (int x = threadIdx.x; x < rows * (D / 4); x += kFewWarps * 32) {
        const int r = x / (D / 4), c = (x - r * (D / 4)) * 4;
        float M = sm_m[0][r];
#pragma unroll
        for (int w = 1; w < kFewWarps; ++w) M = fmaxf(M, sm_m[w][r]);
        float L = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (M != -INFINITY)
#pragma unroll
          for (int w = 0; w < kFewWarps; ++w) {
            const float f = ex2(sm_m[w][r] - M);
            const float4 z = *reinterpret_cast<const float4*>(part + w * (S * 16 * D) + r * D + (c ^ ((r & 3) * 8)));
            L = fmaf(sm_l[w][r], f, L);
            y.x = fmaf(z.x, f, y.x);
            y.y = fmaf(z.y, f, y.y);
            y.z = fmaf(z.z, f, y.z);
            y.w = fmaf(z.w, f, y.w);
          }
        if (whole) {
          const float inv = L == 0.f ? 0.f : __fdiv_rn(1.f, L);
          const int rr = tile * 16 + r, tok = rr / a.rep, hd = rr - tok * a.rep;
          *reinterpret_cast<uint2*>(a.out + (((int64_t)now.b * a.T + tok) * a.nh + kh * a.rep + hd) * D + c) =
              make_uint2(rl::pack_bf16x2(y.x * inv, y.y * inv), rl::pack_bf16x2(y.z * inv, y.w * inv));
        } else {
          // Two floats at a time: D + 2 floats a row keep 8-byte alignment only.
          float2* to = reinterpret_cast<float2*>(slot + 32 + r * D + c);
          to[0] = make_float2(y.x, y.y);
          to[1] = make_float2(y.z, y.w);
          if (c == 0) {
            slot[r] = M;
            slot[16 + r] = L;
          }
        }
      }
      __syncthreads();  // before the stages, sm_m and sm_l are written again
    }
    if (n + 1 < count) now.next(a, groups);
  }
}

// CTA c adds up the partial results of the group that the boundary between
// the shares c and c + 1 cuts, if c is the first that holds part of it.
// Threads (dimension, row); the weights of the parts are worked out once a
// row, a part a thread.
constexpr int kMaxShares = 512;
template <int D>
__global__ void __launch_bounds__(D * 4) join_kernel(const AttnArgs a, int tiles, int G, const float* __restrict__ ws) {
  constexpr int kRows = 16, kSlot = kSlotFloats<D>, kW = D / 32;
  __shared__ float weight[4][kMaxShares], red[2][4][kW];
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const int groups = a.pg.nkv * tiles, c0 = blockIdx.x;
  const UnitAt at = find_unit<D * 4>(a, groups, G, c0 + 1);
  if (at.u >= at.W) return;
  const int64_t g = (at.u - at.start) / at.bl.n, g0 = at.start + g * at.bl.n, g1 = g0 + at.bl.n;
  if (at.u == g0 || share_of(at.W, at.G, g0) != c0) return;  // not cut here, or cut before as well
  const int parts = share_of(at.W, at.G, g1 - 1) - c0 + 1;
  // The first part is in its CTA's second slot where the group began inside
  // that CTA's share.
  const float* first = ws + (2 * (int64_t)c0 + (share_begin(at.W, at.G, c0) < g0 ? 1 : 0)) * kSlot;
  const float* rest = ws + 2 * (int64_t)c0 * kSlot;
  const int kh = (int)(g / tiles), tile = (int)(g - (int64_t)kh * tiles);
  const int rows = min(kRows, a.T * a.rep - tile * kRows);
  const int d = threadIdx.x % D, rs = threadIdx.x / D, lane = d & 31, w = d >> 5;
  for (int r0 = 0; r0 < rows; r0 += 4) {
    const int r = r0 + rs;
    const bool in = r < rows;
    float M = -INFINITY;
    if (in)
      for (int i = d; i < parts; i += D) M = fmaxf(M, __ldcg((i ? rest + (int64_t)i * 2 * kSlot : first) + r));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (lane == 0) red[0][rs][w] = M;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kW; ++x) M = fmaxf(M, red[0][rs][x]);
    float den = 0.f;
    if (in)
      for (int i = d; i < parts; i += D) {
        const float* s = i ? rest + (int64_t)i * 2 * kSlot : first;
        const float f = M == -INFINITY ? 0.f : ex2(__ldcg(s + r) - M);
        weight[rs][i] = f;
        den = fmaf(f, __ldcg(s + kRows + r), den);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
    if (lane == 0) red[1][rs][w] = den;
    __syncthreads();
    den = 0.f;
#pragma unroll
    for (int x = 0; x < kW; ++x) den += red[1][rs][x];
    if (in) {
      const int64_t at_d = 2 * kRows + r * D + d;
      float num = weight[rs][0] * __ldcg(first + at_d);
#pragma unroll 8
      for (int i = 1; i < parts; ++i) num = fmaf(weight[rs][i], __ldcg(rest + (int64_t)i * 2 * kSlot + at_d), num);
      const int rr = tile * kRows + r, tok = rr / a.rep, hd = rr - tok * a.rep;
      a.out[(((int64_t)at.b * a.T + tok) * a.nh + kh * a.rep + hd) * D + d] = f2bf(den == 0.f ? 0.f : num / den);
    }
    __syncthreads();  // weight and red are written again
  }
}

// The launch of a call with few rows: row tiles of 16, CTAs, and whether a
// group can be cut at all.
struct FewPlan {
  int tiles, G;
  bool join;
  uint64_t ws_bytes;
};
FewPlan few_plan(int num_sms, int B, int T, int nh, int nkv, int d, int64_t cap) {
  FewPlan p;
  const int64_t rows = (int64_t)T * (nh / nkv);
  p.tiles = (int)((rows + 15) / 16);
  const int64_t blocks = (cap + kUnitKeys - 1) / kUnitKeys;
  const int64_t most = (int64_t)B * nkv * p.tiles * blocks;
  p.G = (int)std::min<int64_t>(std::min(2 * num_sms, kMaxShares), most);
  p.join = blocks > 1 && p.G > 1;
  p.ws_bytes = p.join ? (uint64_t)2 * p.G * 16 * (d + 2) * sizeof(float) : 0;
  return p;
}

template <int D>
int32_t launch_few(riallm_ctx* ctx, const AttnArgs& a, const FewPlan& p, float* ws, cudaStream_t st) {
  const char* what = "paged_attention";
  if (int s = rl::allow_smem(ctx, what, few_rows_kernel<D>, kFewSmem<D>, D / 64 - 1)) return s;
  if (int s = rl::launched(ctx, what,
                           rl::launch_pdl(few_rows_kernel<D>, dim3(p.G), dim3(kFewWarps * 32), kFewSmem<D>, st, a,
                                          p.tiles, ws)))
    return s;
  if (!p.join) return RIALLM_OK;
  return rl::launched(ctx, what,
                      rl::launch_pdl(join_kernel<D>, dim3(p.G - 1), dim3(D * 4), 0, st, a, p.tiles, p.G,
                                     static_cast<const float*>(ws)));
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
  if (!ctx || B <= 0 || T <= 0 || nkv <= 0 || nh < nkv || max_pages <= 0 || page_size <= 0) return 0;
  return few_plan(ctx->num_sms, B, T, nh, nkv, d, (int64_t)max_pages * page_size).ws_bytes;
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
  if (ctx && (int64_t)B * T == 0) return RIALLM_OK;
  if (!ctx || !q || !k_pages || !v_pages || !pos || !page_table || !out)
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "NULL argument");
  if (!al16(q) || !al16(out) || !al16(k_pages) || !al16(v_pages))
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "buffers must be 16-byte aligned");
  const FewPlan p = few_plan(ctx->num_sms, B, T, nh, nkv, d, (int64_t)max_pages * page_size);
  if (p.ws_bytes && (!workspace || workspace_bytes < p.ws_bytes || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return rl::refuse(ctx, RIALLM_ERR_MEMORY, what, "workspace missing, too small or not 256-byte aligned");
  return rl::guarded(ctx, [&]() -> int32_t {
    AttnArgs a;
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k_pages);
    a.v = static_cast<const uint16_t*>(v_pages);
    a.pos = pos;
    a.pg = make_pages(page_table, table_stride, max_pages, num_pages, nkv, page_size);
    a.B = B, a.T = T, a.nh = nh, a.rep = nh / nkv;
    a.window = window, a.sinks = sinks;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)d));
    a.out = static_cast<uint16_t*>(out);
    float* ws = static_cast<float*>(workspace);
    cudaStream_t st = (cudaStream_t)stream;
    return d == 128 ? launch_few<128>(ctx, a, p, ws, st) : launch_few<64>(ctx, a, p, ws, st);
  });
}

}  // extern "C"
