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

// CTA (rows, heads): up to kAppendRows rows of qkv, row b*T + t at position
// pos[b] + t, and `hg` of its heads. A thread takes 8 dimensions of a head's
// first half and the same 8 of its second (two 16-byte pieces): the pieces of
// its first units are loaded before the angles are worked out, a row's d / 2
// cosines and sines once for all of its heads. qkv is read once and as much
// written: 8192 rows of 40 heads of 64 (84 MB) take 17.6 us, 4.8 TB/s where
// the HBM's 6.45 would take 13.0. Neither the HBM (30 % of its cycles; what is
// written is in the L2 when the kernel ends) nor the issue slots (53 %) are
// full: a CTA is one chain of load, angles, barrier and store, 42 % of the
// warps' places taken. 64 rows take less than their launch.
constexpr int kAppendRows = 4, kAppendThreads = 256, kAppendUnits = 4;  // units a thread
template <int D>
__global__ void __launch_bounds__(kAppendThreads)
    rope_paged_append_kernel(const uint16_t* __restrict__ qkv, const int* __restrict__ pos, Pages pg, int all_rows,
                             int T, int nh, int rows_per_cta, int hg, const float* __restrict__ inv_freq,
                             uint16_t* __restrict__ q_out, uint16_t* __restrict__ kp, uint16_t* __restrict__ vp) {
  constexpr int P = D / 16;  // units of a head
  __shared__ __align__(16) float cs[kAppendRows * D / 2], sn[kAppendRows * D / 2];
  __shared__ int64_t at[kAppendRows];  // pool row of the position, kv head 0; -1
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const int nkv = pg.nkv, heads = nh + 2 * nkv;
  const int row0 = blockIdx.x * rows_per_cta, rows = min(rows_per_cta, all_rows - row0);
  const int h0 = blockIdx.y * hg, hn = min(hg, heads - h0);
  const int units = rows * hn * P;
  uint4 lo[kAppendUnits], hi[kAppendUnits];
#pragma unroll
  for (int x = 0; x < kAppendUnits; ++x) {
    const int u = x * kAppendThreads + threadIdx.x;
    if (u < units) {
      const int hu = u / P, r = hu / hn;
      const uint4* src = reinterpret_cast<const uint4*>(qkv + ((int64_t)(row0 + r) * heads + h0 + (hu - r * hn)) * D);
      lo[x] = __ldcs(src + u % P);
      hi[x] = __ldcs(src + P + u % P);
    }
  }
  if ((int)threadIdx.x < rows * (D / 2)) {
    const int r = threadIdx.x / (D / 2), j = threadIdx.x % (D / 2);
    const int b = (row0 + r) / T;
    const int64_t p = (int64_t)pos[b] + (row0 + r - b * T);
    if (h0 < nh + nkv) rope_angle(p, inv_freq[j], &sn[threadIdx.x], &cs[threadIdx.x]);
    if (j == 0) at[r] = h0 + hn > nh ? pg.row(b, 0, p) : -1;
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < kAppendUnits; ++x) {
    const int u = x * kAppendThreads + threadIdx.x;
    if (u >= units) break;
    const int c = u % P, hu = u / P, r = hu / hn, h = h0 + (hu - r * hn);
    uint4 o1 = lo[x], o2 = hi[x];
    if (h < nh + nkv) {
      const float4* cr = reinterpret_cast<const float4*>(cs + r * (D / 2) + c * 8);
      const float4* sr = reinterpret_cast<const float4*>(sn + r * (D / 2) + c * 8);
      const uint32_t* a1 = reinterpret_cast<const uint32_t*>(&lo[x]);
      const uint32_t* a2 = reinterpret_cast<const uint32_t*>(&hi[x]);
      uint32_t* w1 = reinterpret_cast<uint32_t*>(&o1);
      uint32_t* w2 = reinterpret_cast<uint32_t*>(&o2);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float4 cc = cr[g], ss = sr[g];
        const float* cf = reinterpret_cast<const float*>(&cc);
        const float* sf = reinterpret_cast<const float*>(&ss);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t x1 = a1[2 * g + e], x2 = a2[2 * g + e];
          const float p1 = __uint_as_float(x1 << 16), q1 = __uint_as_float(x1 & 0xffff0000u);
          const float p2 = __uint_as_float(x2 << 16), q2 = __uint_as_float(x2 & 0xffff0000u);
          const float c0 = cf[2 * e], c1 = cf[2 * e + 1], s0 = sf[2 * e], s1 = sf[2 * e + 1];
          w1[2 * g + e] = rl::pack_bf16x2(fmaf(p1, c0, -p2 * s0), fmaf(q1, c1, -q2 * s1));
          w2[2 * g + e] = rl::pack_bf16x2(fmaf(p2, c0, p1 * s0), fmaf(q2, c1, q1 * s1));
        }
      }
    }
    uint16_t* dst;
    if (h < nh) {
      dst = q_out + ((int64_t)(row0 + r) * nh + h) * D;
    } else {
      if (at[r] < 0) continue;
      const int kh = h < nh + nkv ? h - nh : h - nh - nkv;
      dst = (h < nh + nkv ? kp : vp) + (at[r] + ((int64_t)kh << pg.lg)) * D;
    }
    reinterpret_cast<uint4*>(dst)[c] = o1;
    reinterpret_cast<uint4*>(dst)[P + c] = o2;
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
  uint32_t rep_inv;  // 2^32 / rep, rounded up (rep > 1)
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
// Does some row between positions p0 and p1 not see some key of [j0, j1]?
__device__ __forceinline__ bool is_edge(const AttnArgs& a, int64_t p0, int64_t p1, int j0, int j1) {
  return j1 > min(p0, a.pg.cap() - 1) || (a.window > 0 && j0 < p1 - a.window + 1 && j1 >= a.sinks);
}

// The blocks of kBlock keys that some row between two positions sees, in
// order: the first `ns` hold sinks, the others start at block `w0`.
struct Blocks {
  int ns, w0, n;
  Span all;  // what these rows see together
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

// The work of a call: the rows of every sequence in tiles of R; a group is
// one (sequence, tile, kv head). Groups are laid out in that order along a
// line, each as kCost units of fixed cost and then a unit for each of its
// blocks of kBlock keys, and the line is cut into as many equal shares as
// there are CTAs, whatever the sequences' lengths and the tiles' place under
// the causal diagonal. A block belongs to the share that its unit lies in; a
// group with blocks in several shares leaves partial results, which
// join_kernel adds up. The lengths are the device's, so a captured call
// follows them.
template <int R_, int kBlock_, int kCost_>
struct Shape {
  static constexpr int R = R_, kBlock = kBlock_, kCost = kCost_;
};
struct Tile {
  int b, rows;          // sequence; rows of the tile
  int tok0, head0;      // its first row is head head0 (of rep) of token tok0
  int64_t p0, p1;       // positions of the first and last row
  Blocks bl;
};
// Token of row r of a tile, counted from the tile's first: (head0 + r) / rep.
// rep is at most 128 and r below 256, so rounding 1 / rep up adds less than
// 2^-16 to the quotient.
__device__ __forceinline__ int token_of(const AttnArgs& a, const Tile& t, int r) {
  return a.rep == 1 ? r : (int)__umulhi((uint32_t)(t.head0 + r), a.rep_inv);
}
template <typename Sh>
__device__ __forceinline__ Tile tile_of(const AttnArgs& a, int tiles, int x) {
  Tile t;
  t.b = x / tiles;
  const int row0 = (x - t.b * tiles) * Sh::R;
  t.rows = min(Sh::R, a.T * a.rep - row0);
  t.tok0 = row0 / a.rep;
  t.head0 = row0 - t.tok0 * a.rep;
  const int64_t p = a.pos[t.b];
  t.p0 = p + t.tok0;
  t.p1 = t.p0 + token_of(a, t, t.rows - 1);
  t.bl = blocks_of<Sh::kBlock>(a, t.p0, t.p1);
  return t;
}
// Where row r of a tile lies in q and out, in heads.
__device__ __forceinline__ int64_t head_of(const AttnArgs& a, const Tile& t, int kh, int r) {
  const int tok = token_of(a, t, r);
  return ((int64_t)t.b * a.T + t.tok0 + tok) * a.nh + kh * a.rep + (t.head0 + r - tok * a.rep);
}

// x / y of numbers that are not negative; 32-bit where both allow it (a
// 64-bit division is some 300 cycles, and a share begins with several).
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  return ((x | y) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
}
// Share c of G: units [W c / G, W (c+1) / G). The share that unit u is in.
__device__ __forceinline__ int64_t share_begin(int64_t W, int G, int c) { return quotient(W * c, G); }
__device__ __forceinline__ int share_of(int64_t W, int G, int64_t u) { return (int)quotient((u + 1) * G - 1, W); }

// Finds the tile that the first unit of share c (of the call's G shares, fewer
// where there are fewer units) lies in: every thread of a block of N threads
// sums the units of its slab of tiles, and the thread whose slab holds the
// unit walks it.
struct UnitAt {
  int64_t W;      // all units of the call
  int G;          // shares, none of them empty
  int64_t u;      // the share's first unit (W where there is no such share)
  int64_t start;  // first unit of tile x, which holds u
  int x;
};
template <typename Sh, int N>
__device__ __forceinline__ UnitAt find_unit(const AttnArgs& a, int tiles, int G, int c) {
  __shared__ int64_t sums[N / 32];
  __shared__ int64_t sh_start;
  __shared__ int sh_x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int all = a.B * tiles, per = (all + N - 1) / N;
  const int x0 = min(all, (int)threadIdx.x * per), x1 = min(all, x0 + per);
  auto units = [&](int x) { return (int64_t)(tile_of<Sh>(a, tiles, x).bl.n + Sh::kCost) * a.pg.nkv; };
  int64_t mine = 0;
  for (int x = x0; x < x1; ++x) mine += units(x);
  int64_t upto = mine;  // inclusive scan
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
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
    for (int x = x0; x < x1; ++x) {
      const int64_t n = units(x);
      if (at.u < s + n) {
        sh_x = x;
        sh_start = s;
        break;
      }
      s += n;
    }
  }
  if (at.u >= at.W) return at;
  __syncthreads();
  at.x = sh_x;
  at.start = sh_start;
  return at;
}

// Walks the blocks of share c from its first on.
template <typename Sh>
struct Cursor {
  int x, kh, i;
  int64_t at0, end;  // unit of the group's block 0; end of the share
  Tile t;
  __device__ __forceinline__ void init(const AttnArgs& a, int tiles, const UnitAt& at, int c) {
    x = at.x;
    t = tile_of<Sh>(a, tiles, x);
    const int size = t.bl.n + Sh::kCost;
    kh = (int)quotient(at.u - at.start, size);
    at0 = at.start + (int64_t)kh * size + Sh::kCost;
    i = (int)max((int64_t)0, at.u - at0);
    end = share_begin(at.W, at.G, c + 1);
  }
  __device__ __forceinline__ bool valid() const { return at0 + i < end; }
  // Block i is the last of its group, or of the share.
  __device__ __forceinline__ bool last() const { return i + 1 == t.bl.n || at0 + i + 1 >= end; }
  __device__ __forceinline__ void next_group(const AttnArgs& a, int tiles) {
    i = 0;
    at0 += t.bl.n + Sh::kCost;
    if (++kh < a.pg.nkv) return;
    kh = 0;
    if (++x < a.B * tiles) t = tile_of<Sh>(a, tiles, x);
  }
  __device__ __forceinline__ void next(const AttnArgs& a, int tiles) {
    if (++i == t.bl.n) next_group(a, tiles);
  }
};

// The workspace begins with a record for every share: the group that it is
// the first to hold part of, when others hold the rest.
struct alignas(16) Cut {
  int x, kh;   // the group
  int parts;   // shares that hold part of it, this one the first (0: none)
  int second;  // whether this share's part is in its second slot
};
constexpr uint64_t cuts_bytes(int G) { return ((uint64_t)G * sizeof(Cut) + 255) / 256 * 256; }
// The record of share c, which ends at block i1 of the cursor's group.
template <typename Sh>
__device__ __forceinline__ Cut cut_of(const UnitAt& at, const Cursor<Sh>& c, int i0, int i1, int share, bool second) {
  Cut r{c.x, c.kh, 0, second ? 1 : 0};
  if (i0 == 0 && i1 < c.t.bl.n) r.parts = share_of(at.W, at.G, c.at0 + c.t.bl.n - 1) - share + 1;
  return r;
}

// A share leaves at most two partial results, in slots 2c and 2c + 1: of the
// group it begins with, and of one that begins inside it. A slot holds the
// maxima, the sums and the accumulators of a tile's rows, [D][R] (a thread
// that holds a row writes it column by column) or [R][D].
template <typename Sh>
constexpr bool kByColumn = Sh::R > 16;
template <typename Sh, int D>
constexpr int kSlotFloats = Sh::R * (D + 2);

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
using rl::add_f32x2;
using rl::ex2;
using rl::max3;
// Bits e for which j + e <= x (0 <= e < 32).
__device__ __forceinline__ uint32_t bits_upto(int x, int j) {
  const int n = x - j;
  return n < 0 ? 0u : n >= 31 ? 0xffffffffu : (2u << n) - 1u;
}
// 16 bytes, or 16 zero bytes where `bytes` is 0 (src is not read then).
__device__ __forceinline__ void cp_async_16z(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(rl::smem_u32(dst)), "l"(src), "r"(bytes)
               : "memory");
}
// The largest bf16 below a positive x, as the upper half of a float; 0 of 0.
__device__ __forceinline__ uint32_t bf16_below(float x) {
  return (uint32_t)max(__float_as_int(x) - 1, 0) & 0xffff0000u;
}
// Not 0 where either bf16 of x is infinite or NaN: an exponent of all ones
// carries into the sign's place.
__device__ __forceinline__ uint32_t odd16(uint32_t x) { return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

// ---------------------------------------------------------------- few rows
//
// Attention of few rows per sequence (single new tokens, drafted ones): a
// pass over the keys and values, bound by reading them.
//
// In a CTA each of 4 warps takes 16 keys of every unit and is its own
// pipeline: cp.async into its own ring of kStages x (16 keys, 16 values),
// scores and weighted sums on m16n8k16 matrix instructions (the up to
// 16 rows against 16 keys), running maximum and sum in registers, no
// barrier with other warps until a group's end. The products are 1/40 of
// what even these instructions can do at the rate the bytes arrive, so
// nothing is gained by a 128-row tcgen05 tile of which 4 to 16 rows are
// used. 8 kv heads of 128: one sequence of 131071 keys (537 MB) takes 99 us,
// 5.4 TB/s; 96 of up to 16384 (3.3 GB) 564 to 570 us, 5.8 TB/s; 32 of up to
// 2000 (135 MB) 32.3 us, of which the start, the groups' ends and join_kernel
// are about 10. Two CTAs an SM, as 8 warps hide what one warp's chain of load,
// product, maximum and product leaves open.
constexpr int kFewWarps = 4;
using Few = Shape<16, 64, 1>;

template <int D>
constexpr int kFewStages = D == 128 ? 3 : 6;
template <int D>
constexpr int kFewSmem = kFewStages<D> * (kFewWarps * 2 + 1) * 16 * D * 2;

template <int D>
__global__ void __launch_bounds__(kFewWarps * 32, 2)
    few_rows_kernel(const AttnArgs a, int tiles, Cut* __restrict__ cuts, float* __restrict__ ws) {
  constexpr int S = kFewStages<D>, C = D / 8;
  extern __shared__ __align__(128) uint16_t smem[];
  __shared__ float sm_m[kFewWarps][16], sm_l[kFewWarps][16];
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const UnitAt at = find_unit<Few, kFewWarps * 32>(a, tiles, gridDim.x, blockIdx.x);
  if (cuts && threadIdx.x == 0) cuts[blockIdx.x].parts = 0;
  if (at.u >= at.W) return;
  Cursor<Few> now;
  now.init(a, tiles, at, blockIdx.x);
  Cursor<Few> ahead = now;

  uint16_t* ring = smem + warp * (S * 2 * 16 * D);
  uint16_t* queries = smem + kFewWarps * S * 2 * 16 * D;  // S tiles of 16 query rows, for all warps

  // Loads of unit n (of the share) go to stage n % S, and with a group's
  // first unit its query rows, a quarter by each warp. Bit n % 32 of `held`
  // says whether this warp has anything to do in unit n.
  uint32_t held = 0;
  int issued = 0, begun = 0, page = -1;
  auto key0 = [&](const Cursor<Few>& c) { return c.t.bl.index(c.i) * Few::kBlock + warp * 16; };
  auto fetch_page = [&]() {  // the page of the unit that is loaded next
    page = -1;
    if (ahead.valid()) {
      const int j = key0(ahead);
      const Span all = ahead.t.bl.all;
      const bool any = j <= all.hi && (j + 15 >= all.lo || j < a.sinks);
      if (any) page = a.pg.table[ahead.t.b * a.pg.stride + (j >> a.pg.lg)];
    }
  };
  auto issue = [&]() {
    if (ahead.valid()) {
      if (issued == 0 || ahead.i == 0) {
        uint16_t* to = queries + (begun % S) * 16 * D;
#pragma unroll
        for (int x = 0; x < 4 * C / 32; ++x) {
          const int idx = x * 32 + lane, r = warp * 4 + idx / C, c = idx % C;
          const bool in = r < ahead.t.rows;
          cp_async_16z(to + r * D + ((c ^ (r & 7)) * 8), a.q + head_of(a, ahead.t, ahead.kh, in ? r : 0) * D + c * 8,
                       in ? 16 : 0);
        }
        ++begun;
      }
      const bool ok = (unsigned)page < (unsigned)a.pg.num_pages;
      held = (held & ~(1u << (issued & 31))) | ((ok ? 1u : 0u) << (issued & 31));
      if (ok) {
        const int j = key0(ahead);
        const int64_t row = (((int64_t)page * a.pg.nkv + ahead.kh) << a.pg.lg) + (j & ((1 << a.pg.lg) - 1));
        uint16_t* ks = ring + (issued % S) * (2 * 16 * D);
        uint16_t* vs = ks + 16 * D;
#pragma unroll
        for (int x = 0; x < 16 * C / 32; ++x) {
          const int idx = x * 32 + lane, key = idx / C, c = idx % C;
          const bool in = sees(ahead.t.bl.all, a.sinks, j + key);
          const int64_t off = (row + (in ? key : 0)) * D + c * 8;
          const int to = key * D + ((c ^ (key & 7)) * 8);
          cp_async_16z(ks + to, a.k + off, in ? 16 : 0);
          cp_async_16z(vs + to, a.v + off, in ? 16 : 0);
        }
      }
      ++issued;
      ahead.next(a, tiles);
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
  int first = 0, group = 0;
  for (int n = 0; now.valid(); ++n) {
    rl::cp_async_wait<S - 2>();
    if (n == 0 || now.i == 0) {  // a group begins
      __syncthreads();           // every warp's quarter of its query rows has arrived
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
        const int r = h * 8 + (lane >> 2);
        m[h] = -INFINITY;
        l[h] = 0.f;
        sp[h] = r < now.t.rows ? a.span(now.t.p0 + token_of(a, now.t, r)) : Span{0, -1};
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
      const bool edge = is_edge(a, now.t.p0, now.t.p1, j0, j0 + 15);
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
      if (edge && now.t.p1 > now.t.p0) {
        // A value that is not finite, of a key that some rows see and some
        // do not: 0 times it would reach the latter through the product.
        // It is added to the rows that see it and zeroed for the product.
        bool odd = false;
#pragma unroll
        for (int x = 0; x < 16 * C / 32; ++x) {
          const uint4 w = *reinterpret_cast<const uint4*>(vs + (x * 32 + lane) * 8);
          odd |= (odd16(w.x) | odd16(w.y) | odd16(w.z) | odd16(w.w)) != 0;
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
      // keep 15 bits of each weight (one alone costs as much accuracy again
      // as the rounding of the output), and the matrix pipe is idle anyway.
      // The first is cut off below the weight, so that the second is above
      // 0, too: with one of either sign, or 0, an infinite value that the
      // row sees would come out as NaN.
      uint32_t ph[4], pr[4];
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x0 = sc[y][2 * h], x1 = sc[y][2 * h + 1];
          const uint32_t h0 = bf16_below(x0), h1 = bf16_below(x1);
          ph[2 * y + h] = __byte_perm(h0, h1, 0x7632);
          pr[2 * y + h] = rl::pack_bf16x2(x0 - __uint_as_float(h0), x1 - __uint_as_float(h1));
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

    if (now.last()) {
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
      const bool whole = now.i + 1 == now.t.bl.n && now.i == n - first;
      float* slot = ws + (2 * (int64_t)blockIdx.x + (first == 0 ? 0 : 1)) * kSlotFloats<Few, D>;
      const float* part = reinterpret_cast<const float*>(smem) + (n % S) * (16 * D);
      for (int x = threadIdx.x; x < now.t.rows * (D / 4); x += kFewWarps * 32) {
        const int r = x / (D / 4), c = (x - r * (D / 4)) * 4;
        float M = sm_m[0][r];
#pragma unroll
        for (int w = 1; w < kFewWarps; ++w) M = fmaxf(M, sm_m[w][r]);
        // A row that sees nothing has sums of 0, one whose scores are all NaN
        // the same maximum and sums of NaN, which stay.
        const float base = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
          const float f = ex2(sm_m[w][r] - base);
          const float4 z = *reinterpret_cast<const float4*>(part + w * (S * 16 * D) + r * D + (c ^ ((r & 3) * 8)));
          L = fmaf(sm_l[w][r], f, L);
          y.x = fmaf(z.x, f, y.x);
          y.y = fmaf(z.y, f, y.y);
          y.z = fmaf(z.z, f, y.z);
          y.w = fmaf(z.w, f, y.w);
        }
        if (whole) {
          const float inv = L == 0.f ? 0.f : __fdiv_rn(1.f, L);
          *reinterpret_cast<uint2*>(a.out + head_of(a, now.t, now.kh, r) * D + c) =
              make_uint2(rl::pack_bf16x2(y.x * inv, y.y * inv), rl::pack_bf16x2(y.z * inv, y.w * inv));
        } else {
          *reinterpret_cast<float4*>(slot + 32 + r * D + c) = y;
          if (x == 0) cuts[blockIdx.x] = cut_of(at, now, now.i - (n - first), now.i + 1, blockIdx.x, first != 0);
          if (c == 0) {
            slot[r] = M;
            slot[16 + r] = L;
          }
        }
      }
      __syncthreads();  // before the stages, sm_m and sm_l are written again
    }
    now.next(a, tiles);
  }
}

// --------------------------------------------------------------- many rows
//
// Attention of a prompt or of a tile of drafted rows on tcgen05: scores
// S = Q K^T and sums O += P V of 128 rows against blocks of 128 keys, S, P
// and O in tensor memory. Bound by the matrix rate where d = 128 (1024
// cycles for 128 x 128 pairs), and as much by 16384 exponentials at 16 a
// cycle.
//
// Two slots of 128 rows each, so that one's products run while the other's
// weights are worked out:
//   kTwoTiles  : 256 rows a tile, a slot each half, both against every block
//                (a block's keys and values are read once for 256 rows);
//   !kTwoTiles : up to 128 rows a tile, the slots take the blocks in turn
//                and are added up at the group's end, half of the columns by
//                each slot's warps; the next group's queries are loaded
//                meanwhile.
// Roles: warps 0-3 and 4-7 the two slots' weights (a thread a row), warp 8
// loads blocks by TMA, page by page, warp 9 issues the products, warps
// 10 and 11 look through the values of blocks that some row of the tile does
// not see whole. Keys and values share a ring of kStages blocks in smem.
//
// The weights multiply the values as bf16, at most 2^-8 of a weight off and
// 2^-9.5 in the mean: two products, as for few rows, would be half as much
// tensor work again and, on the chain that bounds this, a subtraction and a
// second conversion and store per weight. The result is 2.1e-3 from 64 bits,
// where the output's own rounding is 1.6e-3.
//
// 4096 tokens, 32 heads of 128: 171 us, 800 TFLOP/s. Two times
// 2501 tokens, heads of 64, window 2048: 104 us, 405 TFLOP/s (exponentials
// alone: 36). 16 sequences of 6 tokens, 5 of them drafts, over up to 4001 keys
// (147 MB): 43 us, 3.4 TB/s. A slot's block is a chain of product, maximum,
// exponentials and product, 2500 of its 3700 cycles the weights'; the other
// slot's chain fills what one leaves. 17 to 64 rows on m16n8k16 instead,
// keys split over warps, take 105 us where this takes 43.
constexpr int kManyThreads = 12 * 32;
// Registers: the launch's 168 a thread, of which the third warpgroup (loads,
// products) keeps 72 and the weights' two take 216 (2 * 216 + 72 = 3 * 168).
constexpr int kWeightRegs = 216, kOtherRegs = 72;
constexpr int kMaxStages = 8;
template <bool kTwoTiles>
using Many = Shape<kTwoTiles ? 256 : 128, 128, kTwoTiles ? 4 : 3>;
template <int D>
constexpr int kManyStages = D == 128 ? 4 : 8;  // even: keys and values keep to stages of their own
template <int D>
constexpr int kTileBytes = 128 * D * 2;
// Two query tiles (with !kTwoTiles one group's and the next one's), the ring,
// and slack to start at a multiple of 1024.
template <int D>
constexpr int kManySmem = (2 + kManyStages<D>) * kTileBytes<D> + 1024;

struct ManyBars {
  uint64_t full[kMaxStages], empty[kMaxStages], ok[kMaxStages];  // loaded, read, looked through (values)
  uint64_t q_full, s_full[2], p_full[2][2], pv_done[2], merge_full, merge_empty, drain;  // p_full: slot, half
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
  return __all_sync(0xffffffffu, rl::mbar_wait(bar, parity, abort, status));
}
// True in one lane of the (converged) warp, in a way the compiler knows.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// A bounded wait for work in flight on the way out.
__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = rl::globaltimer_ns();
  while (!rl::mbar_try_wait_suspend(bar, parity, 2000u))
    if (rl::globaltimer_ns() - t0 > rl::kWaitLimitNs) return;
}

// The part of a group that a share holds: blocks [i0, i1).
template <typename Sh>
struct Segments {
  Cursor<Sh> c;
  int i0, i1;
  __device__ __forceinline__ bool take() {
    i0 = c.i;
    i1 = (int)min((int64_t)c.t.bl.n, c.end - c.at0);
    return c.valid();
  }
  // False where the share holds no block.
  __device__ __forceinline__ bool init(const AttnArgs& a, int tiles, const UnitAt& at, int share) {
    c.init(a, tiles, at, share);
    return take();
  }
  __device__ __forceinline__ bool next(const AttnArgs& a, int tiles) {
    c.next_group(a, tiles);
    return take();
  }
};

template <int D, bool kTwoTiles>
__global__ void __launch_bounds__(kManyThreads, 1)
    many_rows_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, int tiles, Cut* __restrict__ cuts,
                     float* __restrict__ ws, int* status) {
  using Sh = Many<kTwoTiles>;
  constexpr int S = kManyStages<D>, H = D / 64, kHalf = 128 * 128;  // a tile is H column halves of 128 x 128 B
  extern __shared__ uint8_t smem_raw[];
  __shared__ ManyBars bars;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  __shared__ uint32_t gone[8];    // block n % 8: its pages that are not held, or that nobody sees
  __shared__ int poison[16];      // segment n % 16: a value that some rows must not meet is not finite
  __shared__ Segments<Sh> at_seg[8], at_next[8];  // of each weights' warp: its registers are for weights
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* qs = smem;  // 2 tiles
  uint8_t* ring = smem + 2 * kTileBytes<D>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  volatile int* abort = &abort_flag;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kMaxStages; ++i) {
      rl::mbar_init(&bars.full[i], 1);
      rl::mbar_init(&bars.empty[i], 1);
      rl::mbar_init(&bars.ok[i], 2);
    }
    rl::mbar_init(&bars.q_full, 8);
    for (int i = 0; i < 2; ++i) {
      rl::mbar_init(&bars.s_full[i], 1);
      rl::mbar_init(&bars.p_full[i][0], 4);
      rl::mbar_init(&bars.p_full[i][1], 4);
      rl::mbar_init(&bars.pv_done[i], 1);
    }
    rl::mbar_init(&bars.merge_full, 8);
    rl::mbar_init(&bars.merge_empty, 8);
    rl::mbar_init(&bars.drain, 1);
    rl::fence_mbar_init();
    abort_flag = 0;
    for (int i = 0; i < 16; ++i) poison[i] = 0;
  }
  if (warp == 9) {
    rl::tmem_alloc(&tmem_base, 512);
    rl::tmem_relinquish();
  }
  rl::tc_fence_before();
  __syncthreads();
  rl::tc_fence_after();
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const uint32_t tm = tmem_base;

  const UnitAt at = find_unit<Sh, kManyThreads>(a, tiles, gridDim.x, blockIdx.x);
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    Segments<Sh> sg;
    const bool work = at.u < at.W && sg.init(a, tiles, at, blockIdx.x);
    if (cuts && !work && warp == 8 && lane == 0) cuts[blockIdx.x].parts = 0;
    if (work && warp == 8) {
      // ------------------------------------------------ loads
      const int per_page = 1 << a.pg.lg, pages = 128 >> a.pg.lg;
      const int none = (int)((int64_t)a.pg.num_pages * a.pg.nkv << a.pg.lg);  // past the pool: zeros
      int n = 0;  // blocks so far; its keys are load 2n of the ring, its values 2n + 1
      int loads = 0;
      bool go = true;
      do {
        for (int i = sg.i0; go && i < sg.i1; ++i, ++n) {
          const int j = sg.c.t.bl.index(i) * 128 + (lane << a.pg.lg);
          int row = none;
          if (lane < pages && j <= sg.c.t.bl.all.hi && (j + per_page > sg.c.t.bl.all.lo || j < a.sinks)) {
            const int64_t r = a.pg.row(sg.c.t.b, sg.c.kh, j);
            if (r >= 0) row = (int)r;
          }
          const uint32_t bad = __ballot_sync(0xffffffffu, lane < pages && row == none);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const int ld = 2 * n + kv, st = ld % S;
            if (ld >= S && !warp_wait(&bars.empty[st], (ld / S - 1) & 1, abort, status)) {
              go = false;
              break;
            }
            if (lane == 0) {
              // Its last reader has given block n - 8's values back.
              if (kv == 0) *(volatile uint32_t*)&gone[n & 7] = bad;
              rl::mbar_arrive_expect_tx(&bars.full[st], kTileBytes<D>);
            }
            __syncwarp();
            ++loads;
            if (lane < pages) {
              uint8_t* to = ring + st * kTileBytes<D> + lane * per_page * 128;
#pragma unroll
              for (int h = 0; h < H; ++h)
                rl::tma_load_2d(to + h * kHalf, kv ? &vmap : &kmap, &bars.full[st], h * 64, row);
            }
          }
        }
      } while (go && sg.next(a, tiles));
      if (!go) {  // loads in flight end before the CTA does
        for (int ld = max(0, loads - S); ld < loads; ++ld) drain_wait(&bars.full[ld % S], (ld / S) & 1);
      }
    } else if (work && warp == 9) {
      // --------------------------------------------- products
      // The whole warp walks the blocks, so that descriptors are uniform; one
      // lane issues. Descriptors of one tile differ in their start address
      // alone (the low word).
      {
        constexpr uint32_t kIdS = rl::idesc_bf16_f32(128, 128);
        constexpr uint32_t kIdO = rl::idesc_bf16_f32(128, D) | (1u << 16);  // B (the values) MN-major
        const bool leader = elect_one();
        const uint64_t q_desc = rl::sdesc_kmajor_sw128(rl::smem_u32(qs));
        const uint64_t k_desc = rl::sdesc_kmajor_sw128(rl::smem_u32(ring));
        const uint64_t v_desc = rl::sdesc_mnmajor_sw128(rl::smem_u32(ring), kHalf);
        int n0 = 0, seg = 0;  // blocks before this segment, segments
        auto scores = [&](int slot, int st) {
          const uint64_t qd = q_desc + (kTwoTiles ? slot : seg & 1) * (kTileBytes<D> >> 4), kd = k_desc + st * (kTileBytes<D> >> 4);
          if (leader) {
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
              const uint32_t off = ((x / 4) * kHalf + (x % 4) * 32) >> 4;
              rl::tc_mma_ss(tm + slot * 128, qd + off, kd + off, kIdS, x > 0);
            }
            rl::tc_commit(&bars.s_full[slot]);
          }
          __syncwarp();
        };
        uint32_t pc[2] = {0, 0};  // blocks of each slot whose weights were waited for
        auto sums = [&](int slot, int st, bool add) {
          const uint64_t vd = v_desc + st * (kTileBytes<D> >> 4);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!warp_wait(&bars.p_full[slot][h], pc[slot] & 1, abort, status)) return false;
            rl::tc_fence_after();
            if (leader) {
#pragma unroll
              for (int x = 4 * h; x < 4 * h + 4; ++x)
                rl::tc_mma_ts(tm + 256 + slot * D, tm + slot * 128 + x * 8, vd + x * (2048 >> 4), kIdO, add || x > 0);
              if (h == 1) rl::tc_commit(&bars.pv_done[slot]);
            }
            __syncwarp();
          }
          ++pc[slot];
          return true;
        };
        auto release = [&](int st) {
          if (leader) rl::tc_commit(&bars.empty[st]);
          __syncwarp();
        };
        bool go = true;
        do {
          const int nb = sg.i1 - sg.i0;
          go = warp_wait(&bars.q_full, seg & 1, abort, status);
          rl::tc_fence_after();
          // Little may come between a slot's last product and the next one
          // that can be issued: what can be waited for is waited for while
          // products are queued.
          if constexpr (kTwoTiles) {
            auto loaded = [&](int j) {  // block j's keys and block j - 1's values
              const int kl = 2 * (n0 + j), vl = kl - 1;
              return (j >= nb || warp_wait(&bars.full[kl % S], (kl / S) & 1, abort, status)) &&
                     (j == 0 || warp_wait(&bars.ok[vl % S], (vl / S) & 1, abort, status));
            };
            go = go && loaded(0);
            if (go) scores(0, 2 * n0 % S);
            if (go) {
              scores(1, 2 * n0 % S);
              release(2 * n0 % S);
            }
            go = go && loaded(1);
            for (int j = 1; go && j <= nb; ++j) {
              const int kl = 2 * (n0 + j), vl = kl - 1;
              go = sums(0, vl % S, j > 1);
              if (go && j < nb) scores(0, kl % S);
              go = go && sums(1, vl % S, j > 1);
              if (go) release(vl % S);
              if (go && j < nb) {
                scores(1, kl % S);
                release(kl % S);
              }
              go = go && (j == nb || loaded(j + 1));
            }

          } else {
            for (int j = 0; go && j < nb + 2; ++j) {
              const int slot = j & 1;
              if (j >= 2) {  // block j - 2
                const int vl = 2 * (n0 + j - 2) + 1;
                go = warp_wait(&bars.ok[vl % S], (vl / S) & 1, abort, status) && sums(slot, vl % S, j >= 4);
                if (!go) break;
                release(vl % S);
              }
              if (j < nb) {
                const int kl = 2 * (n0 + j);
                go = warp_wait(&bars.full[kl % S], (kl / S) & 1, abort, status);
                if (!go) break;
                scores(slot, kl % S);
                release(kl % S);
              }
              if (nb == 1 && j == 0) ++j;  // slot 1 has no block
            }
          }
          n0 += nb;
          ++seg;
        } while (go && sg.next(a, tiles));
        if (leader) rl::tc_commit(&bars.drain);  // nothing in flight when tensor memory is freed
        __syncwarp();
        drain_wait(&bars.drain, 0);
      }
    } else if (work) {
      // ------------------------------------- values looked through
      int n = 0, seg = 0;
      bool go = true;
      do {
        // The last segment's is the one that stays.
        if (cuts && warp == 10 && lane == 0) cuts[blockIdx.x] = cut_of(at, sg.c, sg.i0, sg.i1, blockIdx.x, seg > 0);
        for (int i = sg.i0; go && i < sg.i1; ++i, ++n) {
          const int ld = 2 * n + 1, st = ld % S, j0 = sg.c.t.bl.index(i) * 128;
          go = warp_wait(&bars.full[st], (ld / S) & 1, abort, status);
          if (!go) break;
          if (is_edge(a, sg.c.t.p0, sg.c.t.p1, j0, j0 + 127)) {
            // A weight of 0 times a value that is not finite is not 0. Such
            // values are zeroed; where some row does see their key, the
            // group's end adds them to the rows that do.
            uint4* v = reinterpret_cast<uint4*>(ring + st * kTileBytes<D>);
            bool any = false;
#pragma unroll 1
            for (int x = (warp - 10) * 32 + lane; x < kTileBytes<D> / 16; x += 4 * 64) {
              uint4 w[4];
              uint32_t odd[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) w[y] = v[x + y * 64];
              uint32_t all = 0;
#pragma unroll
              for (int y = 0; y < 4; ++y) all |= odd[y] = odd16(w[y].x) | odd16(w[y].y) | odd16(w[y].z) | odd16(w[y].w);
              if (!all) continue;
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                if (!odd[y]) continue;
                uint16_t* e = reinterpret_cast<uint16_t*>(&v[x + y * 64]);
                for (int z = 0; z < 8; ++z)
                  if ((e[z] & 0x7f80u) == 0x7f80u) e[z] = 0;
                any |= sees(sg.c.t.bl.all, a.sinks, j0 + ((x + y * 64) % (kHalf / 16)) / 8);
              }
            }
            if (__any_sync(0xffffffffu, any) && lane == 0) *(volatile int*)&poison[seg & 15] = 1;
            rl::fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) rl::mbar_arrive(&bars.ok[st]);  // each of the two warps
        }
        // The weights' warps are at most 5 segments behind (a segment has a
        // block or more, the ring holds 4 at most).
        if (warp == 10 && lane == 0) *(volatile int*)&poison[(seg + 8) & 15] = 0;
        ++seg;
      } while (go && sg.next(a, tiles));
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWeightRegs));
    Segments<Sh>& sg = at_seg[warp];
    int work = 0;
    if (lane == 0) {
      Segments<Sh> first;
      work = at.u < at.W && first.init(a, tiles, at, blockIdx.x);
      sg = first;
    }
    work = __shfl_sync(0xffffffffu, work, 0);
    if (work) {
      // ---------------------------------------------- weights
      const int slot = warp >> 2, wr = warp & 3;
      const uint32_t lane_off = (uint32_t)(wr * 32) << 16;
      const uint32_t ts = tm + slot * 128 + lane_off, to = tm + 256 + slot * D + lane_off;
      const int r = (kTwoTiles ? slot * 128 : 0) + wr * 32 + lane;  // row of the tile
      int seg = 0, n0 = 0;  // segments, blocks before this one
      uint32_t sc = 0;      // blocks of this slot so far: phases of s_full and pv_done
      bool go = true;
      // A segment's query rows, 32 by this warp (16 with one tile), 16 bytes a
      // lane.
      auto load_q = [&](const Tile& t, int kh, int segment) {
        constexpr int kRowsPerWarp = kTwoTiles ? 32 : 16, C = D / 8;
        uint8_t* tile = qs + (kTwoTiles ? slot : segment & 1) * kTileBytes<D>;
#pragma unroll
        for (int x = 0; x < kRowsPerWarp * C / 32; ++x) {
          const int rr = warp * kRowsPerWarp + (x * 32 + lane) / C, c = lane % C, lr = rr & 127;
          const bool have = rr < t.rows;
          cp_async_16z(tile + (c / 8) * kHalf + lr * 128 + (((c & 7) ^ (lr & 7)) * 16),
                       a.q + head_of(a, t, kh, have ? rr : 0) * D + c * 8, have ? 16 : 0);
        }
        rl::cp_async_commit();
      };
      do {
        const Tile& t = sg.c.t;
        const int nb = sg.i1 - sg.i0;
        if (kTwoTiles || seg == 0) load_q(t, sg.c.kh, seg);
        rl::cp_async_wait<0>();
        rl::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) rl::mbar_arrive(&bars.q_full);
        const bool in = r < t.rows;
        const Span sp = in ? a.span(t.p0 + token_of(a, t, r)) : Span{0, -1};
        // Blocks that every row of this warp sees whole end at most at
        // whole_hi, and begin at whole_lo or later, or lie in the sinks.
        const int w0 = r - lane, w1 = min(w0 + 31, t.rows - 1);
        const int whole_hi = w1 < w0 ? -1 : a.span(t.p0 + token_of(a, t, w0)).hi;
        const int whole_lo = w1 < w0 ? 0 : a.span(t.p0 + token_of(a, t, w1)).lo;
        float m = -INFINITY, l = 0.f;  // maximum (of scaled scores) that the weights are relative to, and their sum
        int done = 0;                  // blocks of this segment
        const int i0 = sg.i0, i1 = sg.i1;
        for (int i = i0 + (kTwoTiles ? 0 : slot); i < i1; i += kTwoTiles ? 1 : 2) {
          const int j0 = t.bl.index(i) * 128;
          go = warp_wait(&bars.s_full[slot], sc & 1, abort, status);
          if (!go) break;
          rl::tc_fence_after();
          uint32_t x[4][32];
#pragma unroll
          for (int y = 0; y < 4; ++y) rl::tmem_ld_32x32b_x32(ts + y * 32, x[y]);
          rl::tmem_wait_ld();
          // Pages that are not held are loaded as zeros; their scores go too.
          const uint32_t bad = *(volatile uint32_t*)&gone[(n0 + i - i0) & 7];
          if (bad || j0 + 127 > whole_hi || (j0 < whole_lo && j0 + 127 >= a.sinks)) {
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int j = j0 + y * 32;
              uint32_t see = bits_upto(sp.hi, j) & (~bits_upto(sp.lo - 1, j) | bits_upto(a.sinks - 1, j));
              if (a.pg.lg == 4)
                see &= (bad >> (2 * y) & 1 ? 0xffff0000u : 0xffffffffu) & (bad >> (2 * y + 1) & 1 ? 0xffffu : 0xffffffffu);
              else if (bad >> (y * 32 >> a.pg.lg) & 1)
                see = 0;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(see >> e & 1)) x[y][e] = 0xff800000u;
            }
          }
          float top[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            top[y] = __uint_as_float(x[y][0]);
#pragma unroll
            for (int e = 1; e < 31; e += 2)
              top[y] = max3(top[y], __uint_as_float(x[y][e]), __uint_as_float(x[y][e + 1]));
            top[y] = fmaxf(top[y], __uint_as_float(x[y][31]));
          }
          const float mb = fmaxf(max3(top[0], top[1], top[2]), top[3]) * a.scale_log2;
          if (done == 0) {
            m = mb;
          } else if (__any_sync(0xffffffffu, mb > m + 8.f)) {
            // Weights may exceed 1 (by up to 2^8) before the sums so far are
            // brought down to a new maximum: that rarely happens then (the
            // running maximum of Milakov and Gimelshein, 2018, and a
            // threshold, which is published for attention on tensor memory).
            const float mn = mb > m + 8.f ? mb : m;
            const float f = m == mn ? 1.f : ex2(m - mn);
            m = mn;
            l *= f;
            go = warp_wait(&bars.pv_done[slot], (sc - 1) & 1, abort, status);
            if (!go) break;
            rl::tc_fence_after();
#pragma unroll
            for (int y = 0; y < D / 32; ++y) {
              uint32_t v[32];
              rl::tmem_ld_32x32b_x32(to + y * 32, v);
              rl::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
              rl::tmem_st_32x32b_x32(to + y * 32, v);
            }
            rl::tmem_wait_st();
          }
          const float base = m == -INFINITY ? 0.f : m;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t p[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const int f = y * 64 + 2 * e;
              float e0, e1;
              rl::fma_f32x2(e0, e1, __uint_as_float(x[f / 32][f % 32]), __uint_as_float(x[f / 32][f % 32 + 1]),
                            a.scale_log2, a.scale_log2, -base, -base);
              e0 = ex2(e0);
              e1 = ex2(e1);
              add_f32x2(sum[2 * (e & 1)], sum[2 * (e & 1) + 1], e0, e1);
              p[e] = rl::pack_bf16x2(e0, e1);
            }
            // A half of the weights at a time, so that their products begin.
            rl::tmem_st_32x32b_x32(ts + y * 32, p);
            rl::tmem_wait_st();
            rl::tc_fence_before();
            __syncwarp();
            if (lane == 0) rl::mbar_arrive(&bars.p_full[slot][y]);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          ++sc;
          ++done;
        }
        if (!go) break;
        // The group ends, or this CTA's share of it. The next one is found
        // while the last products run; with one tile its queries go where
        // those of the group before this one were.
        int more = 0;
        if (lane == 0) {
          Segments<Sh> after = sg;
          more = after.next(a, tiles);
          at_next[warp] = after;
        }
        __syncwarp();
        more = __shfl_sync(0xffffffffu, more, 0);
        if (!kTwoTiles && more) load_q(at_next[warp].c.t, at_next[warp].c.kh, seg + 1);
        if (done) {
          go = warp_wait(&bars.pv_done[slot], (sc - 1) & 1, abort, status);
          if (!go) break;
          rl::tc_fence_after();
        }
        const bool whole = sg.i0 == 0 && sg.i1 == t.bl.n;
        bool odd = false;
        float* part = ws + (2 * (int64_t)blockIdx.x + (seg == 0 ? 0 : 1)) * kSlotFloats<Sh, D>;
        float f0 = 1.f, f1 = 0.f;  // factors of the slots' sums
        if constexpr (!kTwoTiles) {
          // Both slots' sums are where either's warps can read them: a warp
          // adds up half of the columns of its rows. Maxima and sums go by
          // way of the query tile: when a slot's last block is done, so are
          // all products of scores.
          float* ml = reinterpret_cast<float*>(qs + (seg & 1) * kTileBytes<D>);
          if (done) {
            ml[slot * 256 + r] = m;
            ml[slot * 256 + 128 + r] = l;
          }
          rl::tc_fence_before();
          __syncwarp();
          if (lane == 0) rl::mbar_arrive(&bars.merge_full);
          go = warp_wait(&bars.merge_full, seg & 1, abort, status);
          if (!go) break;
          rl::tc_fence_after();
          const float m0 = ml[r], m1 = nb > 1 ? ml[256 + r] : -INFINITY;  // slot 1 has no block of one
          m = fmaxf(m0, m1);
          const float base = m == -INFINITY ? 0.f : m;
          f0 = ex2(m0 - base);
          f1 = ex2(m1 - base);
          l = ml[128 + r] * f0;
          if (nb > 1) l = fmaf(ml[384 + r], f1, l);
        }
        // Here every block of the segment has been multiplied, the other
        // slot's too, so it has been looked through.
        odd = *(volatile int*)&poison[seg & 15] != 0;
        if (!whole && in && (kTwoTiles || slot == 0)) {
          part[r] = m;
          part[Sh::R + r] = l;
        }
        constexpr int kPieces = kTwoTiles ? D / 32 : D / 64;  // of 32 columns
        const int y0 = kTwoTiles ? 0 : slot * kPieces;
        const bool rows = w0 < t.rows;  // of this warp
#pragma unroll 1
        for (int y = y0; rows && y < y0 + kPieces; ++y) {
          uint32_t v[32];
          if constexpr (kTwoTiles) {
            rl::tmem_ld_32x32b_x32(to + y * 32, v);
            rl::tmem_wait_ld();
          } else {
            rl::tmem_ld_32x32b_x32(tm + 256 + lane_off + y * 32, v);
            rl::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f0);
            if (nb > 1) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t u[16];
                rl::tmem_ld_32x32b_x16(tm + 256 + lane_off + D + y * 32 + h * 16, u);
                rl::tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  v[h * 16 + e] = __float_as_uint(fmaf(__uint_as_float(u[e]), f1, __uint_as_float(v[h * 16 + e])));
              }
            }
          }
          if (!in) continue;
          if (odd) {
            for (int i = sg.i0; i < sg.i1; ++i) {
              const int j0 = t.bl.index(i) * 128;
              if (!is_edge(a, t.p0, t.p1, j0, j0 + 127)) continue;
              for (int j = j0; j < j0 + 128; ++j) {
                const int64_t row = sees(sp, a.sinks, j) ? a.pg.row(t.b, sg.c.kh, j) : -1;
                if (row < 0) continue;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float f = bf2f(a.v[row * D + y * 32 + e]);
                  if (!isfinite(f)) v[e] = __float_as_uint(__uint_as_float(v[e]) + f);
                }
              }
            }
          }
          if (whole) {
            const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
            // Two tiles: by way of the slot's query tile, whose products are
            // done, to write whole rows at a time.
            uint16_t* o = a.out + head_of(a, t, sg.c.kh, r) * D + y * 32;
            uint8_t* row = qs + slot * kTileBytes<D> + (y / 2) * kHalf + (r & 127) * 128;
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 w;
              w.x = rl::pack_bf16x2(__uint_as_float(v[e]) * inv, __uint_as_float(v[e + 1]) * inv);
              w.y = rl::pack_bf16x2(__uint_as_float(v[e + 2]) * inv, __uint_as_float(v[e + 3]) * inv);
              w.z = rl::pack_bf16x2(__uint_as_float(v[e + 4]) * inv, __uint_as_float(v[e + 5]) * inv);
              w.w = rl::pack_bf16x2(__uint_as_float(v[e + 6]) * inv, __uint_as_float(v[e + 7]) * inv);
              if (kTwoTiles)
                *reinterpret_cast<uint4*>(row + ((((y & 1) * 4 + e / 8) ^ (r & 7)) * 16)) = w;
              else
                *reinterpret_cast<uint4*>(o + e) = w;
            }
          } else {
            float* o = part + 2 * Sh::R + y * 32 * Sh::R + r;
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e * Sh::R] = __uint_as_float(v[e]);
          }
        }
        if (kTwoTiles && whole) {
          constexpr int C = D / 8;
          __syncwarp();
#pragma unroll
          for (int x = 0; x < C; ++x) {
            const int rr = w0 + (x * 32 + lane) / C, c = lane % C, lr = rr & 127;
            if (rr < t.rows)
              *reinterpret_cast<uint4*>(a.out + head_of(a, t, sg.c.kh, rr) * D + c * 8) = *reinterpret_cast<const uint4*>(
                  qs + slot * kTileBytes<D> + (c / 8) * kHalf + lr * 128 + (((c & 7) ^ (lr & 7)) * 16));
          }
          __syncwarp();
        }
        rl::tc_fence_before();  // the next group's first product overwrites O
        if constexpr (!kTwoTiles) {
          __syncwarp();
          if (lane == 0) rl::mbar_arrive(&bars.merge_empty);
          go = warp_wait(&bars.merge_empty, seg & 1, abort, status);
          if (!go) break;
        }
        n0 += nb;
        ++seg;
        __syncwarp();
        if (lane == 0) sg = at_next[warp];
        __syncwarp();
        work = more;
      } while (work);
    }
  }
  rl::tc_fence_before();
  __syncthreads();
  rl::tc_fence_after();
  if (warp == 9) rl::tmem_dealloc(tm, 512);
}

// CTA (c, y, z) adds up kRows rows from kRows y on, 4 kCols kPieces columns
// from there times z on, of the partial results of the group that share c's
// record names. A thread takes 4 columns of a row, kPieces times; where a
// group has many parts and few rows, several threads share its parts. Bound by
// latency, so what a CTA does is as much as keeps all CTAs in one wave: 256
// rows of 128 columns in 32 CTAs of one piece take 2 to 4 us more than in 8
// of four (4096 tokens 175 and 172 us, 128 tokens 17.7 and 14.1), and a CTA
// for all columns of 16 or 128 rows, with a thread for all parts, 3 us more
// (131071 keys, 37 parts a group) to 5 (drafted tokens) than this.
constexpr int kMaxShares = 320, kJoinThreads = 256;
template <typename Sh, int D>
constexpr int kJoinPieces = Sh::R == 256 ? D / 32 : 1;
template <typename Sh, int D>
struct Join {
  static constexpr bool kMany = kByColumn<Sh>;
  static constexpr int kRows = kMany ? 32 : 2;
  static constexpr int kCols = kMany ? 8 : D / 4;
  static constexpr int kShared = kJoinThreads / (kRows * kCols);
  static constexpr int kPieces = kJoinPieces<Sh, D>;  // of 4 columns, a thread
  static constexpr int kZ = D / (4 * kCols * kPieces);
  static constexpr int kPer = kMany ? kJoinThreads / kRows : 32;  // threads that work out a row's weights
};
template <typename Sh, int D>
__global__ void __launch_bounds__(kJoinThreads)
    join_kernel(const AttnArgs a, int tiles, const Cut* __restrict__ cuts, const float* __restrict__ ws) {
  using J = Join<Sh, D>;
  constexpr int kSlot = kSlotFloats<Sh, D>;
  __shared__ float weight[J::kRows][kMaxShares / (J::kMany ? 2 : 1) + 1];  // of the parts
  __shared__ float4 red[J::kShared > 1 ? kJoinThreads : 1];
  rl::pdl_wait();
  rl::pdl_launch_dependents();
  const int c0 = blockIdx.x, row0 = blockIdx.y * J::kRows, tid = threadIdx.x;
  const Cut cut = cuts[c0];
  const int parts = cut.parts;
  if (parts == 0) return;
  const Tile t = tile_of<Sh>(a, tiles, cut.x);
  const int rows = min(J::kRows, t.rows - row0);
  if (rows <= 0) return;
  const float* first = ws + (2 * (int64_t)c0 + cut.second) * kSlot;
  const float* rest = ws + 2 * (int64_t)c0 * kSlot;
  {
    const int r = tid / J::kPer, i0 = tid % J::kPer;
    const bool have = r < rows;
    auto part_of = [&](int i) { return (i ? rest + (int64_t)i * 2 * kSlot : first) + row0 + r; };
    // A thread's first part, usually its only one, stays in registers.
    const bool any = have && i0 < parts;
    const float m0 = any ? __ldcg(part_of(i0)) : -INFINITY, l0 = any ? __ldcg(part_of(i0) + Sh::R) : 0.f;
    float M = m0;
    if (have)
      for (int i = i0 + J::kPer; i < parts; i += J::kPer) {
        const float x = __ldcg(part_of(i));
        weight[r][i] = x;
        M = fmaxf(M, x);
      }
#pragma unroll
    for (int o = J::kPer / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float base = M == -INFINITY ? 0.f : M, f0 = ex2(m0 - base);
    float den = f0 * l0;
    if (any) weight[r][i0] = f0;
    if (have)
      for (int i = i0 + J::kPer; i < parts; i += J::kPer) {
        const float f = ex2(weight[r][i] - base);
        weight[r][i] = f;
        den = fmaf(f, __ldcg(part_of(i) + Sh::R), den);
      }
#pragma unroll
    for (int o = J::kPer / 2; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
    const float inv = den == 0.f ? 0.f : __fdiv_rn(1.f, den);
    if (have)
      for (int i = i0; i < parts; i += J::kPer) weight[r][i] *= inv;
  }
  __syncthreads();
  // Neighbours hold neighbouring rows where the parts are stored by column.
  const int r = J::kMany ? tid % J::kRows : tid / J::kCols % J::kRows;
  const int col0 = (blockIdx.z * J::kCols * J::kPieces + (J::kMany ? tid / J::kRows : tid % J::kCols)) * 4;
  const int turn = J::kMany ? 0 : tid / (J::kRows * J::kCols);
  float4 y[J::kPieces];
#pragma unroll
  for (int x = 0; x < J::kPieces; ++x) y[x] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (r < rows) {
#pragma unroll 8 / J::kPieces
    for (int i = turn; i < parts; i += J::kShared) {
      const float* p = (i ? rest + (int64_t)i * 2 * kSlot : first) + 2 * Sh::R;
      float4 z[J::kPieces];
#pragma unroll
      for (int x = 0; x < J::kPieces; ++x) {
        const int c = col0 + x * J::kCols * 4;
        if (J::kMany) {
          const float* e = p + c * Sh::R + row0 + r;
          z[x] = make_float4(__ldcg(e), __ldcg(e + Sh::R), __ldcg(e + 2 * Sh::R), __ldcg(e + 3 * Sh::R));
        } else {
          z[x] = __ldcg(reinterpret_cast<const float4*>(p + (row0 + r) * D + c));
        }
      }
      const float w = weight[r][i];
#pragma unroll
      for (int x = 0; x < J::kPieces; ++x) {
        y[x].x = fmaf(w, z[x].x, y[x].x);
        y[x].y = fmaf(w, z[x].y, y[x].y);
        y[x].z = fmaf(w, z[x].z, y[x].z);
        y[x].w = fmaf(w, z[x].w, y[x].w);
      }
    }
  }
  if (J::kShared > 1) {
    red[tid] = y[0];
    __syncthreads();
    if (turn) return;
    for (int i = 1; i < J::kShared; ++i) {
      const float4 z = red[i * J::kRows * J::kCols + tid];
      y[0].x += z.x, y[0].y += z.y, y[0].z += z.z, y[0].w += z.w;
    }
  }
  if (r < rows)
#pragma unroll
    for (int x = 0; x < J::kPieces; ++x)
      *reinterpret_cast<uint2*>(a.out + head_of(a, t, cut.kh, row0 + r) * D + col0 + x * J::kCols * 4) =
          make_uint2(rl::pack_bf16x2(y[x].x, y[x].y), rl::pack_bf16x2(y[x].z, y[x].w));
}

// The kernel for a call, its row tiles and CTAs, and whether a group can be
// cut at all.
struct Plan {
  enum { kFew, kOneTile, kTwoTile } kind;
  int tiles, G, R;
  bool join;
  uint64_t ws_bytes;
};
Plan make_plan(int num_sms, int B, int T, int nh, int nkv, int d, int64_t cap) {
  Plan p;
  const int64_t rows = (int64_t)T * (nh / nkv);
  p.kind = rows <= 16 ? Plan::kFew : rows <= 128 ? Plan::kOneTile : Plan::kTwoTile;
  p.R = p.kind == Plan::kFew ? Few::R : p.kind == Plan::kOneTile ? 128 : 256;
  const int block = p.kind == Plan::kFew ? Few::kBlock : 128;
  p.tiles = (int)((rows + p.R - 1) / p.R);
  const int64_t blocks = (cap + block - 1) / block;
  const int64_t most = (int64_t)B * nkv * p.tiles * blocks;
  p.G = (int)std::min<int64_t>(p.kind == Plan::kFew ? std::min(2 * num_sms, kMaxShares) : std::min(num_sms, kMaxShares / 2), most);
  p.join = blocks > 1 && p.G > 1;
  p.ws_bytes = p.join ? cuts_bytes(p.G) + (uint64_t)2 * p.G * p.R * (d + 2) * sizeof(float) : 0;
  return p;
}

// The workspace of a call: records, then partial results (NULL where no group
// can be cut).
struct Space {
  Cut* cuts;
  float* slots;
};

template <typename Sh, int D>
int32_t launch_join(riallm_ctx* ctx, const AttnArgs& a, const Plan& p, const Space& ws, cudaStream_t st) {
  if (!p.join) return RIALLM_OK;
  // The last share is nobody's first of several.
  const int rows = std::min<int64_t>(Sh::R, (int64_t)a.T * a.rep);
  return rl::launched(ctx, "paged_attention",
                      rl::launch_pdl(join_kernel<Sh, D>,
                                     dim3(p.G - 1, (rows + Join<Sh, D>::kRows - 1) / Join<Sh, D>::kRows, Join<Sh, D>::kZ),
                                     dim3(kJoinThreads), 0, st, a, p.tiles, static_cast<const Cut*>(ws.cuts),
                                     static_cast<const float*>(ws.slots)));
}

template <int D>
int32_t launch_few(riallm_ctx* ctx, const AttnArgs& a, const Plan& p, const Space& ws, cudaStream_t st) {
  const char* what = "paged_attention";
  if (int s = rl::allow_smem(ctx, what, few_rows_kernel<D>, kFewSmem<D>, D / 64 - 1)) return s;
  if (int s = rl::launched(ctx, what,
                           rl::launch_pdl(few_rows_kernel<D>, dim3(p.G), dim3(kFewWarps * 32), kFewSmem<D>, st, a,
                                          p.tiles, ws.cuts, ws.slots)))
    return s;
  return launch_join<Few, D>(ctx, a, p, ws, st);
}

template <int D, bool kTwoTiles>
int32_t launch_many(riallm_ctx* ctx, const AttnArgs& a, const Plan& p, const Space& ws, cudaStream_t st) {
  const char* what = "paged_attention";
  const auto kernel = many_rows_kernel<D, kTwoTiles>;
  if (int s = rl::allow_smem(ctx, what, kernel, kManySmem<D>, 2 + (D / 64 - 1) * 2 + kTwoTiles)) return s;
  CUtensorMap map[2];
  for (int i = 0; i < 2; ++i) {
    const CUresult r = rl::encode_tensor_map_2d(&map[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, i ? a.v : a.k, D,
                                                (uint64_t)a.pg.num_pages * a.pg.nkv << a.pg.lg, D * 2, 64,
                                                1u << a.pg.lg, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r != CUDA_SUCCESS) return rl::refuse(ctx, RIALLM_ERR_CUDA, what, "cuTensorMapEncodeTiled");
  }
  if (int s = rl::launched(ctx, what,
                           rl::launch_pdl(kernel, dim3(p.G), dim3(kManyThreads), kManySmem<D>, st, a, map[0], map[1],
                                          p.tiles, ws.cuts, ws.slots, ctx->d_status)))
    return s;
  return launch_join<Many<kTwoTiles>, D>(ctx, a, p, ws, st);
}

template <int D>
int32_t launch_attention(riallm_ctx* ctx, const AttnArgs& a, const Plan& p, const Space& ws, cudaStream_t st) {
  return p.kind == Plan::kFew       ? launch_few<D>(ctx, a, p, ws, st)
         : p.kind == Plan::kOneTile ? launch_many<D, false>(ctx, a, p, ws, st)
                                    : launch_many<D, true>(ctx, a, p, ws, st);
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool is_page_size(int32_t n) { return n == 16 || n == 32 || n == 64 || n == 128; }

// What both entry points share: the checks of the cache's geometry.
template <typename Args>
int check_pages(riallm_ctx* ctx, const char* what, const Args& x) {
  const int32_t B = x.B, T = x.T, nh = x.nh, nkv = x.nkv, d = x.d, page_size = x.page_size;
  auto bad = [&](const char* msg) { return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, msg); };
  if (B < 0 || T < 0 || nh <= 0 || nkv <= 0 || nh % nkv != 0)
    return bad("bad dimensions (heads must be a multiple of kv heads)");
  if (nh / nkv > 128) return bad("more than 128 heads per kv head");
  if (d != 64 && d != 128) return bad("head_dim must be 64 or 128");
  if (!is_page_size(page_size)) return bad("page_size must be 16, 32, 64 or 128");
  if (x.num_pages <= 0 || x.max_pages <= 0 || x.table_stride < x.max_pages) return bad("bad page table");
  // The kernels count positions in 32 bits, to the end of the last position's block and a page past it.
  if ((int64_t)x.num_pages * nkv * page_size > INT32_MAX || (int64_t)x.max_pages * page_size > INT32_MAX - 256)
    return bad("more than 2^31 - 257 positions, or 2^31 - 1 cache rows");
  if ((int64_t)B * T > INT32_MAX / 4 || (int64_t)nh + 2 * nkv > 65535) return bad("too many rows or heads");
  return RIALLM_OK;
}

Pages make_pages(const int32_t* table, int64_t stride, int32_t max_pages, int32_t num_pages, int32_t nkv,
                 int32_t page_size) {
  int lg = 4;
  while ((1 << lg) < page_size) ++lg;
  return Pages{table, stride, max_pages, num_pages, nkv, lg};
}

int32_t append(riallm_ctx* ctx, const riallm_rope_paged_append_args& x, cudaStream_t stream) {
  const char* what = "rope_paged_append";
  if (int s = check_pages(ctx, what, x)) return s;
  if (ctx && (int64_t)x.B * x.T == 0) return RIALLM_OK;
  if (!ctx || !x.qkv || !x.pos || !x.page_table || !x.inv_freq || !x.q_out || !x.k_pages || !x.v_pages)
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "NULL argument");
  if (!al16(x.qkv) || !al16(x.q_out) || !al16(x.k_pages) || !al16(x.v_pages))
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "buffers must be 16-byte aligned");
  return rl::guarded(ctx, [&]() -> int32_t {
    const Pages pg = make_pages(x.page_table, x.table_stride, x.max_pages, x.num_pages, x.nkv, x.page_size);
    // Heads per CTA: all of a row's units where they fit, fewer where the
    // rows alone would leave SMs idle; then as many rows as still fit.
    const int rows = x.B * x.T, heads = x.nh + 2 * x.nkv, per_head = x.d / 16, fit = kAppendThreads * kAppendUnits;
    int hg = std::min(heads, fit / per_head);
    const int64_t want = 2ll * ctx->num_sms;
    if ((int64_t)rows * ((heads + hg - 1) / hg) < want)
      hg = (int)std::max<int64_t>(std::min(heads, kAppendThreads / per_head / 4), (int64_t)heads * rows / want);
    hg = std::min(hg, fit / per_head);
    int per_cta = std::min(kAppendRows, fit / (hg * per_head));
    per_cta = (int)std::max<int64_t>(1, std::min<int64_t>(per_cta, rows * (int64_t)((heads + hg - 1) / hg) / want));
    const auto kernel = x.d == 128 ? rope_paged_append_kernel<128> : rope_paged_append_kernel<64>;
    return rl::launched(ctx, what,
                        rl::launch_pdl(kernel, dim3((rows + per_cta - 1) / per_cta, (heads + hg - 1) / hg),
                                       dim3(kAppendThreads), 0, stream, static_cast<const uint16_t*>(x.qkv), x.pos, pg,
                                       rows, x.T, x.nh, per_cta, hg, x.inv_freq, static_cast<uint16_t*>(x.q_out),
                                       static_cast<uint16_t*>(x.k_pages), static_cast<uint16_t*>(x.v_pages)));
  });
}

int32_t attend(riallm_ctx* ctx, const riallm_paged_attention_args& x, void* workspace, uint64_t workspace_bytes,
               cudaStream_t stream) {
  const char* what = "paged_attention";
  if (int s = check_pages(ctx, what, x)) return s;
  if (x.window < 0 || x.sinks < 0)
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "window and sinks must not be negative");
  if ((int64_t)x.B * x.T * (x.nh / x.nkv) > INT32_MAX / 2)
    return rl::refuse(ctx, RIALLM_ERR_CONFIG, what, "too many rows");
  if (ctx && (int64_t)x.B * x.T == 0) return RIALLM_OK;
  if (!ctx || !x.q || !x.k_pages || !x.v_pages || !x.pos || !x.page_table || !x.out)
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "NULL argument");
  if (!al16(x.q) || !al16(x.out) || !al16(x.k_pages) || !al16(x.v_pages))
    return rl::refuse(ctx, RIALLM_ERR_INVALID, what, "buffers must be 16-byte aligned");
  const Plan p = make_plan(ctx->num_sms, x.B, x.T, x.nh, x.nkv, x.d, (int64_t)x.max_pages * x.page_size);
  if (p.ws_bytes && (!workspace || workspace_bytes < p.ws_bytes || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return rl::refuse(ctx, RIALLM_ERR_MEMORY, what, "workspace missing, too small or not 256-byte aligned");
  return rl::guarded(ctx, [&]() -> int32_t {
    AttnArgs a;
    a.q = static_cast<const uint16_t*>(x.q);
    a.k = static_cast<const uint16_t*>(x.k_pages);
    a.v = static_cast<const uint16_t*>(x.v_pages);
    a.pos = x.pos;
    a.pg = make_pages(x.page_table, x.table_stride, x.max_pages, x.num_pages, x.nkv, x.page_size);
    a.B = x.B, a.T = x.T, a.nh = x.nh, a.rep = x.nh / x.nkv;
    a.rep_inv = (uint32_t)(((1ull << 32) + a.rep - 1) / a.rep);
    a.window = x.window, a.sinks = x.sinks;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)x.d));
    a.out = static_cast<uint16_t*>(x.out);
    Space ws{nullptr, nullptr};
    if (p.join)
      ws = Space{static_cast<Cut*>(workspace),
                 reinterpret_cast<float*>(static_cast<char*>(workspace) + cuts_bytes(p.G))};
    return x.d == 128 ? launch_attention<128>(ctx, a, p, ws, stream) : launch_attention<64>(ctx, a, p, ws, stream);
  });
}

}  // namespace

extern "C" {

int64_t riallm_paged_row(const int32_t* page_table, int64_t table_stride, int32_t max_pages, int32_t num_pages,
                         int32_t nkv, int32_t page_size, int32_t b, int32_t kv_head, int64_t position) {
  if (!page_table || !is_page_size(page_size)) return -1;
  return make_pages(page_table, table_stride, max_pages, num_pages, nkv, page_size).row(b, kv_head, position);
}

int32_t riallm_cuda_rope_paged_append(riallm_ctx* ctx, const riallm_rope_paged_append_args* args, void* stream) {
  if (!args) return rl::refuse(ctx, RIALLM_ERR_INVALID, "rope_paged_append", "NULL argument");
  return append(ctx, *args, (cudaStream_t)stream);
}

uint64_t riallm_cuda_paged_attention_workspace(const riallm_ctx* ctx, int32_t B, int32_t T, int32_t nh, int32_t nkv,
                                               int32_t d, int32_t max_pages, int32_t page_size) {
  if (!ctx || B <= 0 || T <= 0 || nkv <= 0 || nh < nkv || max_pages <= 0 || page_size <= 0) return 0;
  return make_plan(ctx->num_sms, B, T, nh, nkv, d, (int64_t)max_pages * page_size).ws_bytes;
}

int32_t riallm_cuda_paged_attention(riallm_ctx* ctx, const riallm_paged_attention_args* args, void* workspace,
                                    uint64_t workspace_bytes, void* stream) {
  if (!args) return rl::refuse(ctx, RIALLM_ERR_INVALID, "paged_attention", "NULL argument");
  return attend(ctx, *args, workspace, workspace_bytes, (cudaStream_t)stream);
}

}  // extern "C"
