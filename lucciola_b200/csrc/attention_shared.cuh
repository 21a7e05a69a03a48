// What the kernels of attention with shared prefixes have in common: the plan of a step, which a kernel makes from the requests' lengths, and
// the combination of the partial results.
//
// A step's requests fall into groups (prefix_of, prefix_lens): the members' first keys are the same pages.  The work is a list of tiles
// of query rows (a row is a token and a head of a kv head's group of G query heads), each with a range of keys:
//     the tokens of a group's members, up to `tile_tokens` of them, with the group's prefix       (one read of the prefix for all rows)
//     up to `tile_tokens` tokens of one request with what the request has behind the prefix       (all its keys, if it shares none)
// The keys of a tile are visited in blocks of 64.  All blocks of all tiles, once for every kv head, stand in one line, and each CTA
// takes an equal piece of it: the cuts fall anywhere, so that every CTA has the same amount of work whatever the lengths are.  What a CTA has
// of a tile is a segment; a tile has a partial result (m, l, o) of each of its segments, in 32 bits, and a last kernel adds them up by token.
// (With every tile's keys cut into a number of parts of its own, some SMs would have a part more than others.)
//
// A group of a single member, or with less than a block of prefix, is none.  Nothing of this comes from the host: a step that is replayed
// from a recorded graph may have other groups and lengths.  The plan is a kernel of its own because the layers of a model share it, and because the
// code that makes it would have to be fetched by every SM in front of its work (instructions are fetched anew by every launch: 9000 cycles
// for the plan and the walk along it, of 45000 in all, at 64 requests behind 8192 keys).
// Block ids outside the pool and keys past a request's table are not there; a row that sees no key gives zeros.
#pragma once

#include "common.cuh"

namespace lb {

constexpr int AS_MAX_SEQS = 512;
constexpr int AS_KEYS = 64;
constexpr int AS_REC = 12;               // integers a token in the combining kernel's list
constexpr int AS_PIECE = 16;             // integers a CTA in the list of their pieces
constexpr int AS_FOLD_ROWS = 32;

struct SharedParams {
  const void* q; void* out;              // [T, heads, dim]
  const void* k_cache; const void* v_cache;      // [pages, cache heads, page_size, dim]
  const int* table; int max_pages, num_pages;    // [S, max_pages]
  const int* cu; const int* ctx; const int* prefix_of; const int* prefix_lens;
  int T, S, heads, kv_heads, group, dim, page_size, page_shift;      // kv_heads x group = heads; page_shift -1: no power of two
  int kv_share;                          // kv head j of this launch reads cache head j / kv_share
  int tile_tokens, lane_tokens;          // tokens of a tile; a tile of more than lane_tokens counts twice
  int min_span;                          // least units a CTA takes
  int tile_start;                        // units that a tile costs beside its blocks
  bool folds;                            // whether tiles of few rows leave several partial results (as_folds), one behind the other
  float scale_log2;
  // Partial results: 4 consecutive dimensions of all rows of a tile, then the next 4 ([dim / 4][rows][4], so that threads with a row each
  // write, and threads with a head each read, side by side), and [rows][2]: the reference value (-inf: no key) and the sum.
  float* part_o; float* part_ml;
  // The plan.  head: {units a kv head, units a CTA, rows a kv head, first token, end of the tokens}; rec [T][AS_REC]: see as_write_records;
  // pieces [CTAs][AS_PIECE]: the CTA's first and last segment, two of nothing, and the first segment itself; segments [..][12]: see Segment;
  // members [T]: the groups' tokens, group by group, and the last key each sees
  int* head; int* rec; int4* pieces; int4* segments; int2* members;
};

// Integers of a plan, and where its parts begin.
struct SharedPlanLayout {
  long long rec, pieces, segments, members, total;
  __host__ SharedPlanLayout(long long tokens, long long seqs, int kv_heads, int tile_tokens, int ctas) {
    const long long most = kv_heads * 2 * (tokens / tile_tokens + seqs) + ctas;        // a tile has one segment more than it has cuts
    rec = 8; pieces = rec + tokens * AS_REC; segments = pieces + AS_PIECE * ctas; members = segments + most * 12; total = members + 2 * tokens;
  }
};

// The tensor-core kernel (attention_shared_tc.cu): what it takes, how it cuts rows, its launch.
bool attention_shared_tc_takes(int dtype, int group, int head_dim, int page_size);
void attention_shared_tc_cut(int group, int& tile_tokens, int& lane_tokens);
cudaError_t attention_shared_tc(const SharedParams& p, int ctas, cudaStream_t stream);

struct SharedPlan {                      // in shared memory, while it is made
  int4 meta[AS_MAX_SEQS];                // prefix_of (-1: none), new tokens, context, tokens of the prefix in this row's table
  int q0[AS_MAX_SEQS];                   // first token
  int lead[AS_MAX_SEQS];                 // the row whose table holds the prefix that this request shares, -1: none
  int rank[AS_MAX_SEQS];                 // tokens of the group in front of this request's
  int led[AS_MAX_SEQS];                  // tokens of the group that this row leads
  int unit[2 * AS_MAX_SEQS], row[2 * AS_MAX_SEQS], tile[2 * AS_MAX_SEQS];      // of entry e (groups by their leader, then requests): where it
                                         // begins in the line, in the list of rows and among all tiles
  int first_member[AS_MAX_SEQS];         // where the tokens of the group that this row leads begin among all groups'
  int units, span, rows, tiles;          // units, rows and tiles of a kv head, units of a CTA
  bool sound;                            // cu_tokens rise: every token belongs to one request at most
};

__device__ __forceinline__ int as_blocks(int lo, int hi) { return hi > lo ? (hi - (lo & ~(AS_KEYS - 1)) + AS_KEYS - 1) / AS_KEYS : 0; }

__device__ __forceinline__ int as_tile_units(const SharedParams& p, int tokens, int blocks) {
  return p.tile_start + (tokens > p.lane_tokens ? 2 * blocks : blocks);
}
// Units of `tokens` tokens in tiles with `blocks` blocks each, and the rows of their partial results.
__device__ __forceinline__ int as_units(const SharedParams& p, int tokens, int blocks) {
  if (tokens <= 0 || blocks <= 0) return 0;
  if (tokens <= p.tile_tokens) return as_tile_units(p, tokens, blocks);
  const int full = (tokens - 1) / p.tile_tokens;
  return full * as_tile_units(p, p.tile_tokens, blocks) + as_tile_units(p, tokens - full * p.tile_tokens, blocks);
}
// Partial results that each CTA leaves of a tile with this many rows: two of one that both halves of the tensor memory work on, a half of
// the blocks each; four of a request's few rows, a quarter of every block's keys each.
__host__ __device__ __forceinline__ int as_folds(const SharedParams& p, bool shared, int rows) {
  return !p.folds || rows > p.lane_tokens * p.group ? 1 : !shared && rows <= AS_FOLD_ROWS ? 4 : 2;
}
__device__ __forceinline__ int as_rows(const SharedParams& p, bool shared, int tokens) {
  if (tokens <= 0) return 0;
  const int last = tokens <= p.tile_tokens ? tokens : tokens - (tokens - 1) / p.tile_tokens * p.tile_tokens;
  return (tokens - last) * p.group + last * p.group * as_folds(p, shared, last * p.group);
}

// An exclusive sum over `n` numbers by one warp, in place; returns the whole.  A lane has a run of them.
__device__ __forceinline__ int as_scan(int* a, int n) {
  const int lane = threadIdx.x & 31, per = (n + 31) >> 5, from = min(lane * per, n), to = min(from + per, n);
  int s = 0;
  for (int i = from; i < to; ++i) s += a[i];
  const int mine = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  const int total = __shfl_sync(0xffffffffu, s, 31);
  s -= mine;
  for (int i = from; i < to; ++i) {
    const int v = a[i];
    a[i] = s;
    s += v;
  }
  return total;
}

// Made by all AS_PLAN_THREADS threads of a CTA; ends with a barrier.
constexpr int AS_PLAN_THREADS = 512;
__device__ __forceinline__ void as_make_plan(const SharedParams& p, SharedPlan& pl, int ctas) {
  const int tid = threadIdx.x, n = p.S;
  const int most = p.max_pages * p.page_size;
  bool falls = false;
  if (tid < n) {
    const int s = tid;
    const int a = __ldcg(p.cu + s), b = __ldcg(p.cu + s + 1), c = __ldcg(p.ctx + s), l = __ldcg(p.prefix_of + s), f = __ldcg(p.prefix_lens + s);
    const int q0 = min(max(a, 0), p.T);
    falls = b < a;
    pl.q0[s] = q0;
    pl.meta[s] = make_int4(l >= 0 && l < n ? l : -1, max(min(b, p.T), q0) - q0, min(max(c, 0), most), min(max(f, 0), most));
  }
  const bool sound = __syncthreads_or(falls) == 0;
  if (tid == 0) pl.sound = sound;
  // Who shares with whom: every request looks at all others (n is a few dozen, a few hundred at most), 1 << k lanes for each.
  const int k = n <= AS_PLAN_THREADS / 8 ? 3 : n <= AS_PLAN_THREADS / 4 ? 2 : n <= AS_PLAN_THREADS / 2 ? 1 : 0;
  const int s = tid >> k, part = tid & ((1 << k) - 1);
  if ((s & ~(31 >> k)) < n) {            // whole warps
    const int4 me = s < n ? pl.meta[s] : make_int4(-1, 0, 0, 0);
    const int l = me.x;
    int rank = 0, all = 0, led = 0, led_tokens = 0;
#pragma unroll 4
    for (int j = part; j < n; j += 1 << k) {
      const int2 o = *reinterpret_cast<const int2*>(&pl.meta[j]);
      const bool same = o.x == l && l >= 0, mine = o.x == s;
      all += same ? 1 : 0;
      rank += same && j < s ? o.y : 0;
      led += mine ? 1 : 0;
      led_tokens += mine ? o.y : 0;
    }
#pragma unroll 1
    for (int o = (1 << k) >> 1; o > 0; o >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, o); rank += __shfl_xor_sync(0xffffffffu, rank, o);
      led += __shfl_xor_sync(0xffffffffu, led, o); led_tokens += __shfl_xor_sync(0xffffffffu, led_tokens, o);
    }
    if (part == 0 && s < n) {
      // A group of one, or a prefix shorter than a block, is not worth a tile of its own.
      const int prefix = l >= 0 ? pl.meta[l].w : 0;
      const bool shares = all >= 2 && prefix >= AS_KEYS, leads = led >= 2 && me.w >= AS_KEYS;
      pl.lead[s] = shares ? l : -1;
      pl.rank[s] = rank;
      pl.led[s] = led_tokens;
      pl.first_member[s] = leads ? led_tokens : 0;
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const int e = i * n + s, tokens = i ? me.y : leads ? led_tokens : 0, blocks = i ? as_blocks(shares ? prefix : 0, me.z) : as_blocks(0, me.w);
        pl.unit[e] = as_units(p, tokens, blocks);
        pl.row[e] = as_rows(p, i == 0, tokens);
        pl.tile[e] = blocks > 0 ? (tokens + p.tile_tokens - 1) / p.tile_tokens : 0;
      }
    }
  }
  __syncthreads();
  const int warp = tid >> 5;
  if (warp < 4) {
    const int sum = as_scan(warp == 0 ? pl.unit : warp == 1 ? pl.row : warp == 2 ? pl.tile : pl.first_member, warp < 3 ? 2 * n : n);
    if ((tid & 31) == 0) {
      if (warp == 0) {
        pl.units = sum;
        pl.span = max((int)(((unsigned)sum * (unsigned)p.kv_heads + (unsigned)ctas - 1u) / (unsigned)ctas), p.min_span);
      }
      if (warp == 1) pl.rows = sum;
      if (warp == 2) pl.tiles = sum;
    }
  }
  __syncthreads();
}

// Rows of partial results of a kv head, at most: a token has its own and those with its prefix, and the last tile of an entry (one a request, one
// a group of two or more) may be folded, into four with up to 32 rows each or two with up to 128.
// Where cu_tokens fall, requests' tokens overlap and there may be more of everything than there is room for: the plan is empty then, and the output stays as it was.
__host__ __device__ __forceinline__ long long as_most_rows(long long tokens, long long seqs, int group, bool folds) {
  const long long rows = tokens * group, more = 256 * seqs;
  return 2 * rows + (!folds ? 0 : more < 4 * rows ? more : 4 * rows);
}
// What the combining kernel has to know of every token, for the prefix and for the request's own keys: the first row of the token's
// tile, the token's first row in the tile, the tile's rows (not folded), the unit of its first block, and how many units further the last block
// begins (-1: no block).  And the groups' tokens.
__device__ __forceinline__ void as_write_records(const SharedParams& p, const SharedPlan& pl, int cta, int ctas, int thread, int threads) {
  if (cta == 0 && thread == 0) {
    p.head[0] = pl.units; p.head[1] = pl.span; p.head[2] = pl.rows;
    p.head[3] = pl.sound ? pl.q0[0] : 0;
    p.head[4] = pl.sound ? pl.q0[p.S - 1] + pl.meta[p.S - 1].y : 0;
  }
  if (!pl.sound) return;
  // Token by token: the request of a token is the last one that begins at it or in front of it and has any.
  const int begin = pl.q0[0], end = pl.q0[p.S - 1] + pl.meta[p.S - 1].y;
  for (int t = begin + cta * threads + thread; t < end; t += ctas * threads) {
    int s = 0;
#pragma unroll 1
    for (int lo = 0, hi = p.S; hi - lo > 1;) {
      const int mid = (lo + hi) >> 1;
      if (pl.q0[mid] <= t) lo = mid; else hi = mid;
      s = lo;
    }
    const int4 me = pl.meta[s];
    const int t0 = pl.q0[s], q = me.y, l = pl.lead[s], i = t - t0;
    const int prefix = l >= 0 ? pl.meta[l].w : 0;
    {
      int4* dst = reinterpret_cast<int4*>(p.rec + (size_t)(t0 + i) * AS_REC);
      int last[2];
#pragma unroll 1
      for (int of = 0; of < 2; ++of) {   // the prefix, the request's own keys
        const int e = of ? p.S + s : l, index = of ? i : pl.rank[s] + i, tokens = of ? q : l >= 0 ? pl.led[l] : 0;
        const int tile = index / p.tile_tokens, first = tile * p.tile_tokens, here = min(tokens - first, p.tile_tokens);
        const int lo = of ? prefix : 0, hi = of ? me.z : prefix;
        const int blocks = as_blocks(lo, of ? min(hi, hi - q + first + here) : hi);            // that the tile's last token sees
        const bool any = of || l >= 0;
        dst[of] = any ? make_int4(pl.row[e] + first * p.group, (index - first) * p.group, here * p.group,
                                  pl.unit[e] + tile * as_tile_units(p, p.tile_tokens, as_blocks(lo, hi)) + p.tile_start) : make_int4(0, 0, 0, 0);
        last[of] = any && blocks > 0 ? (blocks - 1) * (here > p.lane_tokens ? 2 : 1) : -1;
      }
      dst[2] = make_int4(last[0], last[1], 0, 0);
      if (l >= 0) p.members[pl.first_member[l] + pl.rank[s] + i] = make_int2(t0 + i, me.z - q + i);
    }
  }
}

// A run of blocks of one tile and one kv head.
struct Segment {
  int kv_head, request;                  // the row of the block table
  int first, tokens;                     // first token (shared: its place among the groups' tokens), and how many
  int key_lo, key_hi;                    // keys of the tile (of all its rows together)
  int block, blocks;                     // first block of the run (of the tile's), and how many (0: none are there)
  int row_low, row_high;                 // where its partial rows begin, 64 bits
  int shared, position;                  // rows of several requests; else the last key that the first token sees
};
__device__ __forceinline__ Segment as_segment(const int4* at) {
  const int4 a = __ldcg(at), b = __ldcg(at + 1), c = __ldcg(at + 2);
  return Segment{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w};
}
__device__ __forceinline__ Segment as_segment(const SharedParams& p, int i) { return as_segment(p.segments + (size_t)i * 3); }
// The first and the last segment of a CTA's piece of the line, and the first itself (nothing, if there is none): one access to memory in
// front of the first keys less.
__device__ __forceinline__ int2 as_piece(const SharedParams& p, int cta, Segment& first) {
  const int4* at = p.pieces + (size_t)cta * (AS_PIECE / 4);
  const int4 piece = __ldcg(at);
  first = as_segment(at + 1);
  if (piece.y < piece.x) first.blocks = 0;
  return make_int2(piece.x, piece.y);
}
// A token of a segment: its place in the step, and the last key it sees.
__device__ __forceinline__ int2 as_token(const SharedParams& p, int shared, int first, int position, int i) {
  return shared ? __ldcg(p.members + first + i) : make_int2(first + i, position + i);
}

__device__ __forceinline__ void as_store4(float* dst, float a, float b, float c, float d) { *reinterpret_cast<float4*>(dst) = make_float4(a, b, c, d); }
__device__ __forceinline__ void as_store4(bf16* dst, float a, float b, float c, float d) {
  __nv_bfloat162 lo = __floats2bfloat162_rn(a, b), hi = __floats2bfloat162_rn(c, d);
  *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
}

// out[t, h] = sum 2^(m - M) o / sum 2^(m - M) l over the partial results of a row.  A block has one token and kv head; a thread one head
// of the group (neighbouring threads neighbouring heads: rows that lie side by side), four dimensions, and every PARTS-th partial
// result, eight of which are read at once; the threads' sums are added up in shared memory, in a fixed order.  A partial result with
// m = -inf weighs nothing, and its o is not looked at.  Bound by accesses to L2 that wait for one another, and by its own beginning and end: 5 us
// for 2 tokens, 8 for 64 behind 8192 common keys (32 heads of 128).
constexpr int AS_COMBINE_THREADS = 128;
template <typename T, int PARTS>
__global__ void __launch_bounds__(AS_COMBINE_THREADS * PARTS) as_combine_kernel(SharedParams p) {
  __shared__ float4 sums[PARTS][128];
  __shared__ float2 weights[PARTS][128];
  pdl_trigger();
  const int t = blockIdx.x, kv = blockIdx.y, part = threadIdx.x >> 7, lane = threadIdx.x & 127;
  // The plan was complete when the kernel ahead let this one begin (it waits for the plan first), and is read while that kernel still runs.
  const int4* r = reinterpret_cast<const int4*>(p.rec + (size_t)t * AS_REC);
  const int4 a = __ldcg(r), b = __ldcg(r + 1), last = __ldcg(r + 2);
  const int4 hd = __ldcg(reinterpret_cast<const int4*>(p.head));
  const int end = __ldcg(p.head + 4);
  pdl_wait(p.part_o, p.part_ml);
  if (t < hd.w || t >= end) return;                            // rows of no request stay as they were
  const unsigned line = (unsigned)kv * (unsigned)hd.x, span = (unsigned)hd.y;
  const long long step = (long long)p.tile_tokens * p.group;
  const int fa = as_folds(p, true, a.z) - 1, fb = as_folds(p, false, b.z) - 1;       // 0, 1 or 3
  const int ca = (int)((line + a.w) / span), cb = (int)((line + b.w) / span);
  const int na = last.x < 0 ? 0 : ((int)((line + a.w + last.x) / span) - ca + 1) * (fa + 1);
  const int total = na + (last.y < 0 ? 0 : ((int)((line + b.w + last.y) / span) - cb + 1) * (fb + 1));
  const int chunks = p.dim / 4;
  for (int i0 = 0; i0 < p.group * chunks; i0 += 128) {
    const int i = i0 + lane, h = i % p.group, c = i / p.group;
    const bool on = i < p.group * chunks;
    // this thread's first partial result among the prefix's and among its own keys'
    const long long tile_a = (long long)kv * hd.z + a.x + ca * step, tile_b = (long long)kv * hd.z + b.x + cb * step;
    const float2* ml_a = reinterpret_cast<const float2*>(p.part_ml) + tile_a + a.y + h;
    const float2* ml_b = reinterpret_cast<const float2*>(p.part_ml) + tile_b + b.y + h;
    const float4* o_a = reinterpret_cast<const float4*>(p.part_o + tile_a * p.dim) + c * a.z * (fa + 1) + a.y + h;
    const float4* o_b = reinterpret_cast<const float4*>(p.part_o + tile_b * p.dim) + c * b.z * (fb + 1) + b.y + h;
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int z0 = part; on && z0 < total; z0 += 8 * PARTS) {
      float2 ml[8];
      float4 o[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int z = z0 + u * PARTS;
        ml[u] = make_float2(-INFINITY, 0.f);
        o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (z < total) {
          const bool of_a = z < na;
          const int at = of_a ? z : z - na, f = of_a ? fa : fb, copy = (at & f) * (of_a ? a.z : b.z);
          const long long cta = (at >> (f - (f >> 1))) * step;         // shifted by 0, 1 or 2
          ml[u] = __ldcg((of_a ? ml_a : ml_b) + cta + copy);
          o[u] = __ldcg((of_a ? o_a : o_b) + cta * chunks + copy);
        }
      }
      float m = M;
#pragma unroll
      for (int u = 0; u < 8; ++u) m = fmaxf(m, ml[u].x);
      const float ref = m == -INFINITY ? 0.f : m;
      const float f = exp2f(M - ref);                          // (0 at first: M = -inf)
      L *= f; acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
      M = m;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (ml[u].x == -INFINITY) continue;
        const float w = exp2f(ml[u].x - ref);
        L = fmaf(w, ml[u].y, L);
        acc.x = fmaf(w, o[u].x, acc.x); acc.y = fmaf(w, o[u].y, acc.y); acc.z = fmaf(w, o[u].z, acc.z); acc.w = fmaf(w, o[u].w, acc.w);
      }
    }
    if (PARTS > 1) {
      __syncthreads();                                         // the last heads' sums have been read
      sums[part][lane] = acc;
      weights[part][lane] = make_float2(M, L);
      __syncthreads();
      if (part != 0) continue;
      M = -INFINITY;
#pragma unroll
      for (int q = 0; q < PARTS; ++q) M = fmaxf(M, weights[q][lane].x);
      L = 0.f;
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int q = 0; q < PARTS; ++q) {
        const float2 ml = weights[q][lane];
        if (ml.x == -INFINITY) continue;
        const float w = exp2f(ml.x - M);
        const float4 o = sums[q][lane];
        L = fmaf(w, ml.y, L);
        acc.x = fmaf(w, o.x, acc.x); acc.y = fmaf(w, o.y, acc.y); acc.z = fmaf(w, o.z, acc.z); acc.w = fmaf(w, o.w, acc.w);
      }
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    if (on)
      as_store4(reinterpret_cast<T*>(p.out) + ((size_t)t * p.heads + (size_t)kv * p.group + h) * p.dim + 4 * c, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  }
}

}  // namespace lb
