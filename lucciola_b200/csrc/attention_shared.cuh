// What the kernels of attention with shared prefixes have in common: the plan of a step, made by every CTA for itself from the requests'
// lengths, the walk over a CTA's part of it, and the combination of the partial results.
//
// A step's requests fall into groups (prefix_of, prefix_lens): the members' first keys are the same pages.  The work is a list of tiles
// of query rows (a row is a token and a head of a kv head's group of G query heads), each with a range of keys:
//     the tokens of a group's members, up to `tile_tokens` of them, with the group's prefix       (one read of the prefix for all rows)
//     up to `tile_tokens` tokens of one request with what the request has behind the prefix       (all its keys, if it shares none)
// The keys of a tile are visited in blocks of 64.  All blocks of all tiles, once for every kv head, stand in one line, and each CTA
// takes an equal piece of it: the cuts fall anywhere, so that every CTA has the same amount of work whatever the lengths are.  A tile
// whose blocks fall to several CTAs has a partial result (m, l, o) of each, in 32 bits, which a second kernel adds up by token.
//
// A group of a single member, or with less than a block of prefix, is none.  Nothing of this is kept or comes from the host: a step that is replayed from a recorded graph may have other groups and lengths.
// Block ids outside the pool and keys past a request's table are not there; a row that sees no key gives zeros.
#pragma once

#include "common.cuh"

namespace lb {

constexpr int AS_MAX_SEQS = 512;
constexpr int AS_KEYS = 64;
constexpr int AS_REC = 8;                // integers a token in the combining kernel's list

struct SharedParams {
  const void* q; void* out;              // [T, heads, dim]
  const void* k_cache; const void* v_cache;      // [pages, cache heads, page_size, dim]
  const int* table; int max_pages, num_pages;    // [S, max_pages]
  const int* cu; const int* ctx; const int* prefix_of; const int* prefix_lens;
  int T, S, heads, kv_heads, group, dim, page_size, page_shift;      // kv_heads x group = heads; page_shift -1: no power of two
  int kv_share;                          // kv head j of this launch reads cache head j / kv_share
  int tile_tokens, lane_tokens;          // tokens of a tile; a tile of more than lane_tokens counts twice
  int min_span;                          // least units a CTA takes
  float scale_log2;
  float* part_o; float* part_ml;         // [rows][dim], [rows][2]
  int* rec; int* head;                   // [T][AS_REC], {units a kv head, units a CTA, rows a kv head, first token, end of the tokens}
};

// The tensor-core kernel (attention_shared_tc.cu): what it takes, how it cuts rows, its launch.
bool attention_shared_tc_takes(int dtype, int group, int head_dim, int page_size);
void attention_shared_tc_cut(int group, int& tile_tokens, int& lane_tokens);
cudaError_t attention_shared_tc(const SharedParams& p, int ctas, cudaStream_t stream);

struct SharedPlan {
  int q0[AS_MAX_SEQS + 1], ctx[AS_MAX_SEQS];
  int lead[AS_MAX_SEQS];                 // the row whose table holds the prefix this request shares, -1: none
  int rank[AS_MAX_SEQS];                 // tokens of the group in front of this request's
  int member[AS_MAX_SEQS];               // the groups' members, group by group
  int first_member[AS_MAX_SEQS], members[AS_MAX_SEQS], tokens[AS_MAX_SEQS], prefix[AS_MAX_SEQS];     // of the group led by this row
  int unit[2 * AS_MAX_SEQS + 1];         // where the entries begin in the line: groups by their leader, then requests
  int row[2 * AS_MAX_SEQS];              // and in the list of rows
  int scratch[2 * AS_MAX_SEQS];
  int units, span, rows;                 // of a kv head; of a CTA; of a kv head
};

__device__ __forceinline__ int as_blocks(int lo, int hi) { return hi > lo ? (hi - (lo & ~(AS_KEYS - 1)) + AS_KEYS - 1) / AS_KEYS : 0; }
__device__ __forceinline__ int as_visible(const SharedParams& p, int ctx) { return min(ctx, p.max_pages * p.page_size); }

// Units of `tokens` tokens in tiles with `blocks` blocks each.
__device__ __forceinline__ int as_units(const SharedParams& p, int tokens, int blocks) {
  if (tokens <= 0 || blocks <= 0) return 0;
  const int full = (tokens - 1) / p.tile_tokens, last = tokens - full * p.tile_tokens;
  const int twice = p.tile_tokens > p.lane_tokens ? 2 : 1;
  return blocks * (full * twice + (last > p.lane_tokens ? 2 : 1));
}

// An exclusive sum over `n` numbers by one warp, in place; returns the whole.
__device__ __forceinline__ int as_scan(int* a, int n) {
  const int lane = threadIdx.x & 31;
  int total = 0;
  for (int i = 0; i < n; i += 32) {
    const int v = i + lane < n ? a[i + lane] : 0;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    if (i + lane < n) a[i + lane] = total + s - v;
    total += __shfl_sync(0xffffffffu, s, 31);
  }
  return total;
}

// Made by all threads of a CTA (three warps at least); ends with a barrier.
__device__ __forceinline__ void as_make_plan(const SharedParams& p, SharedPlan& pl, int ctas) {
  const int tid = threadIdx.x, n = p.S;
  for (int s = tid; s <= n; s += blockDim.x) pl.q0[s] = min(max(p.cu[s], 0), p.T);
  for (int s = tid; s < n; s += blockDim.x) {
    const int l = p.prefix_of[s];
    pl.lead[s] = l >= 0 && l < n ? l : -1;
    pl.prefix[s] = as_visible(p, max(p.prefix_lens[s], 0));
    pl.ctx[s] = as_visible(p, max(p.ctx[s], 0));
  }
  __syncthreads();
  if (tid < 32) {                        // never falling, whatever the caller's numbers are
    int most = 0;
    for (int i = 0; i <= n; i += 32) {
      int v = i + tid <= n ? pl.q0[i + tid] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, v, o);
        if (tid >= o) v = max(v, t);
      }
      v = max(v, most);
      if (i + tid <= n) pl.q0[i + tid] = v;
      most = __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  // Who shares with whom: every request looks at all others (n is a few dozen, a few hundred at most).
  for (int s = tid; s < n; s += blockDim.x) {
    const int l = pl.lead[s];
    int rank = 0, tokens = 0, before = 0, all = 0;
    int led = 0, led_tokens = 0;
    for (int j = 0; j < n; ++j) {
      const int lj = pl.lead[j], qj = pl.q0[j + 1] - pl.q0[j];
      if (l >= 0 && lj == l) {
        ++all;
        tokens += qj;
        if (j < s) { ++before; rank += qj; }
      }
      if (lj == s) { ++led; led_tokens += qj; }
    }
    pl.rank[s] = rank;
    pl.members[s] = led;
    pl.tokens[s] = led_tokens;
    pl.scratch[s] = before;
  }
  __syncthreads();
  for (int s = tid; s < n; s += blockDim.x) pl.first_member[s] = pl.members[s];
  __syncthreads();
  if (tid < 32) as_scan(pl.first_member, n);
  __syncthreads();
  for (int s = tid; s < n; s += blockDim.x) {
    const int l = pl.lead[s];
    if (l >= 0) pl.member[pl.first_member[l] + pl.scratch[s]] = s;
  }
  __syncthreads();
  // A group of one, or a prefix shorter than a block, is not worth a tile of its own.
  for (int s = tid; s < n; s += blockDim.x)
    if (pl.members[s] < 2 || pl.prefix[s] < AS_KEYS) pl.members[s] = 0;
  __syncthreads();
  for (int s = tid; s < n; s += blockDim.x) {
    const int l = pl.lead[s];
    const bool shares = l >= 0 && pl.members[l] > 0;
    if (!shares) pl.lead[s] = -1;
    const int q = pl.q0[s + 1] - pl.q0[s];
    const bool leads = pl.members[s] > 0;
    pl.unit[s] = leads ? as_units(p, pl.tokens[s], as_blocks(0, pl.prefix[s])) : 0;
    pl.row[s] = leads ? pl.tokens[s] * p.group : 0;
    pl.unit[n + s] = as_units(p, q, as_blocks(shares ? pl.prefix[l] : 0, pl.ctx[s]));
    pl.row[n + s] = q * p.group;
  }
  __syncthreads();
  if (tid < 32) {
    const int u = as_scan(pl.unit, 2 * n);
    if (tid == 0) {
      pl.unit[2 * n] = u;
      pl.units = u;
      pl.span = max((int)(((long long)u * p.kv_heads + ctas - 1) / ctas), p.min_span);
    }
  } else if (tid < 64) {
    const int r = as_scan(pl.row, 2 * n);
    if (tid == 32) pl.rows = r;
  }
  __syncthreads();
}

// What the combining kernel has to know of every token: for the prefix and for the request's own keys, the token's first row, the unit of
// its tile's first block, and how many units further the last block begins (-1: no block).
__device__ __forceinline__ void as_write_records(const SharedParams& p, const SharedPlan& pl, int cta, int ctas) {
  if (cta == 0 && threadIdx.x == 0) { p.head[0] = pl.units; p.head[1] = pl.span; p.head[2] = pl.rows; p.head[3] = pl.q0[0]; p.head[4] = pl.q0[p.S]; }
  for (int s = cta; s < p.S; s += ctas) {
    const int t0 = pl.q0[s], q = pl.q0[s + 1] - t0, l = pl.lead[s];
    for (int i = threadIdx.x; i < q; i += blockDim.x) {
      int r[AS_REC];
      auto place = [&](int* at, int e, int index, int tokens, int row_blocks, int all_blocks) {
        const int tile = index / p.tile_tokens, first = tile * p.tile_tokens;
        const int w = min(tokens - first, p.tile_tokens) > p.lane_tokens ? 2 : 1;
        const int twice = p.tile_tokens > p.lane_tokens ? 2 : 1;
        at[0] = pl.row[e] + index * p.group;
        at[1] = pl.unit[e] + tile * all_blocks * twice;
        at[2] = row_blocks > 0 ? (row_blocks - 1) * w : -1;
      };
      r[0] = r[1] = 0; r[2] = -1;
      if (l >= 0) {
        const int nb = as_blocks(0, pl.prefix[l]);
        place(r, l, pl.rank[s] + i, pl.tokens[l], nb, nb);
      }
      const int lo = l >= 0 ? pl.prefix[l] : 0;
      const int tile_end = min((i / p.tile_tokens + 1) * p.tile_tokens, q);
      const int hi = min(pl.ctx[s], pl.ctx[s] - q + tile_end);      // keys the tile's last token sees
      place(r + 3, p.S + s, i, q, as_blocks(lo, hi), as_blocks(lo, pl.ctx[s]));
      r[6] = r[7] = 0;
      int4* dst = reinterpret_cast<int4*>(p.rec + (size_t)(t0 + i) * AS_REC);
      dst[0] = make_int4(r[0], r[1], r[2], r[3]);
      dst[1] = make_int4(r[4], r[5], r[6], r[7]);
    }
  }
}

// A run of blocks of one tile and one kv head.
struct Segment {
  int kv_head;
  int table_row;
  int shared;                            // leader of the group, -1: rows of one request
  int request;                           // whose rows they are, if not shared
  int first;                             // shared: rank in the group of the first token; else the first token's place in the request
  int tokens;
  int key_lo, key_hi;                    // keys of the tile (of all its rows together)
  int block, blocks;                     // first block of the run (of the tile's), and how many (0: none are there)
  size_t row;                            // where its partial rows begin
};

// The segment at unit x of the line (0 <= x < units * kv_heads), cut off at x_end; x moves behind it.
__device__ __forceinline__ Segment as_next(const SharedParams& p, const SharedPlan& pl, int cta, long long& x, long long x_end) {
  Segment g;
  g.kv_head = (int)(x / pl.units);
  const int u = (int)(x - (long long)g.kv_head * pl.units);
  int a = 0, b = 2 * p.S - 1;            // the last entry that begins at or before u: the one that holds it
  while (a < b) {
    const int mid = (a + b + 1) >> 1;
    if (pl.unit[mid] <= u) a = mid; else b = mid - 1;
  }
  const bool shared = a < p.S;
  const int s = shared ? a : a - p.S;
  const int q = pl.q0[s + 1] - pl.q0[s];
  const int tokens = shared ? pl.tokens[s] : q;
  const int lead = shared ? -1 : pl.lead[s];
  const int lo = lead >= 0 ? pl.prefix[lead] : 0;
  const int nb = shared ? as_blocks(0, pl.prefix[s]) : as_blocks(lo, pl.ctx[s]);
  const int twice = p.tile_tokens > p.lane_tokens ? 2 : 1;
  const int tile = (u - pl.unit[a]) / (nb * twice);
  const int tile_unit = pl.unit[a] + tile * nb * twice;
  g.table_row = s;
  g.shared = shared ? s : -1;
  g.request = s;
  g.first = tile * p.tile_tokens;
  g.tokens = min(tokens - g.first, p.tile_tokens);
  const int w = g.tokens > p.lane_tokens ? 2 : 1;
  g.key_lo = lo;
  g.key_hi = shared ? pl.prefix[s] : min(pl.ctx[s], pl.ctx[s] - q + g.first + g.tokens);
  const long long base = (long long)g.kv_head * pl.units + tile_unit;
  const int there = as_blocks(lo, g.key_hi);           // a portion's earlier tiles see fewer blocks than its last
  // a block belongs to the CTA in whose piece it begins
  const int from = (int)((x - base + w - 1) / w);
  const long long end = min(x_end, base + (long long)nb * w);
  const int to = min((int)((end - base + w - 1) / w), there);
  g.block = from;
  g.blocks = max(to - from, 0);
  g.row = (size_t)g.kv_head * pl.rows + pl.row[a] + (size_t)g.first * p.group + (size_t)cta * p.tile_tokens * p.group;
  x = end;
  return g;
}

// The i-th token of a segment: its place in the step, and the last key it sees.
__device__ __forceinline__ void as_token(const SharedPlan& pl, const Segment& g, int i, int& token, int& position) {
  int s = g.request, at = g.first + i;
  if (g.shared >= 0) {                   // the member whose tokens these are: the last one whose first token is not behind
    int a = pl.first_member[g.shared], b = a + pl.members[g.shared] - 1;
    while (a < b) {
      const int mid = (a + b + 1) >> 1;
      if (pl.rank[pl.member[mid]] <= at) a = mid; else b = mid - 1;
    }
    s = pl.member[a];
    at -= pl.rank[s];
  }
  token = pl.q0[s] + at;
  position = pl.ctx[s] - (pl.q0[s + 1] - pl.q0[s]) + at;
}

__device__ __forceinline__ void as_store4(float* dst, float a, float b, float c, float d) { *reinterpret_cast<float4*>(dst) = make_float4(a, b, c, d); }
__device__ __forceinline__ void as_store4(bf16* dst, float a, float b, float c, float d) {
  __nv_bfloat162 lo = __floats2bfloat162_rn(a, b), hi = __floats2bfloat162_rn(c, d);
  *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
}

// out[t, h] = sum 2^(m - M) o / sum 2^(m - M) l over the partial results of a row, in the order of the line: one warp a row.
// Partial results with m = -inf weigh nothing and their o is not read.
template <typename T>
__global__ void __launch_bounds__(256) as_combine_kernel(SharedParams p) {
  pdl_trigger();
  const int* rec = p.rec;
  const int* head = p.head;
  pdl_wait(rec, head);
  const int lane = threadIdx.x & 31;
  const int item = (blockIdx.x * 256 + threadIdx.x) >> 5;
  if (item >= p.T * p.heads) return;
  const int t = item / p.heads, h = item % p.heads, kv = h / p.group;
  if (t < __ldcg(head + 3) || t >= __ldcg(head + 4)) return;         // rows of no request stay as they were
  const int4 r0 = __ldcg(reinterpret_cast<const int4*>(rec + (size_t)t * AS_REC));
  const int4 r1 = __ldcg(reinterpret_cast<const int4*>(rec + (size_t)t * AS_REC) + 1);
  const int units = __ldcg(head), span = __ldcg(head + 1), rows = __ldcg(head + 2);
  const long long line = (long long)kv * units;
  // the two runs of partial results: first CTA, number, first row
  int c0[2], n[2];
  size_t row[2];
  const int first_row[2] = {r0.x, r0.w}, unit[2] = {r0.y, r1.x}, last[2] = {r0.z, r1.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    c0[i] = (int)((line + unit[i]) / span);
    n[i] = last[i] < 0 ? 0 : (int)((line + unit[i] + last[i]) / span) - c0[i] + 1;
    row[i] = (size_t)kv * rows + first_row[i] + h % p.group + (size_t)c0[i] * p.tile_tokens * p.group;
  }
  const size_t step = (size_t)p.tile_tokens * p.group;
  const int total = n[0] + n[1];
  auto row_of = [&](int i) { return i < n[0] ? row[0] + (size_t)i * step : row[1] + (size_t)(i - n[0]) * step; };
  float M = -INFINITY, L = 0.f;
  for (int i = lane; i < total; i += 32) M = fmaxf(M, __ldcg(p.part_ml + row_of(i) * 2));
  M = warp_max(M);
  T* out = reinterpret_cast<T*>(p.out) + (size_t)item * p.dim;
  float acc[2][4];                       // dimensions lane * 4 + 128 c .. + 3
  const int chunks = (p.dim + 127) / 128;
#pragma unroll
  for (int c = 0; c < 2; ++c) acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
  if (M > -INFINITY) {
    for (int i0 = 0; i0 < total; i0 += 32) {
      const int i = i0 + lane;
      float w = 0.f;
      if (i < total) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + row_of(i) * 2));
        w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
        L += w * ml.y;
      }
      const int here = min(32, total - i0);
      for (int j0 = 0; j0 < here; j0 += 8) {
        float wj[8];
        float4 a[8];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c >= chunks) break;
          const int d = lane * 4 + 128 * c;
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            wj[u] = __shfl_sync(0xffffffffu, w, (j0 + u) & 31);
            if (j0 + u >= here) wj[u] = 0.f;
            a[u] = wj[u] != 0.f && d < p.dim ? __ldcg(reinterpret_cast<const float4*>(p.part_o + row_of(i0 + j0 + u) * p.dim + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            acc[c][0] = fmaf(wj[u], a[u].x, acc[c][0]); acc[c][1] = fmaf(wj[u], a[u].y, acc[c][1]);
            acc[c][2] = fmaf(wj[u], a[u].z, acc[c][2]); acc[c][3] = fmaf(wj[u], a[u].w, acc[c][3]);
          }
        }
      }
    }
  }
  L = warp_sum(L);
  const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int d = lane * 4 + 128 * c;
    if (c < chunks && d < p.dim) as_store4(out + d, acc[c][0] * inv, acc[c][1] * inv, acc[c][2] * inv, acc[c][3] * inv);
  }
}

}  // namespace lb
