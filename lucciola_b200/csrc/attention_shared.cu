// Attention of a step whose requests share prefixes: the entry point, the plan, and the kernel on the ordinary pipes for 32-bit queries, keys
// and values, and bfloat16 ones that the tensor-core kernel does not take.  The plan's layout and the combination are attention_shared.cuh's.
//
// A tile has up to 32 query rows (tokens x heads of a kv head's group; a group of more heads is cut into equal parts that read the same
// cached head).  Queries, a block of 64 keys and its values lie in shared memory as 32-bit numbers.  256 threads: thread (ty, tx) has
// rows 2 ty and 2 ty + 1; of the scores the keys tx, tx + 16, tx + 32, tx + 48, of the result the dimensions 4 tx + 64 c .. + 3.  Sixteen
// threads share a row: its maximum and sum are four shuffles.  Bound by a block's copy and its products, which take turns, and by reads of shared memory (a
// thread reads six 16-byte words for 32 multiplications): 32 requests behind 4096 common keys, 32 heads of 128 on 8 in 32 bits, 246 us (2.2 GFLOP,
// 9 TFLOP/s of the pipes' 70 or so); 6 requests behind 1000, 16 heads of 64 on 4, with plan and combination 15.9 us, most of it three kernels'
// beginnings and ends.
#include "attention_shared.cuh"

#include <atomic>

namespace lb {

constexpr int AP_THREADS = 256;
constexpr int AP_ROWS = 32;
constexpr int AS_FEW_BLOCKS = 296;

__device__ __forceinline__ float4 ap_load4(const float* p) { return __ldcg(reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ float4 ap_load4(const bf16* p) {
  const uint2 w = __ldcg(reinterpret_cast<const uint2*>(p));
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

// floats of dynamic shared memory: queries, keys (rows four further apart, so that the keys of eight threads fall into different banks),
// values, weights; then the page of every key of the block
template <int D> constexpr int ap_smem_bytes() { return (AP_ROWS * D + AS_KEYS * (D + 4) + AS_KEYS * D + AP_ROWS * (AS_KEYS + 4) + AS_KEYS) * 4; }

template <typename T, int D>
__global__ void __launch_bounds__(AP_THREADS) attention_shared_plain_kernel(SharedParams p) {
  extern __shared__ __align__(16) float ap_smem[];
  float* qs = ap_smem;
  float* ks = qs + AP_ROWS * D;
  float* vs = ks + AS_KEYS * (D + 4);
  float* ps = vs + AS_KEYS * D;
  int* page = reinterpret_cast<int*>(ps + AP_ROWS * (AS_KEYS + 4));      // offset of each key's row in the pool's page units, -1: not there
  pdl_wait();
  pdl_trigger();                         // behind the wait: the combining kernel reads the plan before its own
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const T* q = reinterpret_cast<const T*>(p.q);
  const T* kc = reinterpret_cast<const T*>(p.k_cache);
  const T* vc = reinterpret_cast<const T*>(p.v_cache);
  const int d = p.dim, G = p.group, cache_heads = p.kv_heads / p.kv_share;
  Segment g;
  const int2 piece = as_piece(p, blockIdx.x, g);
  for (int at = piece.x; at <= piece.y; ++at) {
    if (at != piece.x) g = as_segment(p, at);
    if (g.blocks == 0) continue;
    const long long first_row = (long long)(uint32_t)g.row_low | (long long)g.row_high << 32;
    const int rows = g.tokens * G;
    __syncthreads();
    for (int i = tid; i < AP_ROWS * (D / 4); i += AP_THREADS) {
      const int r = i / (D / 4), c = i % (D / 4) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows && c < d) {
        const int token = as_token(p, g.shared, g.first, g.position, r / G).x;
        v = ap_load4(q + ((size_t)token * p.heads + g.kv_head * G + r % G) * d + c);
      }
      *reinterpret_cast<float4*>(qs + r * D + c) = v;
    }
    int last[2];                         // the last key each row sees
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      last[e] = 2 * ty + e < rows ? as_token(p, g.shared, g.first, g.position, (2 * ty + e) / G).y : -1;
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float o[2][D / 64][4];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) o[e][c][0] = o[e][c][1] = o[e][c][2] = o[e][c][3] = 0.f;
    const int* bt = p.table + (size_t)g.request * p.max_pages;
    for (int b = g.block; b < g.block + g.blocks; ++b) {
      const int k0 = (g.key_lo & ~(AS_KEYS - 1)) + b * AS_KEYS;
      __syncthreads();                   // the block before has been read
      if (tid < AS_KEYS) {
        const int key = k0 + tid;
        int at = -1;
        if (key >= g.key_lo && key < g.key_hi) {
          const int pi = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
          at = bt[pi];
          if (at >= p.num_pages) at = -1;
        }
        page[tid] = at;
      }
      __syncthreads();
      for (int i = tid; i < AS_KEYS * (D / 4); i += AP_THREADS) {
        const int j = i / (D / 4), c = i % (D / 4) * 4, at = page[j];
        float4 kv = make_float4(0.f, 0.f, 0.f, 0.f), vv = kv;
        if (at >= 0 && c < d) {
          const int key = k0 + j, slot = p.page_shift >= 0 ? key & (p.page_size - 1) : key % p.page_size;
          const size_t off = (((size_t)at * cache_heads + g.kv_head / p.kv_share) * p.page_size + slot) * d + c;
          kv = ap_load4(kc + off);
          vv = ap_load4(vc + off);
        }
        *reinterpret_cast<float4*>(ks + j * (D + 4) + c) = kv;
        *reinterpret_cast<float4*>(vs + j * D + c) = vv;
      }
      __syncthreads();
      float s[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) s[e][0] = s[e][1] = s[e][2] = s[e][3] = 0.f;
#pragma unroll 4
      for (int c = 0; c < D; c += 4) {
        const float4 q0 = *reinterpret_cast<const float4*>(qs + 2 * ty * D + c), q1 = *reinterpret_cast<const float4*>(qs + (2 * ty + 1) * D + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 k = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * (D + 4) + c);
          s[0][j] = fmaf(q0.x, k.x, fmaf(q0.y, k.y, fmaf(q0.z, k.z, fmaf(q0.w, k.w, s[0][j]))));
          s[1][j] = fmaf(q1.x, k.x, fmaf(q1.y, k.y, fmaf(q1.z, k.z, fmaf(q1.w, k.w, s[1][j]))));
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = m[e];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int jj = tx + 16 * j;
          s[e][j] = (k0 + jj <= last[e] && page[jj] >= 0) ? s[e][j] * p.scale_log2 : -INFINITY;
          mx = fmaxf(mx, s[e][j]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float ref = mx == -INFINITY ? 0.f : mx;
        const float f = m[e] == -INFINITY ? 0.f : exp2f(m[e] - ref);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float w = exp2f(s[e][j] - ref);
          sum += w;
          ps[(2 * ty + e) * (AS_KEYS + 4) + tx + 16 * j] = w;
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        m[e] = mx;
        l[e] = l[e] * f + sum;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) { o[e][c][0] *= f; o[e][c][1] *= f; o[e][c][2] *= f; o[e][c][3] *= f; }
      }
      __syncwarp();                      // a row's weights are written and read by one half of a warp
#pragma unroll 4
      for (int j = 0; j < AS_KEYS; ++j) {
        const float w0 = ps[2 * ty * (AS_KEYS + 4) + j], w1 = ps[(2 * ty + 1) * (AS_KEYS + 4) + j];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const float4 v = *reinterpret_cast<const float4*>(vs + j * D + 64 * c + 4 * tx);
          o[0][c][0] = fmaf(w0, v.x, o[0][c][0]); o[0][c][1] = fmaf(w0, v.y, o[0][c][1]); o[0][c][2] = fmaf(w0, v.z, o[0][c][2]); o[0][c][3] = fmaf(w0, v.w, o[0][c][3]);
          o[1][c][0] = fmaf(w1, v.x, o[1][c][0]); o[1][c][1] = fmaf(w1, v.y, o[1][c][1]); o[1][c][2] = fmaf(w1, v.z, o[1][c][2]); o[1][c][3] = fmaf(w1, v.w, o[1][c][3]);
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 2 * ty + e;
      if (r >= rows) continue;
      if (tx == 0) *reinterpret_cast<float2*>(p.part_ml + (first_row + r) * 2) = make_float2(m[e], l[e]);
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        if (64 * c + 4 * tx < d)
          *reinterpret_cast<float4*>(p.part_o + first_row * d + ((16 * c + tx) * rows + r) * 4) = make_float4(o[e][c][0], o[e][c][1], o[e][c][2], o[e][c][3]);
    }
  }
}

// The plan of a step: every CTA makes all of it, and writes a part.  A chain of lookups, not bytes: 5 us at 2 requests and at 32, 7 to 8 where one of them has 2048
// new tokens (plan after plan; in front of the attention a part of it is hidden).
__global__ void __launch_bounds__(AS_PLAN_THREADS) as_plan_kernel(SharedParams p, int ctas) {
  __shared__ SharedPlan pl;
  pdl_trigger();
  pdl_wait();
  as_make_plan(p, pl, ctas);
  as_write_records(p, pl, blockIdx.x, gridDim.x, threadIdx.x, AS_PLAN_THREADS);
  const bool sound = pl.sound;
  const int total = sound ? pl.units * p.kv_heads : 0, span = pl.span;
  if (blockIdx.x == 0)
    for (int c = threadIdx.x; c < ctas; c += AS_PLAN_THREADS)
      if ((long long)c * span >= total) p.pieces[c * (AS_PIECE / 4)] = make_int4(0, -1, 0, 0);
  if (!sound) return;
  // the segments: eight threads have an entry and a kv head, every eighth tile each, or, of a few tiles, every eighth segment
  for (int i = (blockIdx.x * AS_PLAN_THREADS + threadIdx.x) >> 3; i < 2 * p.S * p.kv_heads; i += gridDim.x * AS_PLAN_THREADS >> 3) {
    const int kv = i / (2 * p.S), e = i - kv * (2 * p.S);
    const bool shared = e < p.S;
    const int s = shared ? e : e - p.S;
    const int4 me = pl.meta[s];
    const int end = e + 1 < 2 * p.S ? pl.unit[e + 1] : pl.units;
    if (pl.unit[e] == end) continue;
    const int lead = shared ? -1 : pl.lead[s], lo = lead >= 0 ? pl.meta[lead].w : 0, hi = shared ? me.w : me.z;
    const int tokens = shared ? pl.led[s] : me.y, nb = as_blocks(lo, hi);
    const int units = as_tile_units(p, p.tile_tokens, nb);     // of every tile but the last
    const bool by_tile = tokens > 4 * p.tile_tokens;
    const int mine = threadIdx.x & 7, tile_step = by_tile ? 8 : 1, step = by_tile ? 1 : 8;
#pragma unroll 1
    for (int i_tile = by_tile ? mine : 0; i_tile * p.tile_tokens < tokens; i_tile += tile_step) {
      const int first = i_tile * p.tile_tokens, tile = pl.tile[e] + i_tile, base = kv * pl.units + pl.unit[e] + i_tile * units;
      const int here = min(tokens - first, p.tile_tokens), two = here > p.lane_tokens ? 1 : 0;             // units of a block: 1 << two
      const int key_hi = shared ? hi : min(hi, hi - tokens + first + here), there = as_blocks(lo, key_hi);      // an earlier tile sees fewer blocks
      const int b0 = base + p.tile_start, b1 = base + as_tile_units(p, here, nb);
      const int c0 = (int)((unsigned)base / (unsigned)span), c1 = (int)((unsigned)(b1 - 1) / (unsigned)span);
#pragma unroll 1
      for (int c = c0 + (by_tile ? 0 : mine); c <= c1; c += step) {
        const int x0 = c * span, x1 = (int)min((unsigned)x0 + (unsigned)span, (unsigned)total);
        // a block belongs to the CTA in whose piece it begins
        const int block = max(x0 - b0 + two, 0) >> two, blocks = max(min(max(min(x1, b1) - b0 + two, 0) >> two, there) - block, 0);
        const int at = kv * pl.tiles + tile + c;
        const long long row = (long long)kv * pl.rows + pl.row[e] + (long long)first * p.group + (long long)c * p.tile_tokens * p.group;
        int4* dst = p.segments + (size_t)at * 3;
        int4* piece = p.pieces + c * (AS_PIECE / 4);
        const int4 segment[3] = {make_int4(kv, s, (shared ? pl.first_member[s] : pl.q0[s]) + first, here), make_int4(lo, key_hi, block, blocks),
                                 make_int4((int)(uint32_t)row, (int)(row >> 32), shared ? 1 : 0, shared ? 0 : me.z - tokens + first)};
#pragma unroll
        for (int u = 0; u < 3; ++u) dst[u] = segment[u];
        if (x0 >= base) {
          piece->x = at;
#pragma unroll
          for (int u = 0; u < 3; ++u) piece[1 + u] = segment[u];
        }
        if (x1 <= b1) piece->y = at;
      }
    }
  }
}

static int as_sms() {
  static std::atomic<int> known[64];                           // by device; 0: not asked yet
  int device = 0, n = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 0;
  std::atomic<int>& have = known[device & 63];
  if (device < 64 && (n = have.load()) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
  if (device < 64) have.store(n);
  return n;
}

// How a launch cuts its rows: kv heads that share a cached one, heads of a tile, tokens of a tile and of a part of one.
struct SharedCut { bool tc; int share, group, tile_tokens, lane_tokens; };
static SharedCut as_cut(int dtype, int group, int head_dim, int page_size) {
  SharedCut c{attention_shared_tc_takes(dtype, group, head_dim, page_size), 1, group, 0, 0};
  if (c.tc) {
    attention_shared_tc_cut(group, c.tile_tokens, c.lane_tokens);
    return c;
  }
  while (group % c.share || group / c.share > AP_ROWS) ++c.share;
  c.group = group / c.share;
  c.tile_tokens = c.lane_tokens = AP_ROWS / c.group;
  return c;
}

template <typename T, int D>
static cudaError_t ap_launch(const SharedParams& p, int ctas, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured{0ull};     // a bit a device
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (!(configured.load() >> (device & 63) & 1ull)) {
    e = cudaFuncSetAttribute(attention_shared_plain_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, ap_smem_bytes<D>());
    if (e != cudaSuccess) return e;
    configured.fetch_or(1ull << (device & 63));
  }
  return launch(attention_shared_plain_kernel<T, D>, dim3(ctas), dim3(AP_THREADS), ap_smem_bytes<D>(), stream, p);
}

template <typename T>
static cudaError_t as_combine(const SharedParams& p, cudaStream_t stream) {
  // Few rows: four threads share a row's partial results, so that one round of loads reads them all.  (8 requests behind 8192 keys 24.0 us against
  // 30.4; 64 requests, which are above the border, 39.8 against 44.8 with four, portions 38 against 61.)
  if ((long long)p.T * p.kv_heads <= AS_FEW_BLOCKS)
    return launch(as_combine_kernel<T, 4>, dim3(p.T, p.kv_heads), dim3(4 * AS_COMBINE_THREADS), 0, stream, p);
  return launch(as_combine_kernel<T, 1>, dim3(p.T, p.kv_heads), dim3(AS_COMBINE_THREADS), 0, stream, p);
}


#define AS_CHECK(cond, ...) do { if (!(cond)) { set_error(__VA_ARGS__); return false; } } while (0)
// What all launches of one call have in common; false with the library's message when the sizes are refused.
static bool as_sizes(SharedParams& p, SharedCut& cut, int dtype, int num_tokens, int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                      int page_size, int max_pages) {
  AS_CHECK(valid_dtype(dtype), "attention_shared: unknown element type %d", dtype);
  AS_CHECK(num_tokens >= 0 && num_seqs >= 0 && num_seqs <= AS_MAX_SEQS, "attention_shared: %d tokens of %d requests, at most %d requests",
           num_tokens, num_seqs, AS_MAX_SEQS);
  AS_CHECK(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0, "attention_shared: %d query heads on %d kv heads",
           num_q_heads, num_kv_heads);
  AS_CHECK(head_dim > 0 && head_dim <= 256 && head_dim % 8 == 0, "attention_shared: heads of %d, a multiple of 8 up to 256 is needed", head_dim);
  AS_CHECK(page_size > 0 && max_pages > 0 && (long long)max_pages * page_size < (1ll << 31) - 64, "attention_shared: tables of %d pages of %d tokens",
           max_pages, page_size);
  AS_CHECK((long long)num_tokens * num_q_heads < (1ll << 30), "attention_shared: %d tokens of %d heads", num_tokens, num_q_heads);
  cut = as_cut(dtype, num_q_heads / num_kv_heads, head_dim, page_size);
  p = SharedParams{};
  p.T = num_tokens; p.S = num_seqs; p.heads = num_q_heads; p.kv_heads = num_kv_heads * cut.share; p.group = cut.group; p.dim = head_dim;
  p.page_size = page_size; p.max_pages = max_pages; p.page_shift = -1; p.kv_share = cut.share;
  p.tile_tokens = cut.tile_tokens; p.lane_tokens = cut.lane_tokens;
  // Measured at 64 requests behind 8192 keys, at portions behind 2000 and at 2 requests behind 256 (us, recorded): tiles that cost 2 units beside
  // their blocks 39.1, 38.3 and 17.1, 3 units 38.7, 36.7 and 14.3, 4 units 39.1, 35.5 and 15.4; pieces of at least 4 units 38.5, 36.9 and 15.2, of 8
  // 38.5, 36.8 and 18.2.
  p.min_span = cut.tc ? 5 : 1; p.tile_start = cut.tc ? 3 : 0; p.folds = cut.tc;
  for (int b = 0; b < 31; ++b) if ((1 << b) == page_size) p.page_shift = b;
  // units of the whole line, at most (as_tile_units; places in the line are 32-bit numbers, an end of a CTA's piece may lie a piece further)
  const long long tiles = 2ll * ((long long)num_tokens / p.tile_tokens + num_seqs), blocks = ((long long)max_pages * page_size + AS_KEYS - 1) / AS_KEYS;
  AS_CHECK(tiles * (2 * blocks + p.tile_start) * p.kv_heads < (1ll << 31) - 65536, "attention_shared: %d tokens of %d requests on tables of %d pages are too much for one launch",
           num_tokens, num_seqs, max_pages);
  AS_CHECK(p.kv_heads <= 65535, "attention_shared: %d kv heads", p.kv_heads);
  return true;
}
// The same on the current device.
static bool as_params(SharedParams& p, SharedCut& cut, int& ctas, int dtype, int num_tokens, int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                      int page_size, int max_pages) {
  if (!as_sizes(p, cut, dtype, num_tokens, num_seqs, num_q_heads, num_kv_heads, head_dim, page_size, max_pages)) return false;
  ctas = as_sms();
  AS_CHECK(ctas > 0, "attention_shared: no device");
  return true;
}
#undef AS_CHECK

static void as_plan_parts(SharedParams& p, int* plan, int ctas) {
  const SharedPlanLayout at(p.T, p.S, p.kv_heads, p.tile_tokens, ctas);
  p.head = plan; p.rec = plan + at.rec; p.pieces = reinterpret_cast<int4*>(plan + at.pieces);
  p.segments = reinterpret_cast<int4*>(plan + at.segments); p.members = reinterpret_cast<int2*>(plan + at.members);
}

}  // namespace lb

// 0 if calls of these sizes are taken, else 1 with the message; needs no GPU.
LB_EXPORT int lb_attention_shared_refused(int dtype, int num_tokens, int num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int page_size, int max_pages) {
  lb::SharedParams p;
  lb::SharedCut cut;
  return lb::as_sizes(p, cut, dtype, num_tokens, num_seqs, num_q_heads, num_kv_heads, head_dim, page_size, max_pages) ? 0 : 1;
}

// Elements that a call needs: of the plan (int32) and of the partial results (float32).
LB_EXPORT int lb_attention_shared_sizes(int dtype, int num_tokens, int num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                        int max_pages, long long* ints, long long* floats) {
  lb::SharedParams p;
  lb::SharedCut cut;
  int ctas = 0;
  if (!lb::as_params(p, cut, ctas, dtype, num_tokens, num_seqs, num_q_heads, num_kv_heads, head_dim, page_size, max_pages)) return 1;
  *ints = lb::SharedPlanLayout(num_tokens, num_seqs, p.kv_heads, p.tile_tokens, ctas).total;
  *floats = (lb::as_most_rows(num_tokens, num_seqs, cut.group, cut.tc) * p.kv_heads + (long long)ctas * cut.tile_tokens * cut.group) * (head_dim + 2);
  return 0;
}

static int as_plan(lb::SharedParams p, const lb::SharedCut& cut, int ctas, int* plan, long long num_ints, const int* cu_tokens, const int* context_lens,
                   const int* prefix_of, const int* prefix_lens, cudaStream_t stream) {
  const long long need = lb::SharedPlanLayout(p.T, p.S, p.kv_heads, p.tile_tokens, ctas).total;
  LB_CHECK_ARG(plan && (uintptr_t)plan % 16 == 0 && num_ints >= need, "attention_shared: a plan of %lld integers at a 16-byte boundary is needed, got %lld", need, num_ints);
  p.cu = cu_tokens; p.ctx = context_lens; p.prefix_of = prefix_of; p.prefix_lens = prefix_lens;
  lb::as_plan_parts(p, plan, ctas);
  // A round of segments and of tokens for every thread, up to 32 CTAs (each makes the whole plan first).
  const long long tasks = 2ll * p.S * p.kv_heads * 8, most = tasks > p.T ? tasks : p.T;
  const int blocks = (int)(most < 32 * lb::AS_PLAN_THREADS ? (most + lb::AS_PLAN_THREADS - 1) / lb::AS_PLAN_THREADS : 32);
  lb::launch(lb::as_plan_kernel, dim3(blocks), dim3(lb::AS_PLAN_THREADS), 0, stream, p, ctas);
  LB_CHECK_LAUNCH("attention_shared plan");
  return 0;
}

// The plan of a step for lb_attention_shared, from cu_tokens [S + 1], context_lens, prefix_of and prefix_lens [S], int32.
LB_EXPORT int lb_attention_shared_plan(int dtype, int* plan, long long num_ints, const int* cu_tokens, const int* context_lens, const int* prefix_of,
                                       const int* prefix_lens, int num_tokens, int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                                       int page_size, int max_pages, cudaStream_t stream) {
  lb::SharedParams p;
  lb::SharedCut cut;
  int ctas = 0;
  if (!lb::as_params(p, cut, ctas, dtype, num_tokens, num_seqs, num_q_heads, num_kv_heads, head_dim, page_size, max_pages)) return 1;
  if (num_tokens == 0 || num_seqs == 0) return 0;
  return as_plan(p, cut, ctas, plan, num_ints, cu_tokens, context_lens, prefix_of, prefix_lens, stream);
}

// q, out: [T, heads, dim]; k_cache, v_cache: [pages, kv heads, page_size, dim]; table [S, max_pages] int32; a plan made for these sizes, or, with
// cu_tokens (and the other three), memory for the plan that is made here.  floats: the partial results.  See attention_shared.cuh.
LB_EXPORT int lb_attention_shared(int dtype, const void* q, void* out, const void* k_cache, const void* v_cache, const int* table, int* plan,
                                  long long num_ints, const int* cu_tokens, const int* context_lens, const int* prefix_of, const int* prefix_lens,
                                  int num_tokens, int num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                  int num_pages, int max_pages, float scale, float* floats, long long num_floats, cudaStream_t stream) {
  lb::SharedParams p;
  lb::SharedCut cut;
  int ctas = 0;
  if (!lb::as_params(p, cut, ctas, dtype, num_tokens, num_seqs, num_q_heads, num_kv_heads, head_dim, page_size, max_pages)) return 1;
  LB_CHECK_ARG(num_pages > 0, "attention_shared: a pool of %d pages", num_pages);
  LB_CHECK_ARG(scale > 0.f && scale < 1e30f, "attention_shared: a scale of %f, a positive one is needed", (double)scale);
  if (num_tokens == 0 || num_seqs == 0) return 0;
  LB_CHECK_ARG(((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)floats | (uintptr_t)plan) % 16 == 0,
               "attention_shared: operands must be 16-byte aligned");
  const long long need = lb::SharedPlanLayout(num_tokens, num_seqs, p.kv_heads, p.tile_tokens, ctas).total;
  const long long rows = lb::as_most_rows(num_tokens, num_seqs, cut.group, cut.tc) * p.kv_heads + (long long)ctas * cut.tile_tokens * cut.group;
  LB_CHECK_ARG(plan && floats && num_ints >= need && num_floats >= rows * (head_dim + 2),
               "attention_shared: a plan of %lld integers and a workspace of %lld floats are needed, got %lld and %lld", need, rows * (head_dim + 2),
               num_ints, num_floats);
  if (cu_tokens && as_plan(p, cut, ctas, plan, num_ints, cu_tokens, context_lens, prefix_of, prefix_lens, stream)) return 2;
  p.q = q; p.out = out; p.k_cache = k_cache; p.v_cache = v_cache; p.table = table; p.num_pages = num_pages;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part_o = floats; p.part_ml = floats + rows * head_dim;
  lb::as_plan_parts(p, plan, ctas);
  cudaError_t e;
  if (cut.tc)
    e = lb::attention_shared_tc(p, ctas, stream);
  else if (dtype == LB_F32)
    e = head_dim <= 64 ? lb::ap_launch<float, 64>(p, ctas, stream) : head_dim <= 128 ? lb::ap_launch<float, 128>(p, ctas, stream) : lb::ap_launch<float, 256>(p, ctas, stream);
  else
    e = head_dim <= 64 ? lb::ap_launch<lb::bf16, 64>(p, ctas, stream) : head_dim <= 128 ? lb::ap_launch<lb::bf16, 128>(p, ctas, stream) : lb::ap_launch<lb::bf16, 256>(p, ctas, stream);
  if (e != cudaSuccess) { lb::set_error("attention_shared: launch failed: %s", cudaGetErrorString(e)); return 2; }
  lb::count_launch();
  e = dtype == LB_F32 ? lb::as_combine<float>(p, stream) : lb::as_combine<lb::bf16>(p, stream);
  if (e != cudaSuccess) { lb::set_error("attention_shared: launch of the combination failed: %s", cudaGetErrorString(e)); return 2; }
  lb::count_launch();
  return 0;
}
