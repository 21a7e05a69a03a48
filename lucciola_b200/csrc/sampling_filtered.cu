// Sampling from what top-k, top-p and min-p leave of softmax(logits / T), over 32-bit logits [R, V].
//
// With M the row's largest logit, z_i = (logit_i - M) / T and w_i = exp(z_i), the row's tokens stand in the order of falling logits,
// equal ones by index.  Of this order a row keeps the first top_k; of those the ones in front of which the sum of w is below
// top_p times the sum of all top_k; of those the ones with w >= min_p; and always the first.  All three are prefixes of one order.
// The token is the kept one with the largest z_i - log(-log(u_i)), u_i the samplers' hash (a draw from the kept ones' softmax).
//
// A row belongs to a cluster of CTAs, each with a slice of it in its shared memory: the logits are read once, and what the filters
// need of the whole row (maximum, sums, borders) goes through distributed shared memory.  Two ways through a row:
//   * top_k up to SF_SHORT: the k-th largest of the threads' own maxima bounds the k-th largest logit from below (found to within a
//     bin of a histogram with one entry a thread); the few logits above it go to the cluster's first CTA, which ranks them and
//     decides everything in 64 bits.
//   * otherwise, without sorting: the best score among all tokens (of the first top_k, if there is a border to find by digits) is
//     looked for first, and then whether its token is kept: one sum over the tokens in front of it.  If not, the same again among those;
//     a drawn token is kept with probability top_p, so that this is rarely repeated more than once or twice.
// A score needs a hash and two logarithms, so as few tokens as possible get that far: those whose weight is so small that the sum of
// all not larger is below 1 - top_p, those below min_p, and those that cannot reach the bound below which the best score falls once
// in 10^8 rows (log of the sum minus 3; such a row is done again without the bound) are left out by their logit alone, and of the
// rest those whose 1 - u, a lower bound of -log u, is too large already.
//
// Which token comes out does not depend on the order of sums, and so not on the batch the row stands in: 32-bit scores and sums decide
// only where they differ by more than they can be off by, and 64-bit scores and whole-number sums of 64 bits decide the rest.
#include "sampling.cuh"

#include <atomic>
#include <cfloat>

namespace lb {

constexpr int SF_THREADS = 512;
constexpr int SF_BINS = 256;
constexpr int SF_SHORT = 256;            // most top_k of the short way
constexpr int SF_LIST = 512;             // logits the first CTA ranks, one a thread
constexpr int SF_MAX_LOG2 = 3, SF_MAX_CLUSTER = 1 << SF_MAX_LOG2;
constexpr int SF_SLICE_BYTES = 200 * 1024;     // most logits of a CTA; longer rows are read again where they lie
constexpr int SF_PAIR_BYTES = 100 * 1024;      // with as many, two CTAs share an SM
constexpr float SF_SCORE_MARGIN = 1.f / 32768.f;     // 32-bit scores z + g lie in [-20, 20] and are off by less than 2^-17
constexpr float SF_SUM_MARGIN = 1.f / 32768.f;       // 32-bit sums of w, relative: w within 2^-18 where it counts, four at a time in 32 bits
constexpr float SF_BELOW = 60.f;                     // weights below e^-60 of the largest change no sum of 64 bits

struct FilterParams {
  int* tokens; const float* logits; const float* temperature; const unsigned long long* keys; const int* counters;
  const int* top_k; const float* top_p; const float* min_p;
  long long row_stride; int vocab;
};

__device__ __forceinline__ uint32_t sf_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t sf_size() { uint32_t r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void sf_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// In two parts, at the start: a peer's shared memory may be written when the peer has begun to run.
__device__ __forceinline__ void sf_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void sf_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t sf_remote(const void* local, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
  return a;
}
// A word into a peer's shared memory that is counted by a barrier there.  One way only: a barrier of the whole cluster around plain
// stores is a way there and one back, and a row has four to eight of these (18.8 us against 16.5 for 8 rows of 151936).
__device__ __forceinline__ void sf_send(uint32_t addr, uint32_t v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];" ::"r"(addr), "r"(v), "r"(bar) : "memory");
}
__device__ __forceinline__ bool sf_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ int g_sampling_error = 0;                  // 1 where a wait gave up (lb_sample_filtered_device_error)
constexpr unsigned SF_WAIT_CYCLES = 2000000000u;
__device__ __forceinline__ void sf_expect(unsigned long long* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(bar)), "r"(bytes) : "memory");
}
// A CTA one of whose waits ran out records it and leaves the row's token as it is.  Not at once: its peers may still write to its shared memory or
// read there.  They get no more values from it, so that each of them ends, or gives up its next wait and comes here too; until then a peer passes the
// cluster's barrier SF_BARRIERS times at most, which this CTA passes with it, and then once more.  (CTAs that have ended count as arrived.)
constexpr int SF_BARRIERS = 10;          // between two exchanges of values: one a digit of top_k's border, three of the short way in front of them
__device__ __noinline__ void sf_leave() {
  g_sampling_error = 1;
#pragma unroll 1
  for (int i = 0; i <= SF_BARRIERS; ++i) sf_cluster_sync();
  asm volatile("exit;");
}
// By all threads of a CTA, bounded (about a second); a barrier of the CTA too.
__device__ __forceinline__ void sf_wait(unsigned long long* bar, uint32_t parity) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(bar);
  const unsigned t0 = (unsigned)clock();
  bool lost = false;
  while (!sf_try_wait(at, parity))
    if ((unsigned)clock() - t0 > SF_WAIT_CYCLES) { lost = true; break; }
  if (__syncthreads_or(lost)) sf_leave();
}
__device__ __forceinline__ void sf_st_remote(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t sf_ld_remote(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t sf_add_remote(uint32_t addr, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
  return old;
}

// Values of up to SF_WORDS words a thread, reduced over the cluster; every thread gets the result.  Two sets of slots in turn: a CTA
// writes a peer's set again only when it has that peer's values of the turn between, which the peer sends when it has read the set.
constexpr int SF_WORDS = 6;
struct FilterShared {
  unsigned long long arrived[2];         // barriers of the two sets of slots
  uint32_t warp_part[SF_THREADS / 32][SF_WORDS];
  uint32_t slot[2][SF_MAX_CLUSTER][SF_WORDS];
  uint32_t hist[2][SF_BINS];
  uint32_t scan[SF_THREADS / 32];
  uint32_t list_n, digit, digit_before;
  float list_l[SF_LIST]; int list_i[SF_LIST];
  float rank_l[SF_LIST]; int rank_i[SF_LIST];
  double warp_sum[SF_THREADS / 32];
};

struct FilterGroup {                     // what a thread knows of its cluster
  FilterShared* sh;
  uint32_t rank, size;
  int turn;
};

// Floats as whole numbers of the same order, for the warp's one-instruction maxima and minima.
__device__ __forceinline__ int sf_order(float x) { const int b = __float_as_int(x); return b ^ ((b >> 31) & 0x7fffffff); }
__device__ __forceinline__ float sf_unorder(int o) { return __int_as_float(o ^ ((o >> 31) & 0x7fffffff)); }
__device__ __forceinline__ double sf_warp_sum(double v, int lanes) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The cluster's value from the lanes' values: `lanes` joins the first 32 or SF_THREADS / 32 lanes of a warp (lane 0 has the result), `slots` the CTAs'.
template <typename T, typename L, typename C>
__device__ __forceinline__ T sf_reduce_by(FilterGroup& g, T v, L lanes, C slots) {
  static_assert(sizeof(T) % 4 == 0 && sizeof(T) / 4 <= SF_WORDS, "words of a slot");
  constexpr int W = sizeof(T) / 4;
  union U { T t; uint32_t w[W]; __device__ U() {} };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  U a;
  a.t = lanes(v, 32);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < W; ++i) g.sh->warp_part[warp][i] = a.w[i];
  }
  __syncthreads();
  const int set = g.turn & 1;
  const uint32_t parity = (g.turn >> 1) & 1;
  uint32_t (*slot)[SF_WORDS] = g.sh->slot[set];
  ++g.turn;
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < W; ++i) a.w[i] = g.sh->warp_part[lane & (SF_THREADS / 32 - 1)][i];
    a.t = lanes(a.t, SF_THREADS / 32);                         // (twice the same in the two halves of the warp)
    // lane 0's value to all CTAs, a word a lane
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const uint32_t w = __shfl_sync(0xffffffffu, a.w[i], 0);
      if (lane % W == i) mine = w;
    }
    if (lane == 0) sf_expect(&g.sh->arrived[set], g.size * W * 4);
    for (uint32_t c = lane / W; c < g.size; c += 32 / W)
      if (lane < 32 / W * W) sf_send(sf_remote(&slot[g.rank][lane % W], c), mine, sf_remote(&g.sh->arrived[set], c));
  }
  sf_wait(&g.sh->arrived[set], parity);
#pragma unroll
  for (int i = 0; i < W; ++i) a.w[i] = slot[0][i];
  T out = a.t;
  for (uint32_t c = 1; c < g.size; ++c) {
    U b;
#pragma unroll
    for (int i = 0; i < W; ++i) b.w[i] = slot[c][i];
    out = slots(out, b.t);
  }
  return out;
}
// The same with one way of joining two values.
template <typename T, typename F>
__device__ __forceinline__ T sf_reduce(FilterGroup& g, T v, F join) {
  constexpr int W = sizeof(T) / 4;
  union U { T t; uint32_t w[W]; __device__ U() {} };
  return sf_reduce_by(g, v, [&](T x, int n) {
#pragma unroll 1
    for (int o = n >> 1; o > 0; o >>= 1) {
      U a, b;
      a.t = x;
#pragma unroll
      for (int i = 0; i < W; ++i) b.w[i] = __shfl_xor_sync(0xffffffffu, a.w[i], o);
      x = join(x, b.t);
    }
    return x;
  }, join);
}

// A histogram of the CTA's threads becomes the cluster's, and the first bin with `want` entries in it or in front of it is found:
// returns that bin (SF_BINS if there are not that many) and how many entries lie in front of it.  `hist` is this CTA's; complete when
// every thread has arrived here.
__device__ __forceinline__ int sf_find_bin(FilterGroup& g, uint32_t* hist, uint32_t want, uint32_t& before) {
  sf_cluster_sync();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t n = 0;
  if (tid < SF_BINS)
    for (uint32_t c = 0; c < g.size; ++c) n += sf_ld_remote(sf_remote(hist + tid, c));
  uint32_t s = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  if (lane == 31) g.sh->scan[warp] = s;
  if (tid == 0) { g.sh->digit = SF_BINS; g.sh->digit_before = 0; }
  __syncthreads();
  if (tid < SF_BINS) {
    for (int w = 0; w < warp; ++w) s += g.sh->scan[w];
    if (s >= want && s - n < want) { g.sh->digit = tid; g.sh->digit_before = s - n; }
    if (tid == SF_BINS - 1 && s < want) g.sh->digit_before = s;
  }
  __syncthreads();
  before = g.sh->digit_before;
  return (int)g.sh->digit;
}

// Whole numbers in the order of the logits.
__device__ __forceinline__ uint32_t sf_key(float l) {
  const uint32_t b = __float_as_uint(l + 0.f);            // -0 as 0: they are equal
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sf_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The first of the order's places that are not kept any more; a token is in front of it if its logit is larger, or equal at a smaller index.
struct Border { float l; int i; };
__device__ __forceinline__ bool in_front(float l, int i, const Border& b) { return l > b.l || (l == b.l && i < b.i); }

struct Best { float s; int i; float l; float second; };      // best score, its token and logit; the best score of any other token
struct Best64 { double s; int i; float l; };

template <bool IN_SMEM>
__global__ void __launch_bounds__(SF_THREADS, 2) sample_filtered_kernel(FilterParams p) {
  extern __shared__ __align__(16) float data[];
  __shared__ FilterShared sh;
  pdl_trigger();
  FilterGroup g{&sh, sf_rank(), sf_size(), 0};
  const int tid = threadIdx.x;
  const int row = blockIdx.x / g.size;
  for (int b = tid; b < 2 * SF_BINS; b += SF_THREADS) sh.hist[0][b] = 0;
  if (tid == 0) {
    sh.list_n = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((uint32_t)__cvta_generic_to_shared(&sh.arrived[i])));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  sf_cluster_arrive();
  pdl_wait(p.logits, p.temperature, p.keys, p.counters, p.top_k, p.top_p, p.min_p);

  // ---- the slice: whole 16-byte words of memory, the first and the last of a row partly filled ----------------------------------
  const float* row_ptr = p.logits + (long long)row * p.row_stride;
  const int skew = (int)(((uintptr_t)row_ptr >> 2) & 3);       // the row's first logit is the skew-th of its 16-byte word
  const float* base = row_ptr - skew;
  const int words = (p.vocab + skew + 3) >> 2;
  const int per = (words + (int)g.size - 1) / (int)g.size;
  const int first = min(words, (int)g.rank * per), nq = min(words, first + per) - first;
  // word q of the slice from memory; places outside the row are not there (-inf)
  auto whole = [&](int q) { const int v = 4 * (first + q) - skew; return v >= 0 && v + 4 <= p.vocab; };
  auto fetch = [&](int q) -> float4 {
    if (whole(q)) return __ldcg(reinterpret_cast<const float4*>(base) + first + q);
    const int v = 4 * (first + q) - skew;
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (v + e >= 0 && v + e < p.vocab) ? __ldcg(row_ptr + v + e) : -INFINITY;
    return make_float4(x[0], x[1], x[2], x[3]);
  };
  auto clean = [](float4 x) {                                  // NaN is as -inf
    x.x = fmaxf(x.x, -INFINITY); x.y = fmaxf(x.y, -INFINITY); x.z = fmaxf(x.z, -INFINITY); x.w = fmaxf(x.w, -INFINITY);
    return x;
  };
  float4* data4 = reinterpret_cast<float4*>(data);
  auto word = [&](int q) -> float4 { return IN_SMEM ? data4[q] : clean(fetch(q)); };
  auto index_of = [&](int q, int e) { return 4 * (first + q) - skew + e; };
  // All of a thread's words are requested at once; only that thread reads them.
  if (IN_SMEM) {
#pragma unroll 4
    for (int q = tid; q < nq; q += SF_THREADS) {
      if (whole(q))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(data4 + q)), "l"(base + 4ll * (first + q)) : "memory");
      else
        data4[q] = fetch(q);
    }
  }
  const float temp = p.temperature ? __ldcg(p.temperature + row) : 0.f;
  const int k_asked = p.top_k ? __ldcg(p.top_k + row) : 0;
  const float top_p = p.top_p ? __ldcg(p.top_p + row) : 1.f, min_p = p.min_p ? __ldcg(p.min_p + row) : 0.f;
  const bool by_k = k_asked > 0 && k_asked < p.vocab, by_p = top_p < 1.f, by_m = min_p > 0.f;
  const double t64 = (double)fminf(temp, 1e30f);
  const float inv_t = (float)fmin(1.0 / t64, 3e38);            // (M - M) / T stays 0 and -inf / T -inf
  const float k2 = (float)fmin(1.4426950408889634 / t64, 3e38);
  if (IN_SMEM) asm volatile("cp.async.wait_all;" ::: "memory");

  // ---- largest logit, and where sums are needed the sum of the weights against it, in one pass: each thread against its own largest ------------
  const bool sums = temp > 0.f && !(by_k && k_asked <= SF_SHORT) && (by_p || by_m || by_k);
  float mine = -INFINITY;
  double mine_sum = 0.0;
#pragma unroll 2
  for (int q = tid; q < nq; q += SF_THREADS) {
    float4 x;
    if (IN_SMEM) {
      x = data4[q];
      if (x.x != x.x || x.y != x.y || x.z != x.z || x.w != x.w) data4[q] = x = clean(x);
    } else {
      x = clean(fetch(q));
    }
    const float m = fmaxf(fmaxf(mine, fmaxf(x.x, x.y)), fmaxf(x.z, x.w));
    if (sums && m > -INFINITY) {
      if (m > mine) {
        mine_sum *= (double)exp2_approx((mine - m) * k2);      // (0 before the first)
        mine = m;
      }
      if (m < INFINITY)                                        // (+inf: no sum is asked for)
        mine_sum += (double)((exp2_approx((x.x - m) * k2) + exp2_approx((x.y - m) * k2)) + (exp2_approx((x.z - m) * k2) + exp2_approx((x.w - m) * k2)));
    }
    mine = m;
  }
  sf_cluster_wait();
  struct Most { double sum; float m, least; };                 // sum of the weights against the largest, the largest, and the smallest of the threads' largest
  const auto scaled = [k2](double sum, float from, float to) { return from == to ? sum : sum * (double)exp2_approx((from - to) * k2); };      // (from -inf: 0)
  const Most most = sf_reduce_by(g, Most{mine_sum, mine, mine > -INFINITY ? mine : INFINITY}, [scaled](Most a, int n) {
    const float m = sf_unorder(__reduce_max_sync(0xffffffffu, sf_order(a.m)));
    return Most{sf_warp_sum(scaled(a.sum, a.m, m), n), m, sf_unorder(__reduce_min_sync(0xffffffffu, sf_order(a.least)))};
  }, [scaled](Most a, Most b) {
    const float m = fmaxf(a.m, b.m);
    return Most{scaled(a.sum, a.m, m) + scaled(b.sum, b.m, m), m, fminf(a.least, b.least)};
  });
  const float M = most.m;
  auto finish = [&](int token) { if (g.rank == 0 && tid == 0) p.tokens[row] = token; };

  if (!(M > -INFINITY)) { finish(0); return; }
  if (!(temp > 0.f) || M == INFINITY) {
    int at = 0x7fffffff;
    if (mine == M)
      for (int q = tid; q < nq && at == 0x7fffffff; q += SF_THREADS) {
        const float4 x = word(q);
        const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 3; e >= 0; --e) if (v[e] == M) at = index_of(q, e);
      }
    at = sf_reduce(g, at, [](int a, int b) { return min(a, b); });
    finish(at);
    return;
  }
  const unsigned long long hrow = hash_row(p.keys ? p.keys[row] : 0ull, p.counters ? (unsigned int)p.counters[row] : 0u);
  if (!by_k && !by_p && !by_m) {
    // no filter: what sample_kernel computes, so that a row's token does not change with the other rows' filters
    const float inv = 1.f / temp;
    struct Plain { float s; int i; };
    Plain b{-INFINITY, 0x7fffffff};
    for (int q = tid; q < nq; q += SF_THREADS) {
      const float4 x = word(q);
      const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = index_of(q, e);
        if (!(v[e] > -INFINITY)) continue;
        const float s = gumbel_score(v[e], inv, bits_to_uniform(hash_bits(hrow, (unsigned int)i)));
        if (s > b.s || (s == b.s && i < b.i)) b = Plain{s, i};
      }
    }
    b = sf_reduce(g, b, [](Plain a, Plain c) { return (c.s > a.s || (c.s == a.s && c.i < a.i)) ? c : a; });
    finish(b.i == 0x7fffffff ? 0 : b.i);
    return;
  }
  auto z64 = [&](float l) { return ((double)l - (double)M) / t64; };
  auto score64 = [&](float l, int i) {
    return z64(l) - log(-log(((double)hash_bits(hrow, (unsigned int)i) + 0.5) / 8388608.0));
  };

  // ---- the short way -------------------------------------------------------------------------------------------------------------------
  if (by_k && k_asked <= SF_SHORT) {
    const float low = M - SF_BELOW * fminf(temp, 1e30f), least = fmaxf(most.least, low);
    const float scale = fminf(0.999f * SF_BINS / (M - least), 1e37f);          // (0 times it is 0)
    auto place = [&](float l) { return l > -INFINITY ? (M - l) * scale : INFINITY; };      // grows as the logit falls
    const float at = place(mine);
    if (at < (float)SF_BINS) atomicAdd(&sh.hist[0][(int)at], 1u);
    uint32_t before;
    const int bin = sf_find_bin(g, sh.hist[0], (uint32_t)k_asked, before);
    // the logits at least as large as the k-th largest of the threads' largest, or, with fewer threads than that, all that weigh anything
    auto wanted = [&](float l) { return bin < SF_BINS ? place(l) < (float)(bin + 1) : l >= low; };
    if (wanted(mine)) {                                            // a thread whose largest is behind the end has nothing to send
      const uint32_t n_addr = sf_remote(&sh.list_n, 0);
      for (int q = tid; q < nq; q += SF_THREADS) {
        const float4 x = word(q);
        const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (wanted(v[e])) {
            const uint32_t n = sf_add_remote(n_addr, 1u);
            if (n < SF_LIST) {
              sf_st_remote(sf_remote(&sh.list_l[n], 0), __float_as_uint(v[e]));
              sf_st_remote(sf_remote(&sh.list_i[n], 0), (uint32_t)index_of(q, e));
            }
          }
      }
    }
    sf_cluster_sync();
    const uint32_t sent = sf_ld_remote(sf_remote(&sh.list_n, 0));
    sf_cluster_sync();                                         // nobody reads the first CTA's memory any more
    if (sent <= SF_LIST) {
      if (g.rank != 0) return;
      const int n = (int)sent, kept = min(n, k_asked);
      if (tid < n) {
        const float l = sh.list_l[tid];
        const int i = sh.list_i[tid];
        int r = 0;
        for (int j = 0; j < n; ++j) r += in_front(sh.list_l[j], sh.list_i[j], Border{l, i}) ? 1 : 0;
        sh.rank_l[r] = l;
        sh.rank_i[r] = i;
      }
      __syncthreads();
      const int lane = tid & 31, warp = tid >> 5;
      const float l = tid < kept ? sh.rank_l[tid] : 0.f;
      const int i = tid < kept ? sh.rank_i[tid] : 0x7fffffff;
      const double w = tid < kept ? exp(z64(l)) : 0.0;
      double s = w;                                            // sum of w up to and with this place
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
      }
      if (lane == 31) sh.warp_sum[warp] = s;
      __syncthreads();
      double total = 0.0;
      for (int c = 0; c < SF_THREADS / 32; ++c) {
        if (c == warp) s += total;
        total += sh.warp_sum[c];
      }
      const bool in = tid == 0 || (tid < kept && (!by_p || s - w < (double)top_p * total) && (!by_m || w >= (double)min_p));
      Best64 b{in ? score64(l, i) : -INFINITY, i, l};
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        Best64 c{__shfl_xor_sync(0xffffffffu, b.s, o), __shfl_xor_sync(0xffffffffu, b.i, o), 0.f};
        if (c.s > b.s || (c.s == b.s && c.i < b.i)) b = c;
      }
      __syncthreads();
      if (lane == 0) { sh.warp_sum[warp] = b.s; sh.scan[warp] = (uint32_t)b.i; }
      __syncthreads();
      if (tid == 0) {
        for (int c = 1; c < SF_THREADS / 32; ++c) {
          const double cs = sh.warp_sum[c];
          const int ci = (int)sh.scan[c];
          if (cs > b.s || (cs == b.s && ci < b.i)) { b.s = cs; b.i = ci; }
        }
        p.tokens[row] = b.i;
      }
      return;
    }
  }

  // ---- the border of a large top_k, digit by digit: of the logits, then of the index among equal ones ---------------------------------------
  Border border{-INFINITY, 0};                                 // every token that is there lies in front of it
  if (by_k) {
    uint32_t want = (uint32_t)k_asked, key = 0, index = 0;
    int turn = 0;
    bool all = false, ties = false;
    for (int digit = 0; digit < 7 && !all; ++digit) {          // four of the logit, three of the index
      uint32_t* hist = sh.hist[turn & 1];
      ++turn;
      __syncthreads();
      for (int b = tid; b < SF_BINS; b += SF_THREADS) hist[b] = 0;
      __syncthreads();
      const int shift = digit < 4 ? 24 - 8 * digit : 16 - 8 * (digit - 4);
      for (int q = tid; q < nq; q += SF_THREADS) {
        const float4 x = word(q);
        const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!(v[e] > -INFINITY)) continue;
          const uint32_t kk = sf_key(v[e]), ii = (uint32_t)index_of(q, e);
          if (digit < 4) {
            if (digit == 0 || (kk >> (shift + 8)) == (key >> (shift + 8))) atomicAdd(&hist[255 - ((kk >> shift) & 255)], 1u);
          } else if (kk == key && (ii >> (shift + 8)) == (index >> (shift + 8))) {
            atomicAdd(&hist[(ii >> shift) & 255], 1u);
          }
        }
      }
      uint32_t before;
      const int bin = sf_find_bin(g, hist, want, before);
      if (bin == SF_BINS) { all = true; break; }               // fewer tokens than top_k (first digit only)
      want -= before;
      if (digit < 4) key |= (uint32_t)(255 - bin) << shift;
      else index |= (uint32_t)bin << shift;
      ties = digit >= 4;
    }
    if (!all) border = Border{sf_unkey(key), ties ? (int)index + 1 : 0x7fffffff};
  }

  // ---- rejection ---------------------------------------------------------------------------------------------------------------------------------
  auto weight = [&](float l) { return exp2_approx((l - M) * k2); };
  // the sum of the weights in front of a border, and how many there are
  struct Sum { double s; int n; int pad; };
  auto sum_in_front = [&](const Border& b) {
    double s = 0.0;
    int n = 0;
    for (int q = tid; q < nq && mine >= b.l; q += SF_THREADS) {
      const float4 x = word(q);
      const float v[4] = {x.x, x.y, x.z, x.w};
      if (fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)) < b.l) continue;
      float w4 = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (in_front(v[e], index_of(q, e), b)) { w4 += weight(v[e]); ++n; }
      s += (double)w4;
    }
    return sf_reduce_by(g, Sum{s, n, 0}, [](Sum a, int lanes) {
      // (both halves of warp 0 have the same when it joins the warps' sums: their number is not added up twice)
      const int n = __reduce_add_sync(0xffffffffu, a.n);
      return Sum{sf_warp_sum(a.s, lanes), lanes < 32 ? n / (32 / lanes) : n, 0};
    }, [](Sum a, Sum c) { return Sum{a.s + c.s, a.n + c.n, 0}; });
  };
  // the same of two borders in whole numbers, for what the above cannot tell: units of 2^-unit, the sum of a row below 2^63
  struct Sum64 { unsigned long long inner, outer; };
  auto sums64 = [&](const Border& inner, const Border& outer) {
    const double one = ldexp(1.0, 62 - (32 - __clz(p.vocab)));
    Sum64 s{0ull, 0ull};
    for (int q = tid; q < nq; q += SF_THREADS) {
      const float4 x = word(q);
      const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll 1
      for (int e = 0; e < 4; ++e) {
        if (!(v[e] > -INFINITY) || !in_front(v[e], index_of(q, e), outer)) continue;
        const unsigned long long w = __double2ull_rn(exp(z64(v[e])) * one);
        s.outer += w;
        if (in_front(v[e], index_of(q, e), inner)) s.inner += w;
      }
    }
    return sf_reduce(g, s, [](Sum64 a, Sum64 c) { return Sum64{a.inner + c.inner, a.outer + c.outer}; });
  };

  const Border first_border = border;                          // of all that top_k leaves
  const double total = by_k ? sum_in_front(first_border).s : most.sum;
  double sum = total;                                          // of what is in front of `border`
  for (;;) {
    Best best{-INFINITY, 0x7fffffff, 0.f, -INFINITY};
    const float log_sum = (float)log(sum);
    for (int bounded = 1; bounded >= 0 && best.i == 0x7fffffff; --bounded) {
      // the smallest z that may be drawn: of min-p, of top-p, and of what can reach the bound (-log(-log u) is at most 16.64)
      float zc = -INFINITY;
      if (by_m) zc = fmaxf(zc, logf(min_p) - 1e-4f);
      if (by_p) zc = fmaxf(zc, logf(fmaxf((1.f - top_p) / (float)p.vocab, 1e-37f)) + (float)log(total) - 1e-2f);
      const float bound = log_sum - 3.f;
      if (bounded) zc = fmaxf(zc, bound - 16.7f);
      zc = fminf(zc, 0.f);                                     // the first is always kept
      const float l_cut = M + zc * fminf(temp, 1e30f) - 1e-5f * fabsf(M);
      const float reach = bounded ? exp2f(-bound * 1.4426951f) * 1.01f : INFINITY;       // -log u < w e^-bound for a score above the bound
      const float cut = fmaxf(fmaxf(l_cut, border.l), -FLT_MAX);
      const bool inside = border.l > -INFINITY;
      auto score = [&](float l, int i) {
        // 1 - u = 2 - 2^-24 - (1 + b / 2^23), the bits b as a mantissa
        const uint32_t b = hash_bits(hrow, (unsigned int)i);
        if ((2.f - __uint_as_float(0x3f800000u | b)) - 1.f / 16777216.f <= weight(l) * reach && (!inside || in_front(l, i, border))) {
          const float s = (l - M) * inv_t - logf(-logf(bits_to_uniform(b)));
          if (s > best.s || (s == best.s && i < best.i)) { best.second = fmaxf(best.second, best.s); best.s = s; best.i = i; best.l = l; }
          else best.second = fmaxf(best.second, s);
        }
      };
      // 32 logits at a time: which of them pass the cut is cheap to see, and only those are looked at one by one (a hash is twenty
      // instructions, and where each lane takes its own, few lanes take many).  Scoring all four of a word instead where most pass, and
      // queues that a warp takes 32 from at a time, were both slower: 65 and 77 us for 64 rows of 151936, against 64.
      if (mine >= cut)
        for (int q0 = tid; q0 < nq; q0 += 8 * SF_THREADS) {
          uint32_t pass = 0;
          for (int w = 0; w < 8; ++w) {
            const int q = q0 + w * SF_THREADS;
            if (q >= nq) break;
            const float4 x = word(q);
            pass |= (x.x >= cut ? 1u << (4 * w) : 0u) | (x.y >= cut ? 2u << (4 * w) : 0u) | (x.z >= cut ? 4u << (4 * w) : 0u) | (x.w >= cut ? 8u << (4 * w) : 0u);
          }
          for (; pass; pass &= pass - 1) {
            const int bit = __ffs(pass) - 1, q = q0 + (bit >> 2) * SF_THREADS, i = index_of(q, bit & 3);
            score(IN_SMEM ? data[4 * q + (bit & 3)] : __ldcg(row_ptr + i), i);
          }
        }
      auto better = [](Best a, Best c) {
        const bool swap = c.s > a.s || (c.s == a.s && c.i < a.i);
        const float second = fmaxf(fmaxf(a.second, c.second), fminf(a.s, c.s));
        return swap ? Best{c.s, c.i, c.l, second} : Best{a.s, a.i, a.l, second};
      };
      best = sf_reduce_by(g, best, [](Best a, int) {
        const int order = sf_order(a.s), top = __reduce_max_sync(0xffffffffu, order);
        const int i = __reduce_min_sync(0xffffffffu, order == top ? a.i : 0x7fffffff);
        const bool won = order == top && a.i == i;
        const int from = __ffs(__ballot_sync(0xffffffffu, won)) - 1;
        const int second = __reduce_max_sync(0xffffffffu, sf_order(won ? a.second : a.s));
        return Best{sf_unorder(top), i, __shfl_sync(0xffffffffu, a.l, from), sf_unorder(second)};
      }, better);
      if (bounded && !(best.s >= bound)) best.i = 0x7fffffff;          // what was left out may be better
      if (best.i != 0x7fffffff && best.second > best.s - SF_SCORE_MARGIN) {
        // two scores too near to tell apart: in 64 bits, all that come near the best
        const float near = best.s - SF_SCORE_MARGIN;
        Best64 b{-INFINITY, 0x7fffffff, 0.f};
        for (int q = tid; q < nq; q += SF_THREADS) {
          const float4 x = word(q);
          const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll 1
          for (int e = 0; e < 4; ++e) {
            const int i = index_of(q, e);
            if (!(v[e] >= l_cut) || !(v[e] > -INFINITY) || !in_front(v[e], i, border)) continue;
            const float u = bits_to_uniform(hash_bits(hrow, (unsigned int)i));
            if ((v[e] - M) * inv_t - logf(-logf(u)) < near) continue;
            const double s = score64(v[e], i);
            if (s > b.s || (s == b.s && i < b.i)) b = Best64{s, i, v[e]};
          }
        }
        b = sf_reduce(g, b, [](Best64 a, Best64 c) { return (c.s > a.s || (c.s == a.s && c.i < a.i)) ? c : a; });
        best.i = b.i;
        best.l = b.l;
      }
    }
    const Border at{best.l, best.i};
    bool kept = !by_m || exp(z64(best.l)) >= (double)min_p;
    const Sum before = by_p || !kept ? sum_in_front(at) : Sum{0.0, 1, 0};
    if (by_p && kept) {
      const double room = (double)top_p * total, off = SF_SUM_MARGIN * total;
      if (fabs(before.s - room) > off) {
        kept = before.s < room;
      } else {
        const Sum64 s = sums64(at, first_border);
        kept = (double)s.inner < (double)top_p * (double)s.outer;
      }
    }
    if (kept || before.n == 0) { finish(best.i); return; }
    border = at;
    sum = before.s;
  }
}

static void sf_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, int ctas, int cluster, size_t smem, cudaStream_t stream) {
  cfg = {};
  cfg.gridDim = dim3((unsigned)ctas); cfg.blockDim = dim3(SF_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_pdl_enabled ? 2 : 1;
}

// How many clusters of 1 << log2 CTAs the GPU has room for at a time, with `per_sm` CTAs on an SM.  (A cluster lies within one of the GPU's parts of
// some 18 SMs: 32 clusters of 8, two CTAs an SM, on 148 SMs.)
static cudaError_t sf_room(int device, int log2, int per_sm, int& room) {
  static std::atomic<int> known[64][4][2];                     // 0: not asked yet
  room = device < 64 ? known[device][log2][per_sm - 1].load() : 0;
  if (room > 0) return cudaSuccess;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  sf_config(cfg, attr, 1 << log2, 1 << log2, per_sm == 2 ? SF_PAIR_BYTES : SF_SLICE_BYTES, nullptr);
  cfg.numAttrs = 1;
  const cudaError_t e = cudaOccupancyMaxActiveClusters(&room, sample_filtered_kernel<true>, &cfg);
  if (e != cudaSuccess) return e;
  if (room < 1) room = 1;
  if (device < 64) known[device][log2][per_sm - 1].store(room);
  return cudaSuccess;
}

// The cluster of a row: the one for which the rounds of rows that there is room for take least time, a round of slices of n logits
// 8.5 us + n x 0.4 ns, or 0.62 ns where two CTAs share an SM; with a word a thread at least, and slices that fit shared memory.  Measured (us,
// clusters of 8, 4, 2, 1): 37 rows of 50003 23.4, 17.0, 19.0, 28.9; 128 rows of 32000 48, 32, 25, 34; 64 rows of 151936 50, 60, 222, 431; 8 rows
// of 100000 14.3, 18.9, 30, 167 (slices that do not fit are read from memory each time).
static cudaError_t sf_launch(const FilterParams& p, int rows, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured{0ull};     // a bit a device
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (!(configured.load() >> (device & 63) & 1ull)) {
    e = cudaFuncSetAttribute(sample_filtered_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SF_SLICE_BYTES);
    if (e != cudaSuccess) return e;
    configured.fetch_or(1ull << (device & 63));
  }
  const int words = (p.vocab + 3 + 3) / 4;
  int cluster = 0;
  float least = 0.f;
  for (int log2 = 0; log2 <= SF_MAX_LOG2; ++log2) {
    const int slice = (words + (1 << log2) - 1) >> log2;
    if (slice * 16 > SF_SLICE_BYTES) continue;
    const int per_sm = slice * 16 <= SF_PAIR_BYTES ? 2 : 1;
    int room = 0;
    e = sf_room(device, log2, per_sm, room);
    if (e != cudaSuccess) return e;
    const float time = (float)((rows + room - 1) / room) * (8.5f + (float)slice * (per_sm == 2 ? 4 * 0.62e-3f : 4 * 0.4e-3f));
    if (cluster == 0 || time < least) { cluster = 1 << log2; least = time; }
    if (slice <= SF_THREADS) break;
  }
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  if (cluster == 0) {
    sf_config(cfg, attr, rows << SF_MAX_LOG2, 1 << SF_MAX_LOG2, 0, stream);
    return cudaLaunchKernelEx(&cfg, sample_filtered_kernel<false>, p);
  }
  sf_config(cfg, attr, rows * cluster, cluster, (size_t)((words + cluster - 1) / cluster) * 16, stream);
  return cudaLaunchKernelEx(&cfg, sample_filtered_kernel<true>, p);
}

}  // namespace lb

// tokens[r] = the token drawn for logits[r * row_stride .. + vocab); see the head of this file.  temperature (none: greedy), keys,
// counters, top_k (<= 0 or >= vocab: all), top_p (>= 1: all), min_p (<= 0: all): one a row, each may be null.
LB_EXPORT int lb_sample_filtered(int* tokens, const float* logits, long long row_stride, const float* temperature,
                                 const unsigned long long* keys, const int* counters, const int* top_k, const float* top_p,
                                 const float* min_p, int num_rows, int vocab, cudaStream_t stream) {
  LB_CHECK_ARG(num_rows >= 0 && vocab > 0 && vocab < (1 << 24) && row_stride >= vocab, "sample_filtered: bad sizes rows=%d vocab=%d (at most %d) row stride=%lld",
               num_rows, vocab, (1 << 24) - 1, row_stride);
  if (num_rows == 0) return 0;
  LB_CHECK_ARG(num_rows <= (1 << 24), "sample_filtered: %d rows, at most %d a launch", num_rows, 1 << 24);
  const lb::FilterParams p{tokens, logits, temperature, keys, counters, top_k, top_p, min_p, row_stride, vocab};
  const cudaError_t e = lb::sf_launch(p, num_rows, stream);
  if (e != cudaSuccess) { lb::set_error("sample_filtered: launch failed: %s", cudaGetErrorString(e)); return 2; }
  lb::count_launch();
  return 0;
}

// Reads and clears the flag a bounded wait of this kernel sets when it gives up (0: none).
LB_EXPORT int lb_sample_filtered_device_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, lb::g_sampling_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(lb::g_sampling_error, &zero, sizeof(int));
  return v;
}
