// Attention of a step whose requests share prefixes, on the 5th-generation tensor cores (bfloat16, heads of 64 or 128, up to 128 query
// heads a kv head, pages of 8 tokens and more that are powers of two).  The plan, the walk and the combination are attention_shared.cuh's.
//
// One CTA an SM walks its piece of the line of key blocks, segment after segment.  There are two tiles, A and B, of up to 128 query rows each,
// on which two sets of warps and two halves of tensor memory work: on a segment with more rows both on every block, else on halves of a
// segment's blocks, or on two requests' own keys (a handful of rows each) side by side.  Copies of keys and values run on through all segments.
//     S = Q K^T      tcgen05.mma, operands from shared memory, two S buffers a tile
//     P              one thread a query row, online softmax in 32 bits, P (bfloat16) written over S in tensor memory
//     O += P V       tcgen05.mma, P from tensor memory, V as it lies in the pages; O stays in tensor memory
// The sum of a row's weights is taken before they are rounded to bfloat16 for P V.  A row's reference value is the maximum of its first
// block, and moves (O is rescaled then) when a block's weights against it sum up to 2^15: what the maximum was does not matter to the quotient.
//
// What bounds it: the way of a block through barriers, tensor memory and registers.  A block that both tiles work on takes 2080 cycles, of
// which the tensor cores are at work for 1000 and the exponentials take 1024 (two warps a quarter of the SM); taking the exponentials out
// leaves 1800.  64 requests with a token each behind 8192 common keys, up to 256 keys of their own, 32 heads of 128 on 8: 25 us of the 38.5 that
// the call takes (plan 4.4, combination 6 to 8; recorded), 66 MB read; by the counters the tensor cores are busy for 26 % of the cycles (41 % on
// the SMs that have the prefix), the issue slots for 38 %, DRAM for 25 %.  8 requests: 22.2 us in all; 2 requests behind 256: 14.3.
// Where only one tile works on a block, the copying warps set the pace, 1300 to 1500 cycles a block: their instructions, not the memory (copies that
// read nothing take as long), which is why their loop looks nothing up that it waits for and makes all addresses before the first copy.
//
// Why 128-row tiles even for one request's few rows: a block of 64 keys takes the tensor cores some 500 cycles whatever the rows, and the
// memory 1400 cycles at its full rate shared by all SMs, so rows that are not there cost nothing; one kernel for both kinds of work is what
// lets the line be cut evenly.
//
// Warps: 0 and 3 copy keys, 2 and 5 values (cp.async, 16 bytes a thread, swizzled for the tensor cores; a warp has half of every block, two
// blocks in flight, and a quarter of the SM that no other copying warp has: three groups of 11 behind 2352 keys 37.2 us against 39.1); 1 issues tile
// A's products and owns the tensor memory, 4 tile B's; 6..9 softmax of A, 10..13 of B.  Each goes through the
// segments, which warp 0 finds.  Barriers tell one turn from the next only, so each tile has barriers of its own for the stages of the rings, and a
// copying warp speaks to the tiles that read a block.  All waits are bounded; when one gives up, the CTA records it and every role leaves.
#include "attention_shared.cuh"
#include "attention_tcgen05.cuh"

#include <atomic>

namespace lb {

constexpr int SC_K_STAGES = 4, SC_V_STAGES = 5;                // a block of values stays until its keys' scores have become weights
constexpr int SC_BARS = 2 * (SC_K_STAGES + SC_V_STAGES) + 8;   // barriers of a tile
constexpr int SC_THREADS = 448, SC_SOFTMAX = 6;                // the first of the softmax warps
enum : int { SC_ERR_Q = 401, SC_ERR_KV_FULL = 402, SC_ERR_KV_EMPTY = 403, SC_ERR_S_FULL = 404, SC_ERR_P_FULL = 405, SC_ERR_O_FULL = 406, SC_ERR_O_FREE = 407, SC_ERR_SEGMENT = 408 };

// Shared memory: queries of A and B | ring of keys | ring of values | barriers.  Rows of 128 bytes (64 elements), 128-byte swizzle, the second
// 64 elements of a head a half further on.
template <int D> struct ScLayout {
  static constexpr int HALVES = D / 64;
  static constexpr int KV_HALF = AS_KEYS * 128, KV_TILE = HALVES * KV_HALF;
  static constexpr int Q_TILE = HALVES * TA_HALF_BYTES;
  static constexpr int K_OFF = 2 * Q_TILE, V_OFF = K_OFF + SC_K_STAGES * KV_TILE, BAR_OFF = V_OFF + SC_V_STAGES * KV_TILE;
  static constexpr int BYTES = BAR_OFF + 2 * SC_BARS * 8 + 16;     // and the tensor memory's address and two flags
};

// What the two tiles work on side by side, a part each: halves of one segment's blocks, segments of two requests, or (both) the same blocks
// with other rows.  The parts' blocks alternate in the rings of keys and values, so that neither tile waits for the other's to pass.
// Warp 0, which copies keys, makes steps of the CTA's segments, one ahead of its copies, and leaves them in a ring; the others read them there.
// A slot comes again after SC_SEGMENTS steps.  The rings of keys and values do not hold warp 0 back for a tile that the steps leave out (tile B has
// no block of a segment of one block, nor beside a request's few rows without a partner: 83 such steps in a row at 256 requests in pairs behind
// 64 keys, 32 kv heads).  So every warp that reads the steps gives each half of the ring back when it is through with it, and warp 0 waits for all of them
// before it writes that half again.  It cannot wait for itself: the steps of that half lie SC_SEGMENTS / 2 behind, and all their blocks are handed over.
struct ScPart {                          // a Segment, and
  int kv_head, request, first, tokens;   // tokens 0: nothing for this tile
  int key_lo, key_hi, block, blocks;     // blocks 0 of a part with tokens: it leaves an empty partial result
  int row_low, row_high, position;
  int kind;                              // one of the following, + SC_SHARED
};
struct ScStep { ScPart part[2]; };
enum : int { SC_END = 0, SC_PARTS = 1, SC_BOTH = 2, SC_HALVES = 3, SC_SHARED = 4 };      // of either part
constexpr int SC_SEGMENTS = 32, SC_SEGMENTS_HALF = SC_SEGMENTS / 2;
constexpr int SC_STEP_READERS = 13;      // warps 1 to 13

__device__ __forceinline__ void sc_tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Waits, bounded like those of attention_tcgen05.cuh, in as few instructions as can be: the roles of this kernel are many, and what they
// execute has to stay in the SM's instruction cache (with 138 KB of code most of the time went into fetching it).  What gave up is left in
// shared memory, and reported at the kernel's end.
constexpr unsigned SC_WAIT_CYCLES = 2000000000u;
template <bool SLEEP>
__device__ __forceinline__ bool sc_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  const unsigned t0 = (unsigned)clock();
#pragma unroll 1
  while (!ta_mbar_try_wait(bar, parity)) {
    if (SLEEP) __nanosleep(40);
    if (*abort_flag) return false;
    if ((unsigned)clock() - t0 > SC_WAIT_CYCLES) { *abort_flag = code; return false; }
  }
  return true;
}
// Whether a wait would be over, without any waiting.
__device__ __forceinline__ bool sc_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// A count in shared memory that one thread raises when what it counts has been written, and the others wait for: more than n.
__device__ __forceinline__ void sc_publish(uint32_t addr, int n) { asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(addr), "r"(n) : "memory"); }
__device__ __forceinline__ bool sc_wait_count(uint32_t addr, int n, volatile int* abort_flag) {
  const unsigned t0 = (unsigned)clock();
#pragma unroll 1
  for (;;) {
    int v;
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    if (v > n) return true;
    __nanosleep(40);
    if (*abort_flag) return false;
    if ((unsigned)clock() - t0 > SC_WAIT_CYCLES) { *abort_flag = SC_ERR_SEGMENT; return false; }
  }
}

// The lowest n bits (none below 0, all from 64 on).
__device__ __forceinline__ unsigned long long sc_low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

template <int D>
__global__ void __launch_bounds__(SC_THREADS, 1) attention_shared_tc_kernel(SharedParams p) {
  typedef ScLayout<D> L;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(16) ScStep steps[SC_SEGMENTS];
  __shared__ int steps_found;
  __shared__ unsigned long long steps_read[2];                // barriers of the ring's halves
  __shared__ unsigned long long products_done[2];             // of the tiles: all products there are
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = ta_smem_u32(smem);
  const uint32_t bars = sbase + L::BAR_OFF;
  // of tile t: keys (values) in stage s there, and read; of S buffer b: S complete, P written, P V complete; queries there, O read
  auto k_full = [&](int t, int s) { return bars + 8u * (t * SC_BARS + s); };
  auto k_empty = [&](int t, int s) { return bars + 8u * (t * SC_BARS + SC_K_STAGES + s); };
  auto v_full = [&](int t, int s) { return bars + 8u * (t * SC_BARS + 2 * SC_K_STAGES + s); };
  auto v_empty = [&](int t, int s) { return bars + 8u * (t * SC_BARS + 2 * SC_K_STAGES + SC_V_STAGES + s); };
  auto s_full = [&](int t, int b) { return bars + 8u * (t * SC_BARS + SC_BARS - 8 + b); };
  auto p_full = [&](int t, int b) { return bars + 8u * (t * SC_BARS + SC_BARS - 8 + 2 + b); };
  auto pv_done = [&](int t, int b) { return bars + 8u * (t * SC_BARS + SC_BARS - 8 + 4 + b); };
  auto q_full = [&](int t) { return bars + 8u * (t * SC_BARS + SC_BARS - 8 + 6); };
  auto o_free = [&](int t) { return bars + 8u * (t * SC_BARS + SC_BARS - 8 + 7); };
  uint32_t* tmem_slot = (uint32_t*)(smem + L::BAR_OFF + 2 * SC_BARS * 8);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile int* holes = (volatile int*)(tmem_slot + 2);       // some key of this CTA's segments lies in no page

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      for (int i = 0; i < SC_K_STAGES; ++i) { ta_mbar_init(k_full(t, i), 2); ta_mbar_init(k_empty(t, i), 1); }        // two warps copy the halves of a block
      for (int i = 0; i < SC_V_STAGES; ++i) { ta_mbar_init(v_full(t, i), 2); ta_mbar_init(v_empty(t, i), 1); }
      for (int b = 0; b < 2; ++b) { ta_mbar_init(s_full(t, b), 1); ta_mbar_init(p_full(t, b), 4); ta_mbar_init(pv_done(t, b), 1); }
      ta_mbar_init(q_full(t), 4); ta_mbar_init(o_free(t), 4);
    }
    for (int h = 0; h < 2; ++h) { ta_mbar_init(ta_smem_u32(&steps_read[h]), SC_STEP_READERS); ta_mbar_init(ta_smem_u32(&products_done[h]), 1); }
    *abort_flag = 0;
    *holes = 0;
    steps_found = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ta_smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  pdl_wait();
  pdl_trigger();                               // behind the wait: the combining kernel reads the plan before its own
  const uint32_t tmem = *tmem_slot;            // columns: tile t's S buffers at t * 128 and t * 128 + 64 (P over their first 32), O at 256 + t * 128

  const int G = p.group, per = p.lane_tokens, cta = blockIdx.x;
  const uint32_t found_addr = ta_smem_u32(&steps_found);
  // Tile t's part of the n-th step, when it has been found; false at the end of the line (or when a wait gave up).
  auto step = [&](int n, int t, ScPart& g) -> bool {
    if (!sc_wait_count(found_addr, n, abort_flag)) return false;
    const int4* at = reinterpret_cast<const int4*>(&steps[n % SC_SEGMENTS].part[t]);
    const int4 a = at[0], b = at[1], c = at[2];
    g.kv_head = a.x; g.request = a.y; g.first = a.z; g.tokens = a.w;
    g.key_lo = b.x; g.key_hi = b.y; g.block = b.z; g.blocks = b.w;
    g.row_low = c.x; g.row_high = c.y; g.position = c.z; g.kind = c.w;
    return g.kind != SC_END;
  };
  auto half_read = [&](int n) { return ta_smem_u32(&steps_read[(n / SC_SEGMENTS_HALF) & 1]); };      // of step n's half
  // One thread of a reading warp that needs no step in front of the n-th any more: where that ends a half, the half goes back.
  auto give_back = [&](int n) {
    if (n > 0 && n % SC_SEGMENTS_HALF == 0) ta_mbar_arrive(half_read(n - 1));
  };
  // Where block i of tile t's part lies among the step's: A's and B's in turn, then what the longer part has more.
  auto place = [](int t, int i, int others, int kind) { return (kind & 3) == SC_BOTH ? i : i + min(t ? i + 1 : i, others); };

  if (warp != 1 && warp != 4 && warp < SC_SOFTMAX) {
    // ---- copies: warps 0 and 3 the halves of every block of keys, 2 and 5 of values -----------------------------------------------------
    const bool is_v = warp == 2 || warp == 5;
    const int half = warp >= 3 ? 1 : 0;
    constexpr int CHUNKS = D / 8, RPI = 32 / CHUNKS;           // 16-byte chunks of a row, rows an instruction
    const int c = lane % CHUNKS, rp = lane / CHUNKS;           // a lane copies chunk c of the rows rp, rp + RPI, ... of its half
    const uint8_t* pool = (const uint8_t*)(is_v ? p.v_cache : p.k_cache) + c * 16 + rp * (D * 2);
    const uint32_t ring = sbase + (is_v ? L::V_OFF : L::K_OFF) + (uint32_t)(c >> 3) * L::KV_HALF + (uint32_t)(half * 32 + rp) * 128u;
    uint32_t swizzled[8 / RPI];                // this lane's chunk in its rows of eight
#pragma unroll
    for (int u = 0; u < 8 / RPI; ++u) swizzled[u] = (uint32_t)(RPI * u * 128 + (((c & 7) ^ (rp + RPI * u)) << 4));
    const uint32_t full0 = is_v ? v_full(0, 0) : k_full(0, 0), empty0 = is_v ? v_empty(0, 0) : k_empty(0, 0);
    const int ps = p.page_size, shift = p.page_shift, size = min(ps, 32), bits = min(shift, 5);
    const size_t page_stride = (size_t)p.kv_heads * ps * (D * 2);
    const int stages = is_v ? SC_V_STAGES : SC_K_STAGES;
    int n = 0, handed = 0, seen = 0;           // blocks requested, handed over; steps looked at
    int stage_n = 0, stage_h = 0;              // their stages
    uint32_t used = 0, turns = 0;              // bits 2 s + t: whether tile t reads stage s's block, and the parity of the next wait for it
    // (Of warp 0) the segment to come, requested when the one before it was taken (and looked at when it is needed), and the one after it in the list.
    Segment found;
    const int2 piece = as_piece(p, cta, found);
    int at_segment = piece.x + 1;
    auto request = [&]() {
      if (at_segment <= piece.y) found = as_segment(p, at_segment++);
      else found.blocks = 0;
    };
    auto find_step = [&]() {
      if (seen >= SC_SEGMENTS && seen % SC_SEGMENTS_HALF == 0) {
        const bool go = sc_wait<true>(half_read(seen), (uint32_t)(seen / SC_SEGMENTS - 1) & 1u, abort_flag, SC_ERR_SEGMENT);
        if (__any_sync(0xffffffffu, !go)) return;              // nothing is found: step() sees the flag
      }
      int kind = SC_END;
      bool keep = false;                       // whether the segment at hand is for tile B too, or for the step after this one
      // At most two segments: the second one if it is a request's few rows, as the first.
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        if (t == 1 && !keep) request();
#pragma unroll 1
        while (found.blocks == 0 && at_segment <= piece.y) request();
        const Segment& g = found;
        const bool few = !g.shared && g.tokens * G <= AS_FOLD_ROWS;
        int block = g.block, blocks = g.blocks, tokens = g.tokens;
        keep = false;
        if (t == 0) {
          kind = blocks == 0 ? SC_END : g.tokens > per ? SC_BOTH : few ? SC_PARTS : SC_HALVES;
          if (kind == SC_HALVES) blocks = (blocks + 1) >> 1;
          keep = kind >= SC_BOTH;
        } else if (kind == SC_HALVES) {
          block += (blocks + 1) >> 1;
          blocks >>= 1;
        } else if (kind == SC_PARTS && !(blocks > 0 && few)) {
          keep = true;
          blocks = tokens = 0;
        }
        if (lane == 0) {
          int4* at = reinterpret_cast<int4*>(&steps[seen % SC_SEGMENTS].part[t]);
          at[0] = make_int4(g.kv_head, g.request, g.first, tokens);
          at[1] = make_int4(g.key_lo, g.key_hi, block, blocks);
          at[2] = make_int4(g.row_low, g.row_high, g.position, kind == SC_END ? SC_END : kind + (g.shared ? SC_SHARED : 0));
        }
      }
      if (lane == 0) sc_publish(found_addr, seen + 1);
      if (!keep) request();
      __syncwarp();
    };
    // Tells the tiles that read them that the blocks in front of the `end`-th are there.
    auto hand_over = [&](int end) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");         // visible to the tensor cores
      __syncwarp();
#pragma unroll 1
      for (; handed < end; ++handed) {
        if (lane < 2 && ((used >> (2 * stage_h + lane)) & 1u)) ta_mbar_arrive(full0 + 8u * (uint32_t)(lane * SC_BARS + stage_h));
        if (++stage_h == stages) stage_h = 0;
      }
    };
    // The block to come: this half's first key, the keys of its part, lane i the id of the half's i-th page (-1: no page, or no key of the part in
    // it).  It is looked up before the one at hand is copied, across the ends of steps.
    int left0 = 0, left1 = 0, key0 = 0, key1 = 0, lo0 = 0, lo1 = 0, hi0 = 0, hi1 = 0, turn = 0;
    int kb = 0, lo = 0, hi = 0, id = -1;
    bool looked_up = false;                    // whether id has been read from the table; it is looked at a block later
    uint32_t tiles = 0;
    bool both = false, ok = true, more = true;
    const int* bt0 = nullptr;
    const int* bt1 = nullptr;
    const uint8_t* head0 = nullptr;
    const uint8_t* head1 = nullptr;
    const uint8_t* head = nullptr;
#pragma unroll 1
    while (more && ok) {
      // ---- the block at hand is the one that was looked up; the one after it
      const int kb_now = kb, lo_now = lo, hi_now = hi, ids_now = looked_up && id >= 0 && id < p.num_pages ? id : -1;
      if (looked_up && ids_now < 0) *holes = 1;                // before the block is handed over
      const uint32_t tiles_now = tiles;
      const uint8_t* head_now = head;
      if (left0 + left1 == 0) {
        if (warp == 0) find_step();
        ScPart g;
        more = step(seen, 1, g);
        both = (g.kind & 3) == SC_BOTH;
        left1 = both ? 0 : g.blocks;
        lo1 = g.key_lo; hi1 = g.key_hi;
        key1 = (g.key_lo & ~(AS_KEYS - 1)) + g.block * AS_KEYS + half * 32;
        bt1 = p.table + (size_t)g.request * p.max_pages;
        head1 = pool + (size_t)g.kv_head * ps * (D * 2);
        more = more && step(seen, 0, g);
        left0 = g.blocks;
        lo0 = g.key_lo; hi0 = g.key_hi;
        key0 = (g.key_lo & ~(AS_KEYS - 1)) + g.block * AS_KEYS + half * 32;
        bt0 = p.table + (size_t)g.request * p.max_pages;
        head0 = pool + (size_t)g.kv_head * ps * (D * 2);
        ++seen;
        __syncwarp();
        if (warp != 0 && lane == 0) give_back(seen);
        turn = 0;
      }
      looked_up = false;
      if (more) {
        const bool b = left0 == 0 || (turn && left1 > 0);
        turn = !b;
        lo = b ? lo1 : lo0; hi = b ? hi1 : hi0; kb = b ? key1 : key0;
        head = b ? head1 : head0;
        const int* bt = b ? bt1 : bt0;
        tiles = both ? 3u : b ? 2u : 1u;
        left0 -= !b; left1 -= b;
        key0 += b ? 0 : AS_KEYS; key1 += b ? AS_KEYS : 0;
        const int key = kb + lane * size;
        looked_up = lane * size < 32 && key < hi && key + size > lo;
        if (looked_up) id = bt[key >> shift];
      }
      if (tiles_now == 0) continue;            // nothing at hand yet
      // ---- its stage: the tiles that read the last block there are through with it.  While that has to be waited for, whatever has been requested
      // is handed over.
      const int s = stage_n;
      const uint32_t before = (used >> (2 * s)) & 3u, bar = empty0 + 8u * (uint32_t)((lane & 1) * SC_BARS + s);
      const bool mine = lane < 2 && ((before >> lane) & 1u);
      const uint32_t parity = (turns >> (2 * s + (lane & 1))) & 1u;
      if (__any_sync(0xffffffffu, mine && !sc_test(bar, parity))) {
        if (n > handed) {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          hand_over(n);
        }
        const bool go = !mine || sc_wait<true>(bar, parity, abort_flag, SC_ERR_KV_EMPTY);
        if (__any_sync(0xffffffffu, !go)) { ok = false; break; }
      }
      turns ^= before << (2 * s);
      used = (used & ~(3u << (2 * s))) | (tiles_now << (2 * s));
      // ---- the copies.  Keys outside lo .. hi - 1 and of no page are filled with zeros.
      const uint32_t stage = ring + (uint32_t)s * L::KV_TILE;
      const bool inner = kb_now >= lo_now && kb_now + 32 <= hi_now;        // every key may be seen
      const uint8_t* src[4];
      uint32_t there = 0;                      // bit e: whether those eight rows' page is
#pragma unroll
      for (int e = 0; e < 4; ++e) {            // eight rows at a time: they lie in one page
        const int of = __shfl_sync(0xffffffffu, ids_now, (8 * e) >> bits);
        src[e] = head_now + (size_t)max(of, 0) * page_stride + (uint32_t)((kb_now + 8 * e) & (ps - 1)) * (uint32_t)(D * 2);
        there |= of >= 0 ? 1u << e : 0u;
      }
      if (inner && there == 15u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int u = 0; u < 8 / RPI; ++u)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(stage + (uint32_t)e * 1024u + swizzled[u]), "l"(src[e] + RPI * u * (D * 2)) : "memory");
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int u = 0; u < 8 / RPI; ++u) {
            const int at = kb_now + 8 * e + rp + RPI * u;
            const uint32_t bytes = (there >> e & 1u) && at >= lo_now && at < hi_now ? 16u : 0u;        // 0: sixteen zeros
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                         ::"r"(stage + (uint32_t)e * 1024u + swizzled[u]), "l"(src[e] + RPI * u * (D * 2)), "r"(bytes) : "memory");
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      ++n;
      if (++stage_n == stages) stage_n = 0;
      // ---- the block before it is handed over.  (With one or two more in flight blocks come that much later: 64 requests behind 8192 common keys
      // 39.9 and 43.0 us against 38.9.)
      if (n - handed > 1) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        hand_over(n - 1);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (ok) hand_over(n);
  } else if (warp == 1 || warp == 4) {
    // ---- products, one thread a tile -------------------------------------------------------------------------------------------------
    const int t = warp == 1 ? 0 : 1;
    if (elect_one()) {
      constexpr uint32_t idesc_qk = ta_idesc(0, AS_KEYS), idesc_pv = ta_idesc(1, D);
      const uint32_t s_col = tmem + (uint32_t)t * 128u, o_col = tmem + 256u + (uint32_t)t * 128u;
      const uint32_t qa = sbase + t * L::Q_TILE;
      int n0 = 0, mine = 0, segments = 0;      // blocks of all segments so far, this tile's blocks and segments
      uint32_t k_turn = 0, v_turn = 0;         // bit s: the parity of this tile's next wait for stage s
      bool ok = true;
      ScPart g, other;
#pragma unroll 1
      for (int seen = 0; ok && step(seen, t, g) && step(seen, t ^ 1, other); ++seen) {
        give_back(seen + 1);
        const int all = (g.kind & 3) == SC_BOTH ? g.blocks : g.blocks + other.blocks;
        if (g.blocks > 0) ok = sc_wait<false>(q_full(t), (uint32_t)(segments & 1), abort_flag, SC_ERR_Q);
        // S(i) = Q K(i)^T into S buffer (mine + i) & 1, then O += P V(i - 1): S(i + 1) overwrites P(i - 1), whose product the tensor cores finish first
#pragma unroll 1
        for (int i = 0; i <= g.blocks && g.blocks > 0 && ok; ++i) {
          if (i < g.blocks) {
            const int s = (n0 + place(t, i, other.blocks, g.kind)) % SC_K_STAGES, b = (mine + i) & 1;
            ok = sc_wait<false>(k_full(t, s), (k_turn >> s) & 1u, abort_flag, SC_ERR_KV_FULL);
            if (!ok) break;
            k_turn ^= 1u << s;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t ka = sbase + L::K_OFF + s * L::KV_TILE;
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              ta_umma(s_col + (uint32_t)b * 64u, ta_desc_kmajor(qa + (uint32_t)(k >> 2) * TA_HALF_BYTES + (uint32_t)(k & 3) * 32u),
                      ta_desc_kmajor(ka + (uint32_t)(k >> 2) * L::KV_HALF + (uint32_t)(k & 3) * 32u), idesc_qk, k != 0);
            ta_commit(s_full(t, b));
            ta_commit(k_empty(t, s));
          }
          if (i > 0) {
            const int h = i - 1, s = (n0 + place(t, h, other.blocks, g.kind)) % SC_V_STAGES, b = (mine + h) & 1;
            ok = sc_wait<false>(v_full(t, s), (v_turn >> s) & 1u, abort_flag, SC_ERR_KV_FULL);
            if (ok && h == 0 && segments > 0) ok = sc_wait<false>(o_free(t), (uint32_t)((segments - 1) & 1), abort_flag, SC_ERR_O_FREE);
            ok = ok && sc_wait<false>(p_full(t, b), (uint32_t)(((mine + h) >> 1) & 1), abort_flag, SC_ERR_P_FULL);
            if (!ok) break;
            v_turn ^= 1u << s;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t va = sbase + L::V_OFF + s * L::KV_TILE;
#pragma unroll
            for (int k = 0; k < AS_KEYS / 16; ++k)
              ta_umma_ts(o_col, s_col + (uint32_t)b * 64u + (uint32_t)k * 8u, ta_desc_mnmajor(va + (uint32_t)k * 16u * 128u, L::KV_HALF), idesc_pv, (h | k) != 0);
            ta_commit(pv_done(t, b));
            ta_commit(v_empty(t, s));
          }
        }
        n0 += all;
        mine += g.blocks;
        if (g.blocks > 0) ++segments;
      }
      // Whatever ended this (the line, or a wait that ran out), the CTA's memory is given away behind its last product.
      ta_commit(ta_smem_u32(&products_done[t]));
      ta_mbar_drain(ta_smem_u32(&products_done[t]), 0);
    }
  } else {
    // ---- softmax: thread = query row; warp w reads lanes (w % 4) * 32 .. + 31 of tensor memory ---------------------------------------------
    const int t = (warp - SC_SOFTMAX) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t tlane = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_addr = tmem + tlane + (uint32_t)t * 128u, o_addr = tmem + tlane + 256u + (uint32_t)t * 128u;
    const uint32_t q_rows = sbase + t * L::Q_TILE + (uint32_t)quarter * 32u * 128u;        // this warp's rows
    // Of the part at hand: the step, its blocks, the first one's first key, the first key and the end of those this row sees (of none, if there is
    // no such row), and the least end among the warp's rows.  A request's tile of at most 32 rows is folded: all four warps have all its rows, and
    // each a quarter of a block's keys (the tensor cores work on 128 rows anyway); each leaves a partial result of its own.
    int at_step = -1, blocks = 0, block_key = 0, lo = 0, hi = 0, hi_all = 0, mine = 0;
    bool valid = false, warp_valid = false, folded = false, ok = true;
    float m_ref = -INFINITY, l_run = 0.f;
    bool pending = false;                      // whether the result of the step before has yet to be written
#pragma unroll 1
    for (;;) {
      // ---- the next step.  If this tile's part has blocks, its queries are requested, whole rows side by side.
      ScPart g;
      int from = -1;                           // this row's place among all rows of the queries
      const bool more = step(++at_step, t, g);
      blocks = more ? g.blocks : 0;
      const bool work = blocks > 0;
      if (more && !work && r < g.tokens * G) { // the second half of a single block: an empty partial result
        const long long tile = (long long)(uint32_t)g.row_low | (long long)g.row_high << 32;
        *reinterpret_cast<float2*>(p.part_ml + (tile + g.tokens * G + r) * 2) = make_float2(-INFINITY, 0.f);
      }
      if (work) {
        const int first = (g.kind & 3) == SC_BOTH ? t * per : 0, lane_rows = min(g.tokens - first, per) * G;
        folded = !(g.kind & SC_SHARED) && g.tokens * G <= AS_FOLD_ROWS;
        const int row = folded ? lane : r;     // of this tile's
        valid = row < lane_rows;
        warp_valid = folded || quarter * 32 < lane_rows;
        lo = g.key_lo;
        block_key = (lo & ~(AS_KEYS - 1)) + g.block * AS_KEYS;
        hi = 0x7fffffff;
        if (valid) {
          const int i = row / G;
          const int2 token = as_token(p, g.kind & SC_SHARED, g.first, g.position, first + i);
          from = token.x * p.heads + g.kv_head * G + (row - i * G);
          hi = min(token.y + 1, g.key_hi);
        }
        hi_all = __reduce_min_sync(0xffffffffu, hi);
        constexpr int CHUNKS = D / 8, RPI = 32 / CHUNKS;
        const int c = lane % CHUNKS;
#pragma unroll 4
        for (int i = 0; i < 32 / RPI; ++i) {
          const int rr = i * RPI + lane / CHUNKS, row_at = __shfl_sync(0xffffffffu, from, rr);
          if (row_at >= 0)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                         ::"r"(q_rows + (uint32_t)rr * 128u + (uint32_t)(c >> 3) * TA_HALF_BYTES + (uint32_t)(((c & 7) ^ (rr & 7)) << 4)),
                           "l"((const uint8_t*)p.q + (size_t)row_at * (D * 2) + c * 16) : "memory");
        }
      }
      if (work) {                              // all products with the last part's queries are done: S of this part may come while that one's O is read
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) ta_mbar_arrive(q_full(t));
      }
      // ---- the part of the step before, if it had blocks: its result is written before any later step is looked at
      if (pending) {
        ok = sc_wait<false>(pv_done(t, (mine - 1) & 1), (uint32_t)(((mine - 1) >> 1) & 1), abort_flag, SC_ERR_O_FULL);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const volatile ScPart* was = &steps[(at_step - 1) % SC_SEGMENTS].part[t];
        const int tile_rows = was->tokens * G, kind = was->kind & 3;
        const long long tile = (long long)(uint32_t)was->row_low | (long long)was->row_high << 32;
        const bool fold = !(was->kind & SC_SHARED) && tile_rows <= AS_FOLD_ROWS;
        const int first_row = kind == SC_BOTH ? t * per * G : 0, rows = fold ? 4 * tile_rows : kind == SC_BOTH ? tile_rows : 2 * tile_rows;
        const int in_tile = fold ? lane : r, left = min(tile_rows - first_row, per * G);             // this thread's row of the tile's `left`
        if (fold || quarter * 32 < left) {
          const bool on = in_tile < left;
          const int row = fold ? quarter * tile_rows + lane : (kind == SC_BOTH ? first_row : t * tile_rows) + r;
          if (on) *reinterpret_cast<float2*>(p.part_ml + (tile + row) * 2) = make_float2(m_ref, l_run);
          float4* dst = reinterpret_cast<float4*>(p.part_o + tile * D) + row;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t v[32];
            ta_tmem_ld32(o_addr + (uint32_t)c, v);             // warp-wide: rows without a token take part and write nothing
            if (on) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                dst[(size_t)((c >> 2) + e) * rows] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]), __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
            }
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) ta_mbar_arrive(o_free(t));
      }
      __syncwarp();
      if (lane == 0) give_back(at_step);
      if (!more) break;
      pending = work;
      if (!work) continue;
      // ---- its blocks
      m_ref = -INFINITY;
      l_run = 0.f;
      bool settled = false;                    // every row has a reference
#pragma unroll 1
      for (int i = 0; i < blocks; ++i, block_key += AS_KEYS) {
        const int j = mine + i, b = j & 1;
        ok = sc_wait<false>(s_full(t, b), (uint32_t)((j >> 1) & 1), abort_flag, SC_ERR_S_FULL);
        if (!ok) break;
        if (warp_valid) {                      // (else its rows of P are anything, and nobody reads what comes of them)
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          bool masked = block_key < lo || block_key + AS_KEYS > hi_all;
          unsigned long long seen = sc_low_bits(hi - block_key) & ~sc_low_bits(lo - block_key);        // which of the block's keys the row sees
          if (*holes) {                        // there are pages that are not: a look at this block's
            const volatile ScPart* now = &steps[at_step % SC_SEGMENTS].part[t];
            const int size = min(p.page_size, AS_KEYS), key = block_key + lane * size;
            const bool here = lane * size < AS_KEYS && key < now->key_hi && key + size > lo;
            const int id = here ? p.table[(size_t)now->request * p.max_pages + (key >> p.page_shift)] : 0;
            uint32_t absent = __ballot_sync(0xffffffffu, id < 0 || id >= p.num_pages);
            masked |= absent != 0;
#pragma unroll 1
            for (; absent; absent &= absent - 1) {
              const int first = (__ffs(absent) - 1) * size;
              seen &= ~(sc_low_bits(first + size) & ~sc_low_bits(first));
            }
          }
          uint32_t w[32];
          float sum, f = 1.f;
          bool rescale = false;
          // A row's reference: its maximum so far when that has grown by 2^8.
          auto follow = [&](float mx) {
            const float m_loc = mx * p.scale_log2;
            const bool grow = valid && m_loc > m_ref + TA_RESCALE_STEP;  // also true for the first finite maximum (m_ref = -inf)
            rescale = __any_sync(0xffffffffu, grow);
            if (grow) {
              if (m_ref != -INFINITY) f = exp2f(m_ref - m_loc);
              m_ref = m_loc;
            }
          };
          if (folded) {
            float xs[16];
            {
              uint32_t v[16];
              sc_tmem_ld16(s_addr + (uint32_t)b * 64u + (uint32_t)quarter * 16u, v);
#pragma unroll
              for (int e = 0; e < 16; ++e) xs[e] = __uint_as_float(v[e]);
            }
            if (masked) {
              const uint32_t mask = (uint32_t)(seen >> (quarter * 16));
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (!((mask >> e) & 1u)) xs[e] = -INFINITY;
            }
            float mx = ta_max3(xs[0], xs[1], xs[2]);
#pragma unroll
            for (int e = 3; e < 15; e += 2) mx = ta_max3(mx, xs[e], xs[e + 1]);
            follow(fmaxf(mx, xs[15]));
            const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
            sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {      // the other warps' keys weigh nothing here
              const float p0 = exp2_approx(fmaf(xs[2 * e], p.scale_log2, -m_use)), p1 = exp2_approx(fmaf(xs[2 * e + 1], p.scale_log2, -m_use));
              sum += p0 + p1;
              __nv_bfloat162 b2 = __floats2bfloat162_rn(p0, p1);
              const uint32_t pair = *reinterpret_cast<uint32_t*>(&b2);
#pragma unroll
              for (int q = 0; q < 4; ++q) w[8 * q + e] = q == quarter ? pair : 0u;
            }
          } else {
            // Where every row has a reference, its maximum is not looked for: a sum of 64 weights that stays below 2^15 says that no score is
            // far above the reference.  Otherwise the block is done again from the scores, which still lie in tensor memory, with the maximum.
#pragma unroll 1
            for (bool exact = !settled;; exact = true) {
              float xs[AS_KEYS];
              {
                uint32_t v[AS_KEYS];
                ta_tmem_ld64(s_addr + (uint32_t)b * 64u, v);
#pragma unroll
                for (int e = 0; e < AS_KEYS; ++e) xs[e] = __uint_as_float(v[e]);
              }
              if (masked) {
                const uint32_t low = (uint32_t)seen, high = (uint32_t)(seen >> 32);
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  if (!((low >> e) & 1u)) xs[e] = -INFINITY;
                  if (!((high >> e) & 1u)) xs[32 + e] = -INFINITY;
                }
              }
              if (exact) {
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < AS_KEYS; e += 8) {
#pragma unroll
                  for (int u = 0; u < 4; ++u) mx4[u] = ta_max3(mx4[u], xs[e + 2 * u], xs[e + 2 * u + 1]);
                }
                follow(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])));
                settled = !__any_sync(0xffffffffu, valid && m_ref == -INFINITY);
              }
              const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
              const uint64_t scale2 = ta_pack2(p.scale_log2, p.scale_log2), negm2 = ta_pack2(-m_use, -m_use);
              uint64_t sum2 = ta_pack2(0.f, 0.f);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                float y0, y1;
                ta_unpack2(ta_fma2(ta_pack2(xs[2 * e], xs[2 * e + 1]), scale2, negm2), y0, y1);
                const float p0 = exp2_approx(y0), p1 = exp2_approx(y1);  // 2^-inf = 0 for masked keys
                sum2 = ta_add2(sum2, ta_pack2(p0, p1));
                __nv_bfloat162 b2 = __floats2bfloat162_rn(p0, p1);
                w[e] = *reinterpret_cast<uint32_t*>(&b2);
              }
              float s0, s1;
              ta_unpack2(sum2, s0, s1);
              sum = s0 + s1;
              if (exact || !__any_sync(0xffffffffu, valid && !(sum < 32768.f))) break;
            }
          }
          l_run = l_run * f + sum;
          if (rescale && i > 0) {              // O in the new reference's units, when P V of the block before is complete
            ok = sc_wait<false>(pv_done(t, b ^ 1), (uint32_t)(((j - 1) >> 1) & 1), abort_flag, SC_ERR_O_FULL);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t v[32];
              ta_tmem_ld32(o_addr + (uint32_t)c, v);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
              ta_tmem_st32(o_addr + (uint32_t)c, v);
            }
          }
          ta_tmem_st32(s_addr + (uint32_t)b * 64u, w);
          ta_tmem_wait_st();
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0) ta_mbar_arrive(p_full(t, b));
      }
      if (!ok) break;
      mine += blocks;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) atomicCAS(&g_attention_tc_error, 0, (int)*abort_flag);
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

template <int D>
static cudaError_t sc_launch(const SharedParams& p, int ctas, cudaStream_t stream) {
  constexpr int smem = ScLayout<D>::BYTES + 1024;
  static_assert(smem + sizeof(ScStep) * SC_SEGMENTS + 64 <= 227 * 1024, "shared memory of a CTA");
  static std::atomic<unsigned long long> configured{0ull};     // a bit a device
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (!(configured.load() >> (device & 63) & 1ull)) {
    e = cudaFuncSetAttribute(attention_shared_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    configured.fetch_or(1ull << (device & 63));
  }
  return launch(attention_shared_tc_kernel<D>, dim3(ctas), dim3(SC_THREADS), smem, stream, p);
}

bool attention_shared_tc_takes(int dtype, int group, int head_dim, int page_size) {
  return dtype == LB_BF16 && (head_dim == 64 || head_dim == 128) && group <= TA_ROWS && page_size >= 8 && (page_size & (page_size - 1)) == 0;
}

void attention_shared_tc_cut(int group, int& tile_tokens, int& lane_tokens) {
  lane_tokens = TA_ROWS / group;
  tile_tokens = 2 * lane_tokens;
}

cudaError_t attention_shared_tc(const SharedParams& p, int ctas, cudaStream_t stream) {
  return p.dim == 64 ? sc_launch<64>(p, ctas, stream) : sc_launch<128>(p, ctas, stream);
}

}  // namespace lb

// Reads and clears the flag a bounded wait of this kernel sets when it gives up (0: none).
LB_EXPORT int lb_attention_shared_device_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, lb::g_attention_tc_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(lb::g_attention_tc_error, &zero, sizeof(int));
  return v;
}
