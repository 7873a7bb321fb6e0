// Paged key/value cache: append (with the rotary embedding on the way) and attention of one new token
// per sequence.
//
// Token p of sequence b lives in slot p % page_size of page table[b, p / page_size]; every index that
// comes from device memory (lengths, counts, table entries) is checked against its array before it
// is used, and a token whose place does not exist is left out and reported in g_paged_status.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include <cuda.h>

#include "common.cuh"
#include "ring.h"

namespace moa {
namespace {

constexpr int kStatusAppend = 31, kStatusAttend = 32, kStatusRope = 33, kStatusLength = 34, kStatusWait = 35;
__device__ int32_t g_paged_status[4];

__device__ __noinline__ void report(int code, int64_t b, int64_t at, int more) {
  if (atomicCAS(&g_paged_status[0], 0, code) == 0) {
    g_paged_status[1] = (int32_t)b;
    g_paged_status[2] = (int32_t)min(at, (int64_t)2147483647);
    g_paged_status[3] = more;
  }
}

// What both entry points know about the pool and the tables of the rotary embedding.
struct Pool {
  void *k, *v;
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;   // element strides
  const int32_t* table;
  int64_t table_stride, max_pages;
  int32_t num_pages;
  int shift;                                                // log2(page_size)
  const void *cos, *sin;
  int64_t rope_sb, rope_sn, rope_rows;
  int rope_f32;
};

// Page of position `pos` of a sequence, or -1 where there is none.
__device__ __forceinline__ int32_t page_of(const Pool& p, const int32_t* table_row, int64_t pos) {
  const int64_t i = pos >> p.shift;
  if (pos < 0 || i >= p.max_pages) return -1;
  const int32_t page = table_row[i];
  return (uint32_t)page < (uint32_t)p.num_pages ? page : -1;
}

// Element offset of the table row of token i (at position pos) of sequence b, or -1 where there is none.
__device__ __forceinline__ int64_t rope_row(const Pool& p, int64_t b, int64_t i, int64_t pos) {
  if (p.rope_rows == 0) return b * p.rope_sb + i * p.rope_sn;
  return pos < p.rope_rows ? pos * p.rope_sn : -1;
}

template <typename T>
__device__ __forceinline__ void load_table8(const Pool& p, const void* t, int64_t off, float (&f)[8]) {
  if (p.rope_f32) {
    const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(t) + off);
    const float4 a = s[0], b = s[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    unpack8<T>(*reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(t) + off), f);
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 o;
  o.x = Cvt<T>::pack(f[0], f[1]); o.y = Cvt<T>::pack(f[2], f[3]);
  o.z = Cvt<T>::pack(f[4], f[5]); o.w = Cvt<T>::pack(f[6], f[7]);
  return o;
}

// ---- append ------------------------------------------------------------------------------------
struct AppendParams {
  Pool pool;
  const void *k, *v, *q;
  const int32_t* lengths;
  const int32_t* counts;
  void *q_out, *k_out;
  int64_t k_sb, k_sh, k_sn, v_sb, v_sh, v_sn, q_sb, q_sh, q_sn;
  int H, KV, kv_jobs, jobs;   // jobs of a token: kHeads key/value heads each, then, with q, kHeads query heads each
  int64_t N;
};

// A row of a rope table for the two 8-wide pieces [8c, 8c+8) and [D/2 + 8c, ...) of a row, which the rotation mixes:
//   x'[d] = x[d] cos[d] - x[d + D/2] sin[d],   x'[d + D/2] = x[d + D/2] cos[d + D/2] + x[d] sin[d + D/2]
// in fp32, rounded once to T (that rounding is the cache's storage type).
template <typename T, int D>
struct Turn {
  float cl[8], ch[8], sl[8], sh[8];
  __device__ __forceinline__ void load(const Pool& p, int64_t row, int c) {
    load_table8<T>(p, p.cos, row + c * 8, cl);
    load_table8<T>(p, p.cos, row + D / 2 + c * 8, ch);
    load_table8<T>(p, p.sin, row + c * 8, sl);
    load_table8<T>(p, p.sin, row + D / 2 + c * 8, sh);
  }
  __device__ __forceinline__ void apply(uint4& lo_u, uint4& hi_u) const {
    float lo[8], hi[8], a[8], b[8];
    unpack8<T>(lo_u, lo);
    unpack8<T>(hi_u, hi);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a[j] = fmaf(lo[j], cl[j], -hi[j] * sl[j]);
      b[j] = fmaf(hi[j], ch[j], lo[j] * sh[j]);
    }
    lo_u = pack8<T>(a);
    hi_u = pack8<T>(b);
  }
};

// Bound by memory: every row is read once and written once (1.5 flops a byte).  D/16 threads take kHeads heads of a
// token, of the keys and values or of the queries, and move 16 bytes of either half of each row: with all of a
// thread's loads under way at once (128 bytes) and the token's table row used for all its heads.
constexpr int kAppendThreads = 64, kHeads = 2;

template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int TPR = D / 16;
  const int64_t b = blockIdx.y;
  const uint32_t idx = (blockIdx.x * kAppendThreads + threadIdx.x) / TPR;        // (below 2^31: checked by the host)
  const int c = threadIdx.x % TPR;
  const uint32_t i = idx / p.jobs;
  const int job = (int)(idx - i * p.jobs);
  if (i >= p.N) return;
  const int64_t len = p.lengths[b];
  const int64_t count = len < 0 ? 0 : (p.counts ? min((int64_t)p.counts[b], p.N) : p.N);
  const int64_t pos = len + i;
  const bool counted = i < count;
  int64_t row = 0;
  bool known = counted;                 // the token has a rope row (or needs none)
  if (counted && p.pool.cos) {
    row = rope_row(p.pool, b, i, pos);
    known = row >= 0;
    if (!known && job == 0 && c == 0) report(kStatusRope, b, pos, 0);
  }
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const bool keys = job < p.kv_jobs;
  const int h0 = (keys ? job : job - p.kv_jobs) * kHeads, heads = min((keys ? p.KV : p.H) - h0, kHeads);
  uint4 lo[kHeads], hi[kHeads], vlo[kHeads], vhi[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    lo[h] = hi[h] = vlo[h] = vhi[h] = zero;
    if (!known || h >= heads) continue;
    const T* src = keys ? reinterpret_cast<const T*>(p.k) + b * p.k_sb + (int64_t)(h0 + h) * p.k_sh + i * p.k_sn + c * 8
                        : reinterpret_cast<const T*>(p.q) + b * p.q_sb + (int64_t)(h0 + h) * p.q_sh + i * p.q_sn + c * 8;
    lo[h] = ld_stream16(src);
    hi[h] = ld_stream16(src + D / 2);
    if (keys) {
      src = reinterpret_cast<const T*>(p.v) + b * p.v_sb + (int64_t)(h0 + h) * p.v_sh + i * p.v_sn + c * 8;
      vlo[h] = ld_stream16(src);
      vhi[h] = ld_stream16(src + D / 2);
    }
  }
  int32_t page = -1;
  if (known && keys) {
    page = page_of(p.pool, p.pool.table + b * p.pool.table_stride, pos);
    if (page < 0 && job == 0 && c == 0) report(kStatusAppend, b, pos, 0);
  }
  if (known && p.pool.cos) {
    Turn<T, D> turn;
    turn.load(p.pool, row, c);
#pragma unroll
    for (int h = 0; h < kHeads; ++h) turn.apply(lo[h], hi[h]);
  }
  const int64_t slot = pos & ((1ll << p.pool.shift) - 1);
  T* copy = reinterpret_cast<T*>(keys ? p.k_out : p.q_out);
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (h >= heads) break;
    if (page >= 0) {
      T* kd = reinterpret_cast<T*>(p.pool.k) + page * p.pool.k_page + (int64_t)(h0 + h) * p.pool.k_head + slot * p.pool.k_slot + c * 8;
      T* vd = reinterpret_cast<T*>(p.pool.v) + page * p.pool.v_page + (int64_t)(h0 + h) * p.pool.v_head + slot * p.pool.v_slot + c * 8;
      // evicted first: nothing reads the pages again before the other layers' turn (8x1500 ragged tokens: 18.1 -> 16.4 us)
      __stcs(reinterpret_cast<uint4*>(kd), lo[h]);
      __stcs(reinterpret_cast<uint4*>(kd + D / 2), hi[h]);
      __stcs(reinterpret_cast<uint4*>(vd), vlo[h]);
      __stcs(reinterpret_cast<uint4*>(vd + D / 2), vhi[h]);
    }
    if (copy) {
      T* dst = copy + ((b * (keys ? p.KV : p.H) + h0 + h) * p.N + i) * D + c * 8;
      *reinterpret_cast<uint4*>(dst) = lo[h];
      *reinterpret_cast<uint4*>(dst + D / 2) = hi[h];
    }
  }
}

// lengths[b] += min(counts[b], N), after the append (its own launch: every block of the append reads them).
__global__ void paged_advance_kernel(int32_t* lengths, const int32_t* counts, int64_t N, int B) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= B || lengths[b] < 0) return;
  const int64_t n = counts ? min((int64_t)max(counts[b], 0), N) : N;
  lengths[b] = (int32_t)min((int64_t)lengths[b] + n, (int64_t)2147483647);
}

// ---- attention of one token ----------------------------------------------------------------------
//
//   o = sum_p w_p v_p / sum_p w_p,   w_p = exp(scale q.k_p - max),   p over the head's span
//
// Every key and value row is read once and used for all query heads that share it, G flops a byte: the kernel
// is bound by memory, and is built to keep loads in flight.
//
// Work.  An item is (sequence, key head, tile of up to 8*MT query heads).  Its positions are counted in units of 16;
// all items' units, and kItemCost more per item for its epilogue, are laid out on one line that is cut into
// equal parts, one per block (two blocks of four warps per SM).  A block therefore moves the same number of bytes however
// ragged the lengths are, and the cut is computed on the device from `lengths` alone: nothing is planned on the
// host, and a captured launch stays right when the lengths change.  Items of up to kWholeUnits units are not
// cut (joining would cost more: 122 sequences of 30 tokens 10.8 -> 7.8 us); one that is cut leaves one partial
// result (maximum, sum, sum of values) per block; the block that finishes last joins them, in the blocks'
// order, so results do not depend on timing.  No block waits for another.  When there are more items than blocks
// and the page table allows short ones only, the line is cut into a part per warp, of whole items: nothing is
// shared between warps then and an item costs no barriers (3840 items of up to 34 tokens: 53 us by blocks, 20 by warps).
//
// Loads.  The warps of a block take the units of a segment in turn.  Each warp runs its own ring of kStages
// units in shared memory, filled by a cursor that runs ahead of the arithmetic, over the ends of items too, so the
// epilogue of one item overlaps with the loads of the next.  128 KB are in flight per SM: less leaves bandwidth
// unused, more only makes every load, look-up and join wait longer in the memory's queues (192 KB: 3 % slower).
// A unit that is attended in full comes with TMA (one lane's few instructions), one that is not with cp.async,
// which leaves masked rows zero: what a page holds behind its last token may be anything.  What else an item
// needs (queries, the new token's rows) is fetched while the item before it is worked on.
//
// Arithmetic.  m16n8k16 tensor instructions with the 8 query heads of a tile in rows 0-7 and, where an operand
// does not fit 16 bits, its remainder in rows 8-15: the weights w are held in two 16-bit parts that way (hi + lo),
// and so is the rotated query of the fused step.  Rows 8-15 would idle otherwise (G is small), so the second part costs
// nothing.  A weight is off by 2^-22 of itself in fp16 and by 2^-17 in bf16, whose third part would cost products of its
// own (64 sequences of up to 8192 tokens 174 -> 180 us) and change little: the result is as far from 64 bits with it (1.5e-6
// against 1.6e-6, of sums in the tensor cores).  fp16 has those bits from 2^-14 on only, so its weights are 2^15 times what
// they are, sums and records with them, and the factor falls out at the division: steps of 2^-39 of the largest.
// With 9..16 heads (MT = 2) all rows are heads, and the lower parts are products of their own into the same sums.
//
// An infinite value with a weight is infinite in the result, and a token with a score of -infinity has none.  So a weight's
// upper part is never 0 (fp16: 2^-39 of the largest at least), and what a lower part makes of an infinity (0 * inf, or the
// other sign) must not get into the sum: with MT = 1 it is in a row of its own.  With MT = 2 the lower part has the sign of
// the upper one, which is cut off and not rounded, and is not 0: that costs rotated queries in bf16 a bit (2^-16).  Only the
// weights in bf16 stay rounded, and their lower part meets the largest finite number in place of an infinity.  (38 sequences
// of up to 35129 tokens, 64 heads of 64 on 4: bf16 162 -> 165 us, with a third part instead 184; fp16 166 -> 167, with finite
// numbers instead 172; finite numbers for keys too: 10 % more in the step.)
//
// The fused step's new token is where one warp of the block that ends the item starts from (its score is the first
// maximum, its value the first sum); it is stored into its page at the same time and read from no page.
constexpr int kPerSm = 2;                   // resident blocks per SM
constexpr int kUnit = 16;                   // positions of a unit (k of the second product)
constexpr int kItemCost = 16, kSoloCost = 2;      // an item's epilogue, in units
constexpr int kSoloTokens = 256;            // longest sequence for warps on their own
constexpr int kMinUnits = 8;                // least share of a block: fewer blocks work when there is less
constexpr int kWholeUnits = 16;             // items up to this are not cut: the part that they begin in does them
constexpr int kJoin = 18;                   // partial results joined at once
constexpr int kMaxParts = kJoin * kJoin;    // two levels of joining
constexpr int kCounters = 3;                // per part
constexpr int kRecHeads = 16;
constexpr int kCached = 256;                // lengths and spans held in shared memory; the others are read where they are
constexpr uint32_t kByHand = 0x80000000u;   // in a stage's mask: filled with cp.async
constexpr int64_t kRecFloats = kRecHeads * (128 + 2);

struct DecodeParams {
  Pool pool;
  const void *q, *k_new, *v_new;
  void* out;
  int32_t* lengths;
  const int64_t *sink, *local;
  int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh, o_sb, o_sh;
  int B, H, KV, G, tiles;                   // tiles of query heads per key head
  int capacity;                             // positions that a row of the page table reaches
  float scale_log2;
  int out_f32, advance, tma;
  int* counters;                            // kCounters per part, zero between launches, and one behind them
  float* records;                           // 2 per part
};

// Weights are exp2(score - m) with m the running maximum less 15 in fp16, so that the largest is 2^15.  m is rounded
// before it is used, and the same m is in the records, so that this adds no error; it is rounded up, so that no weight
// is more than 2^15 however large the scores are.
template <typename T>
__device__ __forceinline__ float lifted(float top) {
  return std::is_same<T, __half>::value ? __fsub_ru(top, 15.f) : top;
}

// A flag that the compiler takes to change: loops are not made in two versions for it (the kernel has to be
// fetched through the caches that the keys run through, its size counts).
__device__ __forceinline__ bool opaque(bool flag) {
  int x = flag;
  asm volatile("" : "+r"(x));
  return x != 0;
}

// The lengths and spans as a block sees them.
struct Sizes {
  const DecodeParams& p;
  const int* len;                           // shared memory, kCached each
  const int2* span;
  __device__ __forceinline__ int length(int b) const { return b < kCached ? len[b] : p.lengths[b]; }
  // Tokens of sequence b, the new one included, as far as the page table reaches.
  __device__ __forceinline__ int tokens(int b) const {
    const int n = length(b);
    return n < 0 ? 0 : min(n + (p.k_new && n < p.capacity ? 1 : 0), p.capacity);
  }
  // Whether the new token of sequence b is one of them.
  __device__ __forceinline__ bool fresh(int b) const {
    const int n = length(b);
    return p.k_new && n >= 0 && n < p.capacity;
  }
  static __device__ __forceinline__ int2 clamped(int64_t sink, int64_t local) {
    const int64_t most = 2147483647;
    return make_int2((int)min(max(sink, (int64_t)0), most), (int)min(max(local, (int64_t)0), most));
  }
  __device__ __forceinline__ int2 sink_local(int kh) const {
    return kh < kCached ? span[kh] : clamped(p.sink[kh], p.local[kh]);
  }
};

// The units of one (sequence, key head): 16 positions each, aligned, so that with pages of 16 and more a unit
// lies in one page.  Units 0 .. head-1 hold the first `sink` positions, the others begin at unit `tail` and hold the
// positions from `from` on; positions < n outside both are masked.
struct Span {
  int n, sink, from, head, tail, units;
  __device__ __forceinline__ Span() {}
  __device__ __forceinline__ Span(const Sizes& s, int tokens, int kh) {
    n = sink = from = tokens;
    if (opaque(s.p.sink != nullptr)) {
      const int2 sl = s.sink_local(kh);
      sink = min(sl.x, n);
      from = n - min(sl.y, n);
    }
    const int end = (n + 15) >> 4;
    head = (sink + 15) >> 4;
    tail = from == n ? end : max(head, from >> 4);
    units = head + end - tail;
  }
  __device__ __forceinline__ int unit(int u) const { return u < head ? u : u - head + tail; }
  // Which of the 16 positions of aligned unit `x` are attended.
  __device__ __forceinline__ uint32_t mask(int x) const {
    const int p0 = x * 16;
    return below(n - p0) & (below(sink - p0) | ~below(from - p0));
  }
  static __device__ __forceinline__ uint32_t below(int m) { return m >= 16 ? 0xffffu : m <= 0 ? 0u : (1u << m) - 1u; }
  __device__ __forceinline__ bool sees_last() const { return n > 0 && (sink == n || from < n); }
};

// a / b for b > 0 and 0 <= a: 64-bit division takes some hundred instructions, and nearly always 32 bits do.
__device__ __forceinline__ int64_t divided(int64_t a, int b) {
  return a >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// The line in equal parts, one per team (a block, or a warp on its own); the first `rest` of them are one longer.
struct Cut {
  int64_t each;                             // units of the other parts
  int parts, rest;
  __device__ __forceinline__ Cut(int64_t total, int most, int least) {
    parts = (int)min(max(total / least, (int64_t)1), (int64_t)most);
    each = divided(total, parts);
    rest = (int)(total - each * parts);
  }
  __device__ __forceinline__ int64_t begin(int c) const { return each * c + min(c, rest); }
  // The part in which x is (each >= 1: a part is never empty).
  __device__ __forceinline__ int part_of(int64_t x) const {
    const int64_t longer = (each + 1) * rest;
    return x < longer ? (int)(x / (each + 1)) : rest + (int)((x - longer) / each);
  }
};

// A walk over the items of a part [lo, hi) of the line: of those that begin in it when warps are on their own (`solo`),
// of all that reach into it else.
struct Part {
  int64_t lo, hi;
};
template <bool SOLO>
struct Cursor {
  static constexpr int kCost = SOLO ? kSoloCost : kItemCost;
  int b, kh, tile;
  int n;                                    // tokens of sequence b
  Span span;
  int64_t at;                               // where the item begins on the line
  int u0, u1;                               // the units of the item that are in the part
  __device__ __forceinline__ void enter(const Sizes& s, const Part& part) {
    span = Span(s, n, kh);
    u0 = 0;
    u1 = span.units;
    if (!SOLO) {
      if (span.units <= kWholeUnits) {
        u0 = at >= part.lo ? 0 : u1;
      } else {
        u0 = (int)min(max(part.lo - at, (int64_t)0), (int64_t)u1);
        u1 = (int)min(part.hi - at, (int64_t)u1);
      }
    }
  }
  // To the next item; false when it is not in the part.
  __device__ __forceinline__ bool next(const Sizes& s, const Part& part) {
    at += span.units + kCost;
    if (at >= part.hi) return false;
    if (++tile == s.p.tiles) {
      tile = 0;
      if (++kh == s.p.KV) {
        kh = 0;
        ++b;
        n = s.tokens(b);
      }
    }
    enter(s, part);
    return true;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// orders this thread's ordinary writes to shared memory before later TMA writes to the same place
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void bar_init(uint32_t bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
constexpr long long kWaitCycles = 2000000000ll;       // about a second
// Bounded: a load that never arrives is reported, the warp stops waiting and the kernel goes on to its end.
__device__ __noinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity) {
  const long long start = clock64();
  while (!bar_try(bar, parity))
    if (clock64() - start > kWaitCycles) {
      report(kStatusWait, blockIdx.x, threadIdx.x, 0);
      return false;
    }
  return true;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  return bar_try(bar, parity) || bar_wait_slow(bar, parity);
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int d, int slot, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(d), "r"(slot), "r"(head), "r"(page) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo with both in T, for two values; hi of an fp16 that does not fit is its largest, lo takes the rest.
// (A weight fits: it is 2^15 at most.)
template <typename T, bool LARGE>
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  if (LARGE && std::is_same<T, __half>::value) {
    hi = Cvt<T>::pack(fminf(fmaxf(x0, -65504.f), 65504.f), fminf(fmaxf(x1, -65504.f), 65504.f));
  } else {
    hi = Cvt<T>::pack(x0, x1);
  }
  const float2 h = Cvt<T>::unpack(hi);
  lo = Cvt<T>::pack(x0 - h.x, x1 - h.y);
}
// The same with hi cut off, so that lo has its sign, and lo not 0 (unless x is): hi is one step less where x fits it.
template <typename T>
__device__ __forceinline__ void split_one_sign(float x, uint16_t& hi, uint16_t& lo) {
  if constexpr (std::is_same<T, __half>::value) {
    hi = __half_as_ushort(__float2half_rz(x));
    lo = __half_as_ushort(__float2half_rn(x - __half2float(__ushort_as_half(hi))));
    if ((lo & 0x7fff) == 0 && (hi & 0x7fff) > 1) lo = __half_as_ushort(__float2half_rn(x - __half2float(__ushort_as_half(--hi))));
  } else {
    hi = (uint16_t)(__float_as_uint(x) >> 16);
    lo = __bfloat16_as_ushort(__float2bfloat16_rn(x - __uint_as_float((uint32_t)hi << 16)));
    if ((lo & 0x7fff) == 0 && (hi & 0x7fff) > 1) lo = __bfloat16_as_ushort(__float2bfloat16_rn(x - __uint_as_float((uint32_t)--hi << 16)));
  }
}
template <typename T>
__device__ __forceinline__ void split_one_sign2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  uint16_t h0, l0, h1, l1;
  split_one_sign<T>(x0, h0, l0);
  split_one_sign<T>(x1, h1, l1);
  hi = h0 | (uint32_t)h1 << 16;
  lo = l0 | (uint32_t)l1 << 16;
}
// Two weights as hi + lo for sums that hold both.  fp16: positive, and only of 0 itself 0 (from 2^-24 on a weight is one
// step at least); bf16 is rounded, its lo to be multiplied with finite2(value).
template <typename T>
__device__ __forceinline__ void split_weights2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same<T, __half>::value) {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(x1), "f"(x0));
    const float2 h = Cvt<T>::unpack(hi);
    lo = Cvt<T>::pack(fmaxf(x0 - h.x, fminf(x0, 0x1p-24f)), fmaxf(x1 - h.y, fminf(x1, 0x1p-24f)));
  } else {
    split2<T, false>(x0, x1, hi, lo);
  }
}
// Two bf16 whose infinities have given way to the largest number.
__device__ __forceinline__ uint32_t finite2(uint32_t v) {
  asm("min.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(0x7f7f7f7fu));
  return v;
}
// hi + lo of a sum that was split; an infinity of hi is the result (its lo is inf - inf or 0 * inf).
__device__ __forceinline__ float joined(float hi, float lo) { return isinf(hi) ? hi : hi + lo; }

// A unit's keys (and values) are D/64 panels of 16 rows of 128 bytes, 16-byte chunk c of row r at c ^ (r % 8): TMA's
// 128-byte swizzle, which ldmatrix reads without bank conflicts.
template <int D, int MT, bool SOLO>
struct Layout {
  static constexpr int kWarps = 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kPanelBytes = kUnit * 128, kTileBytes = kUnit * D * 2, kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = D == 64 ? 4 : 2;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kJoinBytes = kWarps * 8 * D * 4;                // a head's row: value d at d ^ 4 * head
  // what an item needs: queries (rows padded by 16 bytes), the new token's key, value, cos and sin, its page
  static constexpr int kQPitch = D * 2 + 16, kKey = 8 * MT * kQPitch, kValue = kKey + D * 2, kCos = kValue + D * 2,
                       kSin = kCos + D * 4, kPage = kSin + D * 4, kItemBytes = kPage + 16;
  static constexpr int kLowBytes = 8 * MT * kQPitch;                   // what rotated queries have beyond 16 bits
  static constexpr int kTeamBytes = 2 * kItemBytes + kLowBytes;
  // shared memory: the ring, its barriers and masks, maxima and sums of the warps, the scan, lengths and spans, the
  // teams' (and behind a block's the join buffer)
  static constexpr int kBar = kRing, kMask = kBar + kWarps * kStages * 8, kMax = kMask + kWarps * kStages * 4,
                       kScan = kMax + 2 * kWarps * 8 * 4, kLen = kScan + 128 + (SOLO ? kThreads * 8 : 0),
                       kTeams = kLen + kCached * 12;
  static constexpr int kBytes = 1024 + kTeams + (SOLO ? kWarps * kTeamBytes : kTeamBytes + kJoinBytes);
  static_assert(kPanelBytes * (D / 64) == kTileBytes, "panels");
  static constexpr bool kFits = kPerSm * (kBytes + 1024) <= 233472;
  static_assert((SOLO || kFits) && kTeams % 16 == 0, "shared memory");
  static __device__ __forceinline__ uint32_t at(int row, int chunk) {
    return (chunk >> 3) * kPanelBytes + row * 128 + (((chunk ^ row) & 7) << 4);
  }
};

// A block, or a warp on its own.
template <bool SOLO, int WARPS>
struct Team {
  static constexpr int warps = SOLO ? 1 : WARPS, size = warps * 32;
  int rank, warp;                                  // thread of the team, warp of the team
  __device__ __forceinline__ Team() : rank(SOLO ? threadIdx.x & 31 : threadIdx.x), warp(SOLO ? 0 : threadIdx.x >> 5) {}
  __device__ __forceinline__ void sync() const {
    if (SOLO) __syncwarp();
    else __syncthreads();
  }
};

// What follows up to the kernel runs once or twice per item and stays out of the loop's registers.

// Four coordinates of head h's result: sum of values over sum of weights (zeros where there is no weight).
template <typename T>
__device__ __forceinline__ void store_out4(const DecodeParams& p, int b, int h, int d, float4 O, float sum) {
  const int64_t off = (int64_t)b * p.o_sb + (int64_t)h * p.o_sh + d;
  if (sum == 0.f) O = make_float4(0.f, 0.f, 0.f, 0.f);
  else O = make_float4(O.x / sum, O.y / sum, O.z / sum, O.w / sum);
  if (p.out_f32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + off) = O;
  else *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + off) = make_uint2(Cvt<T>::pack(O.x, O.y), Cvt<T>::pack(O.z, O.w));
}

// Fetches what an item needs into its buffer, with cp.async; called by the whole team.
template <typename T, int D, int MT, typename TEAM, typename CURSOR>
__device__ __forceinline__ void fetch_item(const DecodeParams& p, const TEAM& team, const CURSOR& c, bool fresh, uint32_t buf) {
  using L = Layout<D, MT, false>;            // (the same for both)
  constexpr int CPR = D / 8;                       // 16-byte chunks per row
  const int h0 = c.kh * p.G + c.tile * 8 * MT, heads = min(p.G - c.tile * 8 * MT, 8 * MT);
#pragma unroll
  for (int i = team.rank; i < 8 * MT * CPR; i += team.size) {
    const int row = i / CPR, chunk = i % CPR;
    const T* src = reinterpret_cast<const T*>(p.q) + (int64_t)c.b * p.q_sb + (int64_t)(h0 + min(row, heads - 1)) * p.q_sh;
    cp_async16(buf + row * L::kQPitch + chunk * 16, src + chunk * 8, row < heads);
  }
  if (fresh) {
    const int64_t pos = c.n - 1;
    if (team.rank < 2 * CPR) {
      const int chunk = team.rank % CPR;
      const T* src = team.rank < CPR ? reinterpret_cast<const T*>(p.k_new) + c.b * p.k_sb + c.kh * p.k_sh
                                     : reinterpret_cast<const T*>(p.v_new) + c.b * p.v_sb + c.kh * p.v_sh;
      cp_async16(buf + (team.rank < CPR ? L::kKey : L::kValue) + chunk * 16, src + chunk * 8, true);
    }
    const int64_t row = p.pool.cos ? rope_row(p.pool, c.b, 0, pos) : -1;
    const int cells = p.pool.rope_f32 ? 4 : 2, chunks = D * cells / 16;      // bytes of a table's value
    if (row >= 0) {
#pragma unroll 1
      for (int i = team.size - 1 - team.rank; i < 2 * chunks; i += team.size) {
        const int chunk = i % chunks;
        const char* src = reinterpret_cast<const char*>(i < chunks ? p.pool.cos : p.pool.sin) + row * cells;
        cp_async16(buf + (i < chunks ? L::kCos : L::kSin) + chunk * 16, src + chunk * 16, true);
      }
    }
    if (team.rank == 0) cp_async4(buf + L::kPage, p.pool.table + (int64_t)c.b * p.pool.table_stride + (pos >> p.pool.shift));
  }
  cp_async_commit();
}

// Two neighbouring values of a table row in shared memory.
template <typename T>
__device__ __forceinline__ float2 table2(const unsigned char* row, int d, bool f32) {
  if (f32) return *reinterpret_cast<const float2*>(row + d * 4);
  return Cvt<T>::unpack(*reinterpret_cast<const uint32_t*>(row + d * 2));
}

// The item's queries are rotated in their buffer, by the whole team: what fits T stays there, the rest goes to `low`.
template <typename T, int D, int MT, typename TEAM>
__device__ __forceinline__ void turn_queries(const DecodeParams& p, const TEAM& team, unsigned char* item, unsigned char* low,
                                             int heads) {
  using L = Layout<D, MT, false>;            // (the same for both)
  const bool f32 = p.pool.rope_f32;
#pragma unroll 1
  for (int i = team.rank; i < heads * (D / 4); i += team.size) {
    const int head = i / (D / 4), d = i % (D / 4) * 2;       // a pair of coordinates of either half
    uint32_t* q = reinterpret_cast<uint32_t*>(item + head * L::kQPitch);
    uint32_t* r = reinterpret_cast<uint32_t*>(low + head * L::kQPitch);
    const float2 a = Cvt<T>::unpack(q[d / 2]), b = Cvt<T>::unpack(q[(d + D / 2) / 2]);
    const float2 cl = table2<T>(item + L::kCos, d, f32), ch = table2<T>(item + L::kCos, d + D / 2, f32);
    const float2 sl = table2<T>(item + L::kSin, d, f32), sh = table2<T>(item + L::kSin, d + D / 2, f32);
    const float2 lo = make_float2(fmaf(a.x, cl.x, -b.x * sl.x), fmaf(a.y, cl.y, -b.y * sl.y));
    const float2 hi = make_float2(fmaf(b.x, ch.x, a.x * sh.x), fmaf(b.y, ch.y, a.y * sh.y));
    if (MT == 1) {
      split2<T, true>(lo.x, lo.y, q[d / 2], r[d / 2]);
      split2<T, true>(hi.x, hi.y, q[(d + D / 2) / 2], r[(d + D / 2) / 2]);
    } else {
      split_one_sign2<T>(lo.x, lo.y, q[d / 2], r[d / 2]);
      split_one_sign2<T>(hi.x, hi.y, q[(d + D / 2) / 2], r[(d + D / 2) / 2]);
    }
  }
}

// The new token's key is rotated in its buffer (a warp's work).
template <typename T, int D, int MT>
__device__ __forceinline__ void turn_key(const DecodeParams& p, unsigned char* item) {
  using L = Layout<D, MT, false>;            // (the same for both)
  const int d = (threadIdx.x & 31) * 2;            // a pair of coordinates of either half
  const bool f32 = p.pool.rope_f32;
  if (d < D / 2) {
    uint32_t* lo = reinterpret_cast<uint32_t*>(item + L::kKey + d * 2);
    uint32_t* hi = reinterpret_cast<uint32_t*>(item + L::kKey + (d + D / 2) * 2);
    const float2 a = Cvt<T>::unpack(*lo), b = Cvt<T>::unpack(*hi);
    const float2 cl = table2<T>(item + L::kCos, d, f32), ch = table2<T>(item + L::kCos, d + D / 2, f32);
    const float2 sl = table2<T>(item + L::kSin, d, f32), sh = table2<T>(item + L::kSin, d + D / 2, f32);
    *lo = Cvt<T>::pack(fmaf(a.x, cl.x, -b.x * sl.x), fmaf(a.y, cl.y, -b.y * sl.y));
    *hi = Cvt<T>::pack(fmaf(b.x, ch.x, a.x * sh.x), fmaf(b.y, ch.y, a.y * sh.y));
  }
}

// The new token's rows go into their page (a warp's work).
template <typename T, int D, int MT>
__device__ __forceinline__ void store_new(const DecodeParams& p, const unsigned char* item, int kh, int slot, int page) {
  using L = Layout<D, MT, false>;            // (the same for both)
  const int lane = threadIdx.x & 31, chunk = lane % (D / 8);
  if (lane >= 2 * (D / 8)) return;
  if (lane < D / 8) {
    T* to = reinterpret_cast<T*>(p.pool.k) + page * p.pool.k_page + kh * p.pool.k_head + slot * p.pool.k_slot;
    *reinterpret_cast<uint4*>(to + chunk * 8) = *reinterpret_cast<const uint4*>(item + L::kKey + chunk * 16);
  } else {
    T* to = reinterpret_cast<T*>(p.pool.v) + page * p.pool.v_page + kh * p.pool.v_head + slot * p.pool.v_slot;
    *reinterpret_cast<uint4*>(to + chunk * 8) = *reinterpret_cast<const uint4*>(item + L::kValue + chunk * 16);
  }
}

// The rows of aligned unit x one by one, with cp.async, and zeros where nothing is attended.  `page`: of the unit, or of
// position lane % 16 when pages are smaller.  Returns `present` without the rows that have no page.  Called by a
// whole warp.
template <typename T, int D, int MT>
__device__ __noinline__ uint32_t load_rows(const DecodeParams& p, int b, int kh, int x, int32_t page, uint32_t present,
                                           uint32_t dst) {
  using L = Layout<D, MT, false>;            // (the same for both)
  constexpr int LPR = D / 8, RPI = 32 / LPR;       // lanes per row, rows per load instruction
  const int lane = threadIdx.x & 31;
  const int pos = x * 16 + (lane & 15);
  bool take = (present >> (lane & 15)) & 1;
  if (take && (uint32_t)page >= (uint32_t)p.pool.num_pages) {
    if (lane < 16) report(kStatusAttend, b, pos, kh);
    take = false;
  }
  const T* ks = reinterpret_cast<const T*>(p.pool.k);
  const T* vs = reinterpret_cast<const T*>(p.pool.v);
  if (take) {
    const int64_t slot = pos & ((1ll << p.pool.shift) - 1);
    ks += page * p.pool.k_page + kh * p.pool.k_head + slot * p.pool.k_slot;
    vs += page * p.pool.v_page + kh * p.pool.v_head + slot * p.pool.v_slot;
  }
  present = __ballot_sync(0xffffffffu, take) & 0xffffu;
#pragma unroll 1
  for (int i = 0; i < kUnit / RPI; ++i) {
    const int row = i * RPI + lane / LPR, chunk = lane % LPR;
    const T* k_row = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(ks), row));
    const T* v_row = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(vs), row));
    cp_async16(dst + L::at(row, chunk), k_row + chunk * 8, (present >> row) & 1);
    cp_async16(dst + L::kTileBytes + L::at(row, chunk), v_row + chunk * 8, (present >> row) & 1);
  }
  __syncwarp();
  return present;
}

// Joins the records that parts c0 .. c1 of the line left of one item (`heads` query heads from h0 of sequence b);
// called by every block that left one.  kJoin neighbours are joined by the last of them, their results by the last
// of those that joined, and so on; no block waits.
template <typename T, int D, int MT>
__device__ __noinline__ void join_parts(const DecodeParams& p, int c0, int c1, int b, int h0, int heads, float* scratch,
                                        int* flag) {
  constexpr int kThreads = Layout<D, MT, false>::kThreads;
  const int tid = threadIdx.x;
  float* weight = scratch;                         // (record, head); then by head
  float* top = scratch + kJoin * kRecHeads;
  float* total = top + kRecHeads;
  // at each level groups of kJoin neighbours; `step` parts lie behind one of them
  int index = (int)blockIdx.x - c0, there = c1 - c0 + 1, step = 1;
  for (int level = 0;; ++level) {
    const int group = index / kJoin, first = group * kJoin * step, count = min(there - group * kJoin, kJoin);
    // counters of a part: of the item that begins in it 0 and 1 by level, of the one that began before 2
    int* counter = p.counters + kCounters * (c0 + first) + (group == 0 ? level : 2);
    const bool final = there <= kJoin;
    // One thread's acquire and release stand for the block's: the barriers around it order the others' records, which
    // are read past L1.
    __syncthreads();
    if (tid == 0) {
      int before;
      asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
      *flag = before == count - 1;
      if (before == count - 1) *counter = 0;
    }
    __syncthreads();
    if (!*flag) return;
    // record i of the group; a part's second record is of the item that begins in it
    float* const records = p.records + (int64_t)(2 * (c0 + first)) * kRecFloats;
    const uint32_t stride = 2 * step * (uint32_t)kRecFloats, shift0 = first == 0 ? (uint32_t)kRecFloats : 0;
    // four coordinates of kAtOnce records at a time (more would take registers from the kernel's loop); the first ones
    // are asked for before the weights are known
    constexpr int kAtOnce = kJoin / 2;
    float4 x[kAtOnce];
    auto load = [&](int e, int i0) {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
        if (i0 + i < count)
          x[i] = __ldcg(reinterpret_cast<const float4*>(records + (i0 + i == 0 ? shift0 : (i0 + i) * stride) + e));
    };
    if (tid * 4 < heads * D) load(tid * 4, 0);
    if (tid < kRecHeads * 8 && tid / 8 < heads) {  // eight threads a head: its maximum, and every record's weight
      const int head = tid / 8;
      float2 ml[(kJoin + 7) / 8];
      float M = -INFINITY;
#pragma unroll
      for (int k = 0; k < (kJoin + 7) / 8; ++k) {
        const int i = tid % 8 + k * 8;
        ml[k] = make_float2(-INFINITY, 0.f);
        if (i < count)
          ml[k] = __ldcg(reinterpret_cast<const float2*>(records + (i == 0 ? shift0 : i * stride) + kRecHeads * 128 + head * 2));
      }
#pragma unroll
      for (int k = 0; k < (kJoin + 7) / 8; ++k) M = fmaxf(M, ml[k].x);
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffu << (tid & 24), M, off));
      const float base = M == -INFINITY ? 0.f : M;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < (kJoin + 7) / 8; ++k) {
        const int i = tid % 8 + k * 8;
        if (i >= count) break;
        const float f = exp2f(ml[k].x - base);
        weight[i * kRecHeads + head] = f;
        sum += f * ml[k].y;
      }
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) sum += __shfl_xor_sync(0xffu << (tid & 24), sum, off);
      if (tid % 8 == 0) {
        top[head] = M;
        total[head] = sum;
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int e = tid * 4; e < heads * D; e += kThreads * 4) {
      const int head = e / D;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int i0 = 0; i0 < count; i0 += kAtOnce) {
        if (e >= kThreads * 4 || i0 > 0) load(e, i0);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
          if (i0 + i < count) {
            const float f = weight[(i0 + i) * kRecHeads + head];
            O.x += f * x[i].x; O.y += f * x[i].y; O.z += f * x[i].z; O.w += f * x[i].w;
          }
      }
      if (final) {
        store_out4<T>(p, b, h0 + head, e % D, O, total[head]);
      } else {
        // (each element of the group's first record is read by the thread that writes it, maxima and sums above)
        float* to = records + shift0;
        *reinterpret_cast<float4*>(to + e) = O;
        if (e % D == 0) *reinterpret_cast<float2*>(to + kRecHeads * 128 + head * 2) = make_float2(top[head], total[head]);
      }
    }
    if (final) return;
    index = group;
    there = (there + kJoin - 1) / kJoin;
    step *= kJoin;
  }
}

// SOLO: a team is a warp, and items are not cut.
template <typename T, int D, int MT, bool SOLO>
__global__ void __launch_bounds__(Layout<D, MT, SOLO>::kThreads, kPerSm)
    paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const __grid_constant__ DecodeParams p) {
  using L = Layout<D, MT, SOLO>;
  constexpr int kStages = L::kStages, kWarps = L::kWarps, kThreads = L::kThreads, kCost = Cursor<SOLO>::kCost;
  constexpr int KS = D / 16;                       // k steps of the first product, pairs of n tiles of the second
  extern __shared__ unsigned char smem_raw[];      // the swizzle goes by the address: panels start at multiples of 1024
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* sm_m = reinterpret_cast<float*>(smem + L::kMax);
  float* sm_l = sm_m + kWarps * 8;
  int64_t* sm_sum = reinterpret_cast<int64_t*>(smem + L::kScan);      // by warp; then where the block's part begins
  int64_t* sm_before = sm_sum + 16;                // (SOLO) by thread
  int* sm_flag = reinterpret_cast<int*>(sm_sum + 12);
  int* sm_len = reinterpret_cast<int*>(smem + L::kLen);
  int2* sm_span = reinterpret_cast<int2*>(sm_len + kCached);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Sizes sizes = {p, sm_len, sm_span};
  const Team<SOLO, kWarps> team;
  unsigned char* sm_item = smem + L::kTeams + (SOLO ? warp * L::kTeamBytes : 0);
  unsigned char* sm_low = sm_item + 2 * L::kItemBytes;
  float* sm_o = reinterpret_cast<float*>(smem + L::kTeams + L::kTeamBytes);

  if (tid == 0 && p.tma) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
  }
  const uint32_t bars = (uint32_t)__cvta_generic_to_shared(smem + L::kBar) + warp * kStages * 8;
  if (lane < kStages) {
    bar_init(bars + lane * 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // So far nothing was read that a kernel before this one may have written: a launch may begin while the one before
  // it ends (1.8 us less from launch to launch), and waits here until all of that one's writes are there.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // ---- the line: its length, and where this team's part begins
#pragma unroll 1
  for (int b = tid; b < min(p.B, kCached); b += kThreads) sm_len[b] = p.lengths[b];
  if (p.sink)
#pragma unroll 1
    for (int kh = tid; kh < min(p.KV, kCached); kh += kThreads) sm_span[kh] = Sizes::clamped(p.sink[kh], p.local[kh]);
  __syncthreads();
  // in rows of items that cost the same: a sequence's, or with spans a (sequence, key head)'s
  const int per_seq = p.sink ? p.KV : 1, items = p.sink ? p.tiles : p.KV * p.tiles;
  const uint32_t rows = (uint32_t)p.B * per_seq, per = (rows - 1) / kThreads + 1;      // (B, KV < 2^16)
  const uint32_t row_lo = min(tid * per, rows), row_hi = row_lo + min(per, rows - row_lo);
  const int b_lo = (int)(row_lo / per_seq), kh_lo = (int)(row_lo - (uint32_t)b_lo * per_seq);
  auto cost_of = [&](int b, int kh) { return Span(sizes, sizes.tokens(b), kh).units + kCost; };
  int64_t mine = 0;
  int b_at = b_lo, kh_at = kh_lo;
#pragma unroll 4
  for (uint32_t r = row_lo; r < row_hi; ++r) {
    mine += (int64_t)items * cost_of(b_at, kh_at);
    if (++kh_at == per_seq) {
      kh_at = 0;
      ++b_at;
    }
  }
  int64_t before = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t other = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += other;
  }
  if (lane == 31) sm_sum[warp] = before;
  before -= mine;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sm_sum[w];
    total += sm_sum[w];
  }
  const Cut cut(total, SOLO ? gridDim.x * kWarps : gridDim.x, SOLO ? 1 : kMinUnits);
  const int number = SOLO ? warp * gridDim.x + blockIdx.x : blockIdx.x;
  if (SOLO) {                                      // (the warps of a block look for different parts)
    sm_before[tid] = before;
    __syncthreads();
  }

  if (number < cut.parts) {
    const Part part = {cut.begin(number), cut.begin(number + 1)};
    Cursor<SOLO> cur;
    // from the first of a thread's rows (b, kh, at) on to the row, and the item of it, in which the part begins
    auto walk = [&](int b, int kh, int64_t at) {
      int cost;
#pragma unroll 1
      for (;;) {
        cost = cost_of(b, kh);
        const int64_t end = at + (int64_t)items * cost;
        if (part.lo < end) break;
        at = end;
        if (++kh == per_seq) {
          kh = 0;
          ++b;
        }
      }
      const int item = items == 1 ? 0 : (int)divided(part.lo - at, cost);
      cur.b = b;
      cur.kh = kh + item;
      cur.tile = 0;
      if (p.tiles > 1) {
        cur.kh = kh + item / p.tiles;
        cur.tile = item % p.tiles;
      }
      cur.at = at + (int64_t)item * cost;
    };
    if (SOLO) {
      int j = 0;                                   // threads whose rows begin at or before the part
#pragma unroll
      for (int k = 0; k < kThreads; k += 32)
        j += __popc(__ballot_sync(0xffffffffu, (k + lane) * per < rows && sm_before[k + lane] <= part.lo));
      const uint32_t row = (j - 1) * per;
      walk((int)(row / per_seq), (int)(row % per_seq), sm_before[j - 1]);
    } else {
      if (before <= part.lo && part.lo < before + mine) {      // one thread
        walk(b_lo, kh_lo, before);
        sm_sum[8] = cur.b;
        sm_sum[9] = (int64_t)cur.kh << 32 | cur.tile;
        sm_sum[10] = cur.at;
      }
      __syncthreads();
      cur.b = (int)sm_sum[8];
      cur.kh = (int)(sm_sum[9] >> 32);
      cur.tile = (int)sm_sum[9];
      cur.at = sm_sum[10];
    }
    cur.n = sizes.tokens(cur.b);
    cur.enter(sizes, part);
    bool any = true;
    if (SOLO && cur.at < part.lo) any = cur.next(sizes, part);      // it begins in the part before
    const uint32_t item_at = (uint32_t)__cvta_generic_to_shared(sm_item);
    if (any) fetch_item<T, D, MT>(p, team, cur, sizes.fresh(cur.b), item_at);

    // ---- loads: a cursor of this warp's own
    Cursor<SOLO> ld = cur;
    bool ld_more = any;
    int ld_u = ld.u0 + team.warp;
    int ld_x = 0;                                  // aligned unit that is loaded next, its attended positions and its page
    uint32_t ld_mask = 0;                          // (of position lane % 16 when pages are smaller than a unit)
    int32_t ld_page = -1;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * kStages * L::kStageBytes;
    uint32_t* my_mask = reinterpret_cast<uint32_t*>(smem + L::kMask) + warp * kStages;

    auto ld_look = [&]() {                         // look up the next unit's page
      ld_x = ld.span.unit(ld_u);
      ld_mask = ld.span.mask(ld_x);
      const int32_t* row = p.pool.table + (int64_t)ld.b * p.pool.table_stride;
      if (opaque(p.pool.shift >= 4)) {
        ld_page = row[ld_x >> (p.pool.shift - 4)];
      } else {
        const int pos = ld_x * 16 + (lane & 15);
        ld_page = (ld_mask >> (lane & 15)) & 1 ? row[pos >> p.pool.shift] : -1;
      }
      if (ld_x == (ld.n - 1) >> 4 && sizes.fresh(ld.b)) ld_mask &= ~(1u << ((ld.n - 1) & 15));    // the new token is in no page
    };
    auto ld_seek = [&]() {                         // to the next unit of this warp
      while (ld_u >= ld.u1) {
        if (!ld.next(sizes, part)) {
          ld_more = false;
          return;
        }
        ld_u = ld.u0 + team.warp;
      }
      ld_look();
    };
    Ring<kStages> loads;
    auto ld_issue = [&](int stage) {
      if (ld_more) {
        const uint32_t dst = ring + stage * L::kStageBytes, bar = bars + stage * 8;
        if (ld_mask == 0xffffu && opaque(p.tma) && (uint32_t)ld_page < (uint32_t)p.pool.num_pages) {
          if (lane == 0) {
            const int slot = (ld_x << 4) & ((1 << p.pool.shift) - 1);
            my_mask[stage] = 0xffffu;              // seen by the other lanes when they have waited on the barrier
            bar_expect(bar, L::kStageBytes);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) tma_load(dst + i * L::kPanelBytes, &map_k, bar, i * 64, slot, ld.kh, ld_page);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) tma_load(dst + L::kTileBytes + i * L::kPanelBytes, &map_v, bar, i * 64, slot, ld.kh, ld_page);
          }
        } else {
          const uint32_t present = load_rows<T, D, MT>(p, ld.b, ld.kh, ld_x, ld_page, ld_mask, dst);
          if (lane == 0) {
            my_mask[stage] = present | kByHand;
            bar_arrive(bar);
          }
        }
        ld_u += team.warps;
        ld_seek();
      }
      cp_async_commit();                           // a group per call, empty or not: they are counted
    };

    if (any) ld_seek();
#pragma unroll 1
    for (int s = 0; s < kStages; ++s) ld_issue(s);

    // ---- items
    const int g = lane >> 2, t = lane & 3;         // row (query head of a tile) and column pair of a fragment
    int buf = 0;
    for (bool more = any; more; buf ^= 1) {
      Cursor<SOLO> next = cur;
      more = next.next(sizes, part);
      cp_async_wait_all();                         // the item's own data; its buffers were fetched an item ago
      team.sync();                                 // (and the item before is through with the join buffer)
      if (more) fetch_item<T, D, MT>(p, team, next, sizes.fresh(next.b), item_at + (buf ^ 1) * L::kItemBytes);

      unsigned char* item = sm_item + buf * L::kItemBytes;
      const int h0 = cur.kh * p.G + cur.tile * 8 * MT;                   // first query head of the item
      const int heads = min(p.G - cur.tile * 8 * MT, 8 * MT);
      const int units = cur.span.units;
      const bool owner = cur.at >= part.lo;        // the item begins in this part
      const bool ends = units == 0 ? owner : cur.u0 < cur.u1 && cur.u1 == units;
      const bool fresh = sizes.fresh(cur.b);
      const bool turn = fresh && p.pool.cos && rope_row(p.pool, cur.b, 0, cur.n - 1) >= 0;
      if (turn) {
        turn_queries<T, D, MT>(p, team, item, sm_low, heads);
        if (team.warp == team.warps - 1 && ends) turn_key<T, D, MT>(p, item);
        team.sync();
      }
      bool with_new = false;                       // this block attends the new token
      if (fresh && ends) {
        const int page = *reinterpret_cast<const int*>(item + L::kPage);
        const bool placed = (uint32_t)page < (uint32_t)p.pool.num_pages && (turn || !p.pool.cos);
        with_new = placed && cur.span.sees_last();
        if (team.warp == team.warps - 1 && cur.tile == 0) {
          if (placed) store_new<T, D, MT>(p, item, cur.kh, (cur.n - 1) & ((1 << p.pool.shift) - 1), page);
          else if (lane == 0) report(p.pool.cos && !turn ? kStatusRope : kStatusAppend, cur.b, cur.n - 1, cur.kh);
        }
      }
      if (owner && cur.kh == 0 && cur.tile == 0 && team.rank == 0) {
        const int64_t wanted = (int64_t)sizes.length(cur.b) + (p.k_new ? 1 : 0);
        if (wanted > p.capacity) report(kStatusLength, cur.b, wanted, 0);
      }

      if (units == 0) {                            // nothing to attend (a part's first item may not be its own)
        if (owner)
#pragma unroll 1
          for (int i = team.rank * 4; i < heads * D; i += team.size * 4)
            store_out4<T>(p, cur.b, h0 + i / D, i % D, make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
      } else if (cur.u0 < cur.u1) {
        float m[MT], l[MT], acc[D / 8][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          m[mt] = -INFINITY;
          l[mt] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
        // coordinates 8j + 2t and the next of query head 8 mt + g
        auto result = [&](int mt, int j) {
          return MT == 1 ? make_float2(joined(acc[j][0], acc[j][2]), joined(acc[j][1], acc[j][3]))
                         : make_float2(acc[j][2 * mt], acc[j][2 * mt + 1]);
        };
        if (cur.u0 + team.warp < cur.u1) {
          // query fragments.  One tile: rows 0-7 the heads, rows 8-15 what a rotated query has beyond 16 bits (without
          // tables those rows are whatever is there, and their scores are not looked at).  Two: 16 heads; what they
          // have beyond 16 bits is a second product, its fragments read when it is made.
          uint32_t qa[KS][4];
          const uint32_t q_row = (lane & 7) * L::kQPitch + (lane >> 4) * 16, q_8 = 8 * L::kQPitch;
          const uint32_t q_at = item_at + buf * L::kItemBytes + q_row, low_at = item_at + 2 * L::kItemBytes + q_row;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) ldmatrix4(qa[ks], ((lane & 8) ? (MT == 1 ? low_at : q_at + q_8) : q_at) + ks * 32);
          auto low_query = [&](int ks, uint32_t(&q)[4]) { ldmatrix4(q, low_at + ((lane & 8) ? q_8 : 0) + ks * 32); };
          if (with_new && team.warp == 0) {        // start from the new token: column 0 of a tile of keys, weight 1
            const uint32_t* key = reinterpret_cast<const uint32_t*>(item + L::kKey);
            float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              const uint32_t k0 = g == 0 ? key[ks * 8 + t] : 0u, k1 = g == 0 ? key[ks * 8 + 4 + t] : 0u;
              mma16816<T>(sc, qa[ks], k0, k1);
              if (MT > 1 && turn) {
                uint32_t q[4];
                low_query(ks, q);
                mma16816<T>(sc, q, k0, k1);
              }
            }
            float w[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              float score = (MT == 1 && turn ? joined(sc[0], sc[2]) : sc[2 * mt]) * p.scale_log2;
              score = __shfl_sync(0xffffffffu, score, lane & ~3);
              m[mt] = lifted<T>(score);
              // (weights of scores that are no numbers follow the formula: exp(inf - inf) and the like)
              w[mt] = score == -INFINITY ? 0.f : exp2f(score - m[mt]);
              l[mt] = t == 0 ? w[mt] : 0.f;
              if (m[mt] != m[mt]) m[mt] = -INFINITY;           // (a maximum passes over NaN)
            }
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
              const float2 v = Cvt<T>::unpack(*reinterpret_cast<const uint32_t*>(item + L::kValue + (j * 8 + 2 * t) * 2));
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                acc[j][2 * mt] = w[mt] * v.x;
                acc[j][2 * mt + 1] = w[mt] * v.y;
              }
            }
          }
          // ldmatrix addresses within a tile: four chunk pairs of a panel, the other panel behind them
          const int mi = lane >> 3, r8 = lane & 7;
          const uint32_t k_at = ((mi >> 1) * 8 + r8) * 128 + (((mi & 1) ^ r8) << 4);
          const uint32_t v_at = L::kTileBytes + ((mi & 1) * 8 + r8) * 128 + (((mi >> 1) ^ r8) << 4);
#pragma unroll 1
          for (int u = cur.u0 + team.warp; u < cur.u1; u += team.warps) {
            if (opaque(!loads.late))
              loads.take([&](int at, uint32_t parity) { return __all_sync(0xffffffffu, bar_wait(bars + at * 8, parity)) != 0; });
            ld_more = ld_more && !loads.late;      // (a late load is reported; the block goes on to its end without others)
            const uint32_t base = ring + loads.stage * L::kStageBytes;
            const uint32_t present = my_mask[loads.stage];
            if (present & kByHand) {
              cp_async_wait<kStages - 1>();        // one group per unit that was asked for after this one may be open
              __syncwarp();
            }
            float sc[2][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[0][e] = sc[1][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              uint32_t kb[4];
              ldmatrix4(kb, ((base + k_at) ^ ((ks & 3) << 5)) + (ks >> 2) * L::kPanelBytes);
              mma16816<T>(sc[0], qa[ks], kb[0], kb[1]);
              mma16816<T>(sc[1], qa[ks], kb[2], kb[3]);
              if (MT > 1 && opaque(turn)) {
                uint32_t q[4];
                low_query(ks, q);
                mma16816<T>(sc[0], q, kb[0], kb[1]);
                mma16816<T>(sc[1], q, kb[2], kb[3]);
              }
            }
            // weights as two 16-bit parts.  One tile: rows 0-7 of a fragment the upper parts, rows 8-15 the lower ones;
            // two: a fragment each, 16 heads.
            uint32_t pa[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              float s[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) s[e] = sc[e >> 1][(e & 1) + 2 * mt];
              if (MT == 1 && opaque(turn)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] = joined(s[e], sc[e >> 1][(e & 1) + 2]);
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) s[e] *= p.scale_log2;
              if (present != 0xffffu) {
                const uint32_t mine16 = present >> (2 * t);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (!((mine16 >> ((e >> 1) * 8 + (e & 1))) & 1)) s[e] = -INFINITY;
              }
              float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
              top = lifted<T>(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)));
              if (__any_sync(0xffffffffu, top > m[mt])) {      // a new maximum: what there is so far is scaled down
                const float m_new = fmaxf(m[mt], top);
                const float corr = m_new == m[mt] ? 1.f : exp2f(m[mt] - m_new);
                m[mt] = m_new;
                l[mt] *= corr;
#pragma unroll
                for (int j = 0; j < D / 8; ++j)
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if (MT == 1 || e >> 1 == mt) acc[j][e] *= corr;
              }
              const float ref = m[mt] == -INFINITY ? 0.f : m[mt];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                s[e] = exp2f(s[e] - ref);
                if (std::is_same<T, __half>::value && s[e] > 0.f) s[e] = fmaxf(s[e], 0x1p-24f);
              }
              l[mt] += (s[0] + s[1]) + (s[2] + s[3]);
              if (MT == 1) {
                split2<T, false>(s[0], s[1], pa[0][0], pa[0][1]);
                split2<T, false>(s[2], s[3], pa[0][2], pa[0][3]);
              } else {
                split_weights2<T>(s[0], s[1], pa[0][mt], pa[MT - 1][mt]);
                split_weights2<T>(s[2], s[3], pa[0][mt + 2], pa[MT - 1][mt + 2]);
              }
            }
#pragma unroll
            for (int j = 0; j < KS; ++j) {
              uint32_t vb[4];
              ldmatrix4_trans(vb, ((base + v_at) ^ ((j & 3) << 5)) + (j >> 2) * L::kPanelBytes);
#pragma unroll
              for (int part16 = 0; part16 < MT; ++part16) {
                if (part16 == 1 && std::is_same<T, __nv_bfloat16>::value)
#pragma unroll
                  for (int i = 0; i < 4; ++i) vb[i] = finite2(vb[i]);
                mma16816<T>(acc[2 * j], pa[part16], vb[0], vb[1]);
                mma16816<T>(acc[2 * j + 1], pa[part16], vb[2], vb[3]);
              }
            }
            if (present & kByHand) proxy_fence();
            __syncwarp();
            ld_issue(loads.stage);
            loads.next();
          }
        }

        if (SOLO) {                           // ---- a warp's own result
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            float sum = l[mt];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (mt * 8 + g >= heads) continue;
            const float f = sum == 0.f ? 0.f : 1.f / sum;
            const int64_t off = (int64_t)cur.b * p.o_sb + (int64_t)(h0 + mt * 8 + g) * p.o_sh + 2 * t;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
              const float2 o = result(mt, j);
              const float x = sum == 0.f ? 0.f : o.x * f, y = sum == 0.f ? 0.f : o.y * f;
              if (p.out_f32) *reinterpret_cast<float2*>(reinterpret_cast<float*>(p.out) + off + j * 8) = make_float2(x, y);
              else *reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + off + j * 8) = Cvt<T>::pack(x, y);
            }
          }
          if (more) cur = next;
          continue;
        }

        // ---- the warps' results joined
        const bool whole = cur.u0 == 0 && cur.u1 == units;
        const int nw = min(kWarps, cur.u1 - cur.u0);
        float* rec = p.records + (int64_t)(2 * blockIdx.x + (owner ? 1 : 0)) * kRecFloats;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int here = min(heads - mt * 8, 8);
          if (MT > 1 && here <= 0) break;
          if (mt > 0) __syncthreads();
          if (warp < nw) {
            float sum = l[mt];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (t == 0) {
              sm_m[warp * 8 + g] = m[mt];
              sm_l[warp * 8 + g] = sum;
            }
            if (g < here) {
              float* o = sm_o + (warp * 8 + g) * D;
#pragma unroll
              for (int j = 0; j < D / 8; ++j)
                *reinterpret_cast<float2*>(o + ((j * 8 + 2 * t) ^ (g << 2))) = result(mt, j);
            }
          }
          __syncthreads();
#pragma unroll 1
          for (int i = tid * 4; i < here * D; i += kThreads * 4) {
            const int head = i / D, d = i % D;
            float M = -INFINITY, Ls = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
              if (w < nw) M = fmaxf(M, sm_m[w * 8 + head]);
            const float base = M == -INFINITY ? 0.f : M;
            float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
              if (w < nw) {
                const float f = exp2f(sm_m[w * 8 + head] - base);
                const float4 x = *reinterpret_cast<const float4*>(sm_o + (w * 8 + head) * D + (d ^ (head << 2)));
                Ls += f * sm_l[w * 8 + head];
                O.x += f * x.x; O.y += f * x.y; O.z += f * x.z; O.w += f * x.w;
              }
            if (whole) {
              store_out4<T>(p, cur.b, h0 + mt * 8 + head, d, O, Ls);
            } else {
              *reinterpret_cast<float4*>(rec + (mt * 8 + head) * D + d) = O;
              if (d == 0) *reinterpret_cast<float2*>(rec + kRecHeads * 128 + (mt * 8 + head) * 2) = make_float2(M, Ls);
            }
          }
        }
        if (!whole)
          join_parts<T, D, MT>(p, cut.part_of(cur.at), cut.part_of(cur.at + units - 1), cur.b, h0, heads, sm_o, sm_flag);
      }
      if (more) cur = next;
    }
    if (loads.late) {                              // one limit for all stages
      const long long start = clock64();
      loads.drain([&](int at, uint32_t parity) {
        while (!bar_try(bars + at * 8, parity))
          if (clock64() - start > kWaitCycles) break;
      });
    }
  }

  if (p.advance) {                                 // the last block to get here: every block has read the lengths
    __syncthreads();
    if (tid == 0) {
      int* done = p.counters + kCounters * kMaxParts;
      *sm_flag = atomicAdd(done, 1) == (int)gridDim.x - 1;
      if (*sm_flag) *done = 0;
    }
    __syncthreads();
    if (*sm_flag)
#pragma unroll 1
      for (int b = tid; b < p.B; b += kThreads) {
        const int len = p.lengths[b];
        if (len >= 0 && len < 2147483647) p.lengths[b] = len + 1;
      }
  }
}

constexpr int kMaxDevices = 64;
// SMs of the current device (kept per device ordinal); 148 where no device can be asked.
int sm_count() {
  static int cached[kMaxDevices];                  // benign race: every writer stores the same value
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices ||
      (cached[dev] == 0 && cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)) {
    (void)cudaGetLastError();
    return 148;
  }
  if (cached[dev] == 0) cached[dev] = std::min(sms, kMaxParts / kPerSm);
  return cached[dev];
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The pool as a tensor (D, slots, heads, pages) that is loaded in panels of 16 rows of 64 values.  False when the
// strides are none that TMA takes.
bool make_map(CUtensorMap* map, const void* base, const DecodeParams& p, int64_t page, int64_t head, int64_t slot, int D,
              bool bf16) {
  static EncodeTiledFn encode = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      ptr = nullptr;
    }
    return reinterpret_cast<EncodeTiledFn>(ptr);
  }();
  if (!encode) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)1 << p.pool.shift, (cuuint64_t)p.KV, (cuuint64_t)p.pool.num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)slot * 2, (cuuint64_t)head * 2, (cuuint64_t)page * 2};
  const cuuint32_t box[4] = {64, kUnit, 1, 1}, step[4] = {1, 1, 1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base),
                dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                // rows of 128 bytes apart from one another: a neighbour's would be fetched for nothing
                D == 64 && slot != D ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, int MT, bool SOLO>
int launch_decode(DecodeParams& p, int grid, cudaStream_t stream) {
  using L = Layout<D, MT, SOLO>;
  static bool ready[kMaxDevices];
  int dev = 0;
  MOA_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices || !ready[dev]) {
    MOA_CUDA_CHECK(cudaFuncSetAttribute(paged_decode_kernel<T, D, MT, SOLO>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
    if (dev >= 0 && dev < kMaxDevices) ready[dev] = true;
  }
  CUtensorMap map_k, map_v;
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  p.tma = p.pool.shift >= 4 &&      // a unit lies in one page
          make_map(&map_k, p.pool.k, p, p.pool.k_page, p.pool.k_head, p.pool.k_slot, D, bf16) &&
          make_map(&map_v, p.pool.v, p, p.pool.v_page, p.pool.v_head, p.pool.v_slot, D, bf16);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)grid);
  config.blockDim = dim3(L::kThreads);
  config.dynamicSmemBytes = L::kBytes;
  config.stream = stream;
  cudaLaunchAttribute early = {};                  // see griddepcontrol.wait in the kernel
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  MOA_CUDA_CHECK(cudaLaunchKernelEx(&config, paged_decode_kernel<T, D, MT, SOLO>, map_k, map_v, p));
  return MOA_OK;
}
template <typename T, int D, int MT>
int launch_decode(DecodeParams& p, int grid, cudaStream_t stream) {
  // Warps on their own where no sequence can be long (the page table reaches kSoloTokens at most) and blocks would have
  // to take several items each.  By blocks and by warps: 120 sequences of 1..34 tokens, 32 heads of 128, 53 and 20 us;
  // 51 of 128 tokens, 16 heads, 31 and 18.5; 20 of 156..318 tokens, 16 heads of 64, 18.0 and 21.1.
  if constexpr (Layout<D, MT, true>::kFits)        // (16 heads of 128: no room)
    if (p.capacity <= kSoloTokens && (int64_t)p.B * p.KV * p.tiles > grid) return launch_decode<T, D, MT, true>(p, grid, stream);
  return launch_decode<T, D, MT, false>(p, grid, stream);
}
template <typename T>
int launch_decode(DecodeParams& p, int D, int grid, cudaStream_t stream) {
  if (D == 128) return p.G > 8 ? launch_decode<T, 128, 2>(p, grid, stream) : launch_decode<T, 128, 1>(p, grid, stream);
  return p.G > 8 ? launch_decode<T, 64, 2>(p, grid, stream) : launch_decode<T, 64, 1>(p, grid, stream);
}

inline bool aligned(const void* p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
inline bool aligned16(const void* p) { return aligned(p, 16); }
inline bool multiples_of_8(std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if (s % 8 != 0 || s < 0) return false;
  return true;
}

// The checks and the translation that both argument structs share.
template <typename A>
int make_pool(const A& a, Pool& p) {
  MOA_REQUIRE(a.k_pages && a.v_pages && a.page_table && a.lengths, "paged: null pointer");
  MOA_REQUIRE(a.B > 0 && a.B <= 65535 && a.KV > 0 && a.KV <= 65535 && a.H > 0 && a.H <= 65535, "paged: bad shape");
  MOA_REQUIRE(a.max_pages > 0 && a.max_pages <= 2147483647LL && a.num_pages > 0 && a.num_pages <= 2147483647LL &&
                  a.table_stride >= 0,
              "paged: bad page table or number of pages");
  MOA_REQUIRE(a.page_size > 0 && a.page_size <= 65536 && (a.page_size & (a.page_size - 1)) == 0,
              "paged: page_size must be a power of two up to 65536");
  MOA_REQUIRE(aligned16(a.k_pages) && aligned16(a.v_pages) &&
                  multiples_of_8({a.kp_page, a.kp_head, a.kp_slot, a.vp_page, a.vp_head, a.vp_slot}),
              "paged: pages must be 16-byte aligned with strides that are multiples of 8 elements");
  MOA_REQUIRE(aligned(a.page_table, 4) && aligned(a.lengths, 4), "paged: page_table and lengths must be 4-byte aligned");
  MOA_REQUIRE((a.rope_cos == nullptr) == (a.rope_sin == nullptr), "paged: rope_cos and rope_sin go together");
  if (a.rope_cos) {
    MOA_REQUIRE(aligned16(a.rope_cos) && aligned16(a.rope_sin) && multiples_of_8({a.rope_sb, a.rope_sn}) && a.rope_rows >= 0,
                "paged: rope tables must be 16-byte aligned with strides that are multiples of 8 elements");
  }
  if (a.D != 64 && a.D != 128) {
    set_error_text("paged: head_dim must be 64 or 128");
    return MOA_ERR_UNSUPPORTED;
  }
  if (a.dtype != MOA_F16 && a.dtype != MOA_BF16) {
    set_error_text("paged: dtype must be MOA_F16 or MOA_BF16");
    return MOA_ERR_UNSUPPORTED;
  }
  p.k = a.k_pages; p.v = a.v_pages;
  p.k_page = a.kp_page; p.k_head = a.kp_head; p.k_slot = a.kp_slot;
  p.v_page = a.vp_page; p.v_head = a.vp_head; p.v_slot = a.vp_slot;
  p.table = a.page_table; p.table_stride = a.table_stride; p.max_pages = a.max_pages;
  p.num_pages = (int32_t)a.num_pages;
  p.shift = 0;
  while ((1ll << p.shift) < a.page_size) ++p.shift;
  p.cos = a.rope_cos; p.sin = a.rope_sin;
  p.rope_sb = a.rope_sb; p.rope_sn = a.rope_sn; p.rope_rows = a.rope_rows; p.rope_f32 = a.rope_f32 != 0;
  return MOA_OK;
}

}  // namespace
}  // namespace moa

extern "C" {

int moa_paged_append(const moa_paged_append_args* args, moa_stream_t stream) {
  using namespace moa;
  MOA_REQUIRE(args != nullptr, "paged_append: null arguments");
  const moa_paged_append_args& a = *args;
  AppendParams p;
  const int rc = make_pool(a, p.pool);
  if (rc != MOA_OK) return rc;
  MOA_REQUIRE(a.k && a.v, "paged_append: null pointer");
  MOA_REQUIRE(a.N > 0 && a.N <= (1ll << 30), "paged_append: bad number of tokens");
  MOA_REQUIRE((a.q == nullptr) == (a.q_out == nullptr) && (a.q == nullptr) == (a.k_out == nullptr),
              "paged_append: q, q_out and k_out go together");
  MOA_REQUIRE(a.q == nullptr || a.rope_cos != nullptr, "paged_append: a query is given to be rotated: tables are needed");
  MOA_REQUIRE(aligned16(a.k) && aligned16(a.v) && aligned16(a.q) && aligned16(a.q_out) && aligned16(a.k_out) &&
                  multiples_of_8({a.k_sb, a.k_sh, a.k_sn, a.v_sb, a.v_sh, a.v_sn, a.q_sb, a.q_sh, a.q_sn}),
              "paged_append: rows must be 16-byte aligned with strides that are multiples of 8 elements");
  MOA_REQUIRE(aligned(a.counts, 4), "paged_append: counts must be 4-byte aligned");
  p.k = a.k; p.v = a.v; p.q = a.q; p.lengths = a.lengths; p.counts = a.counts; p.q_out = a.q_out; p.k_out = a.k_out;
  p.k_sb = a.k_sb; p.k_sh = a.k_sh; p.k_sn = a.k_sn; p.v_sb = a.v_sb; p.v_sh = a.v_sh; p.v_sn = a.v_sn;
  p.q_sb = a.q_sb; p.q_sh = a.q_sh; p.q_sn = a.q_sn;
  p.H = (int)a.H; p.KV = (int)a.KV; p.N = a.N;
  p.kv_jobs = (p.KV + kHeads - 1) / kHeads;
  p.jobs = p.kv_jobs + (a.q ? (p.H + kHeads - 1) / kHeads : 0);
  MOA_REQUIRE(a.N * p.jobs * (a.D / 16) < (1ll << 31) - kAppendThreads, "paged_append: too many rows");
  dim3 grid((unsigned)ceil_div64(a.N * p.jobs * (a.D / 16), kAppendThreads), (unsigned)a.B);
  cudaStream_t st = (cudaStream_t)stream;
  if (a.dtype == MOA_F16) {
    if (a.D == 128) paged_append_kernel<__half, 128><<<grid, kAppendThreads, 0, st>>>(p);
    else paged_append_kernel<__half, 64><<<grid, kAppendThreads, 0, st>>>(p);
  } else {
    if (a.D == 128) paged_append_kernel<__nv_bfloat16, 128><<<grid, kAppendThreads, 0, st>>>(p);
    else paged_append_kernel<__nv_bfloat16, 64><<<grid, kAppendThreads, 0, st>>>(p);
  }
  MOA_CUDA_CHECK(cudaGetLastError());
  if (a.advance) {
    paged_advance_kernel<<<(unsigned)ceil_div64(a.B, 256), 256, 0, st>>>(a.lengths, a.counts, a.N, (int)a.B);
    MOA_CUDA_CHECK(cudaGetLastError());
  }
  return MOA_OK;
}

int64_t moa_paged_decode_workspace_bytes(void) {
  using namespace moa;
  static_assert((kCounters * kMaxParts + 1) * 4 <= MOA_PAGED_COUNTER_BYTES, "counters");
  return MOA_PAGED_COUNTER_BYTES + (int64_t)sm_count() * kPerSm * 2 * kRecFloats * 4;
}

int moa_paged_decode(const moa_paged_decode_args* args, moa_stream_t stream) {
  using namespace moa;
  MOA_REQUIRE(args != nullptr, "paged_decode: null arguments");
  const moa_paged_decode_args& a = *args;
  DecodeParams p;
  const int rc = make_pool(a, p.pool);
  if (rc != MOA_OK) return rc;
  MOA_REQUIRE(a.q && a.out, "paged_decode: null pointer");
  MOA_REQUIRE((a.k_new == nullptr) == (a.v_new == nullptr), "paged_decode: k_new and v_new go together");
  MOA_REQUIRE(a.rope_cos == nullptr || a.k_new != nullptr, "paged_decode: the rotary embedding is for the step with a new token");
  MOA_REQUIRE((a.sink_size == nullptr) == (a.local_size == nullptr), "paged_decode: sink_size and local_size go together");
  MOA_REQUIRE(a.H % a.KV == 0, "paged_decode: the query heads must be a multiple of the key heads");
  MOA_REQUIRE(!a.advance || a.k_new, "paged_decode: advance needs a new token");
  MOA_REQUIRE(aligned16(a.q) && aligned16(a.k_new) && aligned16(a.v_new) &&
                  multiples_of_8({a.q_sb, a.q_sh, a.k_sb, a.k_sh, a.v_sb, a.v_sh}),
              "paged_decode: rows must be 16-byte aligned with strides that are multiples of 8 elements");
  MOA_REQUIRE(aligned16(a.out) && multiples_of_8({a.o_sb, a.o_sh}),
              "paged_decode: rows of out must be 16-byte aligned with strides that are multiples of 8 elements");
  MOA_REQUIRE(aligned(a.sink_size, 8) && aligned(a.local_size, 8), "paged_decode: sink_size and local_size must be 8-byte aligned");
  MOA_REQUIRE(aligned16(a.workspace), "paged_decode: workspace must be 16-byte aligned");
  if (!a.workspace || a.workspace_bytes < moa_paged_decode_workspace_bytes()) {
    set_error_text("paged_decode: workspace missing or smaller than moa_paged_decode_workspace_bytes()");
    return MOA_ERR_WORKSPACE;
  }
  p.q = a.q; p.k_new = a.k_new; p.v_new = a.v_new; p.out = a.out; p.lengths = a.lengths;
  p.sink = a.sink_size; p.local = a.local_size;
  p.q_sb = a.q_sb; p.q_sh = a.q_sh; p.k_sb = a.k_sb; p.k_sh = a.k_sh; p.v_sb = a.v_sb; p.v_sh = a.v_sh;
  p.o_sb = a.o_sb; p.o_sh = a.o_sh;
  p.B = (int)a.B; p.H = (int)a.H; p.KV = (int)a.KV; p.G = p.H / p.KV;
  p.tiles = (p.G + (p.G > 8 ? 15 : 7)) / (p.G > 8 ? 16 : 8);
  p.capacity = (int)std::min(a.max_pages * a.page_size, (int64_t)2147483647 - 64);
  p.scale_log2 = (float)(a.sm_scale * 1.4426950408889634);
  p.out_f32 = a.out_f32 != 0; p.advance = a.advance != 0;
  p.counters = reinterpret_cast<int*>(a.workspace);
  p.records = reinterpret_cast<float*>(reinterpret_cast<char*>(a.workspace) + MOA_PAGED_COUNTER_BYTES);
  // as many blocks as the longest sequences that the table allows could employ
  const int64_t most = a.B * a.KV * p.tiles * (std::min(ceil_div64(p.capacity, kUnit), (int64_t)4096) + kItemCost);
  const int grid = (int)std::max((int64_t)1, std::min((int64_t)sm_count() * kPerSm, most / kMinUnits));
  cudaStream_t st = (cudaStream_t)stream;
  return a.dtype == MOA_F16 ? launch_decode<__half>(p, (int)a.D, grid, st)
                            : launch_decode<__nv_bfloat16>(p, (int)a.D, grid, st);
}

int moa_paged_status(int32_t status[4]) {
  using namespace moa;
  MOA_REQUIRE(status != nullptr, "paged_status: null pointer");
  MOA_CUDA_CHECK(cudaDeviceSynchronize());
  MOA_CUDA_CHECK(cudaMemcpyFromSymbol(status, g_paged_status, sizeof(g_paged_status)));
  if (status[0] != 0) {
    const int32_t zero[4] = {0, 0, 0, 0};
    MOA_CUDA_CHECK(cudaMemcpyToSymbol(g_paged_status, zero, sizeof(zero)));
  }
  return MOA_OK;
}

}  // extern "C"
