// Paged key/value cache: append (with the rotary embedding on the way) and attention of one new token
// per sequence.
//
// Token p of sequence b lives in slot p % page_size of page table[b, p / page_size]; every index that
// comes from device memory (lengths, counts, table entries) is checked against its array before it
// is used, and a token whose place does not exist is left out and reported in g_paged_status.
#include <initializer_list>

#include "common.cuh"

namespace moa {
namespace {

constexpr int kStatusAppend = 31, kStatusAttend = 32, kStatusRope = 33, kStatusLength = 34;
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
  int H, KV, jobs;   // jobs: rows of work per token, KV key/value heads and then, with q, H query heads
  int64_t N;
};

// The two 8-wide pieces [8c, 8c+8) and [D/2 + 8c, ...) of a row, which the rotation mixes:
//   x'[d] = x[d] cos[d] - x[d + D/2] sin[d],   x'[d + D/2] = x[d + D/2] cos[d + D/2] + x[d] sin[d + D/2]
// in fp32, rounded once to T (that rounding is the cache's storage type).
template <typename T, int D>
__device__ __forceinline__ void rotate_pair(const Pool& p, int64_t row, int c, uint4& lo_u, uint4& hi_u) {
  float lo[8], hi[8], cl[8], ch[8], sl[8], sh[8], a[8], b[8];
  unpack8<T>(lo_u, lo);
  unpack8<T>(hi_u, hi);
  load_table8<T>(p, p.cos, row + c * 8, cl);
  load_table8<T>(p, p.cos, row + D / 2 + c * 8, ch);
  load_table8<T>(p, p.sin, row + c * 8, sl);
  load_table8<T>(p, p.sin, row + D / 2 + c * 8, sh);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    a[j] = fmaf(lo[j], cl[j], -hi[j] * sl[j]);
    b[j] = fmaf(hi[j], ch[j], lo[j] * sh[j]);
  }
  lo_u = pack8<T>(a);
  hi_u = pack8<T>(b);
}

// D/16 threads per (token, head) row; each moves 16 bytes of either half of the key row and of the value
// row (or of a query row).  Bound by memory: every row is read once and written once.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int TPR = D / 16;
  const int64_t b = blockIdx.y;
  const int64_t idx = ((int64_t)blockIdx.x * 256 + threadIdx.x) / TPR;
  const int c = threadIdx.x % TPR;
  const int64_t i = idx / p.jobs;
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
  if (job >= p.KV) {                    // a query row
    const int h = job - p.KV;
    uint4 lo = zero, hi = zero;
    if (known) {
      const T* src = reinterpret_cast<const T*>(p.q) + b * p.q_sb + h * p.q_sh + i * p.q_sn + c * 8;
      lo = *reinterpret_cast<const uint4*>(src);
      hi = *reinterpret_cast<const uint4*>(src + D / 2);
      rotate_pair<T, D>(p.pool, row, c, lo, hi);
    }
    T* dst = reinterpret_cast<T*>(p.q_out) + ((b * p.H + h) * p.N + i) * D + c * 8;
    *reinterpret_cast<uint4*>(dst) = lo;
    *reinterpret_cast<uint4*>(dst + D / 2) = hi;
    return;
  }
  uint4 klo = zero, khi = zero, vlo = zero, vhi = zero;
  if (known) {
    const T* ks = reinterpret_cast<const T*>(p.k) + b * p.k_sb + job * p.k_sh + i * p.k_sn + c * 8;
    const T* vs = reinterpret_cast<const T*>(p.v) + b * p.v_sb + job * p.v_sh + i * p.v_sn + c * 8;
    klo = *reinterpret_cast<const uint4*>(ks);
    khi = *reinterpret_cast<const uint4*>(ks + D / 2);
    vlo = *reinterpret_cast<const uint4*>(vs);
    vhi = *reinterpret_cast<const uint4*>(vs + D / 2);
    if (p.pool.cos) rotate_pair<T, D>(p.pool, row, c, klo, khi);
    const int32_t page = page_of(p.pool, p.pool.table + b * p.pool.table_stride, pos);
    if (page >= 0) {
      const int64_t slot = pos & ((1ll << p.pool.shift) - 1);
      T* kd = reinterpret_cast<T*>(p.pool.k) + page * p.pool.k_page + job * p.pool.k_head + slot * p.pool.k_slot + c * 8;
      T* vd = reinterpret_cast<T*>(p.pool.v) + page * p.pool.v_page + job * p.pool.v_head + slot * p.pool.v_slot + c * 8;
      *reinterpret_cast<uint4*>(kd) = klo;
      *reinterpret_cast<uint4*>(kd + D / 2) = khi;
      *reinterpret_cast<uint4*>(vd) = vlo;
      *reinterpret_cast<uint4*>(vd + D / 2) = vhi;
    } else if (job == 0 && c == 0) {
      report(kStatusAppend, b, pos, 0);
    }
  }
  if (p.k_out) {
    T* dst = reinterpret_cast<T*>(p.k_out) + ((b * p.KV + job) * p.N + i) * D + c * 8;
    *reinterpret_cast<uint4*>(dst) = klo;
    *reinterpret_cast<uint4*>(dst + D / 2) = khi;
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
struct DecodeParams {
  Pool pool;
  const void *q, *k_new, *v_new;
  void* out;
  int32_t* lengths;
  const int64_t *sink, *local;
  int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh, o_sb, o_sh;
  int B, H, KV;
  float scale_log2;
  int out_f32;
};

// One block per (query head, sequence): 4 warps walk the rows of the head's span, D/8 lanes a row, with a
// running maximum and sum each; the block joins them.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_decode_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int LPR = D / 8, RPI = 32 / LPR, GROUPS = 4 * RPI;
  __shared__ __align__(16) T sm_q[D], sm_k[D], sm_v[D];
  __shared__ float sm_m[GROUPS], sm_l[GROUPS];
  __shared__ float sm_acc[GROUPS][D];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, li = lane % LPR, g = warp * RPI + lane / LPR;
  const int h = blockIdx.x, G = p.H / p.KV, kh = h / G;
  const int64_t b = blockIdx.y;
  const int32_t* table_row = p.pool.table + b * p.pool.table_stride;
  const int64_t slot_mask = (1ll << p.pool.shift) - 1, capacity = p.pool.max_pages << p.pool.shift;
  const int64_t len = p.lengths[b];
  const bool fused = p.k_new != nullptr;
  int64_t n = fused ? (len < 0 ? 0 : len + 1) : max(len, (int64_t)0);
  const int64_t pos_new = fused && n > 0 ? len : -1;
  if (n > capacity) {
    if (tid == 0 && h == 0) report(kStatusLength, b, n, 0);
    n = capacity;
  }
  bool have_new = pos_new >= 0 && pos_new < n;
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_sb + h * p.q_sh;
  float qf[8];
  if (have_new) {
    const int64_t row = p.pool.cos ? rope_row(p.pool, b, 0, pos_new) : 0;
    const int32_t page = page_of(p.pool, table_row, pos_new);
    if (row < 0 || page < 0) {
      if (tid == 0 && h == 0) report(row < 0 ? kStatusRope : kStatusAppend, b, pos_new, 0);
      have_new = false;
    }
    if (tid < D / 16 && row >= 0) {
      const T* ks = reinterpret_cast<const T*>(p.k_new) + b * p.k_sb + kh * p.k_sh + tid * 8;
      const T* vs = reinterpret_cast<const T*>(p.v_new) + b * p.v_sb + kh * p.v_sh + tid * 8;
      uint4 klo = *reinterpret_cast<const uint4*>(ks), khi = *reinterpret_cast<const uint4*>(ks + D / 2);
      const uint4 vlo = *reinterpret_cast<const uint4*>(vs), vhi = *reinterpret_cast<const uint4*>(vs + D / 2);
      if (p.pool.cos) rotate_pair<T, D>(p.pool, row, tid, klo, khi);
      *reinterpret_cast<uint4*>(sm_k + tid * 8) = klo;
      *reinterpret_cast<uint4*>(sm_k + D / 2 + tid * 8) = khi;
      *reinterpret_cast<uint4*>(sm_v + tid * 8) = vlo;
      *reinterpret_cast<uint4*>(sm_v + D / 2 + tid * 8) = vhi;
      if (have_new && h % G == 0) {
        T* kd = reinterpret_cast<T*>(p.pool.k) + page * p.pool.k_page + kh * p.pool.k_head + (pos_new & slot_mask) * p.pool.k_slot + tid * 8;
        T* vd = reinterpret_cast<T*>(p.pool.v) + page * p.pool.v_page + kh * p.pool.v_head + (pos_new & slot_mask) * p.pool.v_slot + tid * 8;
        *reinterpret_cast<uint4*>(kd) = klo;
        *reinterpret_cast<uint4*>(kd + D / 2) = khi;
        *reinterpret_cast<uint4*>(vd) = vlo;
        *reinterpret_cast<uint4*>(vd + D / 2) = vhi;
      }
    }
    __syncthreads();
    unpack8<T>(*reinterpret_cast<const uint4*>(q + li * 8), qf);
    if (p.pool.cos && row >= 0) {       // the query is rotated in fp32 and not rounded
      float other[8], cf[8], sf[8];
      const bool upper = li >= LPR / 2;
      unpack8<T>(*reinterpret_cast<const uint4*>(q + (upper ? li * 8 - D / 2 : li * 8 + D / 2)), other);
      load_table8<T>(p.pool, p.pool.cos, row + li * 8, cf);
      load_table8<T>(p.pool, p.pool.sin, row + li * 8, sf);
#pragma unroll
      for (int j = 0; j < 8; ++j) qf[j] = fmaf(qf[j], cf[j], (upper ? other[j] : -other[j]) * sf[j]);
    }
  } else {
    unpack8<T>(*reinterpret_cast<const uint4*>(q + li * 8), qf);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) qf[j] *= p.scale_log2;

  int64_t sink = n, rows = n;           // the span: positions [0, sink) and [n - (rows - sink), n)
  if (p.sink) {
    sink = min(max(p.sink[kh], (int64_t)0), n);
    rows = min(n, sink + min(max(p.local[kh], (int64_t)0), n));
  }
  const int64_t gap = n - rows;
  float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  for (int64_t r0 = 0; r0 < rows; r0 += GROUPS) {
    const int64_t r = r0 + g;
    const int64_t pos = r < sink ? r : r + gap;
    uint4 ku = make_uint4(0, 0, 0, 0), vu = ku;
    bool ok = r < rows;
    if (ok && pos == pos_new) {
      ok = have_new;
      ku = *reinterpret_cast<const uint4*>(sm_k + li * 8);
      vu = *reinterpret_cast<const uint4*>(sm_v + li * 8);
    } else if (ok) {
      const int32_t page = page_of(p.pool, table_row, pos);
      ok = page >= 0;
      if (ok) {
        ku = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.pool.k) + page * p.pool.k_page + kh * p.pool.k_head + (pos & slot_mask) * p.pool.k_slot + li * 8);
        vu = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.pool.v) + page * p.pool.v_page + kh * p.pool.v_head + (pos & slot_mask) * p.pool.v_slot + li * 8);
      } else if (li == 0) {
        report(kStatusAttend, b, pos, h);
      }
    }
    float kf[8], vf[8], s = 0.f;
    unpack8<T>(ku, kf);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(qf[j], kf[j], s);
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (ok) {
      unpack8<T>(vu, vf);
      const float m_new = fmaxf(m, s), base = m_new == -INFINITY ? 0.f : m_new;
      const float corr = exp2f(m - base), pr = exp2f(s - base);
      l = l * corr + pr;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = fmaf(pr, vf[j], acc[j] * corr);
      m = m_new;
    }
  }
  if (li == 0) {
    sm_m[g] = m;
    sm_l[g] = l;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sm_acc[g][li * 8 + j] = acc[j];
  __syncthreads();
  if (tid >= D) return;
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int i = 0; i < GROUPS; ++i) M = fmaxf(M, sm_m[i]);
  if (M == -INFINITY) M = 0.f;
  for (int i = 0; i < GROUPS; ++i) {
    const float w = exp2f(sm_m[i] - M);
    L += sm_l[i] * w;
    O += sm_acc[i][tid] * w;
  }
  const float o = L == 0.f ? 0.f : O / L;
  const int64_t off = b * p.o_sb + h * p.o_sh + tid;
  if (p.out_f32) reinterpret_cast<float*>(p.out)[off] = o;
  else reinterpret_cast<T*>(p.out)[off] = static_cast<T>(o);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
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
  p.k = a.k; p.v = a.v; p.q = a.q; p.lengths = a.lengths; p.counts = a.counts; p.q_out = a.q_out; p.k_out = a.k_out;
  p.k_sb = a.k_sb; p.k_sh = a.k_sh; p.k_sn = a.k_sn; p.v_sb = a.v_sb; p.v_sh = a.v_sh; p.v_sn = a.v_sn;
  p.q_sb = a.q_sb; p.q_sh = a.q_sh; p.q_sn = a.q_sn;
  p.H = (int)a.H; p.KV = (int)a.KV; p.N = a.N;
  p.jobs = p.KV + (a.q ? p.H : 0);
  const int64_t blocks = ceil_div64(a.N * p.jobs * (a.D / 16), 256);
  MOA_REQUIRE(blocks <= 2147483647LL, "paged_append: too many rows");
  dim3 grid((unsigned)blocks, (unsigned)a.B);
  cudaStream_t st = (cudaStream_t)stream;
  if (a.dtype == MOA_F16) {
    if (a.D == 128) paged_append_kernel<__half, 128><<<grid, 256, 0, st>>>(p);
    else paged_append_kernel<__half, 64><<<grid, 256, 0, st>>>(p);
  } else {
    if (a.D == 128) paged_append_kernel<__nv_bfloat16, 128><<<grid, 256, 0, st>>>(p);
    else paged_append_kernel<__nv_bfloat16, 64><<<grid, 256, 0, st>>>(p);
  }
  MOA_CUDA_CHECK(cudaGetLastError());
  if (a.advance) {
    paged_advance_kernel<<<(unsigned)ceil_div64(a.B, 256), 256, 0, st>>>(a.lengths, a.counts, a.N, (int)a.B);
    MOA_CUDA_CHECK(cudaGetLastError());
  }
  return MOA_OK;
}

int64_t moa_paged_decode_workspace_bytes(void) { return MOA_PAGED_COUNTER_BYTES; }

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
  if (!a.workspace || a.workspace_bytes < moa_paged_decode_workspace_bytes()) {
    set_error_text("paged_decode: workspace missing or smaller than moa_paged_decode_workspace_bytes()");
    return MOA_ERR_WORKSPACE;
  }
  p.q = a.q; p.k_new = a.k_new; p.v_new = a.v_new; p.out = a.out; p.lengths = a.lengths;
  p.sink = a.sink_size; p.local = a.local_size;
  p.q_sb = a.q_sb; p.q_sh = a.q_sh; p.k_sb = a.k_sb; p.k_sh = a.k_sh; p.v_sb = a.v_sb; p.v_sh = a.v_sh;
  p.o_sb = a.o_sb; p.o_sh = a.o_sh;
  p.B = (int)a.B; p.H = (int)a.H; p.KV = (int)a.KV;
  p.scale_log2 = (float)(a.sm_scale * 1.4426950408889634);
  p.out_f32 = a.out_f32 != 0;
  dim3 grid((unsigned)a.H, (unsigned)a.B);
  cudaStream_t st = (cudaStream_t)stream;
  if (a.dtype == MOA_F16) {
    if (a.D == 128) paged_decode_kernel<__half, 128><<<grid, 128, 0, st>>>(p);
    else paged_decode_kernel<__half, 64><<<grid, 128, 0, st>>>(p);
  } else {
    if (a.D == 128) paged_decode_kernel<__nv_bfloat16, 128><<<grid, 128, 0, st>>>(p);
    else paged_decode_kernel<__nv_bfloat16, 64><<<grid, 128, 0, st>>>(p);
  }
  MOA_CUDA_CHECK(cudaGetLastError());
  if (a.advance) {
    paged_advance_kernel<<<(unsigned)ceil_div64(a.B, 256), 256, 0, st>>>(a.lengths, nullptr, 1, (int)a.B);
    MOA_CUDA_CHECK(cudaGetLastError());
  }
  return MOA_OK;
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
