// paged_ops.cu -- the bookkeeping of a paged K/V cache, on the device.
//
//   paged_update       block tables, slot map and positions of one step, built
//                      from the requests' lengths; pages come from and go back
//                      to a free list.  The paged counterpart of
//                      initialize_past_key_values / the cache-length rollback
//                      (kv_cache.py:72-165, std_qwen25vl.py:923-929).
//   paged_rope_append  RoPE of the new tokens' q and k and the K/V append by
//                      slot: the paged sibling of rope_append
//                      (modeling_qwen2_5_vl.py:690-732, kv_cache.py:54-69).
#include "common.cuh"

namespace stdb {

// ------------------------------ paged_update -------------------------------
// want_b = ceil((past_b + new_b) / page) pages for request b, which holds
// held_b of them.  Returned pages (held_b > want_b) are counted r = 0, 1, ... in
// request and block order, R in all, and page r is put at free[n_free + R-1-r];
// wanted pages are counted a = 0, 1, ... in the same order and page a comes from
// the top, free[n_free + R - 1 - a].  So a return undoes a take exactly, order
// included.  A request whose needs, added to those of the requests before it,
// pass n_free + R is refused (needing none is always granted); the granted ones
// that need pages are therefore a prefix in request order, and a is their plain
// prefix sum.
//
// One block: the work is three prefix sums over the requests and a few hundred
// page moves, all latency.  Prefix sums live in shared memory, and every later
// phase (returns, takes, tokens) is flat over its own items, each finding its
// request by bisection: the time does not depend on how the pages and tokens
// are spread over the requests.  Measured (from a graph): 3.1 us for 8 requests of
// 10 new tokens, 5.5 us for 256 requests with 8192 new tokens.
struct PagedUpdateParams {
  const int32_t* past;
  const int32_t* fresh;
  int32_t* table;  // [B, width]
  int32_t* n_blocks;
  int32_t* free_pages;
  int32_t* n_free;
  int B, width, page, num_pages, max_tokens;
  int32_t* cu_q;
  int32_t* kv_lens;
  int32_t* slots;
  int32_t* positions;
  int32_t* admitted;
  int tokens_here;  // 1: this kernel also writes slots and positions
};

// Last index i in [0, n) with pre[i] <= x (pre ascending, pre[0] <= x): the
// owner of item x when pre are exclusive prefix sums, empty owners skipped.
template <typename Ptr>
STD_DEV int paged_owner(Ptr pre, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Slot and position of a token at position pos of a request whose table row is
// `row`.  A page id outside the pool gives slot -1.
STD_DEV void paged_token(const PagedUpdateParams& p, const int32_t* row, int pos, int t) {
  int slot = -1;
  const int id = row[pos / p.page];
  if (id >= 0 && id < p.num_pages)
    slot = id * p.page + pos % p.page;
  else
    std_set_error(STD_DEVERR_BOUNDS);
  p.slots[t] = slot;
  p.positions[t] = pos;
}

__global__ void __launch_bounds__(1024) paged_update_kernel(const PagedUpdateParams p) {
  pdl_wait();
  extern __shared__ int32_t s_dyn[];
  int32_t* s_cu = s_dyn;             // [B + 1] exclusive sums of the new tokens
  int32_t* s_take = s_cu + p.B + 1;  // [B] exclusive sums of the pages needed
  int32_t* s_back = s_take + p.B;    // [B] exclusive sums of the pages returned
  int32_t* s_past = s_back + p.B;    // [B] past length; -1: refused
  __shared__ long long s_part[3][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nt = blockDim.x, nw = nt >> 5;
  int n_free = *p.n_free;
  if (n_free < 0 || n_free > p.num_pages) {
    if (tid == 0) std_set_error(STD_DEVERR_BOUNDS);
    n_free = n_free < 0 ? 0 : p.num_pages;
  }
  const long long room = static_cast<long long>(p.width) * p.page;
  long long run[3] = {0, 0, 0};  // new tokens, pages needed, pages returned so far
  for (int b0 = 0; b0 < p.B; b0 += nt) {
    const int b = b0 + tid;
    long long v[3] = {0, 0, 0};
    int past = -1;
    if (b < p.B) {
      past = p.past[b];
      const int fresh = p.fresh[b], held = p.n_blocks[b];
      v[0] = fresh > 0 ? fresh : 0;
      const long long len = static_cast<long long>(past) + fresh;
      if (past < 0 || fresh < 0 || len > room || held < 0 || held > p.width) {
        std_set_error(STD_DEVERR_LENGTH);
        past = -1;
      } else {
        const int want = static_cast<int>((len + p.page - 1) / p.page);
        if (want > held) v[1] = want - held;
        if (want < held) v[2] = held - want;
      }
    }
    long long inc[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      inc[i] = v[i];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, inc[i], o);
        if (lane >= o) inc[i] += u;
      }
      if (lane == 31) s_part[i][warp] = inc[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      long long part = lane < nw ? s_part[i][lane] : 0;  // the warps' sums, scanned by every warp
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, part, o);
        if (lane >= o) part += u;
      }
      const long long before = __shfl_sync(0xffffffffu, part, warp > 0 ? warp - 1 : 0);
      inc[i] += run[i] + (warp > 0 ? before : 0);
      run[i] += __shfl_sync(0xffffffffu, part, 31);
    }
    if (b < p.B) {
      // sums beyond int32 are reported below and cut here so that every index stays
      // in range; a request's own tokens are read from `fresh`, not from these
      s_cu[b] = static_cast<int>(min(inc[0] - v[0], 0x7fffffffll));
      s_take[b] = static_cast<int>(inc[1] - v[1]);
      s_back[b] = static_cast<int>(inc[2] - v[2]);
      s_past[b] = past;
    }
    __syncthreads();
  }
  const int back = static_cast<int>(run[2]);
  if (tid == 0) {
    s_cu[p.B] = static_cast<int>(min(run[0], 0x7fffffffll));
    // more tokens than the outputs hold (cu_q, or slots and positions if there are
    // any), or more pages returned than exist
    if (run[0] > (p.max_tokens > 0 ? p.max_tokens : 0x7fffffffll)) std_set_error(STD_DEVERR_LENGTH);
    if (static_cast<long long>(n_free) + back > p.num_pages) std_set_error(STD_DEVERR_BOUNDS);
  }
  // returns: page r of the whole step, ids cleared from the table (unsigned: `back` may
  // come near 2^31 where n_blocks claims more pages than there are)
  for (uint32_t u = tid; u < static_cast<uint32_t>(back); u += nt) {
    const int r = static_cast<int>(u);
    const int b = paged_owner(s_back, p.B, r);
    const int total = (b + 1 < p.B ? s_back[b + 1] : back) - s_back[b];
    int32_t* at = p.table + static_cast<size_t>(b) * p.width + (p.n_blocks[b] - total + (r - s_back[b]));
    const long long to = static_cast<long long>(n_free) + back - 1 - r;
    if (to < p.num_pages) p.free_pages[to] = *at;
    *at = -1;
  }
  const int pool = static_cast<int>(min(static_cast<long long>(n_free) + back, static_cast<long long>(p.num_pages)));
  __syncthreads();
  // takes: the granted requests that need pages are those whose inclusive sum
  // stays within the pool
  const int need = static_cast<int>(run[1]);
  int taken = need;
  if (need > pool) {  // the first request that does not fit ends the prefix
    const int b = paged_owner(s_take, p.B, pool);  // its pages straddle, or begin at, the pool's end
    taken = s_take[b];
  }
  for (int a = tid; a < taken; a += nt) {
    const int b = paged_owner(s_take, p.B, a);
    const int i = p.n_blocks[b] + (a - s_take[b]);
    p.table[static_cast<size_t>(b) * p.width + i] = p.free_pages[pool - 1 - a];
  }
  __syncthreads();  // table complete, n_blocks read
  for (int b = tid; b < p.B; b += nt) {
    const int past = s_past[b], needs = (b + 1 < p.B ? s_take[b + 1] : need) - s_take[b];
    const bool ok = past >= 0 && (needs == 0 || s_take[b] + needs <= taken);
    const long long len = static_cast<long long>(past) + p.fresh[b];
    p.cu_q[b] = s_cu[b];
    p.kv_lens[b] = ok ? static_cast<int>(len) : 0;
    p.admitted[b] = ok ? 1 : 0;
    if (ok) p.n_blocks[b] = static_cast<int>((len + p.page - 1) / p.page);
    if (!ok) s_past[b] = -1;
  }
  if (tid == 0) {
    p.cu_q[p.B] = s_cu[p.B];
    *p.n_free = pool - taken;
  }
  if (p.tokens_here == 0) return;
  __syncthreads();
  const int total = s_cu[p.B];
  for (int t = tid; t < p.max_tokens; t += nt) {
    const int b = t < total ? paged_owner(s_cu, p.B, t) : -1;
    if (b < 0 || s_past[b] < 0) {
      p.slots[t] = -1;
      p.positions[t] = -1;
    } else {
      paged_token(p, p.table + static_cast<size_t>(b) * p.width, s_past[b] + (t - s_cu[b]), t);
    }
  }
}

// Slots and positions from the finished tables, one thread per token, for steps
// with many tokens.
__global__ void __launch_bounds__(256) paged_tokens_kernel(const PagedUpdateParams p) {
  pdl_wait();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= p.max_tokens) return;
  const int b = t < p.cu_q[p.B] ? paged_owner(p.cu_q, p.B, t) : -1;
  if (b < 0 || p.admitted[b] == 0) {
    p.slots[t] = -1;
    p.positions[t] = -1;
  } else {
    paged_token(p, p.table + static_cast<size_t>(b) * p.width, p.kv_lens[b] - p.fresh[b] + (t - p.cu_q[b]), t);
  }
}

// ---------------------------- paged_rope_append ----------------------------
// y_lo = lo cos - hi sin, y_hi = hi cos + lo sin over the two halves of each q
// and k head, in fp32 and rounded once (the contiguous rope_append rounds every
// product to bf16, as the reference's bf16 arithmetic does); v is copied.  A
// thread handles 8 + 8 elements (16-byte loads and stores), a block one token.  The
// row's loads go out before its position is there (28.6 -> 25.7 us).  HBM: 8192
// tokens of 28 + 8 heads 25.7 us = 6.0 TB/s read and written (0.91 of the measured
// copy); 80 tokens 1.6 us.
struct PagedAppendParams {
  const void* qkv;  // [T, (Hq + 2 Hkv) * D]
  const int32_t* positions;
  const int32_t* slots;
  const void* cos_t;  // [max_pos, D / 2]
  const void* sin_t;
  void* q_out;    // [T, Hq, D]
  void* k_pages;  // [num_pages, Hkv, page, D]
  void* v_pages;
  int Hq, Hkv, D, max_pos, page;
  long long total_slots;  // num_pages * page
};

STD_DEV float2 pair_to_float(__nv_bfloat162 v) { return __bfloat1622float2(v); }
STD_DEV float2 pair_to_float(__half2 v) { return __half22float2(v); }
template <typename T>
struct PairOf;
template <>
struct PairOf<__nv_bfloat16> {
  typedef __nv_bfloat162 type;
  static STD_DEV __nv_bfloat162 make(float a, float b) { return __floats2bfloat162_rn(a, b); }
};
template <>
struct PairOf<__half> {
  typedef __half2 type;
  static STD_DEV __half2 make(float a, float b) { return __floats2half2_rn(a, b); }
};
template <typename T>
STD_DEV T to_type(float v);
template <>
STD_DEV __nv_bfloat16 to_type<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
STD_DEV __half to_type<__half>(float v) { return __float2half_rn(v); }
template <typename T>
STD_DEV uint32_t pack_pair(float a, float b) {
  const typename PairOf<T>::type v = PairOf<T>::make(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// A load that stays where it is written.
STD_DEV uint4 ld_global_16b(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

template <typename T>
__global__ void __launch_bounds__(512) paged_append_kernel(const PagedAppendParams p) {
  typedef typename PairOf<T>::type Pair;
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x;
  int pos = p.positions[row];
  const int slot = p.slots[row];
  const bool slot_ok = slot >= 0 && slot < p.total_slots;
  const int heads = p.Hq + 2 * p.Hkv, half = p.D / 2, per_head = half / 8;
  const T* src = static_cast<const T*>(p.qkv) + static_cast<size_t>(row) * heads * p.D;
  for (int i = threadIdx.x; i < heads * per_head; i += blockDim.x) {
    const int h = i / per_head, c = (i % per_head) * 8;
    // (on their way while the position is)
    const uint4 lo = ld_global_16b(src + h * p.D + c), hi = ld_global_16b(src + h * p.D + half + c);
    if (pos < 0) return;  // no token in this row
    if (i == 0 && (slot >= p.total_slots || pos >= p.max_pos)) std_set_error(STD_DEVERR_BOUNDS);
    if (pos >= p.max_pos) pos = p.max_pos - 1;
    T* dst;
    if (h < p.Hq) {
      dst = static_cast<T*>(p.q_out) + (static_cast<size_t>(row) * p.Hq + h) * p.D;
    } else {
      if (!slot_ok) continue;
      const bool is_k = h < p.Hq + p.Hkv;
      const size_t head = static_cast<size_t>(slot / p.page) * p.Hkv + (h - p.Hq - (is_k ? 0 : p.Hkv));
      dst = static_cast<T*>(is_k ? p.k_pages : p.v_pages) + (head * p.page + slot % p.page) * p.D;
      if (!is_k) {
        *reinterpret_cast<uint4*>(dst + c) = lo;
        *reinterpret_cast<uint4*>(dst + half + c) = hi;
        continue;
      }
    }
    const uint4 cv = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.cos_t) + static_cast<size_t>(pos) * half + c);
    const uint4 sv = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.sin_t) + static_cast<size_t>(pos) * half + c);
    const uint32_t *pl = &lo.x, *ph = &hi.x, *pc = &cv.x, *ps = &sv.x;
    uint4 yl, yh;
    uint32_t *ol = &yl.x, *oh = &yh.x;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 a = pair_to_float(*reinterpret_cast<const Pair*>(pl + k));
      const float2 b = pair_to_float(*reinterpret_cast<const Pair*>(ph + k));
      const float2 cs = pair_to_float(*reinterpret_cast<const Pair*>(pc + k));
      const float2 sn = pair_to_float(*reinterpret_cast<const Pair*>(ps + k));
      ol[k] = pack_pair<T>(fmaf(a.x, cs.x, -(b.x * sn.x)), fmaf(a.y, cs.y, -(b.y * sn.y)));
      oh[k] = pack_pair<T>(fmaf(b.x, cs.x, a.x * sn.x), fmaf(b.y, cs.y, a.y * sn.y));
    }
    *reinterpret_cast<uint4*>(dst + c) = yl;
    *reinterpret_cast<uint4*>(dst + half + c) = yh;
  }
}

}  // namespace stdb

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
static bool paged_page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128 || page == 256; }
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A call's arrays: true when one that it writes shares bytes with any other.
struct PagedArray {
  const void* p;
  unsigned long long bytes;
  bool written;
};
template <int N>
static bool paged_overlap(const PagedArray (&a)[N]) {
  for (int i = 0; i < N; ++i)
    for (int j = 0; j < i; ++j) {
      if ((!a[i].written && !a[j].written) || a[i].bytes == 0 || a[j].bytes == 0) continue;
      const unsigned long long x = reinterpret_cast<uintptr_t>(a[i].p), y = reinterpret_cast<uintptr_t>(a[j].p);
      if (x < y + a[j].bytes && y < x + a[i].bytes) return true;
    }
  return false;
}

extern "C" int std_paged_update(const int32_t* past_lens, const int32_t* new_lens, int32_t* block_table,
                                int32_t* n_blocks, int32_t* free_pages, int32_t* n_free, int B, int max_blocks,
                                int page_size, int num_pages, int max_tokens, int32_t* cu_q, int32_t* kv_lens,
                                int32_t* slots, int32_t* positions, int32_t* admitted, void* stream) {
  if (B <= 0 || B > STD_PAGED_MAX_REQUESTS || max_blocks <= 0 || num_pages <= 0 || max_tokens < 0 ||
      !paged_page_ok(page_size))
    return 1;
  // int32 indexes: table entries, slots and positions
  if (static_cast<long long>(B) * max_blocks > 0x7fffffffll ||
      static_cast<long long>(num_pages) * page_size > 0x7fffffffll ||
      static_cast<long long>(max_blocks) * page_size > 0x7fffffffll)
    return 1;
  if (past_lens == nullptr || new_lens == nullptr || block_table == nullptr || n_blocks == nullptr ||
      free_pages == nullptr || n_free == nullptr || cu_q == nullptr || kv_lens == nullptr || admitted == nullptr)
    return 1;
  if (max_tokens > 0 && (slots == nullptr || positions == nullptr)) return 1;
  const unsigned long long n = 4ull * B, nt = 4ull * max_tokens;
  if (paged_overlap<11>({{past_lens, n, false}, {new_lens, n, false}, {block_table, n * max_blocks, true},
                         {n_blocks, n, true}, {free_pages, 4ull * num_pages, true}, {n_free, 4, true}, {cu_q, n + 4, true},
                         {kv_lens, n, true}, {slots, nt, true}, {positions, nt, true}, {admitted, n, true}}))
    return 1;
  stdb::PagedUpdateParams p;
  p.past = past_lens;
  p.fresh = new_lens;
  p.table = block_table;
  p.n_blocks = n_blocks;
  p.free_pages = free_pages;
  p.n_free = n_free;
  p.B = B;
  p.width = max_blocks;
  p.page = page_size;
  p.num_pages = num_pages;
  p.max_tokens = max_tokens;
  p.cu_q = cu_q;
  p.kv_lens = kv_lens;
  p.slots = slots;
  p.positions = positions;
  p.admitted = admitted;
  // Few tokens' slots are written by the one block, many by a second kernel of many
  // blocks (8 requests: 256 tokens 3.2 us against 4.3, 1024 4.3 against 4.5, 4096
  // 6.4 against 4.4; 256 requests: 1024 tokens 4.7 against 5.4, 4096 7.6 against 5.4).
  p.tokens_here = max_tokens <= 1024 ? 1 : 0;
  const size_t smem = (4 * static_cast<size_t>(B) + 1) * 4;
  static SmemGrant grant;
  if (ensure_smem(stdb::paged_update_kernel, grant, smem) != 0) return 3;
  const int items = B > (p.tokens_here ? max_tokens : 0) ? B : max_tokens;
  const int threads = items >= 1024 ? 1024 : ((items < 128 ? 128 : items) + 31) / 32 * 32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (launch_pdl(stdb::paged_update_kernel, dim3(1), dim3(threads), smem, s, p) != cudaSuccess) return 4;
  if (!p.tokens_here &&
      launch_pdl(stdb::paged_tokens_kernel, dim3((max_tokens - 1) / 256 + 1), dim3(256), 0, s, p) != cudaSuccess)
    return 4;
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

extern "C" int std_paged_rope_append(const void* qkv, int T, int Hq, int Hkv, int D, int is_fp16,
                                     const int32_t* positions, const int32_t* slots, const void* cos_t,
                                     const void* sin_t, int max_pos, void* q_out, void* k_pages, void* v_pages,
                                     int num_pages, int page_size, void* stream) {
  if (T < 0 || Hq <= 0 || Hkv <= 0 || Hq > 4096 || Hkv > 4096 || (D != 64 && D != 128) || max_pos <= 0 ||
      num_pages <= 0 || !paged_page_ok(page_size))
    return 1;
  if (static_cast<long long>(num_pages) * page_size > 0x7fffffffll) return 1;
  if (T == 0) return 0;
  if (qkv == nullptr || positions == nullptr || slots == nullptr || cos_t == nullptr || sin_t == nullptr ||
      q_out == nullptr || k_pages == nullptr || v_pages == nullptr)
    return 1;
  if (!aligned16(qkv) || !aligned16(cos_t) || !aligned16(sin_t) || !aligned16(q_out) || !aligned16(k_pages) ||
      !aligned16(v_pages))
    return 1;
  const unsigned long long row = 2ull * D, pool = row * Hkv * num_pages * page_size;
  const bool in_place = T == 1 && q_out == qkv;  // (a thread writes what it has read)
  if (paged_overlap<8>({{qkv, in_place ? 0 : row * T * (Hq + 2 * Hkv), false}, {positions, 4ull * T, false},
                        {slots, 4ull * T, false}, {cos_t, row / 2 * max_pos, false}, {sin_t, row / 2 * max_pos, false},
                        {q_out, row * T * Hq, true}, {k_pages, pool, true}, {v_pages, pool, true}}))
    return 1;
  stdb::PagedAppendParams p;
  p.qkv = qkv;
  p.positions = positions;
  p.slots = slots;
  p.cos_t = cos_t;
  p.sin_t = sin_t;
  p.q_out = q_out;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.D = D;
  p.max_pos = max_pos;
  p.page = page_size;
  p.total_slots = static_cast<long long>(num_pages) * page_size;
  const int work = (Hq + 2 * Hkv) * (D / 16);
  const int threads = work >= 512 ? 512 : (work + 31) / 32 * 32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = is_fp16 ? launch_pdl(stdb::paged_append_kernel<__half>, dim3(T), dim3(threads), 0, s, p)
                                : launch_pdl(stdb::paged_append_kernel<__nv_bfloat16>, dim3(T), dim3(threads), 0, s, p);
  return e == cudaSuccess ? 0 : 4;
}
