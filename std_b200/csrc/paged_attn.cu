// paged_attn.cu -- attention of each request's new tokens over its paged K/V
// cache, on tcgen05 / TMEM: prompt chunks, verify blocks and single tokens, any
// mix of them in one launch.  The paged, ragged counterpart of
// modeling_qwen2_5_vl.py:1096-1133 (repeat_kv + F.sdpa with the causal mask of
// :65-101).
//
// Tiles.  The G = Hq / Hkv query heads of a KV head share its keys, so rows
// are (token, head of the group) pairs: row = t * G + g, TQ = floor(128 / G)
// whole tokens per 128-row tile.  An item is one KV head's span of up to 2 TQ
// tokens of one request: a pair of tiles that share every K/V block or, when at
// most TQ tokens are left, a single one.  Keys come in blocks of 128.
//   S = Q K^T     tcgen05.mma M=128, two halves of N=64 keys, Q and K from
//                 shared memory
//   P = exp2(S * scale * log2e - m), 16 bits, each half written over its S in TMEM
//   O += P V      tcgen05.mma with P as the A operand in TMEM, V MN-major
// Two softmax warpgroups each own a stream of steps with an S and an O of its
// own in TMEM: in a pair, stream s is tile s; in a single, stream s takes the
// blocks j = s mod 2 and the two accumulators are joined at the end.  Either way
// one stream's MMAs run while the other's softmax does.  The running maximum
// is raised lazily, when a block passes it by more than 2^8, so O is normally
// not touched between blocks.
//
// Few rows.  A single item of at most 32 rows (decoding: G rows) is computed
// transposed, keys on the 128 MMA rows and the query rows on N:
//   S^T = K Q^T    M=128 (keys) N=16 or 32, both operands in shared memory
//   O^T += V^T P^T M=128 (head dims), A = V MN-major, B = P^T in shared memory
// A softmax thread then owns one key and N rows, so a block costs N exponentials
// a thread on all 128 threads instead of 128 on the few threads that have a row,
// and the MMAs are N wide instead of 128.
//
// Split.  One CTA per SM.  The items' costs (blocks, weighted) are laid end to
// end and cut into equal shares, one per CTA, at block boundaries; a CTA reads
// the lengths and finds its share itself, so nothing is planned on the host and
// a captured graph follows the lengths.  An item that a cut divides leaves
// fp32 (O, m, l) partials, at most two per CTA, which paged_merge_kernel joins
// in CTA order: no atomics, the same bits for the same inputs.  (Where the cuts
// fall depends on the whole batch, so a request's last bits may too.)
//
// Pages.  A block's pages are fetched by the lanes of one warp, one TMA copy
// per page (or per 128 tokens of a larger page): a 4-D view (64 columns, 8
// rows, D / 64 halves, row groups) puts both halves of 8 rows into adjacent
// 1 KB swizzle atoms, so pages land side by side whatever their size and a tile
// of 128 rows has constant strides.  Only pages with a visible key are read.
// Rows past the last visible key may hold anything: their scores are replaced,
// not added to, and their V rows are cleared before the product.
//
// What bounds it, and what was measured (B200, replayed from a graph; bf16, 28
// query heads on 4 key heads, D 128 unless said).  Long prompts: the softmax warps
// and power; a 2048-token chunk over 31K keys 825 us = 1130 TFLOP/s in a short run
// (0.69 of cuBLAS's burst; 3200 cycles a block of a pair, of which a softmax warp
// works 2900 and the MMAs need 2560; 1.45 GHz) and 924 to 945 us = 990 to 1010 TFLOP/s
// in a long one (0.72 to 0.74 of what cuBLAS sustains under the power cap; 1.3 GHz), an
// 8192-token prompt 508 and 518 to 528 us.  S in halves costs 1.5 x the shared-memory reads of N=128 but keeps
// a half of S ready while the other is multiplied: 866 us with one S of 128 columns a
// step from one issuing thread, 815 with halves and a thread per stream (at the same
// clock, before the sums of O were divided).
// Decoding: HBM; 64 requests of 100 to 8000 keys 85 us = 5.7 TB/s (0.88 of the
// measured copy), one request of 131K keys 50 us = 5.4 TB/s, 8 verify blocks of
// 10 tokens over 33K keys 102 us = 5.3 TB/s (111 in a long run); untransposed, the
// first two took 118 and 67 us, bound by one warp's softmax of 128 columns for 7 live
// rows.  Short contexts: latency, one token and 200 keys 7.6 us with a table for up to
// 512 keys and 8.8 with a wider one, whose call has the merge behind it (half of it
// finding the share, 2 us, and the first page, key and score, 2 us); 8 single tokens
// over 1025 keys 15.0 us whatever the table's width.
#include "common.cuh"

#include <type_traits>

namespace stdb {

constexpr int PA_CTAS = 148;     // one CTA per SM
constexpr int PA_THREADS = 384;  // 2 softmax warpgroups; TMA, two MMA and a scheduler warp
constexpr int PA_BN = 128;       // keys per block
constexpr float PA_RESCALE = 8.0f;  // log2 units
// m is set this far below the maximum, in log2 units: P is 2^top there and stays below
// 2^(top + PA_RESCALE), for fp16 below its 65504.  Weights under 2^(-25 - top) of the
// largest are lost in fp16, which many keys of small weight beside a heavy one notice
// (2^17 keys of 2^-25 each: 0.4 % of the row with top 0).  bf16 has the range of a float.
template <typename T>
constexpr float PA_TOP = std::is_same<T, __half>::value ? 7.0f : 0.0f;
// Cost of a block in a single and in a pair (measured: 2000 to 2400 cycles and
// 3200 to 3700); an item costs PA_OVER blocks more (its queries, first keys and output).
constexpr int PA_W1 = 3, PA_W2 = 5, PA_OVER = 3;
// An item of at most this many blocks is not divided but goes where it begins: a cut
// would cost a partial and the merge (2 us) to save at most two blocks (2 us), and
// calls whose tables allow no longer item (up to 512 keys) need no merge launch: one
// token and 200 keys 7.6 us, 8.8 with a table of 2048 pages of 16.
constexpr int PA_WHOLE = 4;

// Shared memory: two query slots and a ring of K/V blocks.  A slot holds a
// 128-row Q tile (halves of 64 columns, 16 KB apart), or, for few rows, a 32-row
// one (halves 8 KB apart) in its first 16 KB and P^T of stream = slot (a 128-byte
// row per key) in its last 16 KB.
constexpr uint32_t PA_SLOT = 32768, PA_PT = 16384;
template <int D>
struct PagedTile {
  static constexpr uint32_t kv_bytes = PA_BN * D * 2;
  static constexpr int stages = D == 128 ? 5 : 8;
  static constexpr uint32_t smem = 2 * PA_SLOT + stages * kv_bytes + 1024;
};
// Most rows of an item that is computed transposed.  Up to 64 it would still pay by
// itself, but the registers of that variant (64 scores and 64 sums a thread) made
// the compiler spill in the whole-tile softmax beside it: 8 verify blocks over 33K
// keys 105 -> 99 us, an 8192-token prompt 505 -> 455 us without it.
constexpr int PA_FEW = 32;
// Every 3rd pair of exponentials goes to the FMA pipe (the 2048-token chunk in a
// long run: none 972 us, every 8th 950, 4th 947, 3rd 942; every 2nd is slower again).
constexpr int PA_POLY = 3;

// Steps of a stream after which its O is added to a sum in global memory (the slot
// that the item's partial takes, or would take) and started anew.  The tensor core
// cuts its 32-bit sums off instead of rounding them, so a sum of same-signed values
// lags by about 2^-24 of itself with each 16 keys: without this 4.5e-3 over 2^20 keys
// in one CTA, more than half a step of bf16; with it below 3e-4 at any length (8
// verify blocks over 33K keys, which never come here, 1 % slower for the longer code,
// the 2048-token chunk the same).
constexpr int PA_FLUSH = 512;

// What a CTA leaves for the merge about the item that its share ends inside.
struct PagedSplit {
  int first_cta, last_cta;  // where the item's pieces are; last < 0: nothing to merge
  int token0;    // first token row of the item
  int tokens;
  int kvh;
};

struct PagedAttnParams {
  const int32_t* table;  // [B, width]
  const int32_t* cu_q;   // [B + 1]
  const int32_t* kv_lens;
  int T, B, width, page_log2, num_pages, Hq, Hkv, G, TQ, TQ_few, causal;  // TQ_few = floor(32 / G)
  float scale_log2;
  void* out;   // [T, Hq, D]
  int out_32b;    // out is 32-byte aligned
  int unit_log2;  // of the costs
  float* lse;  // [T, Hq], may be null
  float* ws_o;        // [2 * PA_CTAS][256][D]
  float2* ws_ml;      // [2 * PA_CTAS][256]
  PagedSplit* splits;  // [PA_CTAS]
};

// One request's place from its raw entries: token rows [q0, q0 + n), kv keys.
// Lengths that do not fit the tensors are cut; false: they were.
STD_DEV bool paged_request(const PagedAttnParams& p, int q0, int q1, int& kv, int& n) {
  const int room = p.width << p.page_log2;
  const bool fit = q0 >= 0 && q1 <= p.T && q1 >= q0 && kv >= 0 && kv <= room;
  n = q0 < 0 || q1 > p.T || q1 < q0 ? 0 : q1 - q0;
  kv = kv < 0 ? 0 : (kv > room ? room : kv);
  return fit;
}
// Inclusive sums over the warp's lanes.
STD_DEV int warp_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// Item i of a request: its tokens, the last key that any of them sees (+1),
// its blocks and what one costs.
STD_DEV void paged_item(const PagedAttnParams& p, int n, int kv, int i, int& t0, int& nt, int& limit, int& nb, int& w) {
  t0 = i * 2 * p.TQ;
  nt = min(2 * p.TQ, n - t0);
  limit = p.causal ? max(0, kv - n + t0 + nt) : kv;
  nb = max(1, (limit + PA_BN - 1) / PA_BN);
  w = nt > p.TQ ? PA_W2 : PA_W1;
}
// Costs fit 32 bits: the host picks the unit, 2^unit_log2 (1 unless the lengths
// that the tensors allow are extreme).
STD_DEV int paged_item_cost(const PagedAttnParams& p, int n, int kv, int i) {
  int t0, nt, limit, nb, w;
  paged_item(p, n, kv, i, t0, nt, limit, nb, w);
  return ((nb + PA_OVER) * w + (1 << p.unit_log2) - 1) >> p.unit_log2;
}
// The first block at or after cost x of an item: block j lies at (j + PA_OVER) w.
STD_DEV int paged_cut(const PagedAttnParams& p, int x, int w) {
  x <<= p.unit_log2;
  return max(0, (w == PA_W1 ? (x + PA_W1 - 1) / PA_W1 : (x + PA_W2 - 1) / PA_W2) - PA_OVER);
}

// A piece as the other warps see it: nblk blocks from block j0 of one item.
struct PagedPiece {
  int b, h;
  int token0;  // first token row
  int tokens;  // of the item; > TQ: a pair
  int limit;   // last key that any of them sees, + 1
  int first;   // causal: keys that token t of the item sees = first + t
  int j0, nblk;  // nblk 0: no more pieces
  int slot;      // partial's slot, or -1: the item is whole
};
constexpr int PA_PIECES = 4;  // ring of pieces in shared memory

// A CTA's walk over the pieces of its share, by a whole warp.
struct PagedWalk {
  int b, h, i;         // current item
  int q0, n, kv, items;
  int skip;            // cost of the item that earlier CTAs did
  int rem;             // cost left in this CTA's share
  // the current piece
  int t0, nt, limit, nb, w, j0, j1;
  int cut;             // cost of the item up to the end of this piece

  STD_DEV void request(const PagedAttnParams& p) {
    q0 = __ldg(p.cu_q + b);
    kv = __ldg(p.kv_lens + b);
    paged_request(p, q0, __ldg(p.cu_q + b + 1), kv, n);
    items = (n + 2 * p.TQ - 1) / (2 * p.TQ);
  }
  // On to the next request with tokens, 32 at a time, a request per lane (a batch
  // of fixed size may be idle for the most part: 8192 requests, two at each end with
  // tokens: 231 us, and 1583 when they were passed one by one).  False: there is none.
  STD_DEV bool next_request(const PagedAttnParams& p) {
    const int lane = threadIdx.x & 31;
    for (++b; b < p.B; b += 32) {
      int q0_ = 0, kv_ = 0, n_ = 0;
      if (lane < p.B - b) {
        q0_ = __ldg(p.cu_q + b + lane);
        kv_ = __ldg(p.kv_lens + b + lane);
        paged_request(p, q0_, __ldg(p.cu_q + b + lane + 1), kv_, n_);
      }
      const uint32_t some = __ballot_sync(0xffffffffu, n_ > 0);
      if (some != 0) {
        const int src = __ffs(some) - 1;
        b += src;
        q0 = __shfl_sync(0xffffffffu, q0_, src);
        kv = __shfl_sync(0xffffffffu, kv_, src);
        n = __shfl_sync(0xffffffffu, n_, src);
        items = (n + 2 * p.TQ - 1) / (2 * p.TQ);
        return true;
      }
    }
    return false;
  }
  // Advance to the next non-empty piece; false at the end of the share.
  STD_DEV bool next(const PagedAttnParams& p) {
    while (rem > 0) {
      if (i >= items) {  // next head, then next request
        i = 0;
        if (++h >= p.Hkv) {
          h = 0;
          if (!next_request(p)) return false;
        }
      }
      paged_item(p, n, kv, i, t0, nt, limit, nb, w);
      const int cost = paged_item_cost(p, n, kv, i);
      const int end = min(cost, skip + rem);
      j0 = nb <= PA_WHOLE ? (skip > 0 ? nb : 0) : paged_cut(p, skip, w);
      j1 = nb <= PA_WHOLE ? nb : min(nb, paged_cut(p, end, w));
      rem -= end - skip;
      skip = 0;
      cut = end;
      ++i;
      if (j1 > j0) return true;
    }
    return false;
  }
};

// Instruction descriptor for operands of type T (format 1 = bf16, 0 = fp16).
template <typename T>
__host__ __device__ constexpr uint32_t paged_idesc(int M, int N, int a_mn_major, int b_mn_major) {
  return idesc_bf16_f32(M, N, a_mn_major, b_mn_major) &
         (std::is_same<T, __half>::value ? ~((1u << 7) | (1u << 10)) : ~0u);
}
// MMA columns for `rows` few rows.
STD_DEV int paged_few_cols(int rows) { return rows <= 16 ? 16 : 32; }

STD_DEV void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// Static shared memory of a CTA with an ST-stage ring.
template <int ST>
struct PagedShared {
  // mbarriers, by the arrivals that complete a phase
  static constexpr int BARS_1 = 14 + ST + PA_PIECES, BARS_2 = BARS_1 + ST, BARS_3 = BARS_2 + 2,
                       BARS_4 = BARS_3 + 8, BARS = BARS_4 + PA_PIECES;
  union {
    uint64_t bars[BARS];
    struct {
      // one
      uint64_t bar_q_full[2];                  // query slots
      uint64_t bar_s[2][2], bar_o[2];          // per stream: S's halves there, O complete
      uint64_t bar_half[2];                    // whole tiles: the product of an item's last first half done
      uint64_t bar_tail[2], bar_end[2];        // a tail's V there; all MMAs done
      uint64_t bar_full[ST];                   // K/V ring
      uint64_t bar_piece[PA_PIECES];
      // two: both MMA threads have seen the load, and its readers are done
      uint64_t bar_empty[ST];
      // three: both MMA threads have seen the tile, and its reader is done
      uint64_t bar_q_empty[2];
      // four (a stream's warps)
      uint64_t bar_p[2], bar_p2[2];   // P's halves there
      uint64_t bar_join, bar_joined;  // a single's two streams
      uint64_t bar_group[2];          // few rows: the four warps of a stream
      // eleven (the warps that read a piece)
      uint64_t bar_taken[PA_PIECES];
    };
  };
  // A single's statistics, of one use at a time: whole tiles hand them from
  // stream 1 to stream 0, few rows keep theirs here.  A stream's warps write the
  // next piece's only after a barrier that all readers of the last have passed.
  union {
    struct {
      float m[128], l[128];
    };
    struct {
      alignas(16) float ref[2][PA_FEW];    // m of each stream and row; the streams' weights at the join
      alignas(16) float up[2][PA_FEW];     // by how much m was raised last
    };
  };
  float m_sum[2][PA_FEW];  // few rows: m of each stream's sum in global memory
  alignas(16) int flag[2][2][4];  // few rows: a vote per warp, by step parity
  int open[2];                    // few rows: some row's m is not set yet
  PagedPiece piece[PA_PIECES];
  uint32_t tmem;
};

STD_DEV void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
STD_DEV void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
STD_DEV void tmem_ld4(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr)
               : "memory");
}
template <int N>
STD_DEV void tmem_ld_cols(uint32_t taddr, uint32_t* r) {
  if constexpr (N == 16) {
    tmem_ld16(taddr, r);
  } else {
#pragma unroll
    for (int c = 0; c < N / 32; ++c) tmem_ld32(taddr + 32 * c, r + 32 * c);
  }
}
// One thread of a converged warp, the same one each time.  Behind this predicate
// (not behind lane == 0) the compiler knows that a single thread runs and feeds
// tcgen05.mma its uniform registers directly; otherwise it serialises over
// possible threads, ~170 cycles an MMA.
STD_DEV bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
// 32 bytes: one store of a whole sector when the address is 32-byte aligned.
STD_DEV void st_global_32b(void* p, const uint32_t* r, bool aligned) {
  if (aligned)
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(r[0], r[1], r[2], r[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(r[4], r[5], r[6], r[7]);
  }
}
// Two floats in one 64-bit register, for the paired FMA and add.
STD_DEV uint64_t f2_make(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
STD_DEV float2 f2_split(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
STD_DEV uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
STD_DEV uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
STD_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// (NaN if one of them is)
STD_DEV float max2_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^y for two y <= 127 on the FMA and integer pipes, to spare the SFU (16
// results a cycle and SM): y = n + f with n whole and |f| <= 1/2, 2^f = 1 + f q(f)
// with q the degree-4 polynomial that interpolates (2^f - 1) / f at the Chebyshev
// nodes of [-1/2, 1/2] (off by at most 2.1e-7, 2.6e-7 as rounded here), n added
// to the exponent.  At and below -127 (masked: -inf) the sum is exactly 0, since
// 2^0 is exactly 1 here; between that and -126 a number below 2^-126.  A NaN gives
// FLT_MAX: n is added to the bits of a NaN.
STD_DEV float2 ex2_fma2(uint64_t y2) {
  float2 y = f2_split(y2);
  y.x = max2_nan(y.x, -127.f);
  y.y = max2_nan(y.y, -127.f);
  const float MAGIC = 12582912.f;  // 1.5 * 2^23: adding it leaves round(y) in the low bits
  const uint64_t v = f2_make(y.x, y.y);
  const uint64_t t = f2_add(v, f2_make(MAGIC, MAGIC));
  const uint64_t n = f2_add(t, f2_make(-MAGIC, -MAGIC));
  const uint64_t f = f2_fma(n, f2_make(-1.f, -1.f), v);
  uint64_t r = f2_make(1.338130254e-03f, 1.338130254e-03f);
  r = f2_fma(r, f, f2_make(9.666368515e-03f, 9.666368515e-03f));
  r = f2_fma(r, f, f2_make(5.550381014e-02f, 5.550381014e-02f));
  r = f2_fma(r, f, f2_make(2.402234904e-01f, 2.402234904e-01f));
  r = f2_fma(r, f, f2_make(6.931471806e-01f, 6.931471806e-01f));
  r = f2_fma(r, f, f2_make(1.f, 1.f));
  const float2 e = f2_split(r), k = f2_split(t);
  float2 out;
  out.x = __uint_as_float(__float_as_uint(e.x) + (__float_as_uint(k.x) << 23));
  out.y = __uint_as_float(__float_as_uint(e.y) + (__float_as_uint(k.y) << 23));
  return out;
}

// Clears the V rows of a tail that no query sees, up to the multiple of 16 at
// which the products stop (rows last .. of the stage sV), by a stream's 128 threads.
template <int D>
STD_DEV void paged_clear_tail(uint8_t* sV, int last, int thread) {
  constexpr int HALVES = D / 64;
  for (int i = thread; i < (16 - (last & 15)) * HALVES * 8; i += 128) {
    const int r = last + i / (HALVES * 8), ch = i % (HALVES * 8);
    *reinterpret_cast<uint4*>(sV + (r >> 3) * (HALVES * 1024) + (ch >> 3) * 1024 + (r & 7) * 128 + (ch & 7) * 16) =
        make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
}

// A stream's O of whole tiles and its row's sum in global memory: sum = f sum + O,
// O = 0 (begin: there is no sum yet), f = 2^(m of the sum - m of O); or, to end with,
// O += f sum.  For a warp whose products are at rest.  (A call: inlined, it cost the
// loops around it 1 %.)
template <int D>
__device__ __noinline__ void paged_flush(uint32_t tO, float* sum, float f, bool begin, bool end) {
  tc_fence_after();
  uint32_t o[16];
#pragma unroll 1
  for (int c = 0; c < D; c += 16) {
    tmem_ld16(tO + c, o);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      float4* at = reinterpret_cast<float4*>(sum + c + j);
      float4 v = make_float4(__uint_as_float(o[j]), __uint_as_float(o[j + 1]), __uint_as_float(o[j + 2]),
                             __uint_as_float(o[j + 3]));
      if (!begin) {
        const float4 a = *at;
        v = make_float4(fmaf(a.x, f, v.x), fmaf(a.y, f, v.y), fmaf(a.z, f, v.z), fmaf(a.w, f, v.w));
      }
      if (!end) {
        *at = v;
        v = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      o[j] = __float_as_uint(v.x), o[j + 1] = __float_as_uint(v.y);
      o[j + 2] = __float_as_uint(v.z), o[j + 3] = __float_as_uint(v.w);
    }
    tmem_st16(tO + c, o);
  }
  tmem_wait_st();
  tc_fence_before();
}

// Half a step of a whole tile's softmax: 64 columns of S to P, with the row's
// running m and l.  nvis: visible columns; cut: some row of the warp has fewer than
// all (known without a vote, which cost 1 % of an 8192-token prompt).  bar_next: the
// barrier (phase parity `next`) after which the stream's products issued so far are
// complete.  False when a wait ran out.
template <typename T, int D>
STD_DEV bool paged_softmax_half(uint32_t tS, uint32_t tO, float sc, int nvis, bool cut, float& m_run, float& l_run,
                                uint64_t* bar_next, uint32_t next) {
  constexpr int N = PA_BN / 2;
  uint32_t x[N];
  tmem_ld32(tS, x);
  tmem_ld32(tS + 32, x + 32);
  tmem_wait_ld();
  if (cut) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j >= nvis) x[j] = 0xff800000u;  // -inf
  }
  float m4[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) m4[c] = fmaxf(__uint_as_float(x[c]), __uint_as_float(x[4 + c]));
#pragma unroll
  for (int j = 8; j < N; j += 8)
#pragma unroll
    for (int c = 0; c < 4; ++c) m4[c] = max3(m4[c], __uint_as_float(x[j + c]), __uint_as_float(x[j + 4 + c]));
  const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
  const float m_c = fmaf(mx, sc, -PA_TOP<T>);  // scale > 0
  // (the exponent that P gets, not a difference of rounded ones: at 2^24 those are off by
  // 2, and a half would overflow)
  const bool need = m_run != -INFINITY && fmaf(mx, sc, -m_run) > PA_RESCALE + PA_TOP<T>;
  if (__any_sync(0xffffffffu, need)) {
    if (!__all_sync(0xffffffffu, mbar_wait(bar_next, next & 1))) return false;  // O at rest
    tc_fence_after();
    const float alpha = need ? exp2f(m_run - m_c) : 1.0f;
    uint32_t o[32];
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      tmem_ld32(tO + c * 32, o);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
      tmem_st32(tO + c * 32, o);
    }
    if (need) {
      l_run *= alpha;
      m_run = m_c;
    }
  }
  if (m_run == -INFINITY) m_run = m_c;
  // a row that has seen no key yet keeps P = 2^-inf = 0
  const float nm = m_run == -INFINITY ? 0.f : -m_run;
  const uint64_t sc2 = f2_make(sc, sc), nm2 = f2_make(nm, nm);
  uint64_t l2[2] = {f2_make(0.f, 0.f), f2_make(0.f, 0.f)};
  uint32_t pk[N / 2];
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    const uint64_t y = f2_fma(f2_make(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), sc2, nm2);
    float2 e;
    if (j % PA_POLY == PA_POLY - 1) {
      e = ex2_fma2(y);
    } else {
      e = f2_split(y);
      e.x = ex2_approx(e.x);
      e.y = ex2_approx(e.y);
    }
    l2[j & 1] = f2_add(l2[j & 1], f2_make(e.x, e.y));
    pk[j] = pack_pair<T>(e.x, e.y);
  }
  tmem_st32(tS, pk);
  tmem_wait_st();
  tc_fence_before();
  const float2 l = f2_split(f2_add(l2[0], l2[1]));
  // A NaN or +inf score makes its row NaN: it has left a NaN here or, through
  // ex2_fma2, FLT_MAX or more; sums of numbers stay below 2^31 2^(PA_RESCALE + 7).  (-inf has
  // weight 0, as a hidden key.)
  l_run += l.x + l.y;
  if (!(l_run < 1e30f)) l_run = NAN;
  return true;
}

// Combines N <= 32 values of each lane over the warp, halving the rows a lane keeps
// at each step; row `base` is left.
template <int N, typename Op>
STD_DEV int warp_reduce_rows(float* v, int lane, Op op) {
  int base = 0;
#pragma unroll
  for (int o = 16, half = N / 2; o > 0; o >>= 1, half >>= 1) {
    if (half > 0) {
      const bool up = (lane & o) != 0;
      base += up ? half : 0;
#pragma unroll
      for (int i = 0; i < (half > 0 ? half : 1); ++i) {
        const float give = up ? v[i] : v[i + half], keep = up ? v[i + half] : v[i];
        v[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, o));
      }
    } else {
      v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
    }
  }
  return base;
}

// A piece with few rows, for one warp of stream s (thread = key of the block,
// N >= the piece's rows columns).  ns, no, nj, ng: phases used so far of the
// stream's S, O, join and group barriers; bar_q_empty: its query slot's.  False
// when a wait ran out.  sV: the stage of the piece's last V; ntail: tails cleared.
//
// m (sh.ref) is set by the row's maximum over the first block that has one (a
// visible score above -inf: as a rule the first block) and raised when a P would pass
// 2^(PA_RESCALE + PA_TOP), on all four warps: they vote at every block.  Until it is set
// it is 0, the row's P, l and O are 0, and the vote is taken as given.
template <typename T, int D, int N, int ST>
STD_DEV bool paged_few_piece(const PagedAttnParams& p, const PagedPiece& piece, PagedShared<ST>& sh, uint8_t* sQ,
                             uint8_t* sV, uint32_t tS, uint32_t tO, int s, uint64_t* bar_q_empty, uint32_t& ntail,
                             uint32_t& ns, uint32_t& no, uint32_t& nj, uint32_t& ng) {
  const int tid = threadIdx.x, lane = tid & 31, w = (tid >> 5) & 3, key = tid & 127;
  const int rows = piece.tokens * p.G, steps = (piece.nblk - s + 1) >> 1;
  const float sc = p.scale_log2;
  uint8_t* row_p = sQ + s * PA_SLOT + PA_PT + key * 128;
  // [warp][row] values of a stream's warps, where P is not needed (P V done)
  auto red = [&](int stream, int warp, int n) -> float& {
    return reinterpret_cast<float*>(sQ + stream * PA_SLOT + PA_PT)[warp * PA_FEW + n];
  };
  auto group_sync = [&]() -> bool {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.bar_group[s]);
    return __all_sync(0xffffffffu, mbar_wait(&sh.bar_group[s], ng++ & 1));
  };
  float* sum = p.ws_o + (static_cast<size_t>(piece.slot < 0 ? 2 * blockIdx.x + 1 : piece.slot) * 256 + s * 128) * D + key;
  // paged_flush for O^T: thread = head dim, a column per row
  auto flush = [&](bool begin, bool end) -> bool {
    uint32_t o[16];
#pragma unroll 1
    for (int c = 0; c < N; c += 16) {
      tmem_ld16(tO + c, o);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float v = __uint_as_float(o[j]);
        if (key < D) {
          float* at = sum + static_cast<size_t>(c + j) * D;
          // (m only rises; set below 0 after the sum began, the sum is 0)
          if (!begin) v = fmaf(*at, ex2_approx(fminf(sh.m_sum[s][c + j] - sh.ref[s][c + j], 0.f)), v);
          if (!end) *at = v;
        }
        o[j] = end ? __float_as_uint(v) : 0u;
      }
      tmem_st16(tO + c, o);
    }
    tmem_wait_st();
    tc_fence_before();
    if (end) return true;
    if (!group_sync()) return false;
    if (key < N) sh.m_sum[s][key] = sh.ref[s][key];
    return true;  // (m_sum is read again after more group syncs)
  };
  float l[N];
#pragma unroll
  for (int n = 0; n < N; ++n) l[n] = 0.f;
  bool set = false, open = true;  // m of row `key` (key < N); some row's is not set yet
#pragma unroll 1
  for (int k = 0; k < steps; ++k, ++ns) {
    if (!__all_sync(0xffffffffu, mbar_wait(&sh.bar_s[s][0], ns & 1))) return false;
    tc_fence_after();
    if (k > 0 && k % PA_FLUSH == 0 && !flush(k == PA_FLUSH, false)) return false;  // (O is at rest)
    float y[N];
    tmem_ld_cols<N>(tS, reinterpret_cast<uint32_t*>(y));
    tmem_wait_ld();
    // this key is hidden from the tokens before it, hence from rows n < hide
    const int pos = (piece.j0 + 2 * k + s) * PA_BN + key;
    const int hide = pos >= piece.limit ? rows : (p.causal ? max(0, pos - piece.first + 1) * p.G : 0);
    float over = -INFINITY;
#pragma unroll
    for (int n = 0; n < N; n += 4) {
      const float4 m = k > 0 ? *reinterpret_cast<const float4*>(&sh.ref[s][n]) : make_float4(0.f, 0.f, 0.f, 0.f);
      y[n] = n >= hide && n < rows ? fmaf(y[n], sc, -m.x) : -INFINITY;
      y[n + 1] = n + 1 >= hide && n + 1 < rows ? fmaf(y[n + 1], sc, -m.y) : -INFINITY;
      y[n + 2] = n + 2 >= hide && n + 2 < rows ? fmaf(y[n + 2], sc, -m.z) : -INFINITY;
      y[n + 3] = n + 3 >= hide && n + 3 < rows ? fmaf(y[n + 3], sc, -m.w) : -INFINITY;
      over = fmaxf(max3(over, y[n], y[n + 1]), fmaxf(y[n + 2], y[n + 3]));
    }
    bool raise = open;
    if (!open) {
      const bool vote = __any_sync(0xffffffffu, over > PA_RESCALE + PA_TOP<T>);
      if (lane == 0) sh.flag[s][k & 1][w] = vote ? 1 : 0;
      if (!group_sync()) return false;
      const int4 f = *reinterpret_cast<const int4*>(sh.flag[s][k & 1]);
      raise = (f.x | f.y | f.z | f.w) != 0;
    }
    if (raise) {
      float v[N];
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] = y[n];
      const int base = warp_reduce_rows<N>(v, lane, [](float a, float b) { return fmaxf(a, b); });
      red(s, w, base) = v[0];
      if (!group_sync()) return false;
      if (key < N) {
        const float mx = fmaxf(fmaxf(red(s, 0, key), red(s, 1, key)), fmaxf(red(s, 2, key), red(s, 3, key)));
        const float up = mx > (set ? PA_RESCALE + PA_TOP<T> : -INFINITY) ? mx - PA_TOP<T> : 0.f;
        set = set || mx > -INFINITY || key >= rows;
        sh.up[s][key] = up;
        sh.ref[s][key] = k == 0 ? up : sh.ref[s][key] + up;
        const uint32_t unset = __ballot_sync(N == 32 ? 0xffffffffu : (1u << N) - 1, !set);
        if (key == 0) sh.open[s] = unset != 0 ? 1 : 0;
      }
      if (!group_sync()) return false;
      open = sh.open[s] != 0;
#pragma unroll
      for (int n = 0; n < N; ++n) y[n] -= sh.up[s][n];
      if (k > 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) l[n] *= ex2_approx(-fmaxf(sh.up[s][n], 0.f));  // (below 0: l is 0)
        uint32_t o[16];
#pragma unroll 1
        for (int c = 0; c < N; c += 16) {
          tmem_ld16(tO + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            o[j] = __float_as_uint(__uint_as_float(o[j]) * ex2_approx(-fmaxf(sh.up[s][c + j], 0.f)));
          tmem_st16(tO + c, o);
        }
        tmem_wait_st();
      }
    }
#pragma unroll
    for (int n = 0; n < N; n += 8) {
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        e[j] = ex2_approx(y[n + j]);
        l[n + j] += e[j];
      }
      *reinterpret_cast<uint4*>(row_p + (((n >> 3) ^ (key & 7)) << 4)) =
          make_uint4(pack_pair<T>(e[0], e[1]), pack_pair<T>(e[2], e[3]), pack_pair<T>(e[4], e[5]),
                     pack_pair<T>(e[6], e[7]));
    }
    const int left = piece.limit - (pos - key);
    if (left < PA_BN && (left & 15) != 0) {  // the last block, which ends inside a 16-key step
      if (!__all_sync(0xffffffffu, mbar_wait(&sh.bar_tail[s], ntail++ & 1))) return false;
      paged_clear_tail<D>(sV, left, key);
    }
    fence_async_smem();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.bar_p[s]);
  }
  if (steps > 0) {
    if (!__all_sync(0xffffffffu, mbar_wait(&sh.bar_o[s], no++ & 1))) return false;
    if (steps > PA_FLUSH) {
      tc_fence_after();
      flush(false, true);
    }
    const int base = warp_reduce_rows<N>(l, lane, [](float a, float b) { return a + b; });
    red(s, w, base) = l[0];
    fence_async_smem();  // (a TMA load may write here next)
  }
  if (s == 1) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.bar_join);
    if (!__all_sync(0xffffffffu, mbar_wait(&sh.bar_joined, nj++ & 1))) return false;
    // stream 0 is done too, and with it the query slot, P in it included
    if (tid == 128) mbar_arrive(bar_q_empty);
    return true;
  }
  if (!group_sync() || !__all_sync(0xffffffffu, mbar_wait(&sh.bar_join, nj++ & 1))) return false;
  const bool whole = piece.slot < 0, two = piece.nblk > 1;
  const size_t orow0 = static_cast<size_t>(piece.token0) * p.Hq + piece.h * p.G;
  if (key < N) {
    const float la = red(0, 0, key) + red(0, 1, key) + red(0, 2, key) + red(0, 3, key);
    const float lb = two ? red(1, 0, key) + red(1, 1, key) + red(1, 2, key) + red(1, 3, key) : 0.f;
    const float ma = sh.ref[0][key], mb = sh.ref[1][key];
    const float m = la != 0.f ? (lb != 0.f ? fmaxf(ma, mb) : ma) : mb;
    const float wa = la != 0.f ? exp2f(ma - m) : 0.f, wb = lb != 0.f ? exp2f(mb - m) : 0.f;
    const float lt = (la != 0.f ? la * wa : 0.f) + (lb != 0.f ? lb * wb : 0.f);
    const float inv = whole && lt != 0.f ? 1.f / lt : 1.f;
    sh.ref[0][key] = wa * inv;
    sh.ref[1][key] = wb * inv;
    if (key < rows) {
      if (!whole)
        p.ws_ml[static_cast<size_t>(piece.slot) * 256 + key] = make_float2(lt != 0.f ? m : -INFINITY, lt);
      else if (p.lse != nullptr)
        p.lse[orow0 + static_cast<size_t>(key / p.G) * p.Hq + key % p.G] =
            lt != 0.f ? (m + log2f(lt)) * 0.69314718055994530942f : -INFINITY;
    }
  }
  if (!group_sync()) return false;
  tc_fence_after();
  // thread = head dim: O^T's columns are rows
  T* out = static_cast<T*>(p.out) + orow0 * D + key;
  float* part = p.ws_o + static_cast<size_t>(whole ? 0 : piece.slot) * 256 * D + key;
  int g = 0;
#pragma unroll 1
  for (int c = 0; c < rows; c += 4) {
    uint32_t oa[4], ob[4] = {0, 0, 0, 0};
    tmem_ld4(tO + c, oa);
    if (two) tmem_ld4(tO + 128 + c, ob);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float wa = sh.ref[0][c + j], wb = sh.ref[1][c + j];
      const float v = (wa != 0.f ? __uint_as_float(oa[j]) * wa : 0.f) + (wb != 0.f ? __uint_as_float(ob[j]) * wb : 0.f);
      if (c + j < rows && key < D) {
        if (whole)
          *out = to_type<T>(v);
        else
          *part = v;
      }
      out += D;
      part += D;
      if (++g == p.G) {
        g = 0;
        out += static_cast<size_t>(p.Hq - p.G) * D;
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(&sh.bar_joined);
  return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(PA_THREADS, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQfew,
                      const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const PagedAttnParams p) {
  typedef PagedTile<D> Tile;
  constexpr int ST = Tile::stages;
  constexpr int HALVES = D / 64;
  constexpr uint32_t T_O = 256;  // TMEM: S of stream s (P over it) at 128 s, O at 256 + 128 s
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                 // [2][PA_SLOT]
  uint8_t* sKV = smem + 2 * PA_SLOT;  // [ST][kv_bytes]
  __shared__ PagedShared<ST> sh;

  if (tid < PagedShared<ST>::BARS)
    mbar_init(&sh.bars[tid], tid < PagedShared<ST>::BARS_1   ? 1
                             : tid < PagedShared<ST>::BARS_2 ? 2
                             : tid < PagedShared<ST>::BARS_3 ? 3
                             : tid < PagedShared<ST>::BARS_4 ? 4
                                                             : 11);
  if (tid == 64) {
    prefetch_tensormap(&tmQ);
    prefetch_tensormap(&tmQfew);
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
  }
  fence_barrier_init();
  pdl_wait();
  if (warp == 9) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  // Dependents may launch only once this CTA holds its TMEM (verify_attn.cu).
  pdl_launch_dependents();

  // The next piece; false when there is none (or its wait ran out).
  auto next_piece = [&](uint32_t& n, PagedPiece& piece) -> bool {
    const int i = n % PA_PIECES;
    if (!__all_sync(0xffffffffu, mbar_wait(&sh.bar_piece[i], (n / PA_PIECES) & 1))) return false;
    piece = sh.piece[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.bar_taken[i]);
    ++n;
    return piece.nblk > 0;
  };

  if (warp < 8) {
    // ---------------- softmax warpgroups: thread = row ----------------
    const int s = warp >> 2, r = tid & 127;
    const uint32_t trow = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t tS = trow + s * 128, tO = trow + T_O + s * 128;
    const int rt = r / p.G, rg = r % p.G;  // token and head of this row in its tile
    const float sc = p.scale_log2;
    uint32_t npiece = 0, ns = 0, no = 0, nj = 0, ng = 0;  // pieces, steps, results, joins, group syncs so far
    uint32_t ns1 = 0, na = 0;                      // steps' second halves, whole-tile items
    uint32_t nq = 0, ntail = 0, nld = 0;           // query tiles, tails cleared, loads so far
    bool ok = true;
    PagedPiece piece;
    while (ok && next_piece(npiece, piece)) {
      const int nblk = piece.nblk;
      const bool pair = piece.tokens > p.TQ;
      nld += 2 * nblk;
      uint8_t* sV = sKV + (nld - 1) % ST * Tile::kv_bytes;  // the stage of the piece's last V
      if (piece.tokens <= p.TQ_few) {
        const int rows = piece.tokens * p.G;
        if (rows <= 16)
          ok = paged_few_piece<T, D, 16>(p, piece, sh, sQ, sV, tS, tO, s, &sh.bar_q_empty[nq++ & 1], ntail, ns, no, nj, ng);
        else
          ok = paged_few_piece<T, D, 32>(p, piece, sh, sQ, sV, tS, tO, s, &sh.bar_q_empty[nq++ & 1], ntail, ns, no, nj, ng);
        continue;
      }
      nq += pair ? 2 : 1;
      const int tile = pair ? s : 0;
      const int t = tile * p.TQ + rt;  // token of the item
      const bool valid_row = rt < p.TQ && t < piece.tokens;
      const int tile_rows = min(p.TQ, piece.tokens - tile * p.TQ) * p.G;
      const bool live = (warp & 3) * 32 < tile_rows;  // warps without rows only keep the barriers going
      const int limit = p.causal ? min(piece.limit, piece.first + t) : piece.limit;
      const int all_see = __reduce_min_sync(0xffffffffu, limit);  // keys that all rows of the warp see
      const int steps = pair ? nblk : (nblk - s + 1) >> 1;
      float m_run = -INFINITY, l_run = 0.f, m_sum = -INFINITY, l_sum = 0.f;
      // O and l to their sums: begin: the first time; end: and back
      auto flush = [&](bool begin, bool end) {
        float* sum =
            p.ws_o + (static_cast<size_t>(piece.slot < 0 ? 2 * cta + 1 : piece.slot) * 256 + s * 128 + r) * D;
        const float f = m_sum == m_run ? 1.f : exp2f(m_sum - m_run);
        paged_flush<D>(tO, sum, f, begin, end);
        l_sum = fmaf(l_sum, f, l_run);
        l_run = end ? l_sum : 0.f;
        m_sum = m_run;
      };
#pragma unroll 1
      for (int h = 0, h_end = 0; ok && h < 2 * steps;) {
        if (h > 0 && live) {
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_s[s][1], ns1 & 1));  // O at rest
          if (!ok) break;
          flush(h == 2 * PA_FLUSH, false);
        }
        h_end = min(2 * steps, h + 2 * PA_FLUSH);
#pragma unroll 1
        for (; ok && h < h_end; ++h) {  // half steps
          const int half = h & 1, k = h >> 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_s[s][half], (half == 0 ? ns : ns1) & 1));
          if (!ok) break;
          const int k0 = (piece.j0 + (pair ? k : 2 * k + s)) * PA_BN, left = piece.limit - k0;
          if (half == 0) {
            ++ns;
            if (left < PA_BN && (left & 15) != 0) {
              // the last block, which ends inside a 16-key step (both streams of a pair
              // clear its rows, each before its own product)
              ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_tail[s], ntail++ & 1));
              if (!ok) break;
              paged_clear_tail<D>(sV, left, r);
              __syncwarp();
            }
          } else {
            ++ns1;
          }
          if (live) {
            tc_fence_after();
            // (limit - k0: visible keys of this block.)  The products so far are complete
            // once the other half's next S is: it was issued after the last of them.  Behind
            // the last step there is none, and bar_half takes its place.
            const bool at_end = h + 1 == 2 * steps;
            ok = paged_softmax_half<T, D>(tS + half * (PA_BN / 2), tO, sc, limit - k0 - half * (PA_BN / 2),
                                          k0 + (half + 1) * (PA_BN / 2) > all_see, m_run, l_run,
                                          at_end ? &sh.bar_half[s] : &sh.bar_s[s][half ^ 1],
                                          at_end ? na : (half == 0 ? ns1 : ns));
            if (!ok) break;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(half == 0 ? &sh.bar_p[s] : &sh.bar_p2[s]);
        }
      }
      // ---- the item's result ----
      // Every warp waits for every phase of both barriers: nothing says that two commits
      // arrive in the order of their issue, and a wait by parity must not fall two behind.
      // (The next phase of each needs this warp's next P, so neither can be two ahead.)
      if (ok && steps > 0)
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_half[s], na++ & 1)) &&
             __all_sync(0xffffffffu, mbar_wait(&sh.bar_o[s], no++ & 1));
      if (!ok) break;
      if (steps > PA_FLUSH && live) flush(false, true);
      float wa = 1.f, wb = 0.f, m = m_run, l = l_run;
      bool join = false;
      if (!pair) {
        // stream 1, its last product done, hands (m, l) to stream 0, which
        // reads both accumulators
        if (s == 1) {
          sh.m[r] = m_run;
          sh.l[r] = l_run;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.bar_join);
        } else {
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_join, nj & 1));
          if (!ok) break;
          const float mB = sh.m[r], lB = sh.l[r];
          join = __any_sync(0xffffffffu, lB != 0.f);
          m = fmaxf(m_run, mB);
          wa = l_run != 0.f ? exp2f(m_run - m) : 0.f;
          wb = lB != 0.f ? exp2f(mB - m) : 0.f;
          l = (l_run != 0.f ? l_run * wa : 0.f) + (lB != 0.f ? lB * wb : 0.f);
        }
      }
      const bool whole = piece.slot < 0;
      if (live && (pair || s == 0)) {
        tc_fence_after();
        const bool seen = l != 0.f, seen_a = l_run != 0.f, seen_b = join && sh.l[r] != 0.f;
        const float inv = whole && seen ? 1.f / l : 1.f;
        const int token = piece.token0 + t;
        const int head = piece.h * p.G + rg;
        const size_t orow = static_cast<size_t>(token) * p.Hq + head;
        const size_t slot = static_cast<size_t>(whole ? 0 : piece.slot) * 256 + tile * 128 + r;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t oa[32];
          float v[32];
          tmem_ld32(tO + c, oa);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = seen_a ? __uint_as_float(oa[j]) * wa : 0.f;
          if (join) {
            tmem_ld32(tO + 128 + c, oa);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += seen_b ? __uint_as_float(oa[j]) * wb : 0.f;
          }
          if (valid_row) {
            if (whole) {
              T* dst = static_cast<T*>(p.out) + orow * D + c;
              uint32_t pk[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) pk[j] = pack_pair<T>(v[2 * j] * inv, v[2 * j + 1] * inv);
              st_global_32b(dst, pk, p.out_32b);
              st_global_32b(dst + 16, pk + 8, p.out_32b);
            } else {
              float* dst = p.ws_o + slot * D + c;
#pragma unroll
              for (int j = 0; j < 32; j += 8) st_global_32b(dst + j, reinterpret_cast<const uint32_t*>(v) + j, true);
            }
          }
        }
        if (valid_row) {
          if (!whole)
            p.ws_ml[slot] = make_float2(seen ? m : -INFINITY, l);
          else if (p.lse != nullptr)
            p.lse[orow] = seen ? (m + log2f(l)) * 0.69314718055994530942f : -INFINITY;
        }
        tc_fence_before();
      }
      // stream 1 must not start the next item before its O has been read
      if (!pair) {
        if (s == 0) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.bar_joined);
        } else {
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_joined, nj & 1));
          // both streams are done, and with them the query slot
          if (ok && tid == 128) mbar_arrive(&sh.bar_q_empty[(nq - 1) & 1]);
        }
        ++nj;
      }
    }
  } else {
    if (warp == 8) {
      // ---------------- TMA producer: the whole warp, a page per lane ----------------
      const int box_log2 = min(p.page_log2, 7), box = 1 << box_log2;  // rows per copy
      const int per_block = PA_BN >> box_log2;           // copies per block
      const uint32_t copy_bytes = box * D * 2;
      const int groups = 1 << (p.page_log2 - 3);   // 8-row groups per page and head
      uint32_t nld = 0, nq = 0;                    // loads and Q tiles issued
      uint32_t np = 0;
      bool ok = true, was_few = false;
      PagedPiece piece;
      while (ok && next_piece(np, piece)) {
        const int32_t* row = p.table + static_cast<size_t>(piece.b) * p.width;
        const int nblk = piece.nblk, limit = piece.limit;
        const bool pair = piece.tokens > p.TQ, few = piece.tokens <= p.TQ_few;
        // the page of copy `lane` of block j (the copies of one page share it)
        auto page_of = [&](int j) -> int {
          const int key = j * PA_BN + lane * box;
          return lane < per_block && j < piece.j0 + nblk && key < limit ? __ldg(row + (key >> p.page_log2)) : 0;
        };  // (not looked at before it is used: the load is on its way meanwhile)
        int next_id = page_of(piece.j0);
        // queries; between whole tiles and few rows, which use a slot's last half
        // differently (the latter both slots', whichever holds the queries), the last
        // tile has to be done with its slot, not only the one before it
        if (nq > 0 && was_few != few)
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_q_empty[(nq - 1) & 1], ((nq - 1) >> 1) & 1));
        was_few = few;
        for (int s = 0; ok && s < (pair ? 2 : 1); ++s, ++nq) {
          const int st = nq & 1;
          if (nq >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_q_empty[st], ((nq >> 1) - 1) & 1));
          if (ok && lane == 0) {
            mbar_arrive_expect_tx(&sh.bar_q_full[st], (few ? p.TQ_few : p.TQ) * p.G * D * 2);
            for (int hf = 0; hf < HALVES; ++hf)
              tma_load_4d(sQ + st * PA_SLOT + hf * (few ? 8192 : 16384), few ? &tmQfew : &tmQ, &sh.bar_q_full[st], hf * 64,
                          0, piece.h, piece.token0 + s * p.TQ);
          }
        }
        int id = 0, id_before = 0, kk = 0, kv = 0;  // kk, kv: blocks of K, V so far
#pragma unroll 1
        for (int c = 0; ok && c < 2 * nblk; ++c) {
          const bool is_k = kk < nblk && (pair ? kk == kv : kk < kv + 2);
          const int j = piece.j0 + (is_k ? kk : kv);
          if (is_k) {
            id_before = id;
            id = next_id;
            next_id = page_of(j + 1);  // (on its way while this load waits for its stage)
          }
          const int mine = is_k || kk == kv + 1 ? id : id_before;
          const int st = nld % ST;
          if (nld >= ST) ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_empty[st], ((nld / ST) - 1) & 1));
          if (!ok) break;
          const int left = limit - j * PA_BN;
          const int copies = left <= 0 ? 0 : min(per_block, (left + box - 1) >> box_log2);
          if (lane == 0) mbar_arrive_expect_tx(&sh.bar_full[st], copies * copy_bytes);
          __syncwarp();
          if (lane < copies) {
            const int key = j * PA_BN + lane * box;
            const bool in_pool = mine >= 0 && mine < p.num_pages;
            if (!in_pool) std_set_error(STD_DEVERR_BOUNDS);
            const int g = ((in_pool ? mine : 0) * p.Hkv + piece.h) * groups + ((key & ((1 << p.page_log2) - 1)) >> 3);
            tma_load_4d(sKV + st * Tile::kv_bytes + lane * copy_bytes, is_k ? &tmK : &tmV, &sh.bar_full[st], 0, 0, 0,
                        in_pool ? g : p.num_pages * p.Hkv * groups);  // (past the pool: TMA fills zeros)
          }
          ++nld;
          if (is_k)
            ++kk;
          else
            ++kv;
        }
      }
      // never leave a copy in flight, nor a commit that has yet to arrive on a barrier
      for (uint32_t c = nld < ST ? 0 : nld - ST; c < nld; ++c) {
        mbar_wait(&sh.bar_full[c % ST], (c / ST) & 1);
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_empty[c % ST], (c / ST) & 1));
      }
      for (uint32_t c = nq < 2 ? 0 : nq - 2; c < nq; ++c) {
        mbar_wait(&sh.bar_q_full[c & 1], (c >> 1) & 1);
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&sh.bar_q_empty[c & 1], (c >> 1) & 1));
      }
    } else if (warp < 11) {
      // ---------------- MMA issuers: one thread per stream ----------------
      // A stream's S and P V go out in order from one thread, which is what lets S
      // be written over the P that its last P V read.  Per stream, since issuing a
      // step (waits, commits, 16 MMAs beside busy softmax warps) takes one thread
      // about as long as the tensor core needs for two.
      const int s = warp - 9;
      if (elect_one()) {
        constexpr uint32_t idS = paged_idesc<T>(128, PA_BN / 2, 0, 0);
        constexpr uint32_t idO = paged_idesc<T>(128, D, 0, 1);
        // (a descriptor's low bits are the address / 16, so offsets are added to it)
        const uint64_t dKV = sdesc_sw128(smem_u32(sKV), 16, HALVES * 1024);    // K-major
        const uint64_t dVm = sdesc_sw128(smem_u32(sKV), 1024, HALVES * 1024);  // MN-major
        // V as the A operand: D 64 has no second block of 64 columns, rows 64..127 repeat the first
        const uint64_t dVa = sdesc_sw128(smem_u32(sKV), HALVES == 2 ? 1024 : 0, HALVES * 1024);
        const uint64_t dQ0 = sdesc_sw128(smem_u32(sQ), 16, 1024);
        const uint64_t dP = sdesc_sw128(smem_u32(sQ + s * PA_SLOT + PA_PT), 16, 1024);
        const uint32_t tS = tmem + s * 128, tO = tmem + T_O + s * 128;
        uint32_t npiece = 0, nq = 0;      // pieces, query tiles so far
        uint32_t st = 0, ph = 0;                // ring position of the next load, its turn's parity
        uint32_t np = 0, np2 = 0;               // P halves so far
        for (;;) {
          const int ip = npiece % PA_PIECES;
          if (!mbar_wait(&sh.bar_piece[ip], (npiece / PA_PIECES) & 1)) break;
          const PagedPiece piece = sh.piece[ip];
          mbar_arrive(&sh.bar_taken[ip]);
          ++npiece;
          const int nblk = piece.nblk;
          if (nblk <= 0) break;
          const bool pair = piece.tokens > p.TQ, few = piece.tokens <= p.TQ_few;
          // visible keys of the last block: products stop at the next multiple of 16
          const int last = min(PA_BN, piece.limit - (piece.j0 + nblk - 1) * PA_BN);
          const int last_steps = (last + 15) >> 4;
          // query tiles: a pair's stream has its own, a single's share one (whose
          // third release comes from the softmax)
          const uint32_t qs = (nq + (pair ? s : 0)) & 1;
          bool ok = mbar_wait(&sh.bar_q_full[nq & 1], (nq >> 1) & 1);
          ++nq;
          if (pair) {
            ok = ok && mbar_wait(&sh.bar_q_full[nq & 1], (nq >> 1) & 1);
            ++nq;
          }
          mbar_arrive(&sh.bar_q_empty[pair ? qs ^ 1 : qs]);
          const uint64_t dQ = dQ0 + qs * (PA_SLOT / 16);
          // Load `index` of the piece, in its stage `at`.  Loads are waited for in ring
          // order whoever uses them, and not given back before both threads have
          // passed them: a barrier's parity tells neighbouring phases apart, no more,
          // so neither thread may fall a turn behind.
          int pos = 0;
          uint32_t at = 0;
          auto take = [&](int index) -> bool {
            for (;; ++pos) {
              if (!mbar_wait(&sh.bar_full[st], ph)) return false;
              at = st;
              if (++st == ST) {
                st = 0;
                ph ^= 1;
              }
              if (pos == index) break;
              mbar_arrive(&sh.bar_empty[at]);
            }
            ++pos;
            return true;
          };
          // pair: K0 V0 K1 V1 ..; single: K0 K1 V0 K2 V1 .. V, stream s using blocks s, s + 2 ..
          const int step = pair ? 1 : 2;
          int k = pair ? 0 : s;
          if (ok && k < nblk) {
            ok = take(pair || k == 0 ? 0 : 1);
            if (few) {
              const uint32_t n_few = paged_few_cols(piece.tokens * p.G);
              const uint32_t idSt = paged_idesc<T>(128, n_few, 0, 0), idOt = paged_idesc<T>(128, n_few, 1, 1);
#pragma unroll 1
              for (; ok; k += 2) {
                tc_fence_after();
                const uint64_t dK = dKV + at * (Tile::kv_bytes / 16);
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                  umma_bf16(tS, dK + ((ks >> 2) * 1024 + (ks & 3) * 32) / 16,
                            dQ + ((ks >> 2) * 8192 + (ks & 3) * 32) / 16, idSt, ks > 0 ? 1u : 0u);
                umma_commit(&sh.bar_s[s][0]);
                umma_commit(&sh.bar_empty[at]);
                const bool end = k + 1 == nblk;
                ok = take(end ? 2 * nblk - 1 : 2 * k + 2);
                if (!ok) break;
                if (end && (last & 15) != 0) mbar_arrive(&sh.bar_tail[s]);
                ok = mbar_wait(&sh.bar_p[s], np++ & 1);
                if (!ok) break;
                tc_fence_after();
                const uint64_t dV = dVa + at * (Tile::kv_bytes / 16);
                const int ksteps = end ? last_steps : PA_BN / 16;
                uint32_t more = k > 1 ? 1u : 0u;
#pragma unroll 2
                for (int ks = 0; ks < ksteps; ++ks, more = 1u)
                  umma_bf16(tO, dV + ks * (HALVES * 2048 / 16), dP + ks * (2048 / 16), idOt, more);
                umma_commit(&sh.bar_empty[at]);
                if (k + 2 >= nblk) break;
                ok = take(2 * k + 3);
              }
              if (ok) umma_commit(&sh.bar_o[s]);
            } else {
              // S in halves of 64 keys, each a block ahead of its half's product:
              // Sa0 Sb0, PVa0 Sa1 PVb0 Sb1, PVa1 Sa2 ...  The softmax always has a half
              // ready while the other is in the tensor core.
              auto s_half = [&](uint32_t stage, int half) {
                const uint64_t dK = dKV + stage * (Tile::kv_bytes / 16) + half * (8 * HALVES * 1024 / 16);
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                  umma_bf16(tS + half * 64, dQ + ((ks >> 2) * 16384 + (ks & 3) * 32) / 16,
                            dK + ((ks >> 2) * 1024 + (ks & 3) * 32) / 16, idS, ks > 0 ? 1u : 0u);
                umma_commit(&sh.bar_s[s][half]);
              };
              if (ok) {
                tc_fence_after();
                s_half(at, 0);
                s_half(at, 1);
                umma_commit(&sh.bar_empty[at]);
                if (k + step >= nblk && pair) {
                  umma_commit(&sh.bar_q_empty[qs]);
                  umma_commit(&sh.bar_q_empty[qs]);
                }
              }
              uint32_t more = 0;
#pragma unroll 1
              for (; ok; k += step) {
                const bool end = k + 1 == nblk, has_next = k + step < nblk;
                ok = take(pair ? 2 * k + 1 : (end ? 2 * nblk - 1 : 2 * k + 2));
                if (!ok) break;
                const uint32_t at_v = at;
                const uint64_t dV = dVm + at_v * (Tile::kv_bytes / 16);
                if (end && (last & 15) != 0) mbar_arrive(&sh.bar_tail[s]);
                ok = mbar_wait(&sh.bar_p[s], np++ & 1);
                if (!ok) break;
                tc_fence_after();
                if (!end) {
                  umma_bf16_ts(tO, tS, dV, idO, more);
#pragma unroll
                  for (int ks = 1; ks < PA_BN / 32; ++ks)
                    umma_bf16_ts(tO, tS + ks * 8, dV + ks * (HALVES * 2048 / 16), idO, 1u);
                } else {
#pragma unroll 1
                  for (int ks = 0; ks < min(last_steps, PA_BN / 32); ++ks)
                    umma_bf16_ts(tO, tS + ks * 8, dV + ks * (HALVES * 2048 / 16), idO, more | (ks > 0 ? 1u : 0u));
                }
                more = 1u;
                if (has_next) {
                  ok = take(pair ? 2 * k + 2 : 2 * k + 3);
                  if (!ok) break;
                  tc_fence_after();
                  s_half(at, 0);
                } else {
                  umma_commit(&sh.bar_half[s]);  // for a second half that rescales O
                }
                ok = mbar_wait(&sh.bar_p2[s], np2++ & 1);
                if (!ok) break;
                tc_fence_after();
                if (!end) {
#pragma unroll
                  for (int ks = PA_BN / 32; ks < PA_BN / 16; ++ks)
                    umma_bf16_ts(tO, tS + 32 + ks * 8, dV + ks * (HALVES * 2048 / 16), idO, 1u);
                } else {
#pragma unroll 1
                  for (int ks = PA_BN / 32; ks < last_steps; ++ks)
                    umma_bf16_ts(tO, tS + 32 + ks * 8, dV + ks * (HALVES * 2048 / 16), idO, 1u);
                }
                umma_commit(&sh.bar_empty[at_v]);
                if (!has_next) break;
                s_half(at, 1);
                umma_commit(&sh.bar_empty[at]);
                if (k + 2 * step >= nblk && pair) {
                  umma_commit(&sh.bar_q_empty[qs]);
                  umma_commit(&sh.bar_q_empty[qs]);
                }
              }
              if (ok) umma_commit(&sh.bar_o[s]);
            }
          }
          // loads of the other stream that are left
          for (; ok && pos < 2 * nblk; ++pos) {
            ok = mbar_wait(&sh.bar_full[st], ph);
            mbar_arrive(&sh.bar_empty[st]);
            if (++st == ST) {
              st = 0;
              ph ^= 1;
            }
          }
          if (!ok) break;
        }
        // nothing may be in flight when the CTA gives back its TMEM
        umma_commit(&sh.bar_end[s]);
        mbar_wait(&sh.bar_end[s], 0);
      }
      __syncwarp();
    } else {
      // ---------------- scheduler: the pieces of this CTA's share ----------------
      // Costs of the requests, 32 at a time, a request per lane (one of several
      // items is summed by the whole warp): once for their total, and again for
      // the place of this CTA's share.  (Rolled loops: on a first pass the
      // instructions come from L2, and short code is what makes this quick.)
      PagedWalk walk;
      walk.rem = 0;
      int total = 0, share = 1, x0 = 0, off = 0, cost = 0;
#pragma unroll 1
      for (int pass = 0; pass < 2; ++pass) {
        int run = 0;
#pragma unroll 1
        for (int b0 = 0; b0 < p.B; b0 += 32) {
          if (pass == 0 || p.B > 32) {  // (else `cost` still is what pass 0 left)
            const int b = b0 + lane;
            int n = 0, kv = 0;
            if (b < p.B) {
              kv = __ldg(p.kv_lens + b);
              if (!paged_request(p, __ldg(p.cu_q + b), __ldg(p.cu_q + b + 1), kv, n) && cta == 0)
                std_set_error(STD_DEVERR_LENGTH);
            }
            cost = n > 0 && n <= 2 * p.TQ ? paged_item_cost(p, n, kv, 0) : 0;
#pragma unroll 1
            for (uint32_t many = __ballot_sync(0xffffffffu, n > 2 * p.TQ); many != 0; many &= many - 1) {
              const int src = __ffs(many) - 1;
              const int n_ = __shfl_sync(0xffffffffu, n, src), kv_ = __shfl_sync(0xffffffffu, kv, src);
              int sum = 0;
#pragma unroll 1
              for (int i = lane; i * 2 * p.TQ < n_; i += 32) sum += paged_item_cost(p, n_, kv_, i);
              sum = __reduce_add_sync(0xffffffffu, sum);
              if (lane == src) cost = sum;
            }
            cost *= p.Hkv;
          }
          if (pass == 0) {
            total += __reduce_add_sync(0xffffffffu, cost);
            continue;
          }
          const int inc = warp_scan(cost, lane);
          const uint32_t past = __ballot_sync(0xffffffffu, x0 < run + inc);
          if (past != 0) {
            const int src = __ffs(past) - 1;
            walk.b = b0 + src;
            off = x0 - __shfl_sync(0xffffffffu, run + inc - cost, src);
            walk.rem = min(share, total - x0);
            break;
          }
          run += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (pass == 0) {
          // equal shares, of a two-block single at least (its streams take one block each)
          share = max((total + PA_CTAS - 1) / PA_CTAS, ((2 + PA_OVER) * PA_W1) >> p.unit_log2);
          if (total == 0 || cta >= (total + share - 1) / share) break;
          x0 = share * cta;
        }
      }
      if (walk.rem > 0) {
        walk.request(p);
        // KV head and item: the items' costs, a run of `per` of them per lane
        if (walk.items == 1) {
          const int head = paged_item_cost(p, walk.n, walk.kv, 0);
          walk.h = off / head;
          walk.i = 0;
          walk.skip = off - walk.h * head;
        } else {
          const int per = (walk.items + 31) / 32;
          int sum = 0;
#pragma unroll 1
          for (int i = lane * per; i < min((lane + 1) * per, walk.items); ++i)
            sum += paged_item_cost(p, walk.n, walk.kv, i);
          const int inc = warp_scan(sum, lane), head = __shfl_sync(0xffffffffu, inc, 31);
          walk.h = off / head;
          off -= walk.h * head;
          const int src = __ffs(__ballot_sync(0xffffffffu, off < inc)) - 1;
          off -= __shfl_sync(0xffffffffu, inc - sum, src);
#pragma unroll 1
          for (walk.i = src * per;; ++walk.i) {
            const int c = paged_item_cost(p, walk.n, walk.kv, walk.i);
            if (off < c || walk.i + 1 >= walk.items) break;
            off -= c;
          }
          walk.skip = off;
        }
      }
      PagedSplit split = {0, -1, 0, 0, 0};
      bool more = true;
      for (uint32_t n = 0; more; ++n) {
        more = walk.next(p);
        const int i = n % PA_PIECES;
        if (n >= PA_PIECES && !__all_sync(0xffffffffu, mbar_wait(&sh.bar_taken[i], ((n / PA_PIECES) - 1) & 1))) break;
        if (lane == 0) {
          PagedPiece piece = {walk.b, walk.h, walk.q0 + walk.t0, walk.nt, walk.limit, 0, walk.j0, 0, -1};
          if (more) {
            piece.first = walk.kv - walk.n + walk.t0 + 1;
            piece.nblk = walk.j1 - walk.j0;
            if (walk.j0 > 0 || walk.j1 < walk.nb) piece.slot = 2 * cta + (walk.j0 == 0 ? 1 : 0);
          }
          sh.piece[i] = piece;
          mbar_arrive(&sh.bar_piece[i]);
        }
        __syncwarp();
        if (more && walk.j1 < walk.nb) {
          // the share ends inside this item: a block lies with the CTA whose share holds its cost
          const int start = x0 + share - walk.cut;
          split.first_cta = (start + ((PA_OVER * walk.w) >> p.unit_log2)) / share;
          split.last_cta = (start + (((walk.nb - 1 + PA_OVER) * walk.w) >> p.unit_log2)) / share;
          split.token0 = walk.q0 + walk.t0;
          split.tokens = walk.nt;
          split.kvh = walk.h;
        }
      }
      if (lane == 0) p.splits[cta] = split;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of the items that cuts divide: blocks x work at the item that
// CTA x's share ends inside, so an item of many pieces has many blocks.  out =
// sum_c w_c o_c / sum_c w_c l_c with w_c = exp2(m_c - max m), in a fixed order of
// the pieces.  Latency is what counts (a few loads per row, mostly from L2): each
// wave of blocks costs a memory round trip even where there is nothing to join, so
// the grid is one wave (two blocks an item) while no item can be a pair, and two waves
// (four blocks) where one can, whose rows repay it: two blocks against four, mixed
// step 56.3 / 54.9 us, 16 heads of D 64 32.5 / 30.8, 8 verify blocks over 33K keys
// 103.0 / 102.0.  The loads of two rows by two pieces a warp are in flight together, or, for
// an item of many pieces (a long context), a row's pieces over eight warps.
constexpr int PM_THREADS = 512;  // (two blocks per SM)
template <int D>
struct PagedSum {  // a row's running (m, l, o)
  float m, l, o[D / 32];
  STD_DEV PagedSum() : m(-INFINITY), l(0.f) {
#pragma unroll
    for (int k = 0; k < D / 32; ++k) o[k] = 0.f;
  }
  // N pieces at once; one in which the row sees no key has l = 0, m = -inf, o = 0
  template <int N>
  STD_DEV void add(const float2 (&ml)[N], const float (&po)[N][D / 32]) {
    float mx = m;
#pragma unroll
    for (int j = 0; j < N; ++j) mx = fmaxf(mx, ml[j].x);
    const float a = l != 0.f ? exp2f(m - mx) : 0.f;
    l *= a;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) o[k] *= a;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float w = ml[j].y != 0.f ? exp2f(ml[j].x - mx) : 0.f;
      l += w * ml[j].y;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) o[k] += w * po[j][k];
    }
    m = mx;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(PM_THREADS, 2) paged_merge_kernel(const PagedAttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int PER = D / 32;  // columns per lane
  const int cta = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedSplit sp = p.splits[cta];
  // (the rest only if cu_q overlaps itself: the sums it gives may pass 32 bits)
  if (sp.last_cta <= cta || sp.first_cta > cta || sp.first_cta < 0 || sp.last_cta >= PA_CTAS) return;
  const int n = sp.last_cta - sp.first_cta + 1;
  const int block = (cta - sp.first_cta) * gridDim.y + blockIdx.y, blocks = (n - 1) * gridDim.y;  // of this item
  // piece i is CTA first + i's: its continued item (slot 0), or for the first the item begun there (slot 1)
  auto slot = [&](int i) { return (static_cast<size_t>(2 * (sp.first_cta + i)) + (i == 0 ? 1 : 0)) * 256; };
  auto load = [&](size_t row, bool there, float2& ml, float* o) {
    ml = make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int k = 0; k < PER; ++k) o[k] = 0.f;
    if (!there) return;
    ml = __ldcg(p.ws_ml + row);
    const float* src = p.ws_o + row * D + lane * PER;
    if constexpr (PER == 4) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
      o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    } else {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
      o[0] = v.x, o[1] = v.y;
    }
  };
  // rows: tile 0's from 0, tile 1's from 128
  const int rows0 = min(sp.tokens, p.TQ) * p.G, rows1 = (sp.tokens - min(sp.tokens, p.TQ)) * p.G;
  const int end = rows1 > 0 ? 128 + rows1 : rows0;
  auto row_there = [&](int r) { return r < 128 ? r < rows0 : r - 128 < rows1; };
  auto write = [&](int r, const PagedSum<D>& a) {
    const float inv = a.l != 0.f ? 1.f / a.l : 0.f;
    const int t = (r >> 7) * p.TQ + (r & 127) / p.G;
    const size_t orow = static_cast<size_t>(sp.token0 + t) * p.Hq + sp.kvh * p.G + (r & 127) % p.G;
    T* dst = static_cast<T*>(p.out) + orow * D + lane * PER;
    if constexpr (PER == 4)
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(pack_pair<T>(a.o[0] * inv, a.o[1] * inv), pack_pair<T>(a.o[2] * inv, a.o[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack_pair<T>(a.o[0] * inv, a.o[1] * inv);
    if (lane == 0 && p.lse != nullptr)
      p.lse[orow] = a.l != 0.f ? (a.m + log2f(a.l)) * 0.69314718055994530942f : -INFINITY;
  };
  if (n <= 8) {
    constexpr int ROWS = 2, WARPS = PM_THREADS / 32;
    for (int r0 = (block * WARPS + warp) * ROWS; r0 < end; r0 += blocks * WARPS * ROWS) {
      bool there[ROWS];
      PagedSum<D> sum[ROWS];
#pragma unroll
      for (int q = 0; q < ROWS; ++q) there[q] = row_there(r0 + q);
      for (int i = 0; i < n; i += 2) {
        float2 ml[ROWS][2];
        float o[ROWS][2][PER];
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
          load(slot(i) + r0 + q, there[q], ml[q][0], o[q][0]);
          load(slot(i + 1) + r0 + q, there[q] && i + 1 < n, ml[q][1], o[q][1]);
        }
#pragma unroll
        for (int q = 0; q < ROWS; ++q) sum[q].template add<2>(ml[q], o[q]);
      }
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
        if (there[q]) write(r0 + q, sum[q]);
    }
    return;
  }
  constexpr int ROWS = PM_THREADS / 256;  // rows at a time, eight warps each
  __shared__ float s_o[ROWS][8][D];
  __shared__ float2 s_ml[ROWS][8];
  const int q = warp >> 3, part = warp & 7;
  for (int r0 = block * ROWS; r0 < end; r0 += blocks * ROWS) {
    const int r = r0 + q;
    const bool there = row_there(r);
    if (!__syncthreads_or(there ? 1 : 0)) continue;  // (and the last rows' values have been read)
    PagedSum<D> sum;
    for (int i0 = part; i0 < n; i0 += 32) {
      float2 ml[4];
      float o[4][PER];
#pragma unroll
      for (int j = 0; j < 4; ++j) load(slot(i0 + 8 * j) + r, there && i0 + 8 * j < n, ml[j], o[j]);
      sum.template add<4>(ml, o);
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) s_o[q][part][lane * PER + k] = sum.o[k];
    if (lane == 0) s_ml[q][part] = make_float2(sum.m, sum.l);
    __syncthreads();
    if (part == 0 && there) {
      PagedSum<D> all;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float2 ml[4];
        float o[4][PER];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          ml[w] = s_ml[q][4 * h + w];
#pragma unroll
          for (int k = 0; k < PER; ++k) o[w][k] = s_o[q][4 * h + w][lane * PER + k];
        }
        all.template add<4>(ml, o);
      }
      write(r, all);
    }
  }
}

}  // namespace stdb

// ---------------------------------------------------------------------------
// host: tensor maps and C ABI
// ---------------------------------------------------------------------------
static int paged_tmap_4d(CUtensorMap* m, int is_fp16, const void* base, const uint64_t* dims, const uint64_t* strides,
                         const uint32_t* box) {
  PFN_tmapEncodeTiled enc = tmap_encoder();
  if (enc == nullptr) return 3;
  cuuint64_t d[4], st[3];
  cuuint32_t bx[4], es[4] = {1, 1, 1, 1};
  for (int i = 0; i < 4; ++i) d[i] = dims[i], bx[i] = box[i];
  for (int i = 0; i < 3; ++i) st[i] = strides[i];
  const CUresult r =
      enc(m, is_fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base),
          d, st, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 4;
}

static size_t paged_ws_o_bytes(int D) { return static_cast<size_t>(2) * stdb::PA_CTAS * 256 * D * 4; }
static size_t paged_ws_ml_bytes() { return static_cast<size_t>(2) * stdb::PA_CTAS * 256 * 8; }

extern "C" size_t std_paged_attn_workspace_bytes(int D) {
  if (D != 64 && D != 128) return 0;
  return paged_ws_o_bytes(D) + paged_ws_ml_bytes() + stdb::PA_CTAS * sizeof(stdb::PagedSplit);
}

template <typename T, int D>
static int paged_attn_launch(const CUtensorMap& tq, const CUtensorMap& tqf, const CUtensorMap& tk, const CUtensorMap& tv,
                             const stdb::PagedAttnParams& p, cudaStream_t s) {
  static SmemGrant grant;
  if (ensure_smem(stdb::paged_attn_kernel<T, D>, grant, stdb::PagedTile<D>::smem) != 0) return 3;
  if (launch_pdl(stdb::paged_attn_kernel<T, D>, dim3(stdb::PA_CTAS), dim3(stdb::PA_THREADS), stdb::PagedTile<D>::smem,
                 s, tq, tqf, tk, tv, p) != cudaSuccess)
    return 4;
  // nothing to join where no item is long enough to be divided
  if (static_cast<long long>(p.width) << p.page_log2 <= stdb::PA_WHOLE * stdb::PA_BN)
    return cudaGetLastError() == cudaSuccess ? 0 : 4;
  const dim3 mgrid(stdb::PA_CTAS, p.T > p.TQ ? 4 : 2);  // (pairs are possible: two waves)
  if (launch_pdl(stdb::paged_merge_kernel<T, D>, mgrid, dim3(stdb::PM_THREADS), 0, s, p) != cudaSuccess) return 4;
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

extern "C" int std_paged_attn(const void* q, const void* k_pages, const void* v_pages, const int32_t* block_table,
                              const int32_t* cu_q, const int32_t* kv_lens, int T, int B, int Hq, int Hkv, int D,
                              int is_fp16, int num_pages, int page_size, int max_blocks, int causal, float scale,
                              void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  if ((D != 64 && D != 128) || T < 0 || B <= 0 || B > STD_PAGED_MAX_REQUESTS || Hkv <= 0 || Hkv > 65535 || Hq <= 0 ||
      Hq % Hkv != 0 || Hq / Hkv > 128 || num_pages <= 0 || max_blocks <= 0 || !paged_page_ok(page_size))
    return 1;
  if (!(scale > 0.f) || !(scale * 1.4426950408889634f < 3.4e38f)) return 1;
  // int32 indexes: keys of a request, slots, 8-row groups of the pool (one page more: the zero fill)
  if (static_cast<long long>(max_blocks) * page_size > 0x7fffffffll - 1024 ||
      static_cast<long long>(num_pages) * page_size > 0x7fffffffll ||
      (static_cast<long long>(num_pages) + 1) * Hkv * (page_size / 8) > 0x7fffffffll || T > 0x7fffffff / 2)
    return 1;
  // items, each of a cost of one or more, in a total of 32 bits (no memory holds more)
  if ((static_cast<double>(T) / (2 * (128 / (Hq / Hkv))) + B) * Hkv > 5.0e8) return 1;
  if (T == 0) return 0;
  if (q == nullptr || k_pages == nullptr || v_pages == nullptr || block_table == nullptr || cu_q == nullptr ||
      kv_lens == nullptr || out == nullptr || q == out)
    return 1;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out)) return 1;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 31) != 0 ||
      workspace_bytes < std_paged_attn_workspace_bytes(D))
    return 5;
  const unsigned long long rows = static_cast<unsigned long long>(T) * Hq,
                           pool = 2ull * D * Hkv * num_pages * page_size;
  if (paged_overlap<9>({{q, rows * D * 2, false}, {k_pages, pool, false}, {v_pages, pool, false},
                        {block_table, 4ull * B * max_blocks, false}, {cu_q, 4ull * B + 4, false},
                        {kv_lens, 4ull * B, false}, {out, rows * D * 2, true}, {lse, lse == nullptr ? 0 : rows * 4, true},
                        {workspace, std_paged_attn_workspace_bytes(D), true}}))
    return 1;
  const int G = Hq / Hkv, TQ = 128 / G, TQ_few = stdb::PA_FEW / G;
  CUtensorMap tq, tqf, tk, tv;
  {
    const uint64_t e = 2, row = static_cast<uint64_t>(D) * e;
    const uint64_t qd[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(G), static_cast<uint64_t>(Hkv),
                            static_cast<uint64_t>(T)};
    const uint64_t qs[3] = {row, row * G, row * Hq};
    const uint32_t qb[4] = {64, static_cast<uint32_t>(G), 1, static_cast<uint32_t>(TQ)};
    // (one of the two maps is never used where no item, or every item, has few rows)
    int rc = T > TQ_few ? paged_tmap_4d(&tq, is_fp16, q, qd, qs, qb) : 0;
    if (rc != 0) return rc;
    const uint32_t qfb[4] = {64, static_cast<uint32_t>(G), 1, static_cast<uint32_t>(TQ_few)};
    if (TQ_few > 0) rc = paged_tmap_4d(&tqf, is_fp16, q, qd, qs, qfb);
    if (rc != 0) return rc;
    if (T <= TQ_few) tq = tqf;
    if (TQ_few == 0) tqf = tq;
    const uint64_t kd[4] = {64, 8, static_cast<uint64_t>(D / 64),
                            static_cast<uint64_t>(num_pages) * Hkv * (page_size / 8)};
    const uint64_t ks[3] = {row, 128, row * 8};
    const uint32_t box_rows = page_size < stdb::PA_BN ? page_size : stdb::PA_BN;
    const uint32_t kb[4] = {64, 8, static_cast<uint32_t>(D / 64), box_rows / 8};
    rc = paged_tmap_4d(&tk, is_fp16, k_pages, kd, ks, kb);
    if (rc == 0) rc = paged_tmap_4d(&tv, is_fp16, v_pages, kd, ks, kb);
    if (rc != 0) return rc;
  }
  stdb::PagedAttnParams p;
  p.table = block_table;
  p.cu_q = cu_q;
  p.kv_lens = kv_lens;
  p.T = T;
  p.B = B;
  p.width = max_blocks;
  p.page_log2 = 0;
  while ((1 << p.page_log2) < page_size) ++p.page_log2;
  p.num_pages = num_pages;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = G;
  p.TQ = TQ;
  // total cost of the calls that these shapes allow, and its unit
  const double most = (static_cast<double>(T) / (2 * TQ) + B) * Hkv *
                      (static_cast<double>(max_blocks) * page_size / stdb::PA_BN + stdb::PA_OVER + 1) * stdb::PA_W2;
  p.unit_log2 = 0;
  while (most / (1ll << p.unit_log2) + (static_cast<double>(T) / (2 * TQ) + B) * Hkv > 1.0e9) ++p.unit_log2;
  p.TQ_few = TQ_few;
  p.causal = causal != 0 ? 1 : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = out;
  p.out_32b = (reinterpret_cast<uintptr_t>(out) & 31) == 0;
  p.lse = lse;
  char* ws = static_cast<char*>(workspace);
  p.ws_o = reinterpret_cast<float*>(ws);
  p.ws_ml = reinterpret_cast<float2*>(ws + paged_ws_o_bytes(D));
  p.splits = reinterpret_cast<stdb::PagedSplit*>(ws + paged_ws_o_bytes(D) + paged_ws_ml_bytes());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (D == 128)
    return is_fp16 ? paged_attn_launch<__half, 128>(tq, tqf, tk, tv, p, s)
                   : paged_attn_launch<__nv_bfloat16, 128>(tq, tqf, tk, tv, p, s);
  return is_fp16 ? paged_attn_launch<__half, 64>(tq, tqf, tk, tv, p, s)
                 : paged_attn_launch<__nv_bfloat16, 64>(tq, tqf, tk, tv, p, s);
}
