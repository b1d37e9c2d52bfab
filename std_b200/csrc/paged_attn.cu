// paged_attn.cu -- attention of each request's new tokens over its paged K/V
// cache, on tcgen05 / TMEM: prompt chunks, verify blocks and single tokens, any
// mix of them in one launch.  The paged, ragged counterpart of
// modeling_qwen2_5_vl.py:1096-1133 (repeat_kv + F.sdpa with the causal mask of
// :65-101).
//
// Tiles.  The G = Hq / Hkv query heads of a KV head share its keys, so rows
// are (token, head of the group) pairs: row = t * G + g, TQ = floor(128 / G)
// whole tokens per 128-row MMA tile.  An item is one KV head's span of up to
// 2 TQ tokens of one request ("pair": two tiles that share every K/V block) or,
// when at most TQ tokens are left, one tile ("single").  Keys come in blocks of
// 128:
//   S = Q K^T     tcgen05.mma M=128 N=128, Q and K from shared memory
//   P = exp2(S * scale * log2e - m), 16 bits, written over S in TMEM
//   O += P V      tcgen05.mma with P as the A operand in TMEM, V MN-major
// Two softmax warpgroups each own a stream of steps with an S and an O of its
// own in TMEM: in a pair, stream s is tile s; in a single, stream s takes the
// blocks j = s mod 2 and the two accumulators are joined at the end.  Either way
// one stream's MMAs run while the other's softmax does.  The running maximum
// is raised lazily, when a block passes it by more than 2^8, so O is normally
// not touched between blocks.
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
#include "common.cuh"

namespace stdb {

constexpr int PA_CTAS = 148;     // one CTA per SM
constexpr int PA_THREADS = 384;  // 2 softmax warpgroups; TMA, MMA and scheduler warp, one idle
// Registers after the split: 2 * 128 * 208 + 128 * 88 = 384 * 168, the launch's total.
constexpr int PA_REGS_SOFTMAX = 208, PA_REGS_OTHER = 88;
constexpr int PA_BN = 128;       // keys per block
constexpr float PA_RESCALE = 8.0f;  // log2 units
constexpr int PA_W1 = 2, PA_W2 = 3;  // cost of a block in a single and in a pair

template <int D>
struct PagedTile {
  static constexpr uint32_t kv_bytes = PA_BN * D * 2;
  static constexpr uint32_t q_bytes = 128 * D * 2;
  static constexpr int stages = D == 128 ? 5 : 8;
  static constexpr uint32_t smem = 2 * q_bytes + stages * kv_bytes + 1024;
};

// What a CTA leaves for the merge about the item that its share ends inside.
struct PagedSplit {
  int last_cta;  // the item's last piece; < 0: nothing to merge
  int token0;    // first token row of the item
  int tokens;
  int kvh;
};

struct PagedAttnParams {
  const int32_t* table;  // [B, width]
  const int32_t* cu_q;   // [B + 1]
  const int32_t* kv_lens;
  int T, B, width, page, num_pages, Hq, Hkv, G, TQ, causal;
  float scale_log2;
  void* out;   // [T, Hq, D]
  float* lse;  // [T, Hq], may be null
  float* ws_o;        // [2 * PA_CTAS][256][D]
  float2* ws_ml;      // [2 * PA_CTAS][256]
  PagedSplit* splits;  // [PA_CTAS]
};

// One request's place: token rows [q0, q0 + n) and kv keys.  Lengths that do
// not fit the tensors are cut (and reported once, by CTA 0).
STD_DEV void paged_request(const PagedAttnParams& p, int b, int& q0, int& n, int& kv) {
  q0 = __ldg(p.cu_q + b);
  const int q1 = __ldg(p.cu_q + b + 1);
  kv = __ldg(p.kv_lens + b);
  n = q1 - q0;
  if (q0 < 0 || q1 > p.T || n < 0) n = 0;
  const int room = p.width * p.page;
  kv = kv < 0 ? 0 : (kv > room ? room : kv);
}
STD_DEV bool paged_request_bad(const PagedAttnParams& p, int b) {
  const int q0 = p.cu_q[b], q1 = p.cu_q[b + 1], kv = p.kv_lens[b];
  return q0 < 0 || q1 > p.T || q1 < q0 || kv < 0 || kv > p.width * p.page;
}
// Item i of a request: its tokens, the last key that any of them sees (+1).
STD_DEV void paged_item(const PagedAttnParams& p, int n, int kv, int i, int& t0, int& nt, int& limit, int& nb, int& w) {
  t0 = i * 2 * p.TQ;
  nt = min(2 * p.TQ, n - t0);
  limit = p.causal ? max(0, kv - n + t0 + nt) : kv;
  nb = max(1, (limit + PA_BN - 1) / PA_BN);
  w = nt > p.TQ ? PA_W2 : PA_W1;
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

// A CTA's walk over the pieces of its share.
struct PagedWalk {
  int b, h, i;         // current item
  int q0, n, kv, items;
  long long skip;      // cost of the item that earlier CTAs did
  long long rem;       // cost left in this CTA's share
  // the current piece
  int t0, nt, limit, nb, w, j0, j1;
  long long cut;       // cost of the item up to the end of this piece

  STD_DEV void request(const PagedAttnParams& p) {
    paged_request(p, b, q0, n, kv);
    items = (n + 2 * p.TQ - 1) / (2 * p.TQ);
  }
  // Advance to the next non-empty piece; false at the end of the share.
  STD_DEV bool next(const PagedAttnParams& p) {
    while (rem > 0) {
      while (items == 0 || i >= items) {  // next head, then next request
        i = 0;
        if (items == 0 || ++h >= p.Hkv) {
          h = 0;
          if (++b >= p.B) return false;
          request(p);
        }
      }
      paged_item(p, n, kv, i, t0, nt, limit, nb, w);
      const long long cost = static_cast<long long>(nb) * w;
      const long long end = min(cost, skip + rem);
      j0 = static_cast<int>((skip + w - 1) / w);
      j1 = static_cast<int>((end + w - 1) / w);
      rem -= end - skip;
      skip = 0;
      cut = end;
      ++i;
      if (j1 > j0) return true;
    }
    return false;
  }
};

template <typename T>
__host__ __device__ constexpr uint32_t paged_idesc(int M, int N, int b_mn_major);
template <>
__host__ __device__ constexpr uint32_t paged_idesc<__nv_bfloat16>(int M, int N, int b_mn_major) {
  return idesc_bf16_f32(M, N, 0, b_mn_major);
}
template <>
__host__ __device__ constexpr uint32_t paged_idesc<__half>(int M, int N, int b_mn_major) {
  // A and B formats 0 = fp16
  return idesc_bf16_f32(M, N, 0, b_mn_major) & ~((1u << 7) | (1u << 10));
}

STD_DEV void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(PA_THREADS, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const PagedAttnParams p) {
  typedef PagedTile<D> Tile;
  constexpr int ST = Tile::stages;
  constexpr int HALVES = D / 64;
  constexpr uint32_t T_O = 256;  // TMEM: S of stream s (P over it) at 128 s, O at 256 + 128 s
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                     // [2][q_bytes]
  uint8_t* sKV = smem + 2 * Tile::q_bytes;  // [ST][kv_bytes]
  __shared__ __align__(8) uint64_t bar_q_full[2], bar_q_empty[2], bar_full[ST], bar_empty[ST], bar_s[2], bar_p[2],
      bar_o[2], bar_join, bar_joined, bar_piece[PA_PIECES], bar_taken[PA_PIECES], bar_end;
  __shared__ PagedPiece s_piece[PA_PIECES];
  __shared__ uint32_t s_tmem;
  __shared__ float s_m[128], s_l[128];
  __shared__ long long s_warp[PA_THREADS / 32], s_off;
  __shared__ int s_b;

  if (tid == 256) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_q_full[i], 1);
      mbar_init(&bar_q_empty[i], 1);
      mbar_init(&bar_s[i], 1);
      mbar_init(&bar_p[i], 4);
      mbar_init(&bar_o[i], 1);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_empty[i], 1);
    }
    for (int i = 0; i < PA_PIECES; ++i) {
      mbar_init(&bar_piece[i], 1);
      mbar_init(&bar_taken[i], 10);  // the warps that read it
    }
    mbar_init(&bar_join, 4);
    mbar_init(&bar_joined, 4);
    mbar_init(&bar_end, 1);
    fence_barrier_init();
    prefetch_tensormap(&tmQ);
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
    s_b = -1;
  }
  pdl_wait();
  if (warp == 9) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }

  // ---------------- this CTA's share of the blocks ----------------
  // cost of a request: its items' blocks, for all KV heads.  Requests of
  // several items are summed by the whole warp.
  auto request_cost = [&](int b) -> long long {
    int q0 = 0, n = 0, kv = 0;
    if (b < p.B) {
      paged_request(p, b, q0, n, kv);
      if (cta == 0 && paged_request_bad(p, b)) std_set_error(STD_DEVERR_LENGTH);
    }
    const int items = (n + 2 * p.TQ - 1) / (2 * p.TQ);
    int t0, nt, limit, nb, w;
    long long cost = 0;
    if (items == 1) {
      paged_item(p, n, kv, 0, t0, nt, limit, nb, w);
      cost = static_cast<long long>(nb) * w;
    }
    for (uint32_t many = __ballot_sync(0xffffffffu, items > 1); many != 0; many &= many - 1) {
      const int src = __ffs(many) - 1;
      const int n_ = __shfl_sync(0xffffffffu, n, src), kv_ = __shfl_sync(0xffffffffu, kv, src);
      const int items_ = __shfl_sync(0xffffffffu, items, src);
      long long sum = 0;
      for (int i = lane; i < items_; i += 32) {
        paged_item(p, n_, kv_, i, t0, nt, limit, nb, w);
        sum += static_cast<long long>(nb) * w;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == src) cost = sum;
    }
    return cost * p.Hkv;
  };
  long long total = 0, mine = 0, before = 0;  // before: cost of the requests ahead of this thread's
  for (int b0 = 0; b0 < p.B; b0 += PA_THREADS) {
    mine = request_cost(b0 + tid);
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    before = total + inc - mine;
    for (int w = 0; w < PA_THREADS / 32; ++w) {
      if (w < warp) before += s_warp[w];
      total += s_warp[w];
    }
    __syncthreads();
  }
  long long share = (total + PA_CTAS - 1) / PA_CTAS;
  share = max(share, static_cast<long long>(2 * PA_W2));
  const long long x0 = share * cta;
  if (x0 < total) {
    if (p.B <= PA_THREADS) {
      if (x0 >= before && x0 < before + mine) {
        s_b = tid;
        s_off = x0 - before;
      }
    } else {  // a second pass over the requests, in chunks
      long long run = 0;
      for (int b0 = 0; b0 < p.B; b0 += PA_THREADS) {
        const long long c = request_cost(b0 + tid);
        long long inc = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long u = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += u;
        }
        if (lane == 31) s_warp[warp] = inc;
        __syncthreads();
        long long at = run + inc - c;
        for (int w = 0; w < PA_THREADS / 32; ++w) {
          if (w < warp) at += s_warp[w];
          run += s_warp[w];
        }
        if (x0 >= at && x0 < at + c) {
          s_b = b0 + tid;
          s_off = x0 - at;
        }
        __syncthreads();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  // Dependents may launch only once this CTA holds its TMEM (verify_attn.cu).
  pdl_launch_dependents();

  // The next piece; false when there is none (or its wait ran out).
  auto next_piece = [&](uint32_t& n, PagedPiece& piece) -> bool {
    const int i = n % PA_PIECES;
    if (!__all_sync(0xffffffffu, mbar_wait(&bar_piece[i], (n / PA_PIECES) & 1))) return false;
    piece = s_piece[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar_taken[i]);
    ++n;
    return piece.nblk > 0;
  };

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PA_REGS_SOFTMAX));
    // ---------------- softmax warpgroups: thread = row ----------------
    const int s = warp >> 2, r = tid & 127;
    const uint32_t trow = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t tS = trow + s * 128, tO = trow + T_O + s * 128;
    const int rt = r / p.G, rg = r % p.G;  // token and head of this row in its tile
    const float sc = p.scale_log2;
    uint32_t npiece = 0, ns = 0, no = 0, nj = 0;  // pieces, steps, results and joins so far
    bool ok = true;
    PagedPiece piece;
    while (ok && next_piece(npiece, piece)) {
      const int nblk = piece.nblk;
      const bool pair = piece.tokens > p.TQ;
      const int tile = pair ? s : 0;
      const int t = tile * p.TQ + rt;  // token of the item
      const bool valid_row = rt < p.TQ && t < piece.tokens;
      const int tile_rows = min(p.TQ, piece.tokens - tile * p.TQ) * p.G;
      const bool live = (warp & 3) * 32 < tile_rows;  // warps without rows only keep the barriers going
      const int limit = p.causal ? min(piece.limit, piece.first + t) : piece.limit;
      const int steps = pair ? nblk : (nblk - s + 1) >> 1;
      float m_run = -INFINITY, l_run = 0.f;
      for (int k = 0; k < steps; ++k, ++ns) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bar_s[s], ns & 1));
        if (!ok) break;
        if (live) {
          tc_fence_after();
          uint32_t x[PA_BN];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, x + c * 32);
          tmem_wait_ld();
          const int nvis = limit - (piece.j0 + (pair ? k : 2 * k + s)) * PA_BN;  // visible keys of this block
          float mx = -INFINITY;
          if (__any_sync(0xffffffffu, nvis < PA_BN)) {
#pragma unroll
            for (int j = 0; j < PA_BN; ++j) {
              if (j >= nvis) x[j] = 0xff800000u;  // -inf
              mx = fmaxf(mx, __uint_as_float(x[j]));
            }
          } else {
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < PA_BN; j += 4)
#pragma unroll
              for (int c = 0; c < 4; ++c) m4[c] = fmaxf(m4[c], __uint_as_float(x[j + c]));
            mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          }
          const float m_c = mx * sc;  // scale > 0
          // This block's S is issued after the stream's previous P V, and its
          // barrier covers all MMAs before it: O is at rest here.
          const bool need = m_run != -INFINITY && m_c > m_run + PA_RESCALE;
          if (__any_sync(0xffffffffu, need)) {
            const float alpha = need ? exp2f(m_run - m_c) : 1.0f;
            uint32_t o[32];
#pragma unroll
            for (int piece = 0; piece < D / 32; ++piece) {
              tmem_ld32(tO + piece * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
              tmem_st32(tO + piece * 32, o);
            }
            if (need) {
              l_run *= alpha;
              m_run = m_c;
            }
          }
          if (m_run == -INFINITY) m_run = m_c;
          // a row that has seen no key yet: exp2(-inf + 0) = 0 everywhere
          const float nm = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[32];
            float l0 = 0.f, l1 = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float e0 = ex2_approx(fmaf(__uint_as_float(x[c * 64 + 2 * j]), sc, nm));
              const float e1 = ex2_approx(fmaf(__uint_as_float(x[c * 64 + 2 * j + 1]), sc, nm));
              l0 += e0;
              l1 += e1;
              pk[j] = pack_pair<T>(e0, e1);
            }
            l_run += l0 + l1;
            tmem_st32(tS + c * 32, pk);
          }
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_p[s]);
      }
      // ---- the item's result ----
      if (ok && steps > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bar_o[s], no++ & 1));
      if (!ok) break;
      float wa = 1.f, wb = 0.f, m = m_run, l = l_run;
      bool join = false;
      if (!pair) {
        // stream 1, its last product done, hands (m, l) to stream 0, which
        // reads both accumulators
        if (s == 1) {
          s_m[r] = m_run;
          s_l[r] = l_run;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_join);
        } else {
          ok = __all_sync(0xffffffffu, mbar_wait(&bar_join, nj & 1));
          if (!ok) break;
          const float mB = s_m[r], lB = s_l[r];
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
        const bool seen = l != 0.f, seen_a = l_run != 0.f, seen_b = join && s_l[r] != 0.f;
        const float inv = whole && seen ? 1.f / l : 1.f;
        const int token = piece.token0 + t;
        const int head = piece.h * p.G + rg;
        const size_t orow = static_cast<size_t>(token) * p.Hq + head;
        const size_t slot = static_cast<size_t>(whole ? 0 : piece.slot) * 256 + tile * 128 + r;
#pragma unroll
        for (int piece = 0; piece < D / 32; ++piece) {
          uint32_t oa[32];
          float v[32];
          tmem_ld32(tO + piece * 32, oa);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = seen_a ? __uint_as_float(oa[j]) * wa : 0.f;
          if (join) {
            tmem_ld32(tO + 128 + piece * 32, oa);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += seen_b ? __uint_as_float(oa[j]) * wb : 0.f;
          }
          if (valid_row) {
            if (whole) {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + orow * D + piece * 32);
#pragma unroll
              for (int c = 0; c < 4; ++c)
                dst[c] = make_uint4(pack_pair<T>(v[8 * c] * inv, v[8 * c + 1] * inv),
                                    pack_pair<T>(v[8 * c + 2] * inv, v[8 * c + 3] * inv),
                                    pack_pair<T>(v[8 * c + 4] * inv, v[8 * c + 5] * inv),
                                    pack_pair<T>(v[8 * c + 6] * inv, v[8 * c + 7] * inv));
            } else {
              float4* dst = reinterpret_cast<float4*>(p.ws_o + slot * D + piece * 32);
#pragma unroll
              for (int c = 0; c < 8; ++c)
                dst[c] = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
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
          if (lane == 0) mbar_arrive(&bar_joined);
        } else {
          ok = __all_sync(0xffffffffu, mbar_wait(&bar_joined, nj & 1));
        }
        ++nj;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_REGS_OTHER));
    if (warp == 8) {
      // ---------------- TMA producer: the whole warp, a page per lane ----------------
      const int box = min(p.page, PA_BN);          // rows per copy
      const int per_block = PA_BN / box;           // copies per block
      const uint32_t copy_bytes = box * D * 2;
      const int groups = p.page / 8;               // 8-row groups per page and head
      uint32_t nld = 0, nq = 0;                    // loads and Q tiles issued
      uint32_t np = 0;
      bool ok = true;
      PagedPiece piece;
      while (ok && next_piece(np, piece)) {
        const int32_t* row = p.table + static_cast<size_t>(piece.b) * p.width;
        const int nblk = piece.nblk, limit = piece.limit;
        const bool pair = piece.tokens > p.TQ;
        // queries
        for (int s = 0; ok && s < (pair ? 2 : 1); ++s, ++nq) {
          const int st = nq & 1;
          if (nq >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&bar_q_empty[st], ((nq >> 1) - 1) & 1));
          if (ok && lane == 0) {
            mbar_arrive_expect_tx(&bar_q_full[st], p.TQ * p.G * D * 2);
            for (int hf = 0; hf < HALVES; ++hf)
              tma_load_4d(sQ + st * Tile::q_bytes + hf * 16384, &tmQ, &bar_q_full[st], hf * 64, 0, piece.h,
                          piece.token0 + s * p.TQ);
          }
        }
        // the page of copy `lane` of block j (the copies of one page share it)
        auto page_of = [&](int j) -> int {
          const int key = j * PA_BN + lane * box;
          if (lane >= per_block || j >= piece.j0 + nblk || key >= limit) return 0;
          const int id = __ldg(row + key / p.page);
          if (id < 0 || id >= p.num_pages) {
            std_set_error(STD_DEVERR_BOUNDS);
            return p.num_pages;  // past the pool: TMA fills zeros
          }
          return id;
        };
        auto load = [&](const CUtensorMap* map, int j, int id) {
          const int st = nld % ST;
          if (nld >= ST) ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar_empty[st], ((nld / ST) - 1) & 1));
          if (!ok) return;
          const int left = limit - j * PA_BN;
          const int copies = left <= 0 ? 0 : min(per_block, (left + box - 1) / box);
          if (lane == 0) mbar_arrive_expect_tx(&bar_full[st], copies * copy_bytes);
          __syncwarp();
          if (lane < copies) {
            const int key = j * PA_BN + lane * box;
            const int g = (id * p.Hkv + piece.h) * groups + (key % p.page) / 8;
            tma_load_4d(sKV + st * Tile::kv_bytes + lane * copy_bytes, map, &bar_full[st], 0, 0, 0,
                        id >= p.num_pages ? p.num_pages * p.Hkv * groups : g);
          }
          ++nld;
        };
        int id0 = page_of(piece.j0), id1 = page_of(piece.j0 + 1);
        if (ok) load(&tmK, piece.j0, id0);
        for (int k = 0; ok && k < nblk; ++k) {
          const int j = piece.j0 + k;
          const int id2 = page_of(j + 2);
          // a single reads K one block ahead (its two streams start on two blocks)
          if (!pair && k + 1 < nblk) load(&tmK, j + 1, id1);
          if (ok) load(&tmV, j, id0);
          if (ok && pair && k + 1 < nblk) load(&tmK, j + 1, id1);
          id0 = id1;
          id1 = id2;
        }
      }
      // never leave a copy in flight
      for (uint32_t c = nld < ST ? 0 : nld - ST; c < nld; ++c) mbar_wait(&bar_full[c % ST], (c / ST) & 1);
      for (uint32_t c = nq < 2 ? 0 : nq - 2; c < nq; ++c) mbar_wait(&bar_q_full[c & 1], (c >> 1) & 1);
    } else if (warp == 9) {
      // ---------------- MMA issuer (lane 0; the warp clears V rows) ----------------
      constexpr uint32_t idS = paged_idesc<T>(128, PA_BN, 0);
      constexpr uint32_t idO = paged_idesc<T>(128, D, 1);
      uint32_t ld0 = 0, q0 = 0, np[2] = {0, 0};
      uint32_t npiece = 0;
      bool ok = true;
      PagedPiece piece;
      while (ok && next_piece(npiece, piece)) {
        const int nblk = piece.nblk;
        const bool pair = piece.tokens > p.TQ;
        const int steps = pair ? 2 * nblk : nblk;
        auto issue_s = [&](int u) {
          const int s = u & 1;
          const int k = pair ? u >> 1 : u;
          const uint32_t c = ld0 + ((pair || k == 0) ? 2 * k : 2 * k - 1), st = c % ST;
          const uint32_t qi = q0 + (pair ? s : 0), qs = qi & 1;
          if (ok && (!pair || s == 0)) ok = mbar_wait(&bar_full[st], (c / ST) & 1);
          if (ok && (u == 0 || (pair && u == 1))) ok = mbar_wait(&bar_q_full[qs], (qi >> 1) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) return;
          tc_fence_after();
          if (lane == 0) {
            // (a descriptor's low bits are the address / 16, so steps are added to it)
            const uint64_t dQ = sdesc_sw128(smem_u32(sQ + qs * Tile::q_bytes), 16, 1024);
            const uint64_t dK = sdesc_sw128(smem_u32(sKV + st * Tile::kv_bytes), 16, HALVES * 1024);
  #pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              umma_bf16(tmem + s * 128, dQ + ((ks >> 2) * 16384 + (ks & 3) * 32) / 16,
                        dK + ((ks >> 2) * 1024 + (ks & 3) * 32) / 16, idS, ks > 0 ? 1u : 0u);
            umma_commit(&bar_s[s]);
            if (!pair || s == 1) umma_commit(&bar_empty[st]);
            if (pair ? u + 2 >= steps : u + 1 == steps) umma_commit(&bar_q_empty[qs]);
          }
          __syncwarp();
        };
        auto issue_pv = [&](int u) {
          const int s = u & 1;
          const int k = pair ? u >> 1 : u;
          const uint32_t c = ld0 + (pair ? 2 * k + 1 : (k + 1 == nblk ? 2 * nblk - 1 : 2 * k + 2)), st = c % ST;
          const int valid = min(PA_BN, piece.limit - (piece.j0 + k) * PA_BN);  // visible keys of the block
          const int ksteps = (valid + 15) >> 4;
          uint8_t* sV = sKV + st * Tile::kv_bytes;
          if (ok && (!pair || s == 0)) {
            ok = mbar_wait(&bar_full[st], (c / ST) & 1);
            if (ok && (valid & 15) != 0) {
              // rows up to the next multiple of 16 that no query sees
              for (int i = lane; i < (ksteps * 16 - valid) * HALVES * 8; i += 32) {
                const int r = valid + i / (HALVES * 8), ch = i % (HALVES * 8);
                *reinterpret_cast<uint4*>(sV + (r >> 3) * (HALVES * 1024) + (ch >> 3) * 1024 + (r & 7) * 128 +
                                          (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
              }
              fence_async_smem();
            }
          }
          if (ok) ok = mbar_wait(&bar_p[s], np[s] & 1);
          ++np[s];
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) return;
          tc_fence_after();
          if (lane == 0) {
            const uint64_t dV = sdesc_sw128(smem_u32(sV), 1024, HALVES * 1024);
  #pragma unroll
            for (int ks = 0; ks < PA_BN / 16; ++ks)
              if (ks < ksteps)
                umma_bf16_ts(tmem + T_O + s * 128, tmem + s * 128 + ks * 8, dV + ks * (HALVES * 2048 / 16), idO,
                             (u >= 2 || ks > 0) ? 1u : 0u);
            if (!pair || s == 1) umma_commit(&bar_empty[st]);
            if (u + 2 >= steps) umma_commit(&bar_o[s]);
          }
          __syncwarp();
        };
        // S runs two steps ahead: S0 S1 PV0 S2 PV1 S3 ...
  #pragma unroll 1
        for (int v = 0; ok && v < steps + 2; ++v) {
          if (v >= 2) issue_pv(v - 2);
          if (ok && v < steps) issue_s(v);
        }
        ld0 += 2 * nblk;
        q0 += pair ? 2 : 1;
      }
      // nothing may be in flight when the CTA gives back its TMEM
      if (lane == 0) {
        umma_commit(&bar_end);
        mbar_wait(&bar_end, 0);
      }
      __syncwarp();
    } else if (warp == 10) {
      // ---------------- scheduler: the pieces of this CTA's share ----------------
      PagedWalk walk;
      walk.b = s_b;
      walk.rem = 0;
      if (s_b >= 0) {
        walk.rem = min(share, total - x0);
        walk.request(p);
        long long off = s_off;
        long long head = 0;  // cost of one KV head of this request
        {
          int t0, nt, limit, nb, w;
          for (int i = lane; i < walk.items; i += 32) {
            paged_item(p, walk.n, walk.kv, i, t0, nt, limit, nb, w);
            head += static_cast<long long>(nb) * w;
          }
    #pragma unroll
          for (int o = 16; o > 0; o >>= 1) head += __shfl_xor_sync(0xffffffffu, head, o);
          walk.h = static_cast<int>(off / head);
          off -= walk.h * head;
          walk.i = 0;
          for (;;) {
            paged_item(p, walk.n, walk.kv, walk.i, t0, nt, limit, nb, w);
            const long long cost = static_cast<long long>(nb) * w;
            if (off < cost) break;
            off -= cost;
            ++walk.i;
          }
        }
        walk.skip = off;
      }
      PagedSplit split = {-1, 0, 0, 0};
      bool more = true;
      for (uint32_t n = 0; more; ++n) {
        more = walk.next(p);
        const int i = n % PA_PIECES;
        if (n >= PA_PIECES && !__all_sync(0xffffffffu, mbar_wait(&bar_taken[i], ((n / PA_PIECES) - 1) & 1))) break;
        if (lane == 0) {
          PagedPiece piece = {walk.b, walk.h, walk.q0 + walk.t0, walk.nt, walk.limit, 0, walk.j0, 0, -1};
          if (more) {
            piece.first = walk.kv - walk.n + walk.t0 + 1;
            piece.nblk = walk.j1 - walk.j0;
            if (walk.j0 > 0 || walk.j1 < walk.nb) piece.slot = 2 * cta + (walk.j0 == 0 ? 1 : 0);
          }
          s_piece[i] = piece;
          mbar_arrive(&bar_piece[i]);
        }
        __syncwarp();
        if (more && walk.j0 == 0 && walk.j1 < walk.nb) {
          // the share ends inside this item: block j lies with the CTA whose share
          // holds cost j * w of the item
          const long long start = x0 + share - walk.cut;
          split.last_cta = static_cast<int>((start + static_cast<long long>(walk.nb - 1) * walk.w) / share);
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

// Joins the pieces of the items that cuts divide: block x looks at the item
// that CTA x's share ends inside.  A warp per row; out = sum_c w_c o_c / sum_c
// w_c l_c with w_c = exp2(m_c - max m), pieces in CTA order.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedAttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int cta = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedSplit sp = p.splits[cta];
  if (sp.last_cta <= cta) return;
  const int n = sp.last_cta - cta + 1;
  constexpr int PER = D / 32;    // columns per lane
  constexpr int BATCH = 8;
  for (int r = blockIdx.y * 8 + warp; r < 256; r += gridDim.y * 8) {
    const int rt = (r & 127) / p.G, t = (r >> 7) * p.TQ + rt;
    if (rt >= p.TQ || t >= sp.tokens) continue;
    // piece i is CTA cta + i's: its continued item (slot 0), or for the first the item begun there (slot 1)
    const size_t row0 = static_cast<size_t>(2 * cta) * 256 + r;
    auto at = [&](int i) { return row0 + static_cast<size_t>(2 * i + (i == 0 ? 1 : 0)) * 256; };
    float m = -INFINITY;
    for (int i = lane; i < n; i += 32) m = fmaxf(m, __ldcg(p.ws_ml + at(i)).x);
    m = warp_max(m);
    float l = 0.f, acc[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) acc[k] = 0.f;
    for (int i0 = 0; i0 < n; i0 += BATCH) {
      float2 ml[BATCH];
      float o[BATCH][PER];
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        ml[j] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int k = 0; k < PER; ++k) o[j][k] = 0.f;
        if (i0 + j < n) {
          ml[j] = __ldcg(p.ws_ml + at(i0 + j));
          const float* src = p.ws_o + at(i0 + j) * D + lane * PER;
          if constexpr (PER == 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
            o[j][0] = v.x, o[j][1] = v.y, o[j][2] = v.z, o[j][3] = v.w;
          } else {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
            o[j][0] = v.x, o[j][1] = v.y;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        if (ml[j].y == 0.f) continue;  // a piece in which the row sees no key
        const float w = exp2f(ml[j].x - m);
        l += w * ml[j].y;
#pragma unroll
        for (int k = 0; k < PER; ++k) acc[k] += w * o[j][k];
      }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const size_t orow = static_cast<size_t>(sp.token0 + t) * p.Hq + sp.kvh * p.G + (r & 127) % p.G;
    T* dst = static_cast<T*>(p.out) + orow * D + lane * PER;
    if constexpr (PER == 4)
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(pack_pair<T>(acc[0] * inv, acc[1] * inv), pack_pair<T>(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack_pair<T>(acc[0] * inv, acc[1] * inv);
    if (lane == 0 && p.lse != nullptr)
      p.lse[orow] = l != 0.f ? (m + log2f(l)) * 0.69314718055994530942f : -INFINITY;
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
static int paged_attn_launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                             const stdb::PagedAttnParams& p, cudaStream_t s) {
  static SmemGrant grant;
  if (ensure_smem(stdb::paged_attn_kernel<T, D>, grant, stdb::PagedTile<D>::smem) != 0) return 3;
  if (launch_pdl(stdb::paged_attn_kernel<T, D>, dim3(stdb::PA_CTAS), dim3(stdb::PA_THREADS), stdb::PagedTile<D>::smem,
                 s, tq, tk, tv, p) != cudaSuccess)
    return 4;
  // rows that an item can have: all of a pair's 256, or those of all the tokens there are
  const int rows = p.T > p.TQ ? 256 : p.T * p.G;
  const dim3 mgrid(stdb::PA_CTAS, rows >= 64 ? 8 : (rows + 7) / 8);
  if (launch_pdl(stdb::paged_merge_kernel<T, D>, mgrid, dim3(256), 0, s, p) != cudaSuccess) return 4;
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

extern "C" int std_paged_attn(const void* q, const void* k_pages, const void* v_pages, const int32_t* block_table,
                              const int32_t* cu_q, const int32_t* kv_lens, int T, int B, int Hq, int Hkv, int D,
                              int is_fp16, int num_pages, int page_size, int max_blocks, int causal, float scale,
                              void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  if ((D != 64 && D != 128) || T < 0 || B <= 0 || B > STD_PAGED_MAX_REQUESTS || Hkv <= 0 || Hkv > 65535 || Hq <= 0 || Hq % Hkv != 0 ||
      Hq / Hkv > 128 || num_pages <= 0 || max_blocks <= 0 || !paged_page_ok(page_size))
    return 1;
  if (!(scale > 0.f) || !(scale < 3.4e38f)) return 1;
  // int32 indexes: keys of a request, slots, 8-row groups of the pool (one page more: the zero fill)
  if (static_cast<long long>(max_blocks) * page_size > 0x7fffffffll - 1024 ||
      static_cast<long long>(num_pages) * page_size > 0x7fffffffll ||
      (static_cast<long long>(num_pages) + 1) * Hkv * (page_size / 8) > 0x7fffffffll || T > 0x7fffffff / 2)
    return 1;
  if (T == 0) return 0;
  if (q == nullptr || k_pages == nullptr || v_pages == nullptr || block_table == nullptr || cu_q == nullptr ||
      kv_lens == nullptr || out == nullptr || q == out)
    return 1;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out)) return 1;
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < std_paged_attn_workspace_bytes(D)) return 5;
  const int G = Hq / Hkv, TQ = 128 / G;
  CUtensorMap tq, tk, tv;
  {
    const uint64_t e = 2, row = static_cast<uint64_t>(D) * e;
    const uint64_t qd[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(G), static_cast<uint64_t>(Hkv),
                            static_cast<uint64_t>(T)};
    const uint64_t qs[3] = {row, row * G, row * Hq};
    const uint32_t qb[4] = {64, static_cast<uint32_t>(G), 1, static_cast<uint32_t>(TQ)};
    int rc = paged_tmap_4d(&tq, is_fp16, q, qd, qs, qb);
    if (rc != 0) return rc;
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
  p.page = page_size;
  p.num_pages = num_pages;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = G;
  p.TQ = TQ;
  p.causal = causal != 0 ? 1 : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = out;
  p.lse = lse;
  char* ws = static_cast<char*>(workspace);
  p.ws_o = reinterpret_cast<float*>(ws);
  p.ws_ml = reinterpret_cast<float2*>(ws + paged_ws_o_bytes(D));
  p.splits = reinterpret_cast<stdb::PagedSplit*>(ws + paged_ws_o_bytes(D) + paged_ws_ml_bytes());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (D == 128)
    return is_fp16 ? paged_attn_launch<__half, 128>(tq, tk, tv, p, s)
                   : paged_attn_launch<__nv_bfloat16, 128>(tq, tk, tv, p, s);
  return is_fp16 ? paged_attn_launch<__half, 64>(tq, tk, tv, p, s)
                 : paged_attn_launch<__nv_bfloat16, 64>(tq, tk, tv, p, s);
}
