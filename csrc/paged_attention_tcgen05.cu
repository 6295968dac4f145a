// Attention of portions of new tokens over a paged key / value cache, for sm_100a on tcgen05 tensor cores.
//
//   o[i, h] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q[i, h] . k_j - max),   j up to token i of the row
//
// A tile of 128 query rows holds consecutive new tokens of one row with all query heads of a group (token, head), so that a key head's
// pages are read once for the whole group and short portions fill tiles too.  A CTA works on two tiles that share the K / V stream and
// ping-pong on the tensor cores, as in gqa_attention_tcgen05.cu: one query row per soft-max thread, P overwrites S in tensor memory and is
// the A operand of P V (rounded to bf16, the type of the other operand; outputs are 0.0020 to 0.0022 off 64 bits, relative, where their own rounding makes 0.0016), O stays in tensor memory and is rescaled only when the running maximum grows by more than 2^8.
// Bound by the chain of a tile's block, scores -> soft-max -> P V, of which two overlap (2.4 us a pair of blocks of 128 keys and 128 dimensions, 1.1 of them
// products), and in it by the soft-max warps' instructions: an eighth of the exponentials as polynomials on the FMA lanes takes 3 % longer, half of them 19 %,
// and a P V that begins under the last exponentials gains nothing.  32 / 8 heads of 128, whole calls: 1,000 tokens behind 15,000 (255 GFLOP) 247 us = 1,030 TFLOP/s, 0.6
// of the library product's rate; six prompts of 300 to 2,500 tokens (96 GFLOP) 167 us = 575 (162 before scores of any size were told apart), which counts no product of a block that the diagonal halves and all beginnings and
// ends of pieces.  Two soft-max threads a row took 180 us for the latter (from 153), products cut to the diagonal's columns 176 (from 164).
//
// Rows, portions and caches are of any length, so work is dealt out in key blocks: all (row, key head, pair of tiles), each as long as the keys
// that its last token sees and PC_PIECE more for its beginning and end, form one line, and each of 148 CTAs takes an equal stretch of it (272 -> 155 us for the
// six prompts against pairs dealt out by blocks alone).  The roles of a CTA run through the pieces of the stretch independently, so the loads and the first
// scores of the next piece overlap the end of this one.  A pair of tiles that CTAs share leaves fp32 sums in scratch slots, joined by a second launch in the
// order of the line: results do not depend on timing.
// A block on the diagonal, or with the row's last key, holds values that some or all rows of the tiles must not see: a probability of zero does not
// keep a NaN or an infinity out of a product.  Two warps of their own clear such values in shared memory before the product (those that no row
// sees altogether), and a query that does see them adds them to its output at the end; 5 us of the six prompts'.
// Pairs whose second tile is empty (few tokens of a wide group) have one chain under way: 8 rows of 5,000 keys, two tokens each on 52 / 4 heads of 128 39 us = 2.1 TB/s,
// four on 32 / 4 of 64 33 us = 1.2 TB/s.
// Every wait is bounded, whole warps give one up together, and the CTA then unwinds with the status word set; no load uses cluster multicast.
#include "paged_common.cuh"

namespace ats {

constexpr int PC_CTAS = 148;
constexpr int PC_PIECE = 192;    // keys that take as long as the first loads and scores and the outputs of a pair of tiles (4 us, a block of 128 keys 2.4 us)
constexpr int PC_THREADS = 384;  // soft-max A (warps 0-3), soft-max B (4-7), TMA (8), MMA (9), values of blocks on the diagonal (10, 11)

struct PagedPortionArgs {
  PagedRows rows;
  const __nv_bfloat16* v_pages;
  __nv_bfloat16* out;       // [tokens, ldo]
  long long ldo;
  int n_kv, rep, limit;     // rows with more than `limit` query rows (new tokens times rep) are taken
  int tile;                 // tokens of a tile: 128 / rep
  int ctas;
  int zero_tail;            // tokens behind the last row get zeros
  int wide;                 // output rows begin at multiples of 32 bytes
  float scale_log2;
  unsigned long long* total;   // the length of the line
  struct PcPlace* begins;      // [ctas]: where the CTAs' stretches begin
  float* part_o;            // [ctas, 2, 256, D]
  float* part_ml;           // [ctas, 2, 256, 2]
  int* status;
};

// A place on the line: pair `k` of tiles of (row, key head), which begins at `base`.
struct PcPlace {
  int row, hk, k, pad;
  unsigned long long base, pad2;
  __device__ __forceinline__ void find(const PagedPortionArgs& p, int r, unsigned long long row_base, unsigned long long x);   // x within row r
};

constexpr int PC_EDGE = 4;   // blocks of a piece with values that not every row sees: 256 tokens touch three

template <int D>
struct PagedPortionSmem {
  static constexpr int T = D * 256;   // 128 rows
  static constexpr int STAGES = D == 64 ? 4 : 2;
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = 2 * T;
  static constexpr int V_OFF = K_OFF + STAGES * T;
  static constexpr int BAR_OFF = V_OFF + STAGES * T;
  static constexpr int TOTAL = BAR_OFF + 512 + 1024;
};

// The length of pairs of tiles 0 .. k - 1 of a row, each seeing the keys up to its last token (`at` tokens before the portion, `pair` tokens a pair).
__device__ __forceinline__ unsigned long long pc_before(unsigned long long k, unsigned at, unsigned pair) { return k * (at + PC_PIECE) + pair * (k * (k + 1) / 2); }

struct PcRow {
  int first, fresh, keys, at, pairs;
  unsigned long long cost;   // of one key head; 0: the row is empty or another kernel's
  __device__ __forceinline__ PcRow(const PagedPortionArgs& p, int r) {
    paged_row(p.rows, r, &first, &fresh, &keys);
    at = max(keys - fresh, 0);
    const int pair = 2 * p.tile;
    pairs = (long long)fresh * p.rep > p.limit ? (fresh + pair - 1) / pair : 0;
    cost = pairs ? pc_before(pairs - 1, at, pair) + PC_PIECE + at + fresh : 0;
  }
};

// The line shared out: one key more to each of the first `extra` CTAs, and no CTA for less than two blocks.
struct PcShares {
  unsigned long long n, each, extra;
  __device__ __forceinline__ PcShares(const PagedPortionArgs& p, unsigned long long total) {
    n = min((unsigned long long)p.ctas, (total + 255) / 256);
    each = n ? total / n : 0;
    extra = total - each * n;
  }
  __device__ __forceinline__ unsigned long long begin(unsigned long long c) const { return c * each + min(c, extra); }
};

__device__ __forceinline__ void PcPlace::find(const PagedPortionArgs& p, int r, unsigned long long row_base, unsigned long long x) {
  const PcRow w(p, r);
  row = r;
  hk = int((x - row_base) / w.cost);
  base = row_base + hk * w.cost;
  int lo = 0, hi = w.pairs;   // the last pair that begins at or before x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pc_before(mid, w.at, 2 * p.tile) <= x - base) lo = mid;
    else hi = mid;
  }
  k = lo;
  base += pc_before(lo, w.at, 2 * p.tile);
}
// The first key block of a pair that begins at `base` behind place x of the line; `blocks` of them from its end on.
__device__ __forceinline__ int pc_block(unsigned long long base, unsigned long long x, int seen, int blocks) {
  if (x >= base + PC_PIECE + seen) return blocks;
  return x > base + PC_PIECE ? int((x - base - PC_PIECE) >> 7) : 0;
}

// A piece: key blocks [j0, j1) of a pair of tiles (none: the stretch has ended).
struct PcPiece {
  int row, hk, first, fresh, keys, tok0;   // tok0: first token of tile A within the portion
  int j0, j1, blocks;                      // of all the pair's blocks
  int n[2];                                // blocks that the tiles see
  bool opens;                              // the piece that the CTA's stretch begins with
  __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == blocks; }
  __device__ __forceinline__ int end(int x) const { return min(j1, n[x]); }
  // the last key that every row of the piece sees, and the first block with others
  __device__ __forceinline__ int open(const PagedPortionArgs& p) const { return keys - fresh + tok0 + (end(0) > j0 ? 0 : p.tile); }
  __device__ __forceinline__ int edge(const PagedPortionArgs& p) const { return max(open(p) + 1, 0) >> 7; }
};

struct PcWalk {
  const PagedPortionArgs& p;
  PcPlace at;
  unsigned long long lo, hi;
  PcRow w;   // of row at.row: a piece of the row before costs no loads
  __device__ __forceinline__ PcWalk(const PagedPortionArgs& args, const PcPlace& start, unsigned long long from, unsigned long long to)
      : p(args), at(start), lo(from), hi(to), w(args, min(start.row, args.rows.R - 1)) {}
  __device__ __forceinline__ bool next(PcPiece& s) {
    while (at.base < hi) {
      if (w.cost == 0) {
        w = PcRow(p, ++at.row);
        continue;
      }
      const int pair = 2 * p.tile, seen = w.at + min((at.k + 1) * pair, w.fresh);
      s.row = at.row; s.hk = at.hk; s.first = w.first; s.fresh = w.fresh; s.keys = w.keys; s.tok0 = at.k * pair;
      s.blocks = (seen + 127) >> 7;
      s.opens = at.base <= lo;
      s.j0 = pc_block(at.base, lo, seen, s.blocks);
      s.j1 = pc_block(at.base, hi, seen, s.blocks);
      s.n[0] = (w.at + min(s.tok0 + p.tile, w.fresh) + 127) >> 7;
      s.n[1] = s.tok0 + p.tile < w.fresh ? s.blocks : 0;
      at.base += PC_PIECE + seen;
      if (++at.k == w.pairs) {
        at.k = 0;
        if (++at.hk == p.n_kv) {
          at.hk = 0;
          if (at.base < hi) w = PcRow(p, ++at.row);   // (a row is to come)
        }
      }
      if (s.j0 < s.j1) return true;
    }
    return false;
  }
};

template <int D>
__global__ void __launch_bounds__(PC_THREADS, 1) paged_portion_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                      const __grid_constant__ CUtensorMap map_v, const PagedPortionArgs p) {
  using SM = PagedPortionSmem<D>;
  constexpr int T = SM::T, DC = D / 64, ST = SM::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem + SM::Q_OFF;
  uint8_t* sK = smem + SM::K_OFF;
  uint8_t* sV = smem + SM::V_OFF;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::BAR_OFF);
  uint64_t* q_full = bars;              // 1
  uint64_t* q_empty = bars + 1;         // 1: all scores of a piece are done
  uint64_t* k_full = bars + 2;          // [ST]
  uint64_t* k_empty = bars + 6;         // [ST]
  uint64_t* v_full = bars + 10;         // [ST], 2 arrivals
  uint64_t* v_empty = bars + 14;        // [ST]
  uint64_t* v_raw = bars + 18;          // [ST]: values that not every row sees have landed
  uint64_t* s_full = bars + 22;         // [2] per tile
  uint64_t* p_full = bars + 24;         // [2] per tile, 4 arrivals
  uint64_t* o_done = bars + 26;         // [2] per tile: last P V of a piece finished
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 28);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ unsigned long long s_sum[PC_THREADS / 32], s_base;
  __shared__ int s_row;
  // The pieces, told by the producer, which writes a place again when all that read it have said so (nothing else holds it back for the soft-max warps of
  // a tile without keys or the clearing warps of a piece without a diagonal block).
  __shared__ PcPiece s_piece[8];
  __shared__ uint64_t s_told[8], s_through[8];
  // of each: keys whose values the two clearing warps cleared, 128 bits a block from the first block on the diagonal on
  __shared__ uint32_t s_cleared[8][2][PC_EDGE * 4], s_any[8][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PagedRows& rows = p.rows;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (tid == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int x = 0; x < ST; ++x) {
      mbar_init(&v_raw[x], 1);
      mbar_init(&k_full[x], 1);
      mbar_init(&k_empty[x], 1);
      mbar_init(&v_full[x], 2);
      mbar_init(&v_empty[x], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 4);
      mbar_init(&o_done[x], 1);
    }
    for (int x = 0; x < 8; ++x) {
      mbar_init(&s_told[x], 1);
      mbar_init(&s_through[x], 11);   // 8 soft-max warps, MMA, 2 clearing warps
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // where the rows begin on the line: every thread sums up a share of the rows
  const int share = (rows.R + PC_THREADS - 1) / PC_THREADS, r0 = min(tid * share, rows.R), r1 = min(r0 + share, rows.R);
  unsigned long long mine = 0;
  for (int r = r0; r < r1; ++r) mine += PcRow(p, r).cost * p.n_kv;
  unsigned long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_sum[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  unsigned long long total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < PC_THREADS / 32; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  const PcShares shares(p, total);
  const unsigned long long lo = shares.begin(blockIdx.x), hi = blockIdx.x < shares.n ? shares.begin(blockIdx.x + 1) : lo;
  for (int r = r0; r < r1; ++r) {
    const unsigned long long n = PcRow(p, r).cost * p.n_kv;
    if (before <= lo && lo < before + n) s_row = r, s_base = before;
    before += n;
  }
  if (blockIdx.x == 0 && tid == 0) *p.total = total;
  if (p.zero_tail) {
    const int tail = min(max(rows.starts[rows.R], 0), rows.tokens), vecs = p.n_kv * p.rep * (D / 8);
    for (long long i = (long long)blockIdx.x * PC_THREADS + tid; i < (long long)(rows.tokens - tail) * vecs; i += (long long)gridDim.x * PC_THREADS)
      *reinterpret_cast<uint4*>(p.out + (tail + i / vecs) * p.ldo + (i % vecs) * 8) = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  PcPlace start = {};
  if (lo < hi) start.find(p, s_row, s_base, lo);
  else start.base = hi;
  if (tid == 0) p.begins[blockIdx.x] = start;
  auto next_piece = [&](uint32_t n) -> const PcPiece* {   // the n-th, until piece_done(n), or null behind the last one (and where a wait ran out)
    if (!mbar_wait_bounded(&s_told[n & 7], (n >> 3) & 1, abort_flag, p.status, kTimeoutFull)) return nullptr;
    const PcPiece* s = &s_piece[n & 7];
    return s->j0 < s->j1 ? s : nullptr;
  };
  auto piece_done = [&](uint32_t n) { mbar_arrive(&s_through[n & 7]); };   // one lane of each warp
  // columns: S_A [0,128)  S_B [128,256)  O_A [256, 256 + D)  O_B [256 + D, 256 + 2 D)

  if (warp == 8) {
    // ------------------------------------------------------------------ producer: a whole warp, a page's copies from a lane each
    const int page = 1 << rows.page_log, box = min(128, page), copies = 128 / box * DC;   // copies of a block
    const int c = lane % DC, at = lane / DC * box;                                         // 64-column piece and first key of this lane's copy
    uint32_t n_blocks = 0, n_pieces = 0;
    bool ok = true;
    PcWalk walk(p, start, lo, hi);
    PcPiece s;
    while (ok) {
      const bool more = walk.next(s);
      if (!more) s.j0 = s.j1 = 0;
      if (!(ok = mbar_wait_warp(&s_through[n_pieces & 7], ((n_pieces >> 3) & 1) ^ 1, abort_flag, p.status, kTimeoutEmpty))) break;
      if (lane == 0) {
        s_piece[n_pieces & 7] = s;
        mbar_arrive(&s_told[n_pieces & 7]);
      }
      if (!more) break;
      const int edge = s.edge(p);
      const int* table = rows.tables + (long long)s.row * rows.width;
      const int n_pages = (s.keys + page - 1) >> rows.page_log;
      auto look_up = [&](int j) {
        int row = rows.pages << rows.page_log;   // behind the pages: reads as zero
        const int k = j * 128 + at;
        if (lane < copies && (k >> rows.page_log) < n_pages) {
          const int id = table[k >> rows.page_log];
          if (id >= 0 && id < rows.pages) row = (id << rows.page_log) + (k & (page - 1));
          else atomicCAS(p.status, 0, int(kBadArgument));
        }
        return row;
      };
      int where = look_up(s.j0);
      for (int j = s.j0; j < s.j1; ++j, ++n_blocks) {
        const int here = where, st = n_blocks % ST;
        const uint32_t ph = (n_blocks / ST) & 1;
        if (j + 1 < s.j1) where = look_up(j + 1);
        if (!(ok = mbar_wait_warp(&k_empty[st], ph ^ 1, abort_flag, p.status, kTimeoutEmpty))) break;
        if (lane == 0) mbar_expect_tx(&k_full[st], T);
        __syncwarp();
        if (lane < copies) tma_load_3d(sK + st * T + c * 16384 + at * 128, &map_k, &k_full[st], 64 * c, s.hk, here);
        if (!(ok = mbar_wait_warp(&v_empty[st], ph ^ 1, abort_flag, p.status, kTimeoutEmpty))) break;
        uint64_t* bar = j >= edge ? &v_raw[st] : &v_full[st];
        if (lane == 0) {
          mbar_expect_tx(bar, T);
          if (j < edge) mbar_arrive(bar);
        }
        __syncwarp();
        if (lane < copies) tma_load_3d(sV + st * T + c * 16384 + at * 128, &map_v, bar, 64 * c, s.hk, here);
        if (j == s.j0) {   // the queries, once the last piece's scores are done
          if (!(ok = mbar_wait_warp(q_empty, (n_pieces & 1) ^ 1, abort_flag, p.status, kTimeoutEmpty))) break;
          ++n_pieces;
          if (lane == 0) {
            const bool a = s.end(0) > s.j0, b = s.end(1) > s.j0;
            mbar_expect_tx(q_full, (int(a) + int(b)) * p.tile * p.rep * D * 2);
            for (int x = 0; x < 2; ++x)
              if (x ? b : a)
#pragma unroll
                for (int i = 0; i < DC; ++i) tma_load_3d(sQ + x * T + i * 16384, &map_q, q_full, 64 * i, s.hk * p.rep, s.first + s.tok0 + x * p.tile);
          }
        }
      }
    }
    if (*abort_flag) {  // give copies already in flight time to land before the CTA exits
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 20000ull) {
      }
    }
  } else if (warp == 9) {
    if (lane == 0) {
      // ------------------------------------------------------------------ MMA issuer
      const uint32_t idesc_s = make_idesc(128, 128, 1, 1, 0, 0);
      const uint32_t idesc_o = make_idesc(128, D, 1, 1, 0, 1);
      const uint64_t q_k = make_smem_desc_sw128(smem_u32(sQ), 16, 1024), k_k = make_smem_desc_sw128(smem_u32(sK), 16, 1024);
      const uint64_t v_mn = make_smem_desc_sw128(smem_u32(sV), 16384, 1024);
      auto issue_s = [&](int x, uint32_t st) {
        const uint64_t q_d = desc_advance(q_k, uint32_t(x) * T), k_d = desc_advance(k_k, st * T);
#pragma unroll
        for (int k = 0; k < DC * 4; ++k) {
          const uint32_t off = (k >> 2) * 16384 + (k & 3) * 32;
          tc_mma_f16(tmem_base + x * 128, desc_advance(q_d, off), desc_advance(k_d, off), idesc_s, k != 0);
        }
        tc_commit(&s_full[x]);
      };
      auto issue_pv = [&](int x, uint32_t st, bool fresh_sum) {
        const uint64_t v_d = desc_advance(v_mn, st * T);  // MN-major: value dimension contiguous
#pragma unroll
        for (int k = 0; k < 8; ++k)
          tc_mma_f16_ts(tmem_base + 256 + x * D, tmem_base + x * 128 + k * 8, desc_advance(v_d, k * 2048), idesc_o, !(fresh_sum && k == 0));
      };
      uint32_t n_blocks = 0, n_pieces = 0, n_p[2] = {0, 0};
      bool ok = true;
      while (ok) {
        const PcPiece* told = next_piece(n_pieces);
        if (!told) break;
        const int j0 = told->j0, j1 = told->j1, ends[2] = {told->end(0), told->end(1)};
        ok = mbar_wait_bounded(q_full, n_pieces & 1, abort_flag, p.status, kTimeoutFull);
        ok = ok && mbar_wait_bounded(&k_full[n_blocks % ST], (n_blocks / ST) & 1, abort_flag, p.status, kTimeoutFull);
        if (!ok) break;
        piece_done(n_pieces++);
        tc_fence_after();
        for (int x = 0; x < 2; ++x)
          if (j0 < ends[x]) issue_s(x, n_blocks % ST);
        tc_commit(&k_empty[n_blocks % ST]);
        if (j0 + 1 == j1) tc_commit(q_empty);
        for (int j = j0; j < j1; ++j, ++n_blocks) {
          const uint32_t st = n_blocks % ST, nst = (n_blocks + 1) % ST;
          const bool more = j + 1 < j1;
          if (!(ok = mbar_wait_bounded(&v_full[st], (n_blocks / ST) & 1, abort_flag, p.status, kTimeoutFull))) break;
          for (int x = 0; ok && x < 2; ++x) {
            if (j < ends[x]) {
              if (!(ok = mbar_wait_bounded(&p_full[x], n_p[x] & 1, abort_flag, p.status, kTimeoutTmemFull))) break;
              ++n_p[x];
              tc_fence_after();
              issue_pv(x, st, j == j0);
              if (j + 1 == ends[x]) tc_commit(&o_done[x]);
            }
            if (x == 1) tc_commit(&v_empty[st]);
            if (more) {
              if (x == 0 && !(ok = mbar_wait_bounded(&k_full[nst], ((n_blocks + 1) / ST) & 1, abort_flag, p.status, kTimeoutFull))) break;
              tc_fence_after();
              if (j + 1 < ends[x]) issue_s(x, nst);
              if (x == 1) {
                tc_commit(&k_empty[nst]);
                if (j + 2 == j1) tc_commit(q_empty);
              }
            }
          }
          if (!ok) break;
        }
      }
    }
  } else if (warp >= 10) {
    // ------------------------------------------------------------------ values of blocks on the diagonal: every other 32 pieces of 16 bytes each
    const int me = warp - 10;
    uint32_t n_blocks = 0, n_pieces = 0, phases = 0;   // phases: one bit a stage
    bool ok = true;
    for (; ok; ++n_pieces) {
      const PcPiece* told = next_piece(n_pieces);
      if (!__all_sync(0xffffffffu, told != nullptr)) break;
      const PcPiece s = *told;
      const int edge = s.edge(p), open = s.open(p), seen = s.keys - s.fresh + min(s.tok0 + 2 * p.tile, s.fresh);   // keys that some row sees
      uint32_t* cleared = s_cleared[n_pieces & 7][me];
      if (lane < PC_EDGE * 4) cleared[lane] = 0;
      if (lane == 0) s_any[n_pieces & 7][me] = 0;
      __syncwarp();
      for (int j = s.j0; j < s.j1; ++j, ++n_blocks) {
        if (j < edge) continue;
        const int st = n_blocks % ST;
        if (!(ok = mbar_wait_warp(&v_raw[st], phases >> st & 1, abort_flag, p.status, kTimeoutFull))) break;
        phases ^= 1u << st;
        const int live = min(max(seen - j * 128, 0), 128), from = max(open + 1 - j * 128, 0);   // rows [from, live) are some query's but not every one's
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          uint4* rows16 = reinterpret_cast<uint4*>(sV + st * T + c * 16384);   // eight to a row, in an order of their own
#pragma unroll 4
          for (int i = from * 8 + me * 32 + lane; i < live * 8; i += 64) {
            const uint4 w = rows16[i];
            // an exponent of ones carries into the sign's place of its half
            auto up = [](uint32_t v) { return (v & 0x7f807f80u) + 0x00800080u; };
            if ((up(w.x) | up(w.y) | up(w.z) | up(w.w)) & 0x80008000u) {
              auto clear = [&](uint32_t v) { return v & ~(((up(v) & 0x80008000u) >> 15) * 0xffffu); };
              rows16[i] = make_uint4(clear(w.x), clear(w.y), clear(w.z), clear(w.w));
              const int bit = (j - edge) * 128 + (i >> 3);
              if (bit < PC_EDGE * 128) atomicOr(&cleared[bit >> 5], 1u << (bit & 31));
              s_any[n_pieces & 7][me] = 1;
            }
          }
#pragma unroll 4
          for (int i = live * 8 + me * 32 + lane; i < 1024; i += 64) rows16[i] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[st]);
      }
      if (ok && lane == 0) piece_done(n_pieces);
    }
  } else {
    // -------------------------------------------------------------------- soft-max groups
    const int x = warp >> 2;        // 0 = tile A, 1 = tile B
    const int quad = warp & 3;      // TMEM lane quadrant this warp may touch
    const int r = quad * 32 + lane;
    const uint32_t lane_base = uint32_t(quad * 32) << 16;
    const uint32_t tmem_S = tmem_base + x * 128 + lane_base;
    const uint32_t tmem_O = tmem_base + 256 + x * D + lane_base;
    const int my_tok = r / p.rep, my_head = r - my_tok * p.rep;
    uint32_t n_s = 0, n_o = 0, n_pieces = 0;
    bool ok = true;
    for (; ok; ++n_pieces) {
      const PcPiece* told = next_piece(n_pieces);
      if (!__all_sync(0xffffffffu, told != nullptr)) break;
      const PcPiece& s = *told;
      const int tile_tok = s.tok0 + x * p.tile, tok = tile_tok + my_tok;
      const bool live = my_tok < p.tile && tok < s.fresh;
      const int first_pos = s.keys - s.fresh + tile_tok;        // of the tile's first token
      const int my_pos = live ? s.keys - s.fresh + tok : -1;
      const int end = s.end(x);
      float m = -3.402823466e38f, l = 0.f;   // (no finite score is below)
      for (int j = s.j0; j < end; ++j, ++n_s) {
        if (!(ok = mbar_wait_warp(&s_full[x], n_s & 1, abort_flag, p.status, kTimeoutTmemFull))) break;
        tc_fence_after();
        uint32_t v[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(tmem_S + c * 32, reinterpret_cast<uint32_t(&)[32]>(v[c * 32]));
        tmem_ld_wait();
        if (j * 128 + 127 > first_pos) {   // the block holds keys that some token of the tile does not see
          const int seen = my_pos - j * 128;
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c > seen) v[c] = 0xff800000u;  // -inf
        }
        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
        for (int c = 0; c < 128; c += 8) {
          mx0 = fmaxf(mx0, fmaxf(__uint_as_float(v[c]), __uint_as_float(v[c + 1])));
          mx1 = fmaxf(mx1, fmaxf(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])));
          mx2 = fmaxf(mx2, fmaxf(__uint_as_float(v[c + 4]), __uint_as_float(v[c + 5])));
          mx3 = fmaxf(mx3, fmaxf(__uint_as_float(v[c + 6]), __uint_as_float(v[c + 7])));
        }
        const float mnew = fmaxf(m, fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * p.scale_log2);
        // score * scale - m in one rounding leaves the rounding of m in every exponent: a common factor, at most 2^32 up to an m of 2^30.  Beyond, the scores
        // are scaled first, rounded like m itself.
        constexpr float BIG = 1073741824.f;
        float scale = p.scale_log2;
        if (__any_sync(0xffffffffu, live && (mnew > m + 8.f || fabsf(mnew) > BIG))) {   // (what lies behind the portion in the tile has no say)
          const float alpha = exp2f(m - mnew);  // the previous P V of this tile has completed: S(j) was computed after it
          m = mnew;
          l *= alpha;
          if (j > s.j0) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld_32x16(tmem_O + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st_32x16(tmem_O + c * 16, o);
            }
            tmem_st_wait();
          }
          if (__any_sync(0xffffffffu, live && fabsf(m) > BIG)) {
#pragma unroll
            for (int c = 0; c < 128; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * scale);
            scale = 1.f;
          }
        }
        float2 rsa = make_float2(0.f, 0.f), rsb = make_float2(0.f, 0.f);
        const float2 sc2 = make_float2(scale, scale), nm2 = make_float2(-m, -m);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 xs = __ffma2_rn(make_float2(__uint_as_float(v[c * 32 + 2 * e]), __uint_as_float(v[c * 32 + 2 * e + 1])), sc2, nm2);
            const float2 pr = make_float2(exp2f(xs.x), exp2f(xs.y));
            pk[e] = pack_bf16x2(pr.x, pr.y);
            if (e & 1) rsb = __fadd2_rn(rsb, pr);
            else rsa = __fadd2_rn(rsa, pr);
          }
          tmem_st_32x16(tmem_S + c * 16, pk);
        }
        l += (rsa.x + rsa.y) + (rsb.x + rsb.y);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
      }
      if (!ok) break;
      const bool any = end > s.j0;   // the tile sees keys of this piece
      if (any) {
        if (!mbar_wait_warp(&o_done[x], n_o & 1, abort_flag, p.status, kTimeoutTmemFull)) break;
        ++n_o;
        tc_fence_after();
      }
      const bool whole = s.whole();
      const long long slot = ((long long)blockIdx.x * 2 + (s.opens ? 0 : 1)) * 256 + x * 128 + r;
      const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
      __nv_bfloat16* orow = p.out + (long long)(s.first + tok) * p.ldo + (long long)(s.hk * p.rep + my_head) * D;
      float* part = p.part_o + slot * D;
      if (live && !whole) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(any ? m : -INFINITY, l);
      if (any) {
        auto put = [&](int c, const uint32_t (&o)[32]) {
          if (whole) {
            uint4 w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float f[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(o[8 * e + i]) * inv;
              w[e] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
            }
            if (p.wide) {   // whole sectors
              st_global_32B(orow + c * 32, w[0], w[1]);
              st_global_32B(orow + c * 32 + 16, w[2], w[3]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) *reinterpret_cast<uint4*>(orow + c * 32 + e * 8) = w[e];
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              st_global_32B(part + c * 32 + e * 8, make_uint4(o[8 * e], o[8 * e + 1], o[8 * e + 2], o[8 * e + 3]),
                            make_uint4(o[8 * e + 4], o[8 * e + 5], o[8 * e + 6], o[8 * e + 7]));
          }
        };
        if (end <= s.edge(p) || (s_any[n_pieces & 7][0] | s_any[n_pieces & 7][1]) == 0) {   // (written before the values of the first diagonal block were released)
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(tmem_O + c * 32, o);
            tmem_ld_wait();
            if (live) put(c, o);
          }
        } else {   // values that are not finite, of keys that this query sees
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(tmem_O + c * 32, o);
            tmem_ld_wait();
            if (!live) continue;
            for (int bit = 0; bit < PC_EDGE * 128; ++bit) {
              const int key = s.edge(p) * 128 + bit;
              if (key > my_pos || !((s_cleared[n_pieces & 7][0][bit >> 5] | s_cleared[n_pieces & 7][1][bit >> 5]) >> (bit & 31) & 1)) continue;
              const int id = rows.tables[(long long)s.row * rows.width + (key >> rows.page_log)];
              if (id < 0 || id >= rows.pages) continue;
              const __nv_bfloat16* v = p.v_pages + ((((long long)id << rows.page_log) + (key & ((1 << rows.page_log) - 1))) * p.n_kv + s.hk) * D + c * 32;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float f = __bfloat162float(v[e]);
                if ((__float_as_uint(f) & 0x7f800000u) == 0x7f800000u) o[e] = __float_as_uint(__uint_as_float(o[e]) + f);
              }
            }
            put(c, o);
          }
        }
        tc_fence_before();   // O has been read: the next piece's first P, which this warp announces, may be followed by a P V over it
      }
      __syncwarp();
      if (lane == 0) piece_done(n_pieces);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// CTA (c, part): the pair of tiles across the border between stretches c and c + 1, if no earlier border lies in it; 16 of its 256 query rows.
constexpr int PCJ_THREADS = 256, PCJ_ROWS = 16;
template <int D>
__global__ void __launch_bounds__(PCJ_THREADS) paged_portion_join_kernel(const PagedPortionArgs p) {
  __shared__ int s_slots[PC_CTAS], s_n;
  pdl_prologue();
  const PcShares shares(p, *p.total);
  const unsigned c = blockIdx.x;
  if (c + 1 >= shares.n) return;
  const PcPlace at = p.begins[c + 1];
  if (at.base == shares.begin(c + 1) || at.base < shares.begin(c)) return;   // no pair across this border, or an earlier one lies in it too
  const PcRow w(p, at.row);
  const int pair = 2 * p.tile, tok0 = at.k * pair, seen = w.at + min(tok0 + pair, w.fresh), blocks = (seen + 127) >> 7;
  if (threadIdx.x < 32) {   // the slots of its pieces, in order
    int n = 0;
    for (unsigned s0 = c; s0 < shares.n; s0 += 32) {
      const unsigned s = s0 + threadIdx.x;
      const bool in = s < shares.n && shares.begin(s) < at.base + PC_PIECE + seen;
      int from = 0, to = 0;
      if (in) {
        from = pc_block(at.base, shares.begin(s), seen, blocks);
        to = pc_block(at.base, shares.begin(s + 1), seen, blocks);
      }
      const bool piece = from < to, whole = from == 0 && to == blocks;   // (whole: a CTA has finished the pair)
      const unsigned mask = __ballot_sync(0xffffffffu, piece);
      if (piece) s_slots[n + __popc(mask & ((1u << threadIdx.x) - 1))] = 2 * int(s) + (at.base <= shares.begin(s) ? 0 : 1);
      n = __any_sync(0xffffffffu, whole) ? -1 : n + __popc(mask);
      if (n < 0 || !__all_sync(0xffffffffu, in)) break;
    }
    if (threadIdx.x == 0) s_n = n;
  }
  __syncthreads();
  const int n = s_n;
  constexpr int LANES = D / 4;
#pragma unroll
  for (int i = threadIdx.x; i < PCJ_ROWS * LANES; i += PCJ_THREADS) {
    const int q = blockIdx.y * PCJ_ROWS + i / LANES, lane = i % LANES, tile = q >> 7, r = q & 127;
    const int my_tok = r / p.rep, head = r - my_tok * p.rep, tok = tok0 + tile * p.tile + my_tok;
    if (n < 1 || my_tok >= p.tile || tok >= w.fresh) continue;
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int x = 0; x < n; ++x) {
      const long long slot = (long long)s_slots[x] * 256 + q;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot * 2);
      const float4 v = reinterpret_cast<const float4*>(p.part_o + slot * D)[lane];
      if (ml.x == -INFINITY) continue;   // the tile saw no keys of that piece: its sums were not written
      const float top = fmaxf(m, ml.x), keep = exp2f(m - top), f = exp2f(ml.x - top);
      m = top;
      l = l * keep + ml.y * f;
      acc = make_float4(acc.x * keep + v.x * f, acc.y * keep + v.y * f, acc.z * keep + v.z * f, acc.w * keep + v.w * f);
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    *reinterpret_cast<uint2*>(p.out + (long long)(w.first + tok) * p.ldo + (long long)(at.hk * p.rep + head) * D + 4 * lane) =
        make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  }
}

template <int D>
static int launch_paged_portion(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PagedPortionArgs& p, cudaStream_t s) {
  using SM = PagedPortionSmem<D>;
  static_assert(SM::TOTAL <= 227 * 1024, "does not fit an SM");
  static DeviceOnce once;
  cudaError_t ce = once.smem(paged_portion_kernel<D>, SM::TOTAL);
  if (ce == cudaSuccess) ce = launch_pdl(paged_portion_kernel<D>, dim3(p.ctas), dim3(PC_THREADS), SM::TOTAL, s, mq, mk, mv, p);
  if (ce == cudaSuccess && p.ctas > 1) ce = launch_behind(paged_portion_join_kernel<D>, dim3(p.ctas - 1, 256 / PCJ_ROWS), dim3(PCJ_THREADS), s, 0, p);
  if (ce != cudaSuccess) return int(ce);
  return int(cudaGetLastError());
}

}  // namespace ats

using namespace ats;

// Bytes of scratch that `ats_paged_portion` needs (32-byte aligned).
ATS_API long long ats_paged_portion_scratch(int D) { return 32 + PC_CTAS * (long long)sizeof(PcPlace) + 2ll * PC_CTAS * 256 * (D + 2) * 4; }

// Rows whose new tokens times n_q / n_kv are more than `limit`.  q [tokens, ldq], pages [pages * page, n_kv, D] bf16, D 64 or 128, pages of 8 tokens (a power of
// two) or more, up to 128 query heads a group.  zero_tail: tokens behind the last row get zeros.
ATS_API int ats_paged_portion(const void* q, long long ldq, const void* k_pages, const void* v_pages, const int* starts, const int* lengths, const int* tables,
                              void* out, long long ldo, int tokens, int R, int n_q, int n_kv, int D, int width, int pages, int page, int limit, float scale,
                              int zero_tail, void* scratch, int* status, void* stream) {
  if ((D != 64 && D != 128) || tokens < 1 || R < 1 || n_kv < 1 || n_q % n_kv || n_q / n_kv > 128 || (ldq & 7) || (ldo & 7) || off_16(q, k_pages, v_pages, out) || (reinterpret_cast<uintptr_t>(scratch) & 31) ||
      page < 8 || (page & (page - 1)) || (long long)pages * page >= (1ll << 31) - 256 || (long long)width * page >= (1ll << 31) - 256 || tokens > (1 << 30))
    return 1003;
  bind_context();
  PagedPortionArgs p;
  p.rows = {starts, lengths, tables, R, width, pages, __builtin_ctz(page), tokens};
  p.v_pages = static_cast<const __nv_bfloat16*>(v_pages); p.out = static_cast<__nv_bfloat16*>(out); p.ldo = ldo;
  p.n_kv = n_kv; p.rep = n_q / n_kv; p.limit = limit; p.tile = 128 / p.rep; p.ctas = PC_CTAS; p.zero_tail = zero_tail; p.wide = !(reinterpret_cast<uintptr_t>(out) & 31) && !(ldo & 15);
  p.scale_log2 = scale * 1.4426950408889634f; p.status = status;
  static_assert(sizeof(PcPlace) % 32 == 0, "the sums are written 32 bytes at a time");
  p.total = static_cast<unsigned long long*>(scratch);
  p.begins = reinterpret_cast<PcPlace*>(p.total + 4);
  p.part_o = reinterpret_cast<float*>(p.begins + PC_CTAS);
  p.part_ml = p.part_o + 2ll * PC_CTAS * 256 * D;
  CUtensorMap mq, mk, mv;
  int e;
  if ((e = make_tmap_pages(&mk, k_pages, (uint64_t)pages * page, n_kv, D, page < 128 ? page : 128))) return e;
  if ((e = make_tmap_pages(&mv, v_pages, (uint64_t)pages * page, n_kv, D, page < 128 ? page : 128))) return e;
  if ((e = make_tmap_tokens(&mq, q, tokens, n_q, D, ldq, p.rep, p.tile))) return e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return D == 64 ? launch_paged_portion<64>(mq, mk, mv, p, s) : launch_paged_portion<128>(mq, mk, mv, p, s);
}
