// Attention of one or a few new tokens per row over a paged key / value cache, for sm_100a.
//
//   o[i, h] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q[i, h] . k_j - max),   j up to token i of the row
//
// A row takes this kernel when its new tokens times the query heads of a group are at most 8 (or 16): they are the rows of a warp-level MMA
// (m16n8k16), and the step is a stream of the cache, each key and value read once.  Bound by memory: 8 rows x 8 key heads of 128 with 5,000 to 31,000 keys, four
// new tokens each (490 MB) 93 us = 5.3 TB/s, 81 % of a copy's rate (its warps end between 66 and 92 us); short caches by the start (row sums, first table entries
// and copies 3.5 us) and the second launch: 64 rows x 4 key heads of 64, 200 to 2,000 keys (70 MB) 21 us, 11 at the copy's rate; one row of 512 keys 7.1 us.
//
// * Every warp moves units of 8 KB (K and V of 2048 / D keys) by TMA into a ring of its own, 192 KB an SM in flight,
//   and keeps a running softmax; the fragments come out of the swizzled units as in the decode kernel over contiguous rows (inference.cu).
//   The page of a unit comes from the row's table, which the lanes read 32 entries at a time.
// * Probabilities are rounded to bf16 for their product with the values, the type of its other operand (sums of them are not): outputs are 0.0018 to 0.0020
//   off 64 bits, relative, where their own rounding makes 0.0016.
// * Rows of a batch are of any length, so the work is dealt out by units, not by rows: the units of all rows and key heads form one line, and
//   every warp takes an equal stretch of it, its ring running on from one pair (row, key head) to the next.  Pairs that lie in a stretch as a
//   whole are finished there; what it holds of the first and the last goes to a scratch slot, and a second launch joins the slots of each
//   such pair, in the order of the line: results do not depend on timing.
#include "paged_common.cuh"

namespace ats {

constexpr int PD_WARPS = 4, PD_THREADS = 32 * PD_WARPS;
constexpr int PD_UNIT_BYTES = 8192;
// Two CTAs of four warps an SM with a ring of three units each, against three with a ring of two (192 KB in flight either way): 64 rows x 4 key heads of 64,
// 200 to 2,000 keys 21.3 / 24.1 us, one row of 60,000 x 8 of 128 56 / 67 (fewer slots to join), 64 rows x 8 of 128, 2,000 keys 94.7 / 93.8, 128 x 4 of 64,
// 100 to 4,000 55.5 / 54.1; with sixteen MMA rows (twice the sums and queries in registers) 8 rows of 5,000 to 31,000 keys 92 / 100.
constexpr int PD_CTAS = 2, PD_STAGES = 3;
constexpr int PD_SMEM = 1024 + PD_WARPS * PD_STAGES * PD_UNIT_BYTES;

struct PagedDecodeArgs {
  PagedRows rows;
  const __nv_bfloat16* q;   // [tokens, ldq]
  long long ldq;
  __nv_bfloat16* out;       // [tokens, ldo]
  long long ldo;
  int n_kv, rep, limit;     // rows with at most `limit` MMA rows are taken
  int warps;                // of the main launch
  int max_new;              // no row has more new tokens
  int rows_most;            // MMA rows of any row that is taken
  int zero_tail;            // tokens behind the last row get zeros
  int behind;               // the launch before this one is of the same call
  float scale_log2;
  uint32_t* line;           // [R + 1]: where a row's units begin, per key head; the end of the line
  float* part_o;            // [warps, 2, rows of the MMA, D]
  float* part_ml;           // [warps, 2, rows of the MMA, 2]
  int* status;
};

__device__ __forceinline__ void pd_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 pd_lds(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float pd_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pd_from(float m, float base) { return m == -INFINITY ? 0.f : pd_exp2(m - base); }

// The halves of two bf16 values that are not finite, at their signs' places: an exponent of ones carries into these.
__device__ __forceinline__ uint32_t pd_odd(uint32_t v) { return ((v & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

// Units of row r on this kernel's line, per key head (0: the row is empty or another kernel's).
template <int UNIT>
__device__ __forceinline__ int pd_units(const PagedDecodeArgs& p, int r) {
  int first, fresh, keys;
  paged_row(p.rows, r, &first, &fresh, &keys);
  return fresh > 0 && (long long)fresh * p.rep <= p.limit ? (max(keys, 1) + UNIT - 1) / UNIT : 0;
}

template <bool V>
struct PdBool {
  static constexpr bool value = V;
};

// A line of `total` units (below 2^32) shared out over as many warps as there are, one more unit to each of the first `extra`.
struct PdShares {
  uint32_t n, each, extra;
  __device__ __forceinline__ PdShares(const PagedDecodeArgs& p, uint32_t total) {
    n = min(uint32_t(p.warps), total);
    each = n ? total / n : 0;
    extra = total - each * n;
  }
  __device__ __forceinline__ uint32_t begin(uint32_t w) const { return w * each + min(w, extra); }
  __device__ __forceinline__ uint32_t owner(uint32_t x) const {   // the warp whose stretch holds unit x
    const uint32_t longer = extra * (each + 1);
    return x < longer ? x / (each + 1) : extra + (x - longer) / each;
  }
};

template <int D, int NR>  // NR: sets of eight MMA rows (1 or 2)
__global__ void __launch_bounds__(PD_THREADS, PD_CTAS) paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                     const PagedDecodeArgs p) {
  constexpr int UNIT = 2048 / D, NT = UNIT / 8, KB = UNIT / 16, JD = D / 32, RD = D / 64, ROWS = 8 * NR;
  extern __shared__ uint8_t pd_smem[];
  __shared__ uint64_t s_full[PD_WARPS][PD_STAGES];
  __shared__ uint32_t s_sum[PD_WARPS], s_at[PD_WARPS];
  __shared__ int s_row[PD_WARPS], s_abort;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const PagedRows& rows = p.rows;
  uint8_t* base_smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pd_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = base_smem + warp * (PD_STAGES * PD_UNIT_BYTES);
  uint64_t* full = s_full[warp];
  if (lane == 0) {
    for (int i = 0; i < PD_STAGES; ++i) mbar_init(&full[i], 1);
    mbar_fence_init();
  }
  if (tid == 0) {
    s_abort = 0;
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  // where the rows begin on the line: every thread sums up a share of the rows
  const int share = (rows.R + PD_THREADS - 1) / PD_THREADS, r0 = min(tid * share, rows.R), r1 = min(r0 + share, rows.R);
  uint32_t mine = 0;
  for (int r = r0; r < r1; ++r) mine += pd_units<UNIT>(p, r);
  const int fresh_last = r0 < rows.R ? rows.starts[r0 + 1] - rows.starts[r0] : 0;
  uint32_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  uint32_t total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < PD_WARPS; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  total *= p.n_kv;
  const PdShares shares(p, total);
  const uint32_t me0 = blockIdx.x * PD_WARPS;
  for (int r = r0; r < r1; ++r) {
    const uint32_t n = share == 1 ? mine : pd_units<UNIT>(p, r), at = before * p.n_kv;
    if (blockIdx.x == 0) {
      p.line[r] = before;
      if ((share == 1 ? fresh_last : rows.starts[r + 1] - rows.starts[r]) > p.max_new) atomicCAS(p.status, 0, int(kBadArgument));   // more than the caller promised: nobody serves the row
    }
#pragma unroll
    for (int w = 0; w < PD_WARPS; ++w) {
      const uint32_t x = shares.begin(me0 + w);
      if (at <= x && x < at + n * p.n_kv) s_row[w] = r, s_at[w] = at;
    }
    before += n;
  }
  if (blockIdx.x == 0 && tid == 0) p.line[rows.R] = total / p.n_kv;
  __syncthreads();
  auto zero_tail = [&]() {
    const int tail = min(max(rows.starts[rows.R], 0), rows.tokens), vecs = p.n_kv * p.rep * (D / 8);
    for (long long i = (long long)blockIdx.x * PD_THREADS + tid; i < (long long)(rows.tokens - tail) * vecs; i += (long long)gridDim.x * PD_THREADS)
      *reinterpret_cast<uint4*>(p.out + (tail + i / vecs) * p.ldo + (i % vecs) * 8) = make_uint4(0, 0, 0, 0);
  };
  const uint32_t me = me0 + warp;
  if (me >= shares.n) {
    if (p.zero_tail) zero_tail();
    return;
  }
  const uint32_t lo = shares.begin(me);
  const int n_mine = int(shares.begin(me + 1) - lo);

  // ---- requests run ahead of the units that are worked on, into the pairs that follow
  const int page = 1 << rows.page_log, box = min(UNIT, page), per = UNIT / box;   // tokens and number of the copies of a unit's 64-column piece
  const int batch = 32 / per;   // units whose coordinates the lanes hold, copy lane % per of unit lane / per
  int q_row = s_row[warp], q_hk, q_unit, q_units = pd_units<UNIT>(p, q_row), q_pages, q_base = 0, here = 0, asked = 0;
  {
    const uint32_t in_row = lo - s_at[warp];
    q_hk = int(in_row / uint32_t(q_units));
    q_unit = int(in_row) - q_hk * q_units;
  }
  const int w_row = q_row, w_hk = q_hk, w_unit = q_unit;   // the first unit to work on
  auto pages_of = [&](int r) {
    int first, fresh, keys;
    paged_row(rows, r, &first, &fresh, &keys);
    return (keys + page - 1) >> rows.page_log;
  };
  auto look_up = [&](int from) {   // coordinates of units from .. from + batch - 1 of the pair
    q_base = from;
    const int k0 = (from + lane / per) * UNIT + (lane % per) * box, j = k0 >> rows.page_log;
    here = rows.pages << rows.page_log;    // behind the pages: reads as zero
    if (j < q_pages) {
      const int id = rows.tables[(long long)q_row * rows.width + j];
      if (id >= 0 && id < rows.pages) here = (id << rows.page_log) + (k0 & (page - 1));
      else atomicCAS(p.status, 0, int(kBadArgument));
    }
  };
  q_pages = pages_of(q_row);
  look_up(q_unit);
  auto request = [&]() {   // whole warp: the next unit of the stretch
    if (q_unit == q_units) {
      q_unit = 0;
      if (++q_hk == p.n_kv) {
        q_hk = 0;
        do q_units = pd_units<UNIT>(p, ++q_row);   // (a unit is still to come, so a row is)
        while (q_units == 0);
        q_pages = pages_of(q_row);
      }
      look_up(0);
    } else if (q_unit - q_base == batch) {
      look_up(q_unit);
    }
    const uint32_t st = asked % PD_STAGES;
    uint8_t* dst = ring + st * PD_UNIT_BYTES;
    if (lane == 0) mbar_expect_tx(&full[st], PD_UNIT_BYTES);
    for (int s = 0; s < per; ++s) {
      const int c = __shfl_sync(0xffffffffu, here, (q_unit - q_base) * per + s);
      if (lane == 0) {
#pragma unroll
        for (int rd = 0; rd < RD; ++rd) {
          tma_load_3d(dst + (rd * UNIT + s * box) * 128, &map_k, &full[st], 64 * rd, q_hk, c);
          tma_load_3d(dst + PD_UNIT_BYTES / 2 + (rd * UNIT + s * box) * 128, &map_v, &full[st], 64 * rd, q_hk, c);
        }
      }
    }
    ++q_unit;
    ++asked;
  };
  while (asked < min(n_mine, PD_STAGES)) request();

  const uint32_t k_at = smem_u32(ring) + g * 128, v_at = smem_u32(ring) + PD_UNIT_BYTES / 2 + 2 * t * 128;
  // the pieces of key 8 nt + g and of the values' keys 2 t, 2 t + 1 (+ 8), swizzled by their rows modulo eight
  const uint32_t piece[2] = {uint32_t((t ^ g) << 4), uint32_t(((4 + t) ^ g) << 4)};
  const uint32_t vpiece[2] = {uint32_t((g ^ (2 * t)) << 4), uint32_t((g ^ (2 * t + 1)) << 4) + 128};
  int row = w_row, hk = w_hk, u0 = w_unit, done = 0;
#pragma unroll 1
  while (done < n_mine) {
    const int units = pd_units<UNIT>(p, row);
    if (units == 0) {
      ++row;
      continue;
    }
    int first, fresh, keys;
    paged_row(rows, row, &first, &fresh, &keys);
    const int count = min(units - u0, n_mine - done);
    const int n_rows = fresh * p.rep, open = keys - fresh + 1;   // keys below `open` are seen by all new tokens
    // queries of MMA rows g and g + 8, [virtual k-step][pieces of a row]
    uint32_t qa[NR][D / 16][2];
    int last[NR];   // keys up to this one are seen by the row
#pragma unroll
    for (int x = 0; x < NR; ++x) {
      const int i = g + 8 * x, tok = i / p.rep, head = i - tok * p.rep;
      const bool live = i < n_rows;
      last[x] = live ? keys - fresh + tok : -1;
      const uint32_t* qrow = reinterpret_cast<const uint32_t*>(p.q + (long long)(first + (live ? tok : 0)) * p.ldq + (long long)(hk * p.rep + (live ? head : 0)) * D);
#pragma unroll
      for (int j = 0; j < JD; ++j) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (live) w = *reinterpret_cast<const uint4*>(qrow + 4 * (4 * j + t));
        qa[x][2 * j][0] = w.x; qa[x][2 * j][1] = w.y; qa[x][2 * j + 1][0] = w.z; qa[x][2 * j + 1][1] = w.w;
      }
    }
    float oe[RD][4][4], oo[RD][4][4], m[NR], l[NR];
#pragma unroll
    for (int rd = 0; rd < RD; ++rd)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) oe[rd][i][e] = oo[rd][i][e] = 0.f;
#pragma unroll
    for (int x = 0; x < NR; ++x) m[x] = -INFINITY, l[x] = 0.f;
    // EDGE: the unit holds keys that some row does not see
    auto unit = [&](auto edge_c, const int k0, const uint32_t stage) {
      constexpr bool EDGE = decltype(edge_c)::value;
      const uint32_t ks = k_at + stage * PD_UNIT_BYTES, vs = v_at + stage * PD_UNIT_BYTES;
      uint4 vv[KB][RD][4];
      float s[NT][2 * NR];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint4 kv[JD];
#pragma unroll
        for (int j = 0; j < JD; ++j) kv[j] = pd_lds(ks + ((j >> 1) * UNIT + nt * 8) * 128 + piece[j & 1]);
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < JD; ++j) {
          pd_mma(c, qa[0][2 * j][0], NR > 1 ? qa[NR - 1][2 * j][0] : 0u, qa[0][2 * j][1], NR > 1 ? qa[NR - 1][2 * j][1] : 0u, kv[j].x, kv[j].y);
          pd_mma(c, qa[0][2 * j + 1][0], NR > 1 ? qa[NR - 1][2 * j + 1][0] : 0u, qa[0][2 * j + 1][1], NR > 1 ? qa[NR - 1][2 * j + 1][1] : 0u, kv[j].z, kv[j].w);
        }
#pragma unroll
        for (int e = 0; e < 2 * NR; ++e) s[nt][e] = c[e] * p.scale_log2;   // rows g (and g + 8), keys 2t and 2t + 1 of the tile
      }
      // lane (g, t) reads 16 bytes (dims 64 rd + 8 g .. + 7) of four keys
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int rd = 0; rd < RD; ++rd) vv[kb][rd][i] = pd_lds(vs + (rd * UNIT + kb * 16 + (i >> 1) * 8) * 128 + vpiece[i & 1]);
      if (EDGE) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int rd = 0; rd < RD; ++rd)
              if (k0 + kb * 16 + 2 * t + (i & 1) + (i >> 1) * 8 >= keys) vv[kb][rd][i] = make_uint4(0, 0, 0, 0);   // whatever earlier generations left there
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2 * NR; ++e)
            if (k0 + nt * 8 + 2 * t + (e & 1) > last[e >> 1]) s[nt][e] = -INFINITY;
      }
      float keep[NR], ref[NR];
      bool moved = false;
#pragma unroll
      for (int x = 0; x < NR; ++x) {
        float top = m[x];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) top = fmaxf(top, fmaxf(s[nt][2 * x], s[nt][2 * x + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        ref[x] = top == -INFINITY ? 0.f : top;
        moved |= top > m[x];
        keep[x] = pd_from(m[x], ref[x]);
        m[x] = top;
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int x = 0; x < NR; ++x) l[x] *= keep[x];
#pragma unroll
        for (int rd = 0; rd < RD; ++rd)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 2 * NR; ++e) oe[rd][i][e] *= keep[e >> 1], oo[rd][i][e] *= keep[e >> 1];
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2 * NR; ++e) {
          s[nt][e] = pd_exp2(s[nt][e] - ref[e >> 1]);
          l[e >> 1] += s[nt][e];
        }
      // Word i of a V piece holds dims 8 g + 2 i, + 1: the low halves of two keys form the B fragment of the column tile "even dims of
      // word i", the high halves that of "odd dims of word i".
      auto weigh = [&](const float (&pr)[NT][2 * NR], const uint4 (&vv)[KB][RD][4]) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          uint32_t pa[4] = {pack_bf16x2(pr[2 * kb][0], pr[2 * kb][1]), 0u, pack_bf16x2(pr[2 * kb + 1][0], pr[2 * kb + 1][1]), 0u};
          if (NR > 1) pa[1] = pack_bf16x2(pr[2 * kb][2 * NR - 2], pr[2 * kb][2 * NR - 1]), pa[3] = pack_bf16x2(pr[2 * kb + 1][2 * NR - 2], pr[2 * kb + 1][2 * NR - 1]);
#pragma unroll
          for (int rd = 0; rd < RD; ++rd) {
            const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&vv[kb][rd][0]);
            const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&vv[kb][rd][1]);
            const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&vv[kb][rd][2]);
            const uint32_t* w3 = reinterpret_cast<const uint32_t*>(&vv[kb][rd][3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              pd_mma(oe[rd][i], pa[0], pa[1], pa[2], pa[3], __byte_perm(w0[i], w1[i], 0x5410), __byte_perm(w2[i], w3[i], 0x5410));
              pd_mma(oo[rd][i], pa[0], pa[1], pa[2], pa[3], __byte_perm(w0[i], w1[i], 0x7632), __byte_perm(w2[i], w3[i], 0x7632));
            }
          }
        }
      };
      bool odd_unit = false;
      if (EDGE && fresh > 1) {
        // Values that some rows do not see: a probability of zero does not keep one that is not finite out of a product.  Such ones are cleared ...
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (k0 + kb * 16 + 2 * t + (i & 1) + (i >> 1) * 8 >= open)
#pragma unroll
              for (int rd = 0; rd < RD; ++rd) {
                uint32_t* w = reinterpret_cast<uint32_t*>(&vv[kb][rd][i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t odd = pd_odd(w[e]);
                  odd_unit |= odd != 0;
                  w[e] &= ~((odd >> 15) * 0xffffu);
                }
              }
        odd_unit = __any_sync(0xffffffffu, odd_unit);
      }
      weigh(s, vv);
      if (EDGE && odd_unit) {
        // ... and added by the rows that do see them
#pragma unroll 1
        for (int k = max(open - k0, 0); k < min(keys - k0, UNIT); ++k)
#pragma unroll
          for (int rd = 0; rd < RD; ++rd)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint4 piece16 = pd_lds(smem_u32(ring) + stage * PD_UNIT_BYTES + PD_UNIT_BYTES / 2 + (rd * UNIT + k) * 128 + (((2 * t + e) ^ (k & 7)) << 4));
              const uint32_t w[4] = {piece16.x, piece16.y, piece16.z, piece16.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t odd = pd_odd(w[i]);
                const float2 f = unpack_bf16x2(w[i]);
#pragma unroll
                for (int x = 0; x < NR; ++x)
                  if (k0 + k <= last[x]) {
                    if (odd & 0x8000u) oe[rd][i][2 * x + e] += f.x;
                    if (odd & 0x80000000u) oo[rd][i][2 * x + e] += f.y;
                  }
              }
            }
      }
    };
#pragma unroll 1
    for (int u = 0; u < count; ++u, ++done) {
      const uint32_t stage = done % PD_STAGES;
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[stage], (done / PD_STAGES) & 1, &s_abort, p.status, kTimeoutFull))) {
        const uint64_t t0 = globaltimer_ns();   // copies that were issued land before the warp gives its shared memory back
        while (globaltimer_ns() - t0 < 10000000ull) {
        }
        return;
      }
      const int k0 = (u0 + u) * UNIT;
      if (k0 + UNIT > open) unit(PdBool<true>{}, k0, stage);
      else unit(PdBool<false>{}, k0, stage);
      __syncwarp();   // the stage has been read
      if (asked < n_mine) request();
    }
#pragma unroll
    for (int x = 0; x < NR; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      const int i = g + 8 * x;
      if (i >= n_rows) continue;
      // lane (g, t): accumulator column 2t is dim 64 rd + 16 t + 2 i (+ 1 for the odd tile), column 2t + 1 eight dims further
      if (count == units) {
        const int tok = i / p.rep, head = i - tok * p.rep;
        const float inv = l[x] > 0.f ? 1.f / l[x] : 1.f;
        __nv_bfloat16* dst = p.out + (long long)(first + tok) * p.ldo + (long long)(hk * p.rep + head) * D + 16 * t;
#pragma unroll
        for (int rd = 0; rd < RD; ++rd)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<uint4*>(dst + 64 * rd + 8 * e) =
                make_uint4(pack_bf16x2(oe[rd][0][2 * x + e] * inv, oo[rd][0][2 * x + e] * inv), pack_bf16x2(oe[rd][1][2 * x + e] * inv, oo[rd][1][2 * x + e] * inv),
                           pack_bf16x2(oe[rd][2][2 * x + e] * inv, oo[rd][2][2 * x + e] * inv), pack_bf16x2(oe[rd][3][2 * x + e] * inv, oo[rd][3][2 * x + e] * inv));
      } else {
        const long long slot = ((long long)me * 2 + (done == count ? 0 : 1)) * ROWS + i;   // the stretch's first piece, or its last
        if (t == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * slot) = make_float2(m[x], l[x]);
        float* dst = p.part_o + slot * D + 16 * t;
#pragma unroll
        for (int rd = 0; rd < RD; ++rd)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            *reinterpret_cast<float4*>(dst + 64 * rd + 8 * e) = make_float4(oe[rd][0][2 * x + e], oo[rd][0][2 * x + e], oe[rd][1][2 * x + e], oo[rd][1][2 * x + e]);
            *reinterpret_cast<float4*>(dst + 64 * rd + 8 * e + 4) = make_float4(oe[rd][2][2 * x + e], oo[rd][2][2 * x + e], oe[rd][3][2 * x + e], oo[rd][3][2 * x + e]);
          }
      }
    }
    u0 = 0;
    if (++hk == p.n_kv) hk = 0, ++row;
  }
  if (p.zero_tail) zero_tail();
}

// The scratch slots of a pair (row, key head) that several warps shared.  D / 4 lanes hold an MMA row's columns; G such groups take the row's slots
// in turn and are joined in order.  A CTA serves 256 / (G D / 4) MMA rows: many slots (few pairs) want many groups, few slots one or two.
constexpr int PJ_THREADS = 256;
template <int D, int NR, int G>
__global__ void __launch_bounds__(PJ_THREADS) paged_join_kernel(const PagedDecodeArgs p) {
  constexpr int ROWS = 8 * NR, LANES = D / 4, AT_ONCE = PJ_THREADS / (G * LANES), UNIT = 2048 / D;
  __shared__ float4 s_acc[AT_ONCE][G][LANES];
  __shared__ float s_m[AT_ONCE][G], s_l[AT_ONCE][G];
  pdl_prologue();
  const int hk = blockIdx.y, row = blockIdx.z, lane = threadIdx.x % LANES, group = threadIdx.x / LANES % G, sub = threadIdx.x / (LANES * G);
  const int i = blockIdx.x * AT_ONCE + sub;
  int first, fresh, keys;
  paged_row(p.rows, row, &first, &fresh, &keys);
  const uint32_t units = pd_units<UNIT>(p, row);
  const uint32_t total = p.line[p.rows.R] * p.n_kv, a = p.line[row] * p.n_kv + hk * units;
  if (units == 0) return;
  const PdShares shares(p, total);
  const uint32_t w0 = shares.owner(a), w1 = shares.owner(a + units - 1);
  if (w0 == w1) return;   // finished by that warp
  const bool live = i < fresh * p.rep;
  const uint32_t s0 = 2 * w0 + (shares.begin(w0) >= a ? 0 : 1);   // the first one's slot: its first piece unless its stretch began before the pair
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
#pragma unroll 4
    for (uint32_t w = w0 + group; w <= w1; w += G) {
      const long long at = (long long)(w == w0 ? s0 : 2 * w) * ROWS + i;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * at);
      const float4 v = reinterpret_cast<const float4*>(p.part_o + at * D)[lane];
      const float top = fmaxf(m, ml.x), ref = top == -INFINITY ? 0.f : top, keep = pd_from(m, ref), f = pd_from(ml.x, ref);
      m = top;
      l = l * keep + ml.y * f;
      acc = make_float4(acc.x * keep + v.x * f, acc.y * keep + v.y * f, acc.z * keep + v.z * f, acc.w * keep + v.w * f);
    }
  }
  float sum = l;
  float4 o = acc;
  if (G > 1) {
    s_acc[sub][group][lane] = acc;
    if (lane == 0) s_m[sub][group] = m, s_l[sub][group] = l;
    __syncthreads();
    if (group > 0) return;
    float top = m;
#pragma unroll
    for (int x = 1; x < G; ++x) top = fmaxf(top, s_m[sub][x]);
    const float ref = top == -INFINITY ? 0.f : top;
    sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < G; ++x) {
      const float f = pd_from(s_m[sub][x], ref);
      const float4 v = s_acc[sub][x][lane];
      sum += s_l[sub][x] * f;
      o = make_float4(o.x + v.x * f, o.y + v.y * f, o.z + v.z * f, o.w + v.w * f);
    }
  }
  if (!live) return;
  const float inv = sum > 0.f ? 1.f / sum : 1.f;
  const int tok = i / p.rep, head = i - tok * p.rep;
  *reinterpret_cast<uint2*>(p.out + (long long)(first + tok) * p.ldo + (long long)(hk * p.rep + head) * D + 4 * lane) =
      make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

template <int D, int NR, int G>
static cudaError_t launch_paged_join(const PagedDecodeArgs& p, cudaStream_t s) {
  constexpr int AT_ONCE = PJ_THREADS / (G * D / 4);
  const int n = min(p.limit, p.rows_most);
  return launch_behind(paged_join_kernel<D, NR, G>, dim3((n + AT_ONCE - 1) / AT_ONCE, p.n_kv, p.rows.R), dim3(PJ_THREADS), s, 0, p);
}

template <int D, int NR>
static int launch_paged_decode(const CUtensorMap& mk, const CUtensorMap& mv, const PagedDecodeArgs& p, cudaStream_t s) {
  static DeviceOnce once;
  cudaError_t ce = once.smem(paged_decode_kernel<D, NR>, PD_SMEM);
  const dim3 grid((p.warps + PD_WARPS - 1) / PD_WARPS), block(PD_THREADS);
  if (ce == cudaSuccess) ce = p.behind ? launch_behind(paged_decode_kernel<D, NR>, grid, block, s, PD_SMEM, mk, mv, p) : launch_pdl(paged_decode_kernel<D, NR>, grid, block, PD_SMEM, s, mk, mv, p);
  // slots of a pair, if the rows are about as long as each other
  const int slots = p.warps / (p.rows.R * p.n_kv);
  if (ce == cudaSuccess) ce = slots >= 8 ? launch_paged_join<D, NR, 8>(p, s) : launch_paged_join<D, NR, 2>(p, s);
  if (ce != cudaSuccess) return int(ce);
  return int(cudaGetLastError());
}

// Warps of the main launch for up to `keys` keys in each of R rows: as many as run at once, but no more than there are units.
static int paged_decode_warps(int R, int n_kv, int D, long long keys) {
  const int most = 148 * PD_CTAS * PD_WARPS;
  const long long units = (keys + 2048 / D - 1) / (2048 / D) * R * n_kv;
  return int(units < 1 ? 1 : units > most ? most : units);
}

}  // namespace ats

using namespace ats;

// Bytes of scratch that `ats_paged_decode` needs (16-byte aligned).
ATS_API long long ats_paged_decode_scratch(int R, int n_kv, int D, long long max_keys, int limit) {
  return (R + 4ll) / 4 * 16 + 2ll * paged_decode_warps(R, n_kv, D, max_keys) * (limit > 8 ? 16 : 8) * (D + 2) * 4;
}

// Rows whose new tokens times n_q / n_kv are at most `limit` (8 or 16).  q [tokens, ldq], pages [pages * page, n_kv, D] bf16, D 64 or 128, pages of 8 tokens
// (a power of two) or more; max_keys: no row has more.  zero_tail: tokens behind the last row get zeros.  behind: ats_paged_portion of the same call is the
// stream's last launch, so this one is set up while it ends.
ATS_API int ats_paged_decode(const void* q, long long ldq, const void* k_pages, const void* v_pages, const int* starts, const int* lengths, const int* tables,
                             void* out, long long ldo, int tokens, int R, int n_q, int n_kv, int D, int width, int pages, int page, long long max_keys, int max_new, int limit,
                             float scale, int zero_tail, int behind, void* scratch, int* status, void* stream) {
  if ((D != 64 && D != 128) || tokens < 1 || R < 1 || R > 65535 || n_kv < 1 || n_kv > 65535 || n_q % n_kv || (ldq & 7) || (ldo & 7) || page < 8 || (page & (page - 1)) ||
      (limit != 8 && limit != 16) || off_16(q, k_pages, v_pages, out, scratch) || max_new < 1 || max_keys < 1 || ((long long)width * page / 16 + 1) * R * n_kv >= (1ll << 32) || (long long)pages * page >= (1ll << 31) - 256 || (long long)width * page >= (1ll << 31) - 256)
    return 1003;
  bind_context();
  const int unit = 2048 / D;
  CUtensorMap mk, mv;
  int e;
  if ((e = make_tmap_pages(&mk, k_pages, (uint64_t)pages * page, n_kv, D, page < unit ? page : unit))) return e;
  if ((e = make_tmap_pages(&mv, v_pages, (uint64_t)pages * page, n_kv, D, page < unit ? page : unit))) return e;
  PagedDecodeArgs p;
  p.rows = {starts, lengths, tables, R, width, pages, __builtin_ctz(page), tokens};
  p.q = static_cast<const __nv_bfloat16*>(q); p.ldq = ldq; p.out = static_cast<__nv_bfloat16*>(out); p.ldo = ldo;
  p.n_kv = n_kv; p.rep = n_q / n_kv; p.limit = limit; p.max_new = max_new; p.rows_most = int(min((long long)max_new * p.rep, (long long)limit)); p.warps = paged_decode_warps(R, n_kv, D, max_keys); p.zero_tail = zero_tail; p.behind = behind;
  p.scale_log2 = scale * 1.4426950408889634f; p.status = status;
  p.line = static_cast<uint32_t*>(scratch);
  p.part_o = reinterpret_cast<float*>(p.line + (R + 4) / 4 * 4);
  p.part_ml = p.part_o + 2ll * p.warps * (limit > 8 ? 16 : 8) * D;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (limit > 8) return D == 64 ? launch_paged_decode<64, 2>(mk, mv, p, s) : launch_paged_decode<128, 2>(mk, mv, p, s);
  return D == 64 ? launch_paged_decode<64, 1>(mk, mv, p, s) : launch_paged_decode<128, 1>(mk, mv, p, s);
}
