// Attention of one or a few new tokens per row over a paged key / value cache, for sm_100a.
//
//   o[i, h] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q[i, h] . k_j - max),   j up to token i of the row
//
// A row takes this kernel when its new tokens times the query heads of a group are at most 8 (or 16): they are the rows of a warp-level MMA
// (m16n8k16), and the step is a stream of the cache, each key and value read once.  Bound by memory.
//
// * Every warp moves units of 8 KB (K and V of 2048 / D keys) by TMA into a ring of two of its own, 192 KB an SM in flight over three CTAs,
//   and keeps a running softmax; the fragments come out of the swizzled units as in the decode kernel over contiguous rows (inference.cu).
//   The page of a unit comes from the row's table, which the lanes read 32 entries at a time.
// * Rows of a batch are of any length, so the work is dealt out by units, not by rows: the units of all rows and key heads form one line, and
//   every CTA takes an equal stretch of it.  A stretch's pairs (row, key head) that lie in it as a whole are finished there; what it holds of the
//   first and the last goes to a scratch slot, and a second launch joins the slots of each such pair, in the order of the line: results do
//   not depend on timing.
#include "paged_common.cuh"

namespace ats {

constexpr int PD_WARPS = 4, PD_THREADS = 32 * PD_WARPS;
constexpr int PD_STAGES = 2, PD_UNIT_BYTES = 8192;
constexpr int PD_SMEM = 1024 + PD_WARPS * PD_STAGES * PD_UNIT_BYTES;

struct PagedDecodeArgs {
  PagedRows rows;
  const __nv_bfloat16* q;   // [tokens, ldq]
  long long ldq;
  __nv_bfloat16* out;       // [tokens, ldo]
  long long ldo;
  int n_kv, rep, limit;     // rows with at most `limit` MMA rows are taken
  int grid;                 // CTAs of the main launch
  int zero_tail;            // tokens behind the last row get zeros
  float scale_log2;
  float* part_o;            // [grid, 2, rows of the MMA, D]
  float* part_ml;           // [grid, 2, rows of the MMA, 2]
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

// Units of row r on this kernel's line, per key head (0: the row is empty or another kernel's).
template <int UNIT>
__device__ __forceinline__ int pd_units(const PagedDecodeArgs& p, int r) {
  int first, fresh, keys;
  paged_row(p.rows, r, &first, &fresh, &keys);
  return fresh > 0 && (long long)fresh * p.rep <= p.limit ? (max(keys, 1) + UNIT - 1) / UNIT : 0;
}

// Sum of the units of all rows, and for every thread that of the rows in front of its own share [*r0, *r1).
template <int UNIT, int THREADS>
__device__ __forceinline__ long long pd_scan(const PagedDecodeArgs& p, int* r0, int* r1, long long* before, long long* s_sum) {
  const int share = (p.rows.R + THREADS - 1) / THREADS, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  *r0 = min(tid * share, p.rows.R);
  *r1 = min(*r0 + share, p.rows.R);
  long long mine = 0;
  for (int r = *r0; r < *r1; ++r) mine += pd_units<UNIT>(p, r);
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  long long total = 0;
  *before = incl - mine;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) *before += s_sum[w];
    total += s_sum[w];
  }
  return total;
}

// CTAs that share a line of `total` units: at least a unit for each of their warps, as long as there are that many.
__device__ __forceinline__ int pd_ctas(const PagedDecodeArgs& p, long long total) { return int(min((long long)p.grid, (total + PD_WARPS - 1) / PD_WARPS)); }

template <int D, int NR>  // NR: sets of eight MMA rows (1 or 2)
__global__ void __launch_bounds__(PD_THREADS, 3) paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                     const PagedDecodeArgs p) {
  constexpr int UNIT = 2048 / D, NT = UNIT / 8, KB = UNIT / 16, JD = D / 32, RD = D / 64, ROWS = 8 * NR;
  static_assert(ROWS * D * 4 <= PD_STAGES * PD_UNIT_BYTES, "a warp's result fits its ring");
  extern __shared__ uint8_t pd_smem[];
  __shared__ uint64_t s_full[PD_WARPS][PD_STAGES];
  __shared__ float s_m[PD_WARPS][ROWS], s_l[PD_WARPS][ROWS];
  __shared__ long long s_sum[PD_WARPS], s_at;
  __shared__ int s_row, s_abort;
  pdl_prologue();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const PagedRows& rows = p.rows;
  uint8_t* base_smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pd_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = base_smem + warp * (PD_STAGES * PD_UNIT_BYTES);
  uint64_t* full = s_full[warp];
  if (lane == 0) {
    for (int i = 0; i < PD_STAGES; ++i) mbar_init(&full[i], 1);
    mbar_fence_init();
  }
  if (tid == 0) s_abort = 0, s_row = rows.R, s_at = 0;
  if (p.zero_tail) {
    const int tail = min(max(rows.starts[rows.R], 0), rows.tokens), vecs = p.n_kv * p.rep * (D / 8);
    for (long long i = (long long)blockIdx.x * PD_THREADS + tid; i < (long long)(rows.tokens - tail) * vecs; i += (long long)gridDim.x * PD_THREADS)
      *reinterpret_cast<uint4*>(p.out + (tail + i / vecs) * p.ldo + (i % vecs) * 8) = make_uint4(0, 0, 0, 0);
  }
  // this CTA's stretch of the line
  int r0, r1;
  long long before;
  const long long total = pd_scan<UNIT, PD_THREADS>(p, &r0, &r1, &before, s_sum) * p.n_kv;
  const int ctas = pd_ctas(p, total);
  if (int(blockIdx.x) >= ctas) return;
  const long long lo = blockIdx.x * total / ctas, hi = (blockIdx.x + 1) * total / ctas;   // (not empty)
  long long at = before * p.n_kv;   // where the row's units begin
  for (int r = r0; r < r1; ++r) {
    const long long n = (long long)pd_units<UNIT>(p, r) * p.n_kv;
    if (n > 0 && at <= lo && lo < at + n) s_row = r, s_at = at;
    at += n;
  }
  __syncthreads();
  int row = s_row;
  at = s_at;
  const int box = min(UNIT, 1 << rows.page_log), per = UNIT / box;   // tokens and number of the copies of a unit's 64-column piece
  uint32_t stage = 0, parity = 0;
  bool ok = true;
  int first_seg = 1;
  long long cur = lo;
  while (cur < hi && row < rows.R) {
    int first, fresh, keys;
    paged_row(rows, row, &first, &fresh, &keys);
    const int units = pd_units<UNIT>(p, row);
    if (units == 0 || cur >= at + (long long)units * p.n_kv) {   // (the same for all threads)
      at += (long long)units * p.n_kv;
      ++row;
      continue;
    }
    const int hk = int((cur - at) / units), u0 = int((cur - at) - (long long)hk * units), u1 = int(min((long long)units, u0 + (hi - cur)));
    const bool whole = u0 == 0 && u1 == units;
    const int n_rows = fresh * p.rep, open = keys - fresh + 1;   // keys below `open` are seen by all new tokens
    const int* table = rows.tables + (long long)row * rows.width;
    const int n_pages = (keys + (1 << rows.page_log) - 1) >> rows.page_log;
    const int count = u1 - u0 > warp ? (u1 - u0 - warp + PD_WARPS - 1) / PD_WARPS : 0;   // units of this warp: u0 + warp, + 4, ..
    // coordinates of the warp's copies, one per lane, `batch` units at a time
    const int batch = 32 / per;
    auto coordinate = [&](int first_unit) {   // of copy `lane % per` of the warp's unit first_unit + lane / per
      const int i = first_unit + lane / per;
      const int k0 = (u0 + warp + i * PD_WARPS) * UNIT + (lane % per) * box;
      int c = rows.pages << rows.page_log;    // behind the pages: reads as zero
      if (i < count && (k0 >> rows.page_log) < n_pages) {
        const int id = table[k0 >> rows.page_log];
        if (id >= 0 && id < rows.pages) c = (id << rows.page_log) + (k0 & ((1 << rows.page_log) - 1));
        else atomicCAS(p.status, 0, int(kBadArgument));
      }
      return c;
    };
    int here = coordinate(0), next = count > batch ? coordinate(batch) : 0, base_unit = 0;
    auto request = [&](int i, uint32_t st) {   // whole warp; units in order
      if (i - base_unit >= batch) {
        base_unit += batch;
        here = next;
        if (base_unit + batch < count) next = coordinate(base_unit + batch);
      }
      uint8_t* dst = ring + st * PD_UNIT_BYTES;
      if (lane == 0) mbar_expect_tx(&full[st], PD_UNIT_BYTES);
      for (int s = 0; s < per; ++s) {
        const int c = __shfl_sync(0xffffffffu, here, (i - base_unit) * per + s);
        if (lane == 0) {
#pragma unroll
          for (int rd = 0; rd < RD; ++rd) {
            tma_load_3d(dst + (rd * UNIT + s * box) * 128, &map_k, &full[st], 64 * rd, hk, c);
            tma_load_3d(dst + PD_UNIT_BYTES / 2 + (rd * UNIT + s * box) * 128, &map_v, &full[st], 64 * rd, hk, c);
          }
        }
      }
    };
    for (int i = 0; i < min(count, PD_STAGES); ++i) request(i, (stage + i) % PD_STAGES);
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
    const uint32_t k_at = smem_u32(ring) + g * 128, v_at = smem_u32(ring) + PD_UNIT_BYTES / 2 + 2 * t * 128;
    // the pieces of key 8 nt + g and of the values' keys 2 t, 2 t + 1 (+ 8), swizzled by their rows modulo eight
    const uint32_t piece[2] = {uint32_t((t ^ g) << 4), uint32_t(((4 + t) ^ g) << 4)};
    const uint32_t vpiece[2] = {uint32_t((g ^ (2 * t)) << 4), uint32_t((g ^ (2 * t + 1)) << 4) + 128};
#pragma unroll 1
    for (int u = 0; u < count; ++u) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[stage], parity, &s_abort, p.status, kTimeoutFull));
      if (!ok) break;
      const int k0 = (u0 + warp + u * PD_WARPS) * UNIT;
      const uint32_t ks = k_at + stage * PD_UNIT_BYTES, vs = v_at + stage * PD_UNIT_BYTES;
      const bool edge = k0 + UNIT > open;   // the unit holds keys that some row does not see
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
      if (edge) {
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
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        uint32_t pa[4] = {pack_bf16x2(s[2 * kb][0], s[2 * kb][1]), 0u, pack_bf16x2(s[2 * kb + 1][0], s[2 * kb + 1][1]), 0u};
        if (NR > 1) pa[1] = pack_bf16x2(s[2 * kb][2 * NR - 2], s[2 * kb][2 * NR - 1]), pa[3] = pack_bf16x2(s[2 * kb + 1][2 * NR - 2], s[2 * kb + 1][2 * NR - 1]);
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
      __syncwarp();   // the stage has been read
      if (u + PD_STAGES < count) request(u + PD_STAGES, stage);
      if (++stage == PD_STAGES) stage = 0, parity ^= 1;
    }
    if (!ok) {   // copies that were issued land before the CTA gives its shared memory back
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 10000000ull) {
      }
    }
#pragma unroll
    for (int x = 0; x < NR; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    // the warps' results lie in their rings, which are empty
    auto red = [&](int w, int i, int d) { return reinterpret_cast<float*>(base_smem + w * (PD_STAGES * PD_UNIT_BYTES)) + i * D + d; };
    // lane (g, t): accumulator column 2t is dim 64 rd + 16 t + 2 i (+ 1 for the odd tile), column 2t + 1 eight dims further
#pragma unroll
    for (int x = 0; x < NR; ++x) {
      const int i = g + 8 * x;
      if (t == 0) s_m[warp][i] = m[x], s_l[warp][i] = l[x];
#pragma unroll
      for (int rd = 0; rd < RD; ++rd) {
        float* dst = red(warp, i, 64 * rd + 16 * t);
        *reinterpret_cast<float4*>(dst) = make_float4(oe[rd][0][2 * x], oo[rd][0][2 * x], oe[rd][1][2 * x], oo[rd][1][2 * x]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(oe[rd][2][2 * x], oo[rd][2][2 * x], oe[rd][3][2 * x], oo[rd][3][2 * x]);
        *reinterpret_cast<float4*>(dst + 8) = make_float4(oe[rd][0][2 * x + 1], oo[rd][0][2 * x + 1], oe[rd][1][2 * x + 1], oo[rd][1][2 * x + 1]);
        *reinterpret_cast<float4*>(dst + 12) = make_float4(oe[rd][2][2 * x + 1], oo[rd][2][2 * x + 1], oe[rd][3][2 * x + 1], oo[rd][3][2 * x + 1]);
      }
    }
    __syncthreads();
    const long long slot = (long long)blockIdx.x * 2 + (first_seg ? 0 : 1);
    for (int e = tid; e < n_rows * D; e += PD_THREADS) {
      const int i = e / D, d = e - i * D;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < PD_WARPS; ++w) top = fmaxf(top, s_m[w][i]);
      const float ref = top == -INFINITY ? 0.f : top;
      float acc = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < PD_WARPS; ++w) {
        const float f = pd_from(s_m[w][i], ref);
        acc += *red(w, i, d) * f;
        sum += s_l[w][i] * f;
      }
      if (whole) {
        const int tok = i / p.rep, head = i - tok * p.rep;
        p.out[(long long)(first + tok) * p.ldo + (long long)(hk * p.rep + head) * D + d] = __float2bfloat16(sum > 0.f ? acc / sum : acc);
      } else {
        p.part_o[(slot * ROWS + i) * D + d] = acc;
        if (d == 0) p.part_ml[(slot * ROWS + i) * 2] = top, p.part_ml[(slot * ROWS + i) * 2 + 1] = sum;
      }
    }
    fence_proxy_async_smem();   // plain accesses to the rings come before the next copies into them
    __syncthreads();
    if (s_abort) return;
    first_seg = 0;
    cur += u1 - u0;
  }
}

// One CTA per (key head, row): the scratch slots of a pair that several CTAs shared, joined in the order of the line.
constexpr int PJ_THREADS = 128;
template <int D, int NR>
__global__ void __launch_bounds__(PJ_THREADS) paged_join_kernel(const PagedDecodeArgs p) {
  constexpr int UNIT = 2048 / D, ROWS = 8 * NR;
  __shared__ long long s_sum[PJ_THREADS / 32], s_at;
  pdl_prologue();
  const int hk = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const int units = pd_units<UNIT>(p, row);
  if (units == 0) return;
  int r0, r1;
  long long before;
  const long long total = pd_scan<UNIT, PJ_THREADS>(p, &r0, &r1, &before, s_sum) * p.n_kv;
  if (r0 <= row && row < r1) {
    for (int r = r0; r < row; ++r) before += pd_units<UNIT>(p, r);
    s_at = before;
  }
  __syncthreads();
  const long long a = s_at * p.n_kv + (long long)hk * units, b = a + units;
  const int ctas = pd_ctas(p, total);
  auto owner = [&](long long x) { return ((x + 1) * ctas - 1) / total; };   // the CTA whose stretch holds x: the largest c with c total / ctas <= x
  const long long c0 = owner(a), c1 = owner(b - 1);
  if (c0 == c1) return;   // finished by that CTA
  const long long s0 = 2 * c0 + (c0 * total / ctas >= a ? 0 : 1);   // the first CTA's slot: its first piece unless its stretch began before the pair
  int first, fresh, keys;
  paged_row(p.rows, row, &first, &fresh, &keys);
  for (int e = tid; e < fresh * p.rep * D; e += PJ_THREADS) {
    const int i = e / D, d = e - i * D;
    float top = p.part_ml[(s0 * ROWS + i) * 2];
    for (long long c = c0 + 1; c <= c1; ++c) top = fmaxf(top, p.part_ml[(2 * c * ROWS + i) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
    float acc = 0.f, sum = 0.f;
#pragma unroll 4
    for (long long c = c0; c <= c1; ++c) {
      const long long at = (c == c0 ? s0 : 2 * c) * ROWS + i;
      const float f = pd_from(p.part_ml[at * 2], ref);
      acc += p.part_o[at * D + d] * f;
      sum += p.part_ml[at * 2 + 1] * f;
    }
    const int tok = i / p.rep, head = i - tok * p.rep;
    p.out[(long long)(first + tok) * p.ldo + (long long)(hk * p.rep + head) * D + d] = __float2bfloat16(sum > 0.f ? acc / sum : acc);
  }
}

template <int D, int NR>
static int launch_paged_decode(const CUtensorMap& mk, const CUtensorMap& mv, const PagedDecodeArgs& p, cudaStream_t s) {
  cudaError_t ce = cudaFuncSetAttribute(paged_decode_kernel<D, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, PD_SMEM);
  if (ce == cudaSuccess) ce = launch_pdl(paged_decode_kernel<D, NR>, dim3(p.grid), dim3(PD_THREADS), PD_SMEM, s, mk, mv, p);
  if (ce == cudaSuccess) ce = launch_pdl(paged_join_kernel<D, NR>, dim3(p.n_kv, p.rows.R), dim3(PJ_THREADS), 0, s, p);
  if (ce != cudaSuccess) return int(ce);
  return int(cudaGetLastError());
}

// CTAs of the main launch for up to `keys` keys in each of R rows: three an SM, but no more than have a unit for each of their warps.
static int paged_decode_grid(int R, int n_kv, int D, long long keys) {
  const long long units = (keys + 2048 / D - 1) / (2048 / D) * R * n_kv;
  const long long n = (units + PD_WARPS - 1) / PD_WARPS;
  return int(n < 1 ? 1 : n > 444 ? 444 : n);
}

}  // namespace ats

using namespace ats;

// Floats of scratch that `ats_paged_decode` needs: part_o this many, part_ml 2 / D as many.
ATS_API long long ats_paged_decode_scratch(int R, int n_kv, int D, long long max_keys, int limit) {
  return 2ll * paged_decode_grid(R, n_kv, D, max_keys) * (limit > 8 ? 16 : 8) * D;
}

// Rows whose new tokens times n_q / n_kv are at most `limit` (8 or 16).  q [tokens, ldq], pages [pages * page, n_kv, D] bf16, D 64 or 128, pages of 8 tokens
// (a power of two) or more; max_keys: no row has more.  zero_tail: tokens behind the last row get zeros.
ATS_API int ats_paged_decode(const void* q, long long ldq, const void* k_pages, const void* v_pages, const int* starts, const int* lengths, const int* tables,
                             void* out, long long ldo, int tokens, int R, int n_q, int n_kv, int D, int width, int pages, int page, long long max_keys, int limit,
                             float scale, int zero_tail, float* part_o, float* part_ml, int* status, void* stream) {
  if ((D != 64 && D != 128) || tokens < 1 || R < 1 || R > 65535 || n_kv < 1 || n_q % n_kv || (ldq & 7) || (ldo & 7) || page < 8 || (page & (page - 1)) ||
      (limit != 8 && limit != 16) || (long long)pages * page >= (1ll << 31) - 256 || (long long)width * page >= (1ll << 31) - 256)
    return 1003;
  static thread_local bool ctx_bound = false;
  if (!ctx_bound) {
    cudaFree(0);
    ctx_bound = true;
  }
  const int unit = 2048 / D;
  CUtensorMap mk, mv;
  int e;
  if ((e = make_tmap_pages(&mk, k_pages, (uint64_t)pages * page, n_kv, D, page < unit ? page : unit))) return e;
  if ((e = make_tmap_pages(&mv, v_pages, (uint64_t)pages * page, n_kv, D, page < unit ? page : unit))) return e;
  PagedDecodeArgs p;
  p.rows = {starts, lengths, tables, R, width, pages, __builtin_ctz(page), tokens};
  p.q = static_cast<const __nv_bfloat16*>(q); p.ldq = ldq; p.out = static_cast<__nv_bfloat16*>(out); p.ldo = ldo;
  p.n_kv = n_kv; p.rep = n_q / n_kv; p.limit = limit; p.grid = paged_decode_grid(R, n_kv, D, max_keys); p.zero_tail = zero_tail;
  p.scale_log2 = scale * 1.4426950408889634f; p.part_o = part_o; p.part_ml = part_ml; p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (limit > 8) return D == 64 ? launch_paged_decode<64, 2>(mk, mv, p, s) : launch_paged_decode<128, 2>(mk, mv, p, s);
  return D == 64 ? launch_paged_decode<64, 1>(mk, mv, p, s) : launch_paged_decode<128, 1>(mk, mv, p, s);
}
