// Serving from a paged key / value cache, for sm_100a: the pages of every row, the write of new tokens into them, and attention over them
// for any head width and in true 32-bit.
//
// A pool holds N pages of `page` tokens; row r of the table lists the pages of row r in order, so that token i of the row lies in slot
// table[r][i / page] * page + i % page.  Free pages are a stack.
//
// * ats_page_plan: what a step with `fresh` new tokens per row needs: pages taken from the stack (and given back by rows that are closed),
//   packed starts of the rows, slot and position of every new token.
// * ats_paged_append: rotary embedding of the new tokens' queries and keys; keys and values go to their slots.
// * ats_paged_attn_any: causal grouped-query attention of the new tokens over their rows' pages (the general form).
#include "paged_common.cuh"
#include "typed.cuh"

namespace ats {

// ------------------------------------------------------------------------------------------------
// Page plan.  With held = pages a row has, need = pages it gains and freed = pages it gives back, all of a step follows from three
// prefix sums over the rows: packed starts, taken pages, returned pages.  The stack after the returns is free[0 .. n) followed by the
// returned pages in row order; page a of the step comes from its top, n + returned - 1 - a.  What is read (stack below n, table entries
// below held) and what is written (stack from n on, entries from held on) never overlap, so every CTA works out its share of tokens and
// pages from the sums alone and none waits for another; with `commit` the last CTA to finish writes the counters that all have read.
// A step that does not fit is refused as a whole: no row has tokens in it and nothing changes.
// Bound by latency, a chain of dependent loads: counters and lengths, the sums, then a table or stack entry per token.  64 rows of a token each 2.7 us (a launch
// that does next to nothing takes about two); 500 rows with 14,500 tokens 5.7 us, whose 191 KB would take 0.03.  So a token a thread on up to 148 CTAs, each
// of which does the sums over the rows for itself: with several tokens a thread and the sums in steps of 256 rows the latter took 10.0 us.
// ------------------------------------------------------------------------------------------------
constexpr int PLAN_THREADS = 256;
constexpr int PLAN_MAX_ROWS = 4096;

struct PlanArgs {
  int* lengths;        // [R] tokens a row holds
  const int* fresh;    // [R] tokens to come; -1: the row is closed
  int* tables;         // [R, width]
  int* free;           // [pages] stack
  int* state;          // {free pages, refusal of the last committed step, CTAs done, -}
  int* starts;         // [R + 1]
  int* slots;          // [tokens]
  int* positions;      // [tokens]
  int* lengths_out;    // [R]
  int* info;           // {free pages after the step, refusal}
  int R, width, pages, page_log, tokens, commit;
};

__device__ __forceinline__ int last_le(const int* prefix, int n, int x) {   // largest i < n with prefix[i] <= x (prefix[0] = 0, not decreasing)
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(const PlanArgs p) {
  pdl_prologue();
  extern __shared__ int plan_smem[];
  int* starts = plan_smem;                 // [R + 1] each: the row's first token, first taken page, first returned page
  int* taken = starts + p.R + 1;
  int* returned = taken + p.R + 1;
  __shared__ int s_warp[3][PLAN_THREADS / 32];
  __shared__ int s_bad, s_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int page = 1 << p.page_log;
  const long long room = (long long)p.width << p.page_log;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  const int n_free = p.state[0];
  // every thread sums up a share of consecutive rows
  const int share = (p.R + PLAN_THREADS - 1) / PLAN_THREADS, r0 = min(tid * share, p.R), r1 = min(r0 + share, p.R);
  auto row = [&](int old, int fresh, int (&v)[3]) {   // tokens, pages taken, pages returned
    v[0] = v[1] = v[2] = 0;
    // 1: more tokens than the row's table or the packed batch holds (or a length that no row has)
    if (old < 0 || old > room || fresh < -1 || fresh > p.tokens || old + (long long)max(fresh, 0) > room) {
      s_bad = 1;
      return;
    }
    const int held = (old + page - 1) >> p.page_log;
    v[0] = max(fresh, 0);
    if (fresh < 0) v[2] = held;
    else v[1] = ((old + fresh + page - 1) >> p.page_log) - held;
  };
  int sum[3] = {0, 0, 0}, v[3];
#pragma unroll 4
  for (int r = r0; r < r1; ++r) {
    row(p.lengths[r], p.fresh[r], v);
    sum[0] += v[0], sum[1] += v[1], sum[2] += v[2];
  }
  int carry[3], before[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    int incl = sum[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) s_warp[i][warp] = incl;
    before[i] = incl - sum[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    carry[i] = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 32; ++w) {
      if (w < warp) before[i] += s_warp[i][w];
      carry[i] += s_warp[i][w];
    }
  }
  for (int r = r0; r < r1; ++r) {
    starts[r] = before[0], taken[r] = before[1], returned[r] = before[2];
    row(p.lengths[r], p.fresh[r], v);
    before[0] += v[0], before[1] += v[1], before[2] += v[2];
  }
  if (tid == 0) starts[p.R] = carry[0], taken[p.R] = carry[1], returned[p.R] = carry[2];
  __syncthreads();
  int refused = s_bad;
  if (!refused && carry[0] > p.tokens) refused = 1;
  if (!refused && carry[1] > carry[2] + n_free) refused = 2;   // 2: not enough free pages
  if (!refused && (n_free < 0 || n_free + carry[2] > p.pages)) refused = 3;   // 3: more pages on the stack than there are
  const int total = refused ? 0 : carry[0], n_taken = refused ? 0 : carry[1], n_returned = refused ? 0 : carry[2];
  auto stack = [&](int i) {   // the stack after the returns
    if (i < n_free) return p.free[i];
    const int r = last_le(returned, p.R, i - n_free);
    return p.tables[(long long)r * p.width + (i - n_free - returned[r])];
  };
  const int me = int(blockIdx.x) * PLAN_THREADS + tid, step = int(gridDim.x) * PLAN_THREADS;
  for (int t = me; t < p.tokens; t += step) {
    int slot = -1, pos = 0;
    if (t < total) {
      const int r = last_le(starts, p.R, t);
      const int old = p.lengths[r], held = (old + page - 1) >> p.page_log;
      pos = old + t - starts[r];
      const int j = pos >> p.page_log;
      const int id = j < held ? p.tables[(long long)r * p.width + j] : stack(n_free + n_returned - 1 - (taken[r] + j - held));
      if (id >= 0 && id < p.pages) slot = (id << p.page_log) + (pos & (page - 1));
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
  for (int a = me; a < n_taken; a += step) {
    const int r = last_le(taken, p.R, a);
    const int held = (p.lengths[r] + page - 1) >> p.page_log;
    p.tables[(long long)r * p.width + held + a - taken[r]] = stack(n_free + n_returned - 1 - a);
  }
  const int n_after = n_free + n_returned - n_taken;
  for (int i = n_free + me; i < n_after; i += step) p.free[i] = stack(i);
  bool last = gridDim.x == 1;
  if (p.commit && !last) {
    __threadfence();
    __syncthreads();
    if (tid == 0) s_last = atomicAdd(&p.state[2], 1) == int(gridDim.x) - 1;
    __syncthreads();
    last = s_last;
  } else if (!p.commit) {
    last = blockIdx.x == 0;
  }
  if (!last) return;
  __syncthreads();
  for (int r = tid; r <= p.R; r += PLAN_THREADS) {
    p.starts[r] = refused ? 0 : starts[r];
    if (r < p.R) {
      const int old = p.lengths[r], fresh = p.fresh[r];
      p.lengths_out[r] = refused ? old : fresh < 0 ? 0 : old + fresh;
    }
  }
  if (tid == 0) {
    p.info[0] = n_after;
    p.info[1] = refused;
    if (p.commit) p.state[0] = n_after, p.state[1] = refused, p.state[2] = 0;
  }
}

// ------------------------------------------------------------------------------------------------
// Append.  (a, b) of a head's halves become (a cos - b sin, b cos + a sin), fp32, rounded once to the stored type.  A CTA takes every so many-th token, a thread
// of it always the same item: eight columns of a head's first half and the eight that they are rotated with, or sixteen columns that
// only move.  A thread asks for the next token's columns before it works on this one's; a warp's lanes cover whole halves of consecutive heads, so that every
// access is whole sectors.  Bound by memory: the projection is read once, queries, keys and values are written once.  8,200 tokens of 32 / 8 heads of 128
// (202 MB): 36 us = 5.6 TB/s, 87 % of a copy's rate; 40.8 with a CTA a token and nothing asked for ahead, 48.3 with the items of all tokens in one line.
// 64 tokens of 32 / 4 heads of 64: 1.9 us, the launch.
// ------------------------------------------------------------------------------------------------
constexpr int APP_MAX_THREADS = 512;

struct AppendArgs {
  const void* qkv;         // [tokens, ld]: n_q query heads, n_kv key heads, n_kv value heads of d
  long long ld;
  const float* cos_t;      // [table, d / 2], or null: queries and keys are rotated already and no queries are written
  const float* sin_t;
  const int* positions;
  const int* slots;
  void* q_out;             // [tokens, n_q * d]
  void* k_pages;           // [pages * page, n_kv, d]
  void* v_pages;
  int tokens, n_q, n_kv, d, table;
  long long n_slots;
  int* status;
};

template <typename T>
__global__ void __launch_bounds__(APP_MAX_THREADS) paged_append_kernel(const AppendArgs p) {
  pdl_prologue();
  using Raw = typename Typed<T>::Raw8;
  const int half = p.d >> 1;
  const int lanes = half >> 3, turned = p.cos_t ? (p.n_q + p.n_kv) * lanes : 0;   // lanes of a head, items that are rotated
  const int from = p.cos_t ? (p.n_q + p.n_kv) * p.d : p.n_q * p.d;                // first column that only moves
  const int pieces = ((p.n_q + 2 * p.n_kv) * p.d - from) >> 3, items = turned + ((pieces + 1) >> 1);
  const int keys = (p.n_q + p.n_kv) * p.d;   // columns up to here are queries and keys
  for (int i = threadIdx.x; i < items; i += blockDim.x) {
    const bool turn = i < turned;
    const int h = turn ? i / lanes : 0, c = turn ? (i - h * lanes) * 8 : 0;
    const int c0 = turn ? h * p.d + c : from + (i - turned) * 16, c1 = turn ? c0 + half : c0 + 8;
    const bool second = turn || 2 * (i - turned) + 1 < pieces;
    // where the item's columns go, as far as the slot does not matter
    T* base = turn && h < p.n_q ? static_cast<T*>(p.q_out) : c0 < keys ? static_cast<T*>(p.k_pages) : static_cast<T*>(p.v_pages);
    T* base1 = turn ? base + half : c1 < keys ? static_cast<T*>(p.k_pages) : static_cast<T*>(p.v_pages);
    const bool to_q = turn && h < p.n_q;
    const int off = to_q ? h * p.d + c : c0 < keys ? c0 - p.n_q * p.d : c0 - keys, off1 = turn ? off : c1 < keys ? c1 - p.n_q * p.d : c1 - keys;
    auto fetch = [&](int t, Raw& a, Raw& b, int& slot, int& pos) {
      const T* row = static_cast<const T*>(p.qkv) + (long long)t * p.ld;
      a = Typed<T>::raw8(row + c0);
      b = Typed<T>::raw8(row + (second ? c1 : c0));
      slot = p.slots[t];
      pos = p.positions[t];
    };
    Raw a, b, a_next, b_next;
    int slot, pos, slot_next = -1, pos_next = 0;
    int t = blockIdx.x;
    fetch(t, a, b, slot, pos);
    for (; t < p.tokens; t += gridDim.x, a = a_next, b = b_next, slot = slot_next, pos = pos_next) {
      if (t + int(gridDim.x) < p.tokens) fetch(t + gridDim.x, a_next, b_next, slot_next, pos_next);   // the next token's, under this one's
      if (slot >= p.n_slots || pos < 0 || (p.cos_t && pos >= p.table)) {   // a plan of another pool, or positions that the tables do not reach
        if (i == 0) atomicCAS(p.status, 0, int(kBadArgument));
        continue;
      }
      if (!to_q && slot < 0) continue;
      const long long place = to_q ? (long long)t * p.n_q * p.d : (long long)slot * p.n_kv * p.d;
      if (turn) {
        float u[8], w[8], cs[8], sn[8], x[8], y[8];
        Typed<float>::load8(p.cos_t + (long long)pos * half + c, cs);
        Typed<float>::load8(p.sin_t + (long long)pos * half + c, sn);
        Typed<T>::unpack8(a, u);
        Typed<T>::unpack8(b, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = u[e] * cs[e] - w[e] * sn[e];
          y[e] = w[e] * cs[e] + u[e] * sn[e];
        }
        Typed<T>::store8(base + place + off, x);
        Typed<T>::store8(base1 + place + off1, y);
      } else {
        Typed<T>::store_raw8(base + place + off, a);
        if (second) Typed<T>::store_raw8(base1 + place + off1, b);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Attention, general form: any head width that is a multiple of 8 up to 256, any group, any page size, bf16 or fp32 with fp32 sums.
// A CTA serves one token and up to four query heads of a group.  Its four warps take blocks of 32 keys in turn: a lane scores one key for
// all heads, then the lanes share out the value's columns; softmax as a running maximum and sum per warp, warps joined at the end.  Bound by its fp32 FMAs
// and the latency of its loads.  Few tokens: a row's blocks of 128 keys are shared out over `splits` CTAs, as many as make eight
// an SM but no more than the longest row has blocks; their sums are joined in order by a second launch.  One row of 32,000 keys x 8 heads of 96 in bf16 111 us (one
// CTA a token and group 4,800), 64 rows of 200 to 2,000 keys x 8 of 96 251 (373), x 4 of 64 in fp32 186 (282); with four an SM 112, 372, 283 and 8 rows of 4,000 x 8 of
// 128 in fp32 164 instead of 179; with twelve 113, 244, 180 and 188.  Portions: a CTA a token, each of which reads its keys again (from L2): 500 tokens x 8 heads of 96 245 us, 2,000 3,026.
// Tokens behind the last row get zeros (or stay, `keep_tail`), as does a token that sees no key.
// ------------------------------------------------------------------------------------------------
constexpr int ANY_WARPS = 4, ANY_HEADS = 4, ANY_BLOCK = 32 * ANY_WARPS, ANY_MAX_SPLITS = 64;

struct PagedAnyArgs {
  const void* q;         // [tokens, ldq]
  long long ldq;
  const void* k_pages;   // [pages * page, n_kv, d]
  const void* v_pages;
  const int* starts;     // [R + 1]
  const int* lengths;    // [R] tokens of a row, the new ones among them
  const int* tables;     // [R, width]
  void* out;             // [tokens, ldo]
  long long ldo;
  int tokens, R, n_q, n_kv, d, width, pages, page_log, keep_tail;
  int splits;
  float* part;           // [splits, tokens, n_q, d + 2]: sums, largest score, sum of weights (one split: not used)
  float scale;
  int* status;
};


template <typename T>
__global__ void __launch_bounds__(32 * ANY_WARPS) paged_attn_any_kernel(const PagedAnyArgs p) {
  pdl_prologue();
  const int groups = (p.n_q / p.n_kv + ANY_HEADS - 1) / ANY_HEADS;
  const int t = blockIdx.x, hk = blockIdx.y / groups, rep = p.n_q / p.n_kv, h0 = (blockIdx.y % groups) * ANY_HEADS;
  const int nh = min(ANY_HEADS, rep - h0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, d = p.d;
  extern __shared__ float any_smem[];
  float* sq = any_smem;                               // [ANY_HEADS][d], scaled
  float* sp = sq + ANY_HEADS * d;                     // [ANY_WARPS][ANY_HEADS][32]
  float* so = sp + ANY_WARPS * ANY_HEADS * 32;        // [ANY_WARPS][ANY_HEADS][d]
  __shared__ float s_m[ANY_WARPS][ANY_HEADS], s_l[ANY_WARPS][ANY_HEADS];
  T* orow = static_cast<T*>(p.out) + (long long)t * p.ldo + (long long)(hk * rep + h0) * d;
  int n = 0, r = 0;
  const int tail = p.starts[p.R];
  if (t < tail) {
    r = last_le(p.starts, p.R, t);
    n = p.lengths[r] - (p.starts[r + 1] - t) + 1;      // keys that this token sees
    n = (int)min((long long)n, (long long)p.width << p.page_log);
  } else if (p.keep_tail) {
    return;
  }
  float* part = p.part + (((long long)blockIdx.z * p.tokens + t) * p.n_q + hk * rep + h0) * (d + 2);
  const int blocks = (max(n, 0) + ANY_BLOCK - 1) / ANY_BLOCK;
  const int from = int((long long)blocks * blockIdx.z / p.splits) * ANY_BLOCK;
  n = min(n, int((long long)blocks * (blockIdx.z + 1) / p.splits) * ANY_BLOCK);   // (keys of this CTA end here)
  if (n <= from) {
    if (p.splits > 1)
      for (int i = tid; i < nh * (d + 2); i += 32 * ANY_WARPS) part[i] = i % (d + 2) == d ? -INFINITY : 0.f;
    else
      for (int i = tid; i < nh * d; i += 32 * ANY_WARPS) Typed<T>::store(orow + i, 0.f);
    return;
  }
  const T* qrow = static_cast<const T*>(p.q) + (long long)t * p.ldq + (long long)(hk * rep + h0) * d;
  for (int i = tid; i < nh * d; i += 32 * ANY_WARPS) sq[i] = Typed<T>::load(qrow + i) * p.scale;
  __syncthreads();
  float m[ANY_HEADS], l[ANY_HEADS], acc[ANY_HEADS][8];
#pragma unroll
  for (int h = 0; h < ANY_HEADS; ++h) {
    m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[h][e] = 0.f;
  }
  float* wp = sp + warp * ANY_HEADS * 32;
  const int* table = p.tables + (long long)r * p.width;
  const long long ld = (long long)p.n_kv * d;
  for (int k0 = from + warp * 32; k0 < n; k0 += ANY_BLOCK) {
    const int j = k0 + lane;
    float s[ANY_HEADS];
#pragma unroll
    for (int h = 0; h < ANY_HEADS; ++h) s[h] = 0.f;
    long long at = -1;
    if (j < n) {
      const int id = table[j >> p.page_log];
      if (id >= 0 && id < p.pages) at = (((long long)id << p.page_log) + (j & ((1 << p.page_log) - 1))) * ld + (long long)hk * d;
      else atomicCAS(p.status, 0, int(kBadArgument));
    }
    if (at >= 0) {
      const T* krow = static_cast<const T*>(p.k_pages) + at;
#pragma unroll 4
      for (int c = 0; c < d; c += 8) {   // (loads of several pieces under way at once: few warps share an SM where tokens are few)
        float kv[8];
        Typed<T>::load8(krow + c, kv);
#pragma unroll
        for (int h = 0; h < ANY_HEADS; ++h)
          if (h < nh) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s[h] = fmaf(sq[h * d + c + e], kv[e], s[h]);
          }
      }
    }
#pragma unroll
    for (int h = 0; h < ANY_HEADS; ++h) {
      if (h >= nh) break;
      if (at < 0) s[h] = -INFINITY;
      const float top = fmaxf(m[h], warp_max(s[h]));
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = expf(m[h] - base), pr = expf(s[h] - base);
      m[h] = top;
      l[h] = l[h] * keep + warp_sum(pr);
      wp[h * 32 + lane] = pr;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[h][e] *= keep;
    }
    __syncwarp();
    const int cnt = min(32, n - k0);
    for (int i = 0; i < cnt; i += 4) {   // (keys from cnt on: no place, no weight)
      const T* vrow[4];
      bool there[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long vat = __shfl_sync(0xffffffffu, at, i + j);
        there[j] = vat >= 0;
        vrow[j] = static_cast<const T*>(p.v_pages) + vat;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = lane + 32 * e;
        if (c < d) {
          float vv[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) vv[j] = there[j] ? Typed<T>::load(vrow[j] + c) : 0.f;
#pragma unroll
          for (int h = 0; h < ANY_HEADS; ++h)
            if (h < nh) {
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[h][e] = fmaf(wp[h * 32 + i + j], vv[j], acc[h][e]);
            }
        }
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int h = 0; h < ANY_HEADS; ++h) {
    if (h >= nh) break;
    if (lane == 0) s_m[warp][h] = m[h], s_l[warp][h] = l[h];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < d) so[(warp * ANY_HEADS + h) * d + lane + 32 * e] = acc[h][e];
  }
  __syncthreads();
  for (int i = tid; i < nh * d; i += 32 * ANY_WARPS) {
    const int h = i / d, c = i - h * d;
    float top = -INFINITY;
    for (int w = 0; w < ANY_WARPS; ++w) top = fmaxf(top, s_m[w][h]);
    const float base = top == -INFINITY ? 0.f : top;
    float o = 0.f, sum = 0.f;
    for (int w = 0; w < ANY_WARPS; ++w) {
      const float f = expf(s_m[w][h] - base);
      o += so[(w * ANY_HEADS + h) * d + c] * f;
      sum += s_l[w][h] * f;
    }
    if (p.splits > 1) {
      part[h * (d + 2) + c] = o;
      if (c == 0) part[h * (d + 2) + d] = top, part[h * (d + 2) + d + 1] = sum;
    } else {
      Typed<T>::store(orow + i, sum > 0.f ? o / sum : o);   // (a sum that is no number stays one)
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(128) paged_any_join_kernel(const PagedAnyArgs p) {
  pdl_prologue();
  const int t = blockIdx.x, h = blockIdx.y, d = p.d;
  if (p.keep_tail && t >= p.starts[p.R]) return;
  const float* part = p.part + ((long long)t * p.n_q + h) * (d + 2);
  const long long step = (long long)p.tokens * p.n_q * (d + 2);
  float top = -INFINITY, sum = 0.f;
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, part[s * step + d]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int s = 0; s < p.splits; ++s) sum += part[s * step + d + 1] * expf(part[s * step + d] - base);
  for (int c = threadIdx.x; c < d; c += 128) {
    float o = 0.f;
    for (int s = 0; s < p.splits; ++s) o += part[s * step + c] * expf(part[s * step + d] - base);
    Typed<T>::store(static_cast<T*>(p.out) + (long long)t * p.ldo + (long long)h * d + c, sum > 0.f ? o / sum : o);
  }
}

}  // namespace ats

using namespace ats;

ATS_API int ats_page_plan(int* lengths, const int* fresh, int* tables, int* free_stack, int* state, int* starts, int* slots, int* positions, int* lengths_out,
                          int* info, int R, int width, int pages, int page, int tokens, int commit, void* stream) {
  if (R < 1 || R > PLAN_MAX_ROWS || width < 1 || pages < 1 || page < 1 || (page & (page - 1)) || tokens < 0 || tokens > (1 << 18) ||
      (long long)R * width >= (1ll << 31) || (long long)pages * page >= (1ll << 31) || (long long)width * page >= (1ll << 31))
    return 1003;
  PlanArgs p;
  p.lengths = lengths; p.fresh = fresh; p.tables = tables; p.free = free_stack; p.state = state; p.starts = starts; p.slots = slots;
  p.positions = positions; p.lengths_out = lengths_out; p.info = info;
  p.R = R; p.width = width; p.pages = pages; p.page_log = __builtin_ctz(page); p.tokens = tokens; p.commit = commit;
  const int blocks = max(1, min(148, (max(tokens, R) + PLAN_THREADS - 1) / PLAN_THREADS));   // (a token a thread: chains of dependent loads run side by side)
  const size_t smem = 3 * size_t(R + 1) * sizeof(int);
  cudaError_t ce = cudaSuccess;
  if (smem > 48 * 1024) ce = cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (ce == cudaSuccess) ce = launch_pdl(page_plan_kernel, dim3(blocks), dim3(PLAN_THREADS), smem, static_cast<cudaStream_t>(stream), p);
  if (ce != cudaSuccess) return int(ce);
  return int(cudaGetLastError());
}

// fp32: 0 = bf16.  cos_t null: no rotation, q_out is not written.  d a multiple of 16 (of 8 without rotation), at most 256.
ATS_API int ats_paged_append(const void* qkv, long long ld, const float* cos_t, const float* sin_t, int table, const int* positions, const int* slots, void* q_out,
                             void* k_pages, void* v_pages, int tokens, int n_q, int n_kv, int d, long long n_slots, int fp32, int* status, void* stream) {
  if (tokens < 1 || n_q < 1 || n_kv < 1 || d < 8 || d > 256 || (d & (cos_t ? 15 : 7)) || (ld & 7) || off_16(qkv, cos_t, sin_t, k_pages, v_pages) || (cos_t && off_16(q_out))) return 1003;
  AppendArgs p;
  p.qkv = qkv; p.ld = ld; p.cos_t = cos_t; p.sin_t = sin_t; p.positions = positions; p.slots = slots; p.q_out = q_out; p.k_pages = k_pages;
  p.v_pages = v_pages; p.tokens = tokens; p.n_q = n_q; p.n_kv = n_kv; p.d = d; p.table = table; p.n_slots = n_slots; p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int items = cos_t ? (n_q + n_kv) * (d >> 4) + (n_kv * (d >> 3) + 1) / 2 : n_kv * (d >> 3);
  const dim3 threads(min(APP_MAX_THREADS, (items + 31) / 32 * 32));
  const dim3 grid(min(tokens, 148 * max(1, 1536 / int(threads.x))));
  const cudaError_t ce = fp32 ? launch_pdl(paged_append_kernel<float>, grid, threads, 0, s, p)
                              : launch_pdl(paged_append_kernel<__nv_bfloat16>, grid, threads, 0, s, p);
  if (ce != cudaSuccess) return int(ce);
  return int(cudaGetLastError());
}

// CTAs that share a token's keys, of which there are `keys` at most.
ATS_API long long ats_paged_any_splits(int tokens, int n_q, int n_kv, long long keys) {
  const long long ctas = (long long)tokens * n_kv * ((n_q / n_kv + ANY_HEADS - 1) / ANY_HEADS);
  const long long splits = min((keys + ANY_BLOCK - 1) / ANY_BLOCK, 8 * 148 / max(ctas, 1ll));
  return max(1ll, min(splits, (long long)ANY_MAX_SPLITS));
}

// splits > 1: `part` is scratch of splits * tokens * n_q * (d + 2) floats.
ATS_API int ats_paged_attn_any(const void* q, long long ldq, const void* k_pages, const void* v_pages, const int* starts, const int* lengths, const int* tables,
                               void* out, long long ldo, int tokens, int R, int n_q, int n_kv, int d, int width, int pages, int page, float scale, int keep_tail,
                               int fp32, int splits, float* part, int* status, void* stream) {
  if (splits < 1 || splits > ANY_MAX_SPLITS || (splits > 1 && !part) || n_q > 65535 || tokens < 1 || R < 1 || n_kv < 1 || n_q % n_kv || d < 8 || d > 256 || (d & 7) || (ldq & 7) || (ldo & 7) || page < 1 || (page & (page - 1)) || off_16(k_pages, v_pages)) return 1003;
  const int groups = (n_q / n_kv + ANY_HEADS - 1) / ANY_HEADS;
  if ((long long)n_kv * groups > 65535) return 1003;
  PagedAnyArgs p;
  p.q = q; p.ldq = ldq; p.k_pages = k_pages; p.v_pages = v_pages; p.starts = starts; p.lengths = lengths; p.tables = tables; p.out = out; p.ldo = ldo;
  p.tokens = tokens; p.R = R; p.n_q = n_q; p.n_kv = n_kv; p.d = d; p.width = width; p.pages = pages; p.page_log = __builtin_ctz(page);
  p.keep_tail = keep_tail; p.scale = scale; p.splits = splits; p.part = part; p.status = status;
  const size_t smem = sizeof(float) * (ANY_HEADS * d + ANY_WARPS * ANY_HEADS * 32 + ANY_WARPS * ANY_HEADS * d);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(tokens, n_kv * groups, splits);
  cudaError_t ce = fp32 ? launch_pdl(paged_attn_any_kernel<float>, grid, dim3(32 * ANY_WARPS), smem, s, p)
                        : launch_pdl(paged_attn_any_kernel<__nv_bfloat16>, grid, dim3(32 * ANY_WARPS), smem, s, p);
  if (ce == cudaSuccess && splits > 1)
    ce = fp32 ? launch_behind(paged_any_join_kernel<float>, dim3(tokens, n_q), dim3(128), s, 0, p) : launch_behind(paged_any_join_kernel<__nv_bfloat16>, dim3(tokens, n_q), dim3(128), s, 0, p);
  if (ce != cudaSuccess) return int(ce);
  return int(cudaGetLastError());
}
