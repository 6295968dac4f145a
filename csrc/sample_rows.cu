// Next tokens from given random numbers, every row with sampling numbers of its own, for sm_100a.
//
// A row's scores x (penalised where the row's history says so) are put in order: larger first, lower index first among equals.  Three rules
// cut the order to a leading run: the first k tokens; the tokens with mass before them <= top_p Z, Z the mass of those k; the tokens with
// mass >= min_p of the first one's.  The answer is the lowest index whose cumulative mass over the kept tokens, in index order, exceeds
// u times their total.  A temperature <= 0 takes the first token of the order.
//
// * The order is that of one 64-bit number per token: (order-preserving image of x) * 2^32 + (2^32 - 1 - index); all are distinct.
// * The mass of a token is exp((x - max) / T) in fixed point, 42 bits behind the point, from a 64-bit exponential.  Integer sums do not depend
//   on their order, so results repeat whatever the split over threads, and a random number next to a border falls where a 64-bit
//   evaluation puts it: the rounding of all masses together moves a border by 2^-43 sqrt(V) of the largest mass or so.
//   2^42 times 2^20 tokens stays below 2^63.
// * NaN counts as -infinity (mass 0), -0 as 0.
//
// One cluster per row, a contiguous slice of the vocabulary per CTA, read once into shared memory where it fits.  No sort of the vocabulary:
// tokens are counted by how far below the largest they lie (4,095 bins over the 30.5 T that have any mass, and one for the rest), which brackets a
// cut between two bins; only the tokens of the bracket are collected and cut exactly.
//   top-k           the largest of every eight tokens is counted: k of these above a bin mean k tokens above it, and the tokens from there up are a
//                   little more than k (k above half of the eights: all tokens are counted).  They are all that is kept, so nothing but these few needs an exponential.
//   top-p alone     one pass sums the masses by distance, exactly (integers, two bins in one), so one bin holds the cut and everything above it is known,
//                   for the row and for each CTA; the draw then looks into the slice of one CTA.
//   neither         one pass of masses.
// Up to 256 collected tokens are compared with one another, up to 2,048 are cut by weights counted over 512 places of the keys' range, then over the place that holds
// the cut (sorting them took 30 us instead of 5).  Cuts whose brackets hold more (thousands of equal scores, k above 1,024) are found by bisection over the 64-bit order.
// The draw works on sums per 256 consecutive tokens and looks into one of them.
// Bound by latency rather than by a unit: over rows of all kinds memory is busy to 6 %, the FP64 pipe to 9, the SMs' issue to 32; warps wait at barriers first (three to
// five of the cluster; while one CTA cuts the list the others have nothing to do), and 256 rows are 3.5 waves of clusters.  Rows without top-k add 13 FP64 operations and
// 45 others a token and counts in shared memory (rows of equal scores meet in a bin).  64 registers a thread, for two CTAs an SM, leave 30 words of it in local memory.  256 x 131,072 bf16 (67 MB, 10 us at a copy's rate): greedy 30 us, top-k 50 66, no cut 88, k = 1,000 119, top-p alone 160 to
// 290, rows of all kinds 145 to 149; 64 x 100,003 fp32, all with top-k 34 to 36; 4 x 32,000 12.  With bounds from counts alone and a second sum for what they leave open the rows
// of all kinds took 170 us (top-p alone 154 to 365), with two tokens at a time in the passes with exponentials 158; the first form, a bisection with a pass over the
// row per step, took 8,146, 2,761 and 543 us.
#include "paged_common.cuh"

namespace ats {

constexpr int SR_THREADS = 512, SR_WARPS = SR_THREADS / 32;
constexpr int SR_MASS_BITS = 42;
constexpr int SR_MAX_VOCAB = 1 << 20;
constexpr int SR_BINS = 4096;          // the last one: no mass
constexpr float SR_RANGE = 30.5f;      // in units of T: exp(-30.49) 2^42 rounds to nothing
constexpr int SR_MASS_BINS = SR_BINS / 2;
constexpr int SR_LIST = 2048;
static_assert(SR_LIST >= SR_MASS_BINS);
constexpr int SR_MAX_K = 1024;
constexpr int SR_FEW = SR_THREADS / 2;
constexpr int SR_CHUNK = 256;
constexpr int SR_MAX_CLUSTER = 8;
constexpr int SR_CACHED = 131072 + SR_CHUNK * 8;   // bytes of a slice that is kept in shared memory at most

struct SampleRowsArgs {
  const void* logits;   // [B, ld] bf16 or fp32
  long long ld;
  int V, slice;         // tokens of a CTA (a multiple of SR_CHUNK)
  int cached;           // the slice is kept in shared memory
  const float* uniform;       // [B]
  const float* temperature;   // [B], or null: the number beside it
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* penalty;
  float temperature1, top_p1, min_p1, penalty1;
  int top_k1;
  const long long* history;   // [B, hist_ld] token ids, ids outside [0, V) are ignored; or null
  long long hist_ld;
  int hist_len;
  long long* out;             // [B]
};

template <typename T>
struct SampleRowsSmem {   // byte offsets of the dynamic shared memory
  int hist, list, chunks, seen, raw, total;
  __host__ __device__ SampleRowsSmem(int slice, bool cached) {
    hist = 0;                            // u32 [SR_BINS], or halves of SR_MASS_BINS masses; later u64 [SR_LIST]: this CTA's tokens of the bracket
    list = hist + SR_BINS * 4;           // u64 [SR_LIST]: the cluster's tokens of the bracket (rank 0); before that the cluster's masses by distance
    chunks = list + SR_LIST * 8;         // u64 [slice / SR_CHUNK]
    seen = chunks + slice / SR_CHUNK * 8;        // one bit per token of the slice
    raw = (seen + slice / 8 + 15) / 16 * 16;     // the slice
    total = raw + (cached ? slice * int(sizeof(T)) : 0);
  }
};

__device__ __forceinline__ uint64_t sr_ld_u64(const void* local, uint32_t rank) {   // the same place in another CTA of the cluster
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(local), rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t sr_ld_u32(const void* local, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(local), rank)) : "memory");
  return v;
}
__device__ __forceinline__ void sr_st_u64(void* local, uint32_t rank, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_u32(local), rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void sr_st_u32(void* local, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(smem_u32(local), rank)), "r"(v) : "memory");
}
__device__ __forceinline__ uint64_t sr_warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the block (valid in all threads); two barriers, so `red` [SR_WARPS] may be used again at once.
__device__ __forceinline__ uint64_t sr_block_sum(uint64_t v, uint64_t* red) {
  v = sr_warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int i = 0; i < SR_WARPS; ++i) t += red[i];
  return t;
}
// Exclusive prefix over the block's threads; *total: the sum.
template <typename N>
__device__ __forceinline__ N sr_block_scan(N v, N* red, N* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  N incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();
  if (lane == 31) red[warp] = incl;
  __syncthreads();
  N before = incl - v, all = 0;
#pragma unroll
  for (int w = 0; w < SR_WARPS; ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  *total = all;
  return before;
}

// order-preserving image of a float without NaN
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// exp(-w) for w >= 0 (from 44 on, and for NaN, exp(-44): no mass): w = n ln 2 / 32 - z, |z| <= ln 2 / 64; exp(z) by its Taylor series to the fifth power (the next term is below 2^-48), 2^-(n mod 32)/32
// from a table.
__device__ __forceinline__ double sr_exp_neg(double w, const double* table) {
  constexpr double magic = 6755399441055744.0;   // 1.5 * 2^52
  w = __hiloint2double(int(min(uint32_t(__double2hiint(w)), 0x40460000u)), __double2loint(w));   // (the upper half of 44.0)
  const double t = fma(w, 32 * 1.4426950408889634074, magic);
  const int n = __double2loint(t);
  const double z = fma(t - magic, 0.69314718055994530942 / 32, -w);
  double r = fma(z, 1.0 / 120, 1.0 / 24);
  r = fma(r, z, 1.0 / 6);
  r = fma(r, z, 0.5);
  r = fma(r, z, 1.0);
  r = fma(r, z, 1.0) * table[n & 31];
  return __hiloint2double(__double2hiint(r) - ((n >> 5) << 20), __double2loint(r));   // (n / 32 stays far from the smallest exponents)
}

template <typename T>
__global__ void __launch_bounds__(SR_THREADS, 2) sample_rows_kernel(const SampleRowsArgs p) {
  pdl_prologue();
  extern __shared__ __align__(16) uint8_t sr_smem[];
  __shared__ uint64_t red[SR_WARPS], s_range[SR_WARPS], s_top, s_sum[2], s_cut;
  __shared__ double s_table[32];
  __shared__ uint32_t red_u[SR_WARPS], s_count, s_found, s_base;   // tokens of the bracket: this CTA's, the cluster's (rank 0), in front of this CTA's
  __shared__ int s_bracket[2], s_place;
  __shared__ uint32_t s_few;
  constexpr int PER = 16 / sizeof(T);
  const int C = gridDim.x, rank = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = p.V, groups = p.slice / 8;
  const SampleRowsSmem<T> at(p.slice, p.cached);
  uint32_t* hist = reinterpret_cast<uint32_t*>(sr_smem + at.hist);
  uint64_t* near = reinterpret_cast<uint64_t*>(sr_smem + at.hist);
  uint64_t* list = reinterpret_cast<uint64_t*>(sr_smem + at.list);
  uint64_t* chunks = reinterpret_cast<uint64_t*>(sr_smem + at.chunks);
  uint32_t* seen = reinterpret_cast<uint32_t*>(sr_smem + at.seen);
  T* raw = reinterpret_cast<T*>(sr_smem + at.raw);
  auto csync = [&]() {
    if (C > 1) cluster_sync_all();
    else __syncthreads();
  };
  const float temp = p.temperature ? p.temperature[b] : p.temperature1;
  const int top_k = p.top_k ? p.top_k[b] : p.top_k1;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p1;
  const double low = double(fminf(p.min_p ? p.min_p[b] : p.min_p1, 1.f));   // the first token always stays
  const float pen = p.penalty ? p.penalty[b] : p.penalty1;
  const bool penalise = p.history != nullptr && pen != 1.f;
  const T* row = static_cast<const T*>(p.logits) + (long long)b * p.ld;
  // Slices are cut so that they begin at whole 16 bytes: token i0 + j is the slice's j-th; places before token 0 and behind the last hold -infinity.
  const int i0 = rank * p.slice - int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));

  // ---- the slice into shared memory, the history's bits
  auto fetch = [&](int v) -> uint4 {   // 16 bytes of the row: tokens i0 + v * PER ..
    const int i = i0 + v * PER;
    if (i >= 0 && i + PER <= V) return *reinterpret_cast<const uint4*>(row + i);
    uint4 out;
    T* o = reinterpret_cast<T*>(&out);
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] = i + e >= 0 && i + e < V ? row[i + e] : T(-INFINITY);
    return out;
  };
  if (p.cached) {
#pragma unroll 4
    for (int v = tid; v < p.slice / PER; v += SR_THREADS) reinterpret_cast<uint4*>(raw)[v] = fetch(v);
  }
  if (penalise)
    for (int i = tid; i < p.slice / 32; i += SR_THREADS) seen[i] = 0;
  for (int i = tid; i < SR_BINS; i += SR_THREADS) hist[i] = 0;
  if (tid < 32) s_table[tid] = exp2(-double(tid) / 32);
  if (tid == 0) s_count = 0, s_found = 0;
  __syncthreads();
  if (penalise) {
    for (int j = tid; j < p.hist_len; j += SR_THREADS) {
      const long long id = p.history[b * p.hist_ld + j], tok = id - i0;
      if (id >= 0 && id < V && tok >= 0 && tok < p.slice) atomicOr(&seen[tok >> 5], 1u << (tok & 31));
    }
    __syncthreads();
  }
  bool infinite = false;   // the largest score is +infinity: such tokens count as 0, all others as -infinity
  auto load8 = [&](int g, float (&x)[8]) {   // the scores of the slice's tokens 8 g ..
    uint4 w[8 / PER];
#pragma unroll
    for (int e = 0; e < 8 / PER; ++e) w[e] = p.cached ? reinterpret_cast<const uint4*>(raw)[g * (8 / PER) + e] : fetch(g * (8 / PER) + e);
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(u[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[2 * e] = __uint_as_float(u[e] << 16), x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
    }
    if (penalise) {
      const uint32_t bits = reinterpret_cast<const uint8_t*>(seen)[g];
      if (bits) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (bits >> e & 1) x[e] = x[e] > 0.f ? __fdiv_rn(x[e], pen) : __fmul_rn(x[e], pen);
      }
    }
    if (infinite) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] == INFINITY ? 0.f : -INFINITY;
    }
  };
  auto key_of = [&](float x, int j) -> uint64_t { return (uint64_t(order_key(x + 0.f)) << 32) | (0xffffffffu - uint32_t(i0 + j)); };

  // ---- the first token of the order
  {
    float best = -INFINITY;
    int j_best = -1;
    for (int g = tid; g < groups; g += SR_THREADS) {
      float x[8];
      load8(g, x);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (x[e] > best) best = x[e], j_best = 8 * g + e;
    }
    uint64_t k = j_best >= 0 ? key_of(best, j_best) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t u = __shfl_xor_sync(0xffffffffu, k, o);
      k = u > k ? u : k;
    }
    if (lane == 0) red[warp] = k;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < SR_WARPS; ++w) k = red[w] > k ? red[w] : k;
      s_top = k;
    }
  }
  csync();
  uint64_t top = 0;
  for (int r = 0; r < C; ++r) {
    const uint64_t k = sr_ld_u64(&s_top, r);
    top = k > top ? k : top;
  }
  const int arg = top ? int(0xffffffffu - uint32_t(top)) : 0;   // (0: nothing above -infinity)
  float x_max = key_value(uint32_t(top >> 32));
  if (x_max == INFINITY) infinite = true, x_max = 0.f, top = (uint64_t(order_key(0.f)) << 32) | uint32_t(top);

  const double inv_t = 1.0 / double(temp), x_top = double(x_max);
  const float per_bin = float(SR_BINS - 1) / (SR_RANGE * temp);
  auto bin_of = [&](float x) -> int {   // does not fall as x falls; fp32 rounding moves a border by less than a hundredth of a bin.  NaN: the last one
    const float d = x == x_max ? 0.f : (x_max - x) * per_bin;
    return int(fminf(d, float(SR_BINS - 1)));
  };
  auto weight = [&](float x) -> double { return sr_exp_neg((x_top - double(x)) * inv_t, s_table); };   // relative to the first token's
  auto fixed = [&](double w) -> uint64_t {   // round(w * 2^42)
    return uint64_t(__double_as_longlong(fma(w, double(1ll << SR_MASS_BITS), 4503599627370496.0))) & ((1ull << 52) - 1);
  };
  auto mass = [&](float x) -> uint64_t { return bin_of(x) == SR_BINS - 1 ? 0 : fixed(weight(x)); };
  auto cluster_sum = [&](uint64_t v, int slot) -> uint64_t {   // (one barrier; the slots take turns)
    const uint64_t mine = sr_block_sum(v, red);
    if (tid == 0) s_sum[slot] = mine;
    csync();
    uint64_t t = 0;
    for (int r = 0; r < C; ++r) t += sr_ld_u64(&s_sum[slot], r);
    return t;
  };
  const double u = fmax(double(p.uniform[b]), 0.0);
  auto target_of = [&](uint64_t total) -> uint64_t {
    const double want = u * double(total);
    return want < double(total) ? min(uint64_t(want), total - 1) : total - 1;
  };
  // The bracket's tokens: each CTA notes its own (`stage`, room for `room`), then hand_over() puts them into rank 0's list and returns how many there are
  // in all (more than SR_LIST: some did not fit).
  uint64_t* stage = near;
  uint32_t room = SR_LIST;
  auto collect = [&](float x, int j) {
    const uint32_t i = atomicAdd(&s_count, 1u);
    if (i < room) stage[i] = key_of(x, j);
  };
  auto hand_over = [&]() -> uint32_t {
    __syncthreads();
    const uint32_t n = s_count;
    if (tid == 0) {
      uint32_t at;
      asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(at) : "r"(mapa_shared(smem_u32(&s_found), 0)), "r"(n > room ? SR_LIST + 1 : n) : "memory");
      s_base = at;
    }
    __syncthreads();
    const uint32_t base = s_base;
    if (n <= room && base + n <= SR_LIST)
      for (uint32_t i = tid; i < n; i += SR_THREADS) sr_st_u64(&list[base + i], 0, stage[i]);
    csync();
    const uint32_t found = sr_ld_u32(&s_found, 0);
    csync();   // everybody has read: a list that holds all that is kept needs no other CTA any more
    return found;
  };
  // what is kept, per SR_CHUNK consecutive tokens (one group a lane): `kept(x, j)` says whether the token is, as far as min-p does not
  auto sum_chunks = [&](auto kept) {
    for (int g = tid; g < groups; g += SR_THREADS) {
      float x[8];
      load8(g, x);
      uint64_t v = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double w = weight(x[e]);
        v += kept(x[e], 8 * g + e) && !(w < low) ? fixed(w) : 0;
      }
      v = sr_warp_sum(v);
      if (lane == 0) chunks[g >> 5] = v;
    }
    __syncthreads();
  };

  const bool by_k = top_k > 0 && top_k < V, by_p = top_p < 1.f;
  if (!(temp > 0.f) || top == 0) {
    if (rank == 0 && tid == 0) p.out[b] = arg;
    if (C > 1) cluster_sync_all();   // nobody leaves while its shared memory is read
    return;
  }
  bool bisect = by_k && top_k > SR_MAX_K, listed = false;   // listed: the answer is among the list's tokens
  int b_lo = 0;
  uint64_t cut = 0, z = 0, above = 0, own_kept = 0;   // tokens with at least the key `cut` are kept; this CTA's mass of them
  // rank 0, with `found` tokens in the list, `above` the mass of what is in front of them: the cut, and the answer if nothing is in front of them
  auto finish_list = [&](uint32_t found) {
    if (found <= SR_FEW) {
      // Few tokens: two threads compare one with all others, half of them each, twice: by score for the cuts, by index for the draw.
      uint64_t* few = list + SR_FEW;   // masses of the list's tokens; behind them the other half's sums
      const int i = tid % SR_FEW, half = tid / SR_FEW, mid = int(found + 1) / 2, from = half ? mid : 0, to = half ? int(found) : mid;
      const bool mine = i < int(found);
      const uint64_t k = mine ? list[i] : 0;
      const float x = key_value(uint32_t(k >> 32));
      uint64_t m = mine ? mass(x) : 0;
      __syncthreads();
      if (half == 0) few[i] = m;
      __syncthreads();
      uint64_t before = 0;
      uint32_t rank_of = 0;
      if (mine)
        for (int j = from; j < to; ++j) {
          const bool in_front = list[j] > k;
          before += in_front ? few[j] : 0;
          rank_of += in_front;
        }
      if (half) few[SR_FEW + i] = before, few[2 * SR_FEW + i] = rank_of;
      __syncthreads();
      before += few[SR_FEW + i] + above;
      rank_of += uint32_t(few[2 * SR_FEW + i]);
      const bool first_k = half == 0 && mine && (!by_k || rank_of < uint32_t(top_k));
      const uint64_t all = by_k ? sr_block_sum(first_k ? m : 0, red) : z;
      const bool in = first_k && (!by_p || double(before) <= double(fmaxf(top_p, 0.f)) * double(all));   // (both rules keep a leading run)
      if (!in || (low > 0 && !(weight(x) >= low))) m = 0;
      if (!listed) {   // the smallest key that is kept
        uint64_t last = in ? k : ~0ull;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t other = __shfl_xor_sync(0xffffffffu, last, o);
          last = other < last ? other : last;
        }
        __syncthreads();
        if (lane == 0) red[warp] = last;
        __syncthreads();
        if (tid == 0) {
          for (int w = 1; w < SR_WARPS; ++w) last = red[w] < last ? red[w] : last;
          s_cut = last;
        }
        return;
      }
      const uint64_t target = target_of(sr_block_sum(half == 0 ? m : 0, red));
      if (half == 0) few[i] = m;
      __syncthreads();
      before = 0;
      if (mine)
        for (int j = from; j < to; ++j) before += uint32_t(list[j]) > uint32_t(k) ? few[j] : 0;   // (the lower half falls as the index grows)
      if (half) few[SR_FEW + i] = before;
      __syncthreads();
      before += few[SR_FEW + i];
      if (half == 0 && before <= target && target < before + m) p.out[b] = int(0xffffffffu - uint32_t(k));
      return;
    }
    // More tokens: four a thread, in registers.  A cut is where the cumulative weight in falling order of a key passes a limit; it is found by counting
    // weights over 512 places of the keys' range, then over the one place that holds the cut, until that holds one token.
    constexpr int EACH = SR_LIST / SR_THREADS;
    uint32_t* lower = reinterpret_cast<uint32_t*>(list);      // [SR_THREADS] each: halves of the weights' sums, tokens
    uint32_t* upper = lower + SR_THREADS;
    uint32_t* many = upper + SR_THREADS;
    uint64_t* few = list + 2 * SR_THREADS;
    uint64_t v[EACH], w[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) v[e] = tid + e * SR_THREADS < found ? list[tid + e * SR_THREADS] : 0;
    // the smallest key (of tokens whose key is not 0; they are all different) with at most `limit` of weight in front of it, `run` of which is there already; ~0: none
    auto narrow = [&](const uint64_t (&key)[EACH], auto weight_at, uint64_t run, auto within) -> uint64_t {
      uint64_t lo = 1, hi = ~0ull;
      uint32_t left = 0;   // (of 0: the range is not known to be a narrow one)
      for (;;) {
        if (left == 0) {   // the ends of what there is
          uint64_t first = ~0ull, last = 0;
#pragma unroll
          for (int e = 0; e < EACH; ++e)
            if (key[e] >= lo && key[e] <= hi) first = key[e] < first ? key[e] : first, last = key[e] > last ? key[e] : last;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            const uint64_t a = __shfl_xor_sync(0xffffffffu, first, o), c = __shfl_xor_sync(0xffffffffu, last, o);
            first = a < first ? a : first, last = c > last ? c : last;
          }
          __syncthreads();
          if (lane == 0) red[warp] = first, s_range[warp] = last;
          __syncthreads();
          lo = ~0ull, hi = 0;
#pragma unroll
          for (int i = 0; i < SR_WARPS; ++i) lo = red[i] < lo ? red[i] : lo, hi = s_range[i] > hi ? s_range[i] : hi;
          if (hi == 0) return ~0ull;
        }
        const int shift = max(0, 55 - __clzll((long long)(hi - lo)));   // places of 2^shift keys: at most 512
        lower[tid] = 0, upper[tid] = 0, many[tid] = 0;
        if (tid == 0) s_place = -1;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < EACH; ++e)
          if (key[e] && key[e] >= lo && key[e] <= hi) {
            const int at = SR_THREADS - 1 - int((key[e] - lo) >> shift);
            const uint64_t weight = weight_at(e);
            const uint32_t was = atomicAdd(&lower[at], uint32_t(weight)), more = uint32_t(weight >> 32) + (was + uint32_t(weight) < was);
            if (more) atomicAdd(&upper[at], more);
            atomicAdd(&many[at], 1u);
          }
        __syncthreads();
        uint64_t all;
        const uint64_t before = run + sr_block_scan<uint64_t>((uint64_t(upper[tid]) << 32) + lower[tid], red, &all);
        const uint32_t ok = __ballot_sync(0xffffffffu, many[tid] > 0 && within(before));   // (a leading run of the places that hold tokens)
        if (ok && lane == 31 - __clz(ok)) atomicMax(&s_place, tid);
        __syncthreads();
        const int place = s_place;
        if (place < 0) return ~0ull;
        if (tid == place) s_sum[0] = before;
        if (tid == 0) s_few = 0;
        const uint64_t from = lo + (uint64_t(SR_THREADS - 1 - place) << shift);
        const uint32_t n = many[place];
        __syncthreads();
        if (n <= 32) {   // a warp compares each with all
#pragma unroll
          for (int e = 0; e < EACH; ++e)
            if (key[e] >= from && key[e] <= hi && (key[e] - from) >> shift == 0) {
              const uint32_t i = atomicAdd(&s_few, 1u);
              few[i] = key[e], few[32 + i] = weight_at(e);
            }
          __syncthreads();
          if (warp == 0) {
            const uint64_t k = lane < n ? few[lane] : 0, m = lane < n ? few[32 + lane] : 0;
            uint64_t in_front = s_sum[0];
            for (uint32_t j = 0; j < n; ++j) {
              const uint64_t k_j = __shfl_sync(0xffffffffu, k, j), m_j = __shfl_sync(0xffffffffu, m, j);
              in_front += k_j > k ? m_j : 0;
            }
            uint64_t best = lane < n && within(in_front) ? k : ~0ull;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
              const uint64_t c = __shfl_xor_sync(0xffffffffu, best, o);
              best = c < best ? c : best;
            }
            if (lane == 0) s_cut = best;
          }
          __syncthreads();
          return s_cut;
        }
        run = s_sum[0];
        const uint64_t to = from + ((1ull << shift) - 1);   // (more than one key: shift is not 0)
        lo = from, hi = to < hi ? to : hi;
        left = n > found / 2 ? 0 : 1;   // most of them in one place: many equal scores, whose keys differ in the lowest bits alone
      }
    };
    if (!listed) {   // the smallest key that is kept: by_p without by_k
#pragma unroll
      for (int e = 0; e < EACH; ++e) w[e] = v[e] ? mass(key_value(uint32_t(v[e] >> 32))) : 0;
      const double limit = double(fmaxf(top_p, 0.f)) * double(z);
      const uint64_t last = narrow(v, [&](int e) { return w[e]; }, above, [&](uint64_t before) { return double(before) <= limit; });
      __syncthreads();
      if (tid == 0) s_cut = last;
      return;
    }
    if (by_k && found > uint32_t(top_k)) {
      const uint64_t last = narrow(v, [](int) { return 1ull; }, 0, [&](uint64_t before) { return before < uint64_t(top_k); });
#pragma unroll
      for (int e = 0; e < EACH; ++e) v[e] = v[e] >= last ? v[e] : 0;
    }
    uint64_t own = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      w[e] = v[e] ? mass(key_value(uint32_t(v[e] >> 32))) : 0;
      own += w[e];
    }
    if (by_p) {
      const uint64_t all = by_k ? sr_block_sum(own, red) : z;
      const double limit = double(fmaxf(top_p, 0.f)) * double(all);
      const uint64_t last = narrow(v, [&](int e) { return w[e]; }, 0, [&](uint64_t before) { return double(before) <= limit; });
#pragma unroll
      for (int e = 0; e < EACH; ++e) w[e] = v[e] >= last ? w[e] : 0;
    }
    own = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      if (low > 0 && w[e] && !(weight(key_value(uint32_t(v[e] >> 32))) >= low)) w[e] = 0;
      own += w[e];
      v[e] = w[e] ? uint32_t(v[e]) : 0;   // the order of the indices, lowest first
    }
    const uint64_t target = target_of(sr_block_sum(own, red));
    const uint64_t drawn = narrow(v, [&](int e) { return w[e]; }, 0, [&](uint64_t before) { return before <= target; });
    if (tid == 0) p.out[b] = int(0xffffffffu - uint32_t(drawn));
  };

  if (by_k && !bisect) {
    // ---- counts of the largest of every eight tokens (of all tokens where k is more than half of the eights), eight bins in one
    constexpr int WIDE = SR_BINS / SR_THREADS;
    const bool all_tokens = top_k > V / 16;
    for (int g = tid; g < groups; g += SR_THREADS) {
      float x[8];
      load8(g, x);
      if (all_tokens) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int bin = bin_of(x[e]);
          if (bin < SR_BINS - 1) atomicAdd(&hist[bin / WIDE], 1u);
        }
      } else {
        float m = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) m = fmaxf(m, x[e]);
        const int bin = bin_of(m);
        if (bin < SR_BINS - 1) atomicAdd(&hist[bin / WIDE], 1u);
      }
    }
    csync();
    uint32_t c = 0, all;
    for (int r = 0; r < C; ++r) c += sr_ld_u32(&hist[tid], r);
    const uint32_t before = sr_block_scan<uint32_t>(c, red_u, &all);
    if (tid == 0) s_bracket[1] = SR_BINS - 2;   // fewer than k with any mass: all that have some
    __syncthreads();
    if (before < uint32_t(top_k) && before + c >= uint32_t(top_k)) s_bracket[1] = min((tid + 1) * WIDE - 1, SR_BINS - 2);
    __syncthreads();
    const int b_hi = s_bracket[1];
    stage = near + SR_THREADS / 2;   // (behind the counts, which the other CTAs may still read)
    room = SR_LIST - SR_THREADS / 2;
    for (int g = tid; g < groups; g += SR_THREADS) {
      float x[8];
      load8(g, x);
      float m = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) m = fmaxf(m, x[e]);
      if (bin_of(m) <= b_hi) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (bin_of(x[e]) <= b_hi) collect(x[e], 8 * g + e);
      }
    }
    const uint32_t found = hand_over();
    bisect = found > SR_LIST;
    listed = !bisect;
    if (listed) {
      if (rank == 0) finish_list(found);
      return;
    }
  } else if (by_p && !bisect) {
    // ---- masses by distance, two bins in one: lower halves of the sums, then upper ones
    uint32_t* lower = hist;
    uint32_t* upper = hist + SR_MASS_BINS;
    for (int g = tid; g < groups; g += SR_THREADS) {
      float x[8];
      load8(g, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int bin = bin_of(x[e]);
        const uint64_t m = fixed(weight(x[e]));
        if (bin < SR_BINS - 1 && m) {
          const uint32_t was = atomicAdd(&lower[bin / 2], uint32_t(m)), more = uint32_t(m >> 32) + (was + uint32_t(m) < was);
          if (more) atomicAdd(&upper[bin / 2], more);
        }
      }
    }
    csync();
    // a share of the bins each, into rank 0's list
    for (int i = rank * (SR_MASS_BINS / C) + tid; i < (rank + 1) * (SR_MASS_BINS / C); i += SR_THREADS) {
      uint32_t up[SR_MAX_CLUSTER], low_[SR_MAX_CLUSTER];
#pragma unroll
      for (int r = 0; r < SR_MAX_CLUSTER; ++r) up[r] = r < C ? sr_ld_u32(&upper[i], r) : 0, low_[r] = r < C ? sr_ld_u32(&lower[i], r) : 0;
      uint64_t v = 0;
#pragma unroll
      for (int r = 0; r < SR_MAX_CLUSTER; ++r) v += (uint64_t(up[r]) << 32) + low_[r];
      sr_st_u64(&list[i], 0, v);
    }
    csync();
    if (rank == 0) {   // the last bin whose first token is kept holds the cut
      constexpr int EACH = SR_MASS_BINS / SR_THREADS;
      uint64_t v[EACH], own = 0, all, before = 0;
#pragma unroll
      for (int e = 0; e < EACH; ++e) v[e] = list[tid * EACH + e], own += v[e];
      uint64_t run = sr_block_scan<uint64_t>(own, red, &all);
      const double limit = double(fmaxf(top_p, 0.f)) * double(all);
      int at_bin = -1;
      uint64_t in_bin = 0;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        if (v[e] && double(run) <= limit) at_bin = tid * EACH + e, before = run, in_bin = v[e];
        run += v[e];
      }
      if (tid == 0) s_place = -1;
      __syncthreads();
      const uint32_t ok = __ballot_sync(0xffffffffu, at_bin >= 0);
      if (ok && lane == 31 - __clz(ok)) atomicMax(&s_place, at_bin);
      __syncthreads();
      if (at_bin >= 0 && at_bin == s_place) {
        // all tokens up to the bin's end have at least this mass each (rounding moves a border by less than a hundredth of a bin): do so many fit the list?
        const double least = sr_exp_neg(double(SR_RANGE) / (SR_BINS - 1) * (2 * at_bin + 2.02), s_table) * double(1ll << SR_MASS_BITS) - 1.0;
        const bool fit = double(before + in_bin) <= SR_LIST * 0.999 * least;
        s_bracket[0] = fit ? 0 : 2 * at_bin;
        s_bracket[1] = min(2 * at_bin + 1, SR_BINS - 2);
        s_sum[0] = fit ? 0 : before;
        s_sum[1] = all;
      }
    }
    csync();
    b_lo = int(sr_ld_u32(&s_bracket[0], 0));
    const int b_hi = int(sr_ld_u32(&s_bracket[1], 0));
    above = sr_ld_u64(&s_sum[0], 0);
    z = sr_ld_u64(&s_sum[1], 0);
    uint64_t part = 0;
    for (int i = tid; i < b_lo / 2; i += SR_THREADS) part += (uint64_t(upper[i]) << 32) + lower[i];
    own_kept = sr_block_sum(part, red);   // (and the counts have been read: the bracket's tokens take their place)
    for (int g = tid; g < groups; g += SR_THREADS) {
      float x[8];
      load8(g, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int bin = bin_of(x[e]);
        if (bin >= b_lo && bin <= b_hi) collect(x[e], 8 * g + e);
      }
    }
    const uint32_t found = hand_over();
    bisect = found > SR_LIST;
    listed = !bisect && b_lo == 0;
    if (listed) {
      if (rank == 0) finish_list(found);
      return;
    }
    if (!bisect) {
      if (rank == 0) finish_list(found);
      csync();
      cut = sr_ld_u64(&s_cut, 0);
      part = 0;
      if (low > 0) sum_chunks([&](float x, int j) -> bool { return key_of(x, j) >= cut; });
      else
        for (uint32_t i = tid; i < s_count; i += SR_THREADS)   // the bracket's part of what is kept
          if (near[i] >= cut) part += mass(key_value(uint32_t(near[i] >> 32)));
      own_kept += sr_block_sum(part, red);
    }
  }
  {
    const bool summed = !bisect && by_p && !(low > 0);   // this CTA's part of what is kept is known, not yet where it lies
    int slot = 0;
    if (bisect) {
      csync();   // the sum last taken may still be read
      auto total_of = [&](auto f) {
        uint64_t v = 0;
        for (int g = tid; g < groups; g += SR_THREADS) {
          float x[8];
          load8(g, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = x[e] == x[e] ? x[e] : -INFINITY;
            const int i = i0 + 8 * g + e;
            if (i >= 0 && i < V) v += f(y, 8 * g + e);
          }
        }
        slot ^= 1;
        return cluster_sum(v, slot);
      };
      cut = 0;
      if (by_k) {   // the k-th largest key, bit by bit
        for (int bit = 63; bit >= 0; --bit) {
          const uint64_t trial = cut | (1ull << bit);
          if (total_of([&](float x, int j) -> uint64_t { return key_of(x, j) >= trial; }) >= uint64_t(top_k)) cut = trial;
        }
      }
      if (by_p) {   // the smallest key with mass above it <= top_p Z
        const uint64_t zz = total_of([&](float x, int j) -> uint64_t { return key_of(x, j) >= cut ? mass(x) : 0; });
        const double limit = double(fmaxf(top_p, 0.f)) * double(zz);
        uint64_t lo = cut, hi = top;
        while (lo < hi) {
          const uint64_t mid = lo + ((hi - lo) >> 1);
          if (double(total_of([&](float x, int j) -> uint64_t { return key_of(x, j) > mid ? mass(x) : 0; })) <= limit) hi = mid;
          else lo = mid + 1;
        }
        cut = lo;
      }
    }
    const bool cuts = bisect || by_p;
    auto is_kept = [&](float x, int j) -> bool { return !cuts || key_of(x, j) >= cut; };
    if (!cuts) sum_chunks([](float, int) { return true; });
    else if (bisect) sum_chunks(is_kept);
    uint64_t mine = 0;
    if (!summed)
      for (int c = tid; c < p.slice / SR_CHUNK; c += SR_THREADS) mine += chunks[c];
    // (the sums of the CTAs one by one: where the target lies)
    const uint64_t own = summed ? own_kept : sr_block_sum(mine, red);
    if (tid == 0) s_sum[slot ^ 1] = own;
    csync();
    uint64_t total = 0, before = 0;
    for (int r = 0; r < C; ++r) {
      const uint64_t v = sr_ld_u64(&s_sum[slot ^ 1], r);
      if (r < rank) before += v;
      total += v;
    }
    const uint64_t target = target_of(total);
    const bool here = own > 0 && target >= before && target < before + own;
    if (here && summed) sum_chunks(is_kept);
    if (here && warp == 0) {
      // one warp: the chunk, 32 at a time, then the group of eight, then the token
      uint64_t run = before;
      auto step = [&](uint64_t v, int* which) -> bool {   // the lane whose value covers the target, or go on behind all of them
        uint64_t incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t w = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += w;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, run + incl > target);
        const int from = hit ? __ffs(hit) - 1 : 31;
        run += __shfl_sync(0xffffffffu, hit ? incl - v : incl, from);
        *which = from;
        return hit != 0;
      };
      const int n_chunks = p.slice / SR_CHUNK;
      int w = 0, pick = arg;
      bool found = false;
      int c = 0;
      for (; c < n_chunks && !found; c += 32) found = step(c + lane < n_chunks ? chunks[c + lane] : 0, &w);
      if (found) {
        const int chunk = c - 32 + w, g = chunk * 32 + lane;
        float x[8];
        load8(g, x);
        uint64_t m[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double wt = weight(x[e]);
          m[e] = is_kept(x[e], 8 * g + e) && wt >= low ? fixed(wt) : 0;
          sum += m[e];
        }
        if (step(sum, &w)) {
          if (lane == w) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (run <= target && target < run + m[e]) pick = i0 + 8 * g + e;
              run += m[e];
            }
          }
          pick = __shfl_sync(0xffffffffu, pick, w);
        }
      }
      if (lane == 0) p.out[b] = pick;
    }
  }
  if (C > 1) cluster_sync_all();   // nobody leaves while its shared memory is read
}

template <typename T>
static int launch_sample_rows(SampleRowsArgs& p, int B, cudaStream_t s) {
  // As many CTAs a row as keep its slices in shared memory (64 KB each, so that an SM holds two), more while the rows leave SMs idle and a CTA
  // keeps 2,048 tokens.
  int C = 1;
  while (C < SR_MAX_CLUSTER && (long long)p.V * sizeof(T) > C * 65536ll) C *= 2;
  while (C < SR_MAX_CLUSTER && 2 * C * B <= 148 && p.V > C * 2048) C *= 2;
  p.slice = (p.V + 7 + C * SR_CHUNK - 1) / (C * SR_CHUNK) * SR_CHUNK;   // (up to seven places in front of the first token)
  p.cached = (long long)p.slice * sizeof(T) <= SR_CACHED;
  const SampleRowsSmem<T> at(p.slice, p.cached);
  static DeviceOnce once;   // (for the largest slice, whatever this call's: the limit is one for all threads.  A slice that is not kept takes a third of it)
  cudaError_t ce = once.smem(sample_rows_kernel<T>, SampleRowsSmem<T>(SR_CACHED / sizeof(T), true).total);
  if (ce != cudaSuccess) return int(ce);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C, B);
  cfg.blockDim = dim3(SR_THREADS);
  cfg.dynamicSmemBytes = at.total;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  ce = cudaLaunchKernelEx(&cfg, sample_rows_kernel<T>, p);
  if (ce != cudaSuccess) return int(ce);
  return int(cudaGetLastError());
}

}  // namespace ats

using namespace ats;

// logits [B, ld] (bf16, or fp32) -> out [B].  Sampling numbers: one per row, or null and the single number for all rows.
ATS_API int ats_sample_rows(const void* logits, int fp32, long long ld, int B, int V, const float* uniform, const float* temperature, float temperature1,
                            const int* top_k, int top_k1, const float* top_p, float top_p1, const float* min_p, float min_p1, const float* penalty, float penalty1,
                            const long long* history, int hist_len, long long hist_ld, long long* out, void* stream) {
  if (B < 1 || B > 65535 || V < 1 || V > SR_MAX_VOCAB || hist_len < 0) return 1003;
  SampleRowsArgs p;
  p.logits = logits; p.ld = ld; p.V = V; p.uniform = uniform;
  p.temperature = temperature; p.temperature1 = temperature1; p.top_k = top_k; p.top_k1 = top_k1; p.top_p = top_p; p.top_p1 = top_p1;
  p.min_p = min_p; p.min_p1 = min_p1; p.penalty = penalty; p.penalty1 = penalty1;
  p.history = hist_len > 0 ? history : nullptr; p.hist_len = hist_len; p.hist_ld = hist_ld; p.out = out;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return fp32 ? launch_sample_rows<float>(p, B, s) : launch_sample_rows<__nv_bfloat16>(p, B, s);
}
