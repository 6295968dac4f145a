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
#include "common.cuh"

namespace ats {

constexpr int SR_THREADS = 1024;
constexpr int SR_MASS_BITS = 42;
constexpr int SR_MAX_VOCAB = 1 << 20;

struct SampleRowsArgs {
  const void* logits;   // [B, ld] bf16 or fp32
  long long ld;
  int fp32, V;
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

__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  __syncthreads();
  if (l == 0) red[w] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int i = 0; i < SR_THREADS / 32; ++i) t += red[i];
  return t;
}

__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  __syncthreads();
  if (l == 0) red[w] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int i = 0; i < SR_THREADS / 32; ++i) t = red[i] > t ? red[i] : t;
  return t;
}

// order-preserving image of a float without NaN
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

__global__ void __launch_bounds__(SR_THREADS) sample_rows_kernel(const SampleRowsArgs p) {
  pdl_prologue();
  extern __shared__ uint32_t s_seen[];   // one bit per token of the history
  __shared__ uint64_t red[SR_THREADS / 32];
  __shared__ int s_pick;
  const int b = blockIdx.x, tid = threadIdx.x, V = p.V;
  const float temp = p.temperature ? p.temperature[b] : p.temperature1;
  const int top_k = p.top_k ? p.top_k[b] : p.top_k1;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p1;
  const float min_p = fminf(p.min_p ? p.min_p[b] : p.min_p1, 1.f);   // the first token always stays
  const float pen = p.penalty ? p.penalty[b] : p.penalty1;
  const bool penalise = p.history != nullptr && pen != 1.f;
  if (penalise) {
    for (int i = tid; i < (V + 31) / 32; i += SR_THREADS) s_seen[i] = 0;
    __syncthreads();
    for (int j = tid; j < p.hist_len; j += SR_THREADS) {
      const long long tok = p.history[b * p.hist_ld + j];
      if (tok >= 0 && tok < V) atomicOr(&s_seen[tok >> 5], 1u << (tok & 31));
    }
    __syncthreads();
  }
  auto key = [&](int i) -> uint64_t {
    float x = p.fp32 ? static_cast<const float*>(p.logits)[b * p.ld + i] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[b * p.ld + i]);
    if (penalise && (s_seen[i >> 5] >> (i & 31) & 1)) x = x > 0.f ? __fdiv_rn(x, pen) : __fmul_rn(x, pen);
    if (x != x) x = -INFINITY;
    x += 0.f;
    return (uint64_t(order_key(x)) << 32) | (0xffffffffu - uint32_t(i));
  };
  uint64_t top = 0;
  for (int i = tid; i < V; i += SR_THREADS) {
    const uint64_t k = key(i);
    top = k > top ? k : top;
  }
  top = block_max_u64(top, red);
  const int arg = int(0xffffffffu - uint32_t(top));
  const float x_max = key_value(uint32_t(top >> 32));
  if (!(temp > 0.f) || x_max == -INFINITY) {
    if (tid == 0) p.out[b] = arg;
    return;
  }
  const double inv_t = 1.0 / double(temp);
  auto weight = [&](uint64_t k) -> double {   // relative to the first token's
    const float x = key_value(uint32_t(k >> 32));
    return x == x_max ? 1.0 : exp((double(x) - double(x_max)) * inv_t);
  };
  auto mass = [&](uint64_t k) -> uint64_t { return uint64_t(__double2ll_rn(weight(k) * double(1ll << SR_MASS_BITS))); };
  uint64_t cut = 0;   // tokens with at least this key stay
  if (top_k > 0 && top_k < V) {   // the k-th largest key, bit by bit
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t trial = cut | (1ull << bit);
      uint64_t c = 0;
      for (int i = tid; i < V; i += SR_THREADS) c += key(i) >= trial;
      if (block_sum_u64(c, red) >= uint64_t(top_k)) cut = trial;
    }
  }
  if (top_p < 1.f) {   // the smallest key with mass above it <= top_p Z
    uint64_t z = 0;
    for (int i = tid; i < V; i += SR_THREADS) {
      const uint64_t k = key(i);
      if (k >= cut) z += mass(k);
    }
    const double limit = double(fmaxf(top_p, 0.f)) * double(block_sum_u64(z, red));
    uint64_t lo = cut, hi = top;
    while (lo < hi) {
      const uint64_t mid = lo + ((hi - lo) >> 1);
      uint64_t above = 0;
      for (int i = tid; i < V; i += SR_THREADS) {
        const uint64_t k = key(i);
        if (k > mid) above += mass(k);
      }
      if (double(block_sum_u64(above, red)) <= limit) hi = mid;
      else lo = mid + 1;
    }
    cut = lo;
  }
  const double low = double(min_p);
  auto kept_mass = [&](int i) -> uint64_t {
    const uint64_t k = key(i);
    if (k < cut) return 0;
    const double w = weight(k);
    return w >= low ? uint64_t(__double2ll_rn(w * double(1ll << SR_MASS_BITS))) : 0;
  };
  // in index order: a run of tokens per thread
  const int seg = (V + SR_THREADS - 1) / SR_THREADS, i0 = min(tid * seg, V), i1 = min(i0 + seg, V);
  uint64_t mine = 0;
  for (int i = i0; i < i1; ++i) mine += kept_mass(i);
  const uint64_t total = block_sum_u64(mine, red);
  uint64_t incl = mine;
  const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  __syncthreads();
  if (lane == 31) red[warp] = incl;
  if (tid == 0) s_pick = arg;
  __syncthreads();
  uint64_t before = incl - mine;
  for (int w = 0; w < warp; ++w) before += red[w];
  const double u = fmax(double(p.uniform[b]), 0.0);
  const double want = u * double(total);
  const uint64_t target = want < double(total) ? min((uint64_t)want, total - 1) : total - 1;
  if (mine > 0 && target >= before && target < before + mine) {
    uint64_t run = before;
    for (int i = i0; i < i1; ++i) {
      run += kept_mass(i);
      if (run > target) {
        s_pick = i;
        break;
      }
    }
  }
  __syncthreads();
  if (tid == 0) p.out[b] = s_pick;
}

}  // namespace ats

using namespace ats;

// logits [B, ld] (bf16, or fp32) -> out [B].  Sampling numbers: one per row, or null and the single number for all rows.
ATS_API int ats_sample_rows(const void* logits, int fp32, long long ld, int B, int V, const float* uniform, const float* temperature, float temperature1,
                            const int* top_k, int top_k1, const float* top_p, float top_p1, const float* min_p, float min_p1, const float* penalty, float penalty1,
                            const long long* history, int hist_len, long long hist_ld, long long* out, void* stream) {
  if (B < 1 || V < 1 || V > SR_MAX_VOCAB || hist_len < 0) return 1003;
  SampleRowsArgs p;
  p.logits = logits; p.ld = ld; p.fp32 = fp32; p.V = V; p.uniform = uniform;
  p.temperature = temperature; p.temperature1 = temperature1; p.top_k = top_k; p.top_k1 = top_k1; p.top_p = top_p; p.top_p1 = top_p1;
  p.min_p = min_p; p.min_p1 = min_p1; p.penalty = penalty; p.penalty1 = penalty1;
  p.history = hist_len > 0 ? history : nullptr; p.hist_len = hist_len; p.hist_ld = hist_ld; p.out = out;
  const size_t smem = p.history ? size_t((V + 31) / 32) * 4 : 0;
  cudaError_t ce = cudaSuccess;
  if (smem > 40 * 1024) ce = cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (ce == cudaSuccess) ce = launch_pdl(sample_rows_kernel, dim3(B), dim3(SR_THREADS), smem, static_cast<cudaStream_t>(stream), p);
  if (ce != cudaSuccess) return int(ce);
  return int(cudaGetLastError());
}
