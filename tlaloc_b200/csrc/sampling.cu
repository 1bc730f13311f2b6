// One token drawn from each row of logits (include/tlaloc_b200.h, tlaloc_b200_sample): temperature, the k most likely, the shortest run of them that holds a share p of
// their mass, a least share of the most likely one's probability, and the inverse of the distribution function at a given random number.
//
//   w_i = exp((x_i - max x) / T);  kept: rank_i < k,  mass of the better ranked < p * mass of the k,  w_i >= min_p
//   token = first i whose running sum of kept w, in index order, exceeds u * their whole sum
//
// Ranks go by value, equal values by index.  So what is kept is all values above some value and, of those equal to it, the ones up to some index.
// Weights and sums are f64: a row has as many borders between tokens as it has tokens, and a draw that sums 10^5 weights in f32 lands on the wrong side of one in
// about one row of a hundred.
#include <algorithm>

#include "common.cuh"

namespace tlaloc_b200 {
namespace {

struct SampleArgs {
  const void* logits;
  int64_t ld;
  const float* uniforms;
  const float* temperature;  // a row's own settings, or null: the ones below for all
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int* out;
  int n;
};

constexpr int kSampleThreads = 1024, kSampleWarps = kSampleThreads / 32;

// Values in an order of unsigned numbers: -0 as 0, NaN as -infinity (never drawn).
__device__ __forceinline__ uint32_t KeyOf(float x)
{
  if (!(x == x)) x = -INFINITY;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) != 0u ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float ValueOf(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) != 0u ? 0x80000000u : 0xffffffffu)); }

template <typename T>
__device__ __forceinline__ T BlockSumAll(T v, T* red)
{
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  T r = 0;
  for (int w = 0; w < kSampleWarps; ++w) r += red[w];
  return r;
}

template <typename XT>
__global__ void __launch_bounds__(kSampleThreads) SampleKernel(const __grid_constant__ SampleArgs a)
{
  GridDependencySync();
  __shared__ double red[kSampleWarps];
  __shared__ int ired[kSampleWarps];
  __shared__ uint32_t kred[kSampleWarps];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n;
  const XT* x = static_cast<const XT*>(a.logits) + row * a.ld;
  const float temperature = a.temperature != nullptr ? __ldg(a.temperature + row) : a.temperature_all;
  const int top_k = a.top_k != nullptr ? __ldg(a.top_k + row) : a.top_k_all;
  const float top_p = a.top_p != nullptr ? __ldg(a.top_p + row) : a.top_p_all;
  const float min_p = a.min_p != nullptr ? __ldg(a.min_p + row) : a.min_p_all;
  const int per = (n + kSampleWarps - 1) / kSampleWarps;  // a warp's stretch of the row
  const int lo = min(warp * per, n), hi = min(lo + per, n);

  // The largest value, and the first place of it.
  uint32_t best = 0;
  for (int i = lo + lane; i < hi; i += 32) best = max(best, KeyOf(ToF32(x[i])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) kred[warp] = best;
  __syncthreads();
  for (int w = 0; w < kSampleWarps; ++w) best = max(best, kred[w]);
  const float top = ValueOf(best);
  if (!(temperature > 0.f) || top == -INFINITY) {  // greedy, or nothing to draw: the first of the largest, index 0 of a row without one
    int at = 0x7fffffff;
    for (int i = lo + lane; i < hi; i += 32)
      if (KeyOf(ToF32(x[i])) == best) at = min(at, i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, o));
    if (lane == 0) ired[warp] = at;
    __syncthreads();
    for (int w = 0; w < kSampleWarps; ++w) at = min(at, ired[w]);
    if (tid == 0) a.out[row] = top == -INFINITY ? 0 : at;
    return;
  }
  const double inv = 1.0 / static_cast<double>(temperature), dtop = static_cast<double>(top);
  auto weight = [&](uint32_t key) -> double {
    const float v = ValueOf(key);
    if (v == top) return 1.0;
    if (v == -INFINITY || top == INFINITY) return 0.0;
    return exp((static_cast<double>(v) - dtop) * inv);
  };
  auto count_from = [&](uint32_t key) {  // how many are as large as `key` or larger
    int c = 0;
    for (int i = lo + lane; i < hi; i += 32) c += KeyOf(ToF32(x[i])) >= key ? 1 : 0;
    return BlockSumAll(c, ired);
  };
  auto mass_from = [&](uint32_t key) {  // and their mass
    double m = 0.0;
    for (int i = lo + lane; i < hi; i += 32) {
      const uint32_t k = KeyOf(ToF32(x[i]));
      if (k >= key) m += weight(k);
    }
    return BlockSumAll(m, red);
  };
  // Kept: keys above `edge`, and the first `quota` of those equal to it.
  uint32_t edge = 0;
  int quota = n;
  double mass = 0.0;
  const bool by_k = top_k > 0 && top_k < n, by_p = top_p < 1.f;
  if (by_k) {  // the largest key that k are as large as
    uint32_t a0 = 0, a1 = best;
    while (a0 < a1) {
      const uint32_t mid = a0 + (a1 - a0 + 1) / 2;
      if (count_from(mid) >= top_k) a0 = mid;
      else a1 = mid - 1;
    }
    edge = a0;
    quota = top_k - (edge == best ? 0 : count_from(edge + 1));
  }
  if (by_p) {
    mass = by_k ? (edge == best ? 0.0 : mass_from(edge + 1)) + quota * weight(edge) : mass_from(0);
    const double share = fmax(static_cast<double>(top_p), 0.0) * mass;
    // The smallest key whose betters hold less than the share; the best one always does.
    uint32_t a0 = edge, a1 = best;
    while (a0 < a1) {
      const uint32_t mid = a0 + (a1 - a0) / 2;
      if (mass_from(mid + 1) < share) a1 = mid;
      else a0 = mid + 1;
    }
    const double above = a0 == best ? 0.0 : mass_from(a0 + 1), w = weight(a0);
    if (a0 != edge) quota = n;
    // The j-th of the equal ones stays while above + j w < share.
    if (w > 0.0) {
      double most = ceil((share - above) / w);
      if (most > 1.0 && above + (most - 1.0) * w >= share) most -= 1.0;
      if (above + most * w < share) most += 1.0;
      quota = static_cast<int>(fmin(static_cast<double>(quota), fmax(most, 1.0)));
    }
    edge = a0;
  }
  // Up to which place the equal ones stay.
  int equal = 0;
  for (int i = lo + lane; i < hi; i += 32) equal += KeyOf(ToF32(x[i])) == edge ? 1 : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) equal += __shfl_xor_sync(0xffffffffu, equal, o);
  __syncthreads();
  if (lane == 0) ired[warp] = equal;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < warp; ++w) before += ired[w];
  const double least = min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) : 0.0;
  // A warp walks its stretch in order, 32 at a time; what(i, w) gets every kept place of a lane and its weight (0 for the others).
  auto walk = [&](auto&& what) {
    int seen = before;
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t key = i < hi ? KeyOf(ToF32(x[i])) : 0u;
      const unsigned ties = __ballot_sync(0xffffffffu, i < hi && key == edge);
      const bool in = i < hi && (key > edge || (key == edge && seen + __popc(ties & ((1u << lane) - 1u)) < quota));
      seen += __popc(ties);
      double w = 0.0;
      if (in) {
        w = weight(key);
        if (w < least) w = 0.0;
      }
      if (what(i, w)) return;
    }
  };
  double mine = 0.0;
  walk([&](int, double w) {
    mine += w;
    return false;
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) red[warp] = mine;
  __syncthreads();
  double total = 0.0;
  int last = 0;  // the last warp that keeps any
  for (int w = 0; w < kSampleWarps; ++w) {
    total += red[w];
    if (red[w] > 0.0) last = w;
  }
  const float u = __ldg(a.uniforms + row);
  const double target = (u > 0.f ? fmin(static_cast<double>(u), 1.0) : 0.0) * total;
  double sum = 0.0;
  int chosen = last;
  double in_front = 0.0;
  for (int w = 0; w < kSampleWarps; ++w) {
    if (red[w] > 0.0 && sum + red[w] > target) {
      chosen = w;
      in_front = sum;
      break;
    }
    if (w == last) in_front = sum;
    sum += red[w];
  }
  if (warp != chosen) return;
  int token = -1;
  double run = in_front;
  walk([&](int i, double w) {
    double up = w;  // sums up to this lane
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += t;
    }
    const unsigned past = __ballot_sync(0xffffffffu, w > 0.0 && run + up > target), any = __ballot_sync(0xffffffffu, w > 0.0);
    if (past != 0u) {
      token = i - lane + __ffs(past) - 1;
      return true;
    }
    if (any != 0u) token = i - lane + 31 - __clz(any);  // the last one kept, where roundings leave the target out of reach
    run += __shfl_sync(0xffffffffu, up, 31);
    return false;
  });
  if (lane == 0) a.out[row] = max(token, 0);
}

}  // namespace
}  // namespace tlaloc_b200

using namespace tlaloc_b200;

extern "C" int tlaloc_b200_sample(const void* logits, int64_t ld, int32_t dtype, const float* uniforms, const float* temperature, const int32_t* top_k,
                                  const float* top_p, const float* min_p, float temperature_all, int32_t top_k_all, float top_p_all, float min_p_all,
                                  int32_t* out, int32_t rows, int32_t n, void* stream)
{
  const char* op = "SAMPLE";
  if (!logits || !uniforms || !out) return Fail(kInvalid, "%s: a required device pointer is null", op);
  if (!IsFloatType(dtype)) return Fail(kInvalid, "%s: logits must be f32 or bf16", op);
  if (rows < 0 || n < 1 || ld < n) return Fail(kInvalid, "%s: bad sizes", op);
  if (rows == 0) return kOk;
  const SampleArgs a = {logits, ld, uniforms, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all, out, n};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == TLALOC_B200_F32 ? LaunchChained(SampleKernel<float>, rows, kSampleThreads, 0, st, a)
                                                 : LaunchChained(SampleKernel<__nv_bfloat16>, rows, kSampleThreads, 0, st, a);
  if (e != cudaSuccess) return CudaFail("SAMPLE launch", e);
  CountLaunches(1);
  return kOk;
}
