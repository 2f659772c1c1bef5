// Next tokens from logits on gfx950: temperature, top-k, top-p, min-p and the
// draw from a given random number.
//
// A row's weights are whole numbers,
//   W_i = rint(2^42 exp((x_i - max x) / T)),
// so that every sum of them is exact, whatever its order and however it is
// split over threads, and one rule decides what a border falls on.  The
// tokens in the order (logit descending, index ascending) are cut to a
// prefix three times: the first k; of these the tokens whose sum of weights
// before them lies below p times their total; of these the tokens with
// W_i >= 2^42 min_p.  The token is the smallest index whose running sum of
// the remaining weights, in index order, exceeds u times their total.
// A vocabulary of up to 2^20 keeps sums within 2^62; tokens below 2^-43 of
// the likeliest have weight 0.
//
// A prefix of that order is (key K, ties kept m): every logit above K and
// the first m that equal it.  K is found by a radix select on the ordered
// bits of the logits whose histogram adds counts (top-k) or weights (top-p);
// no row is sorted.

#include "tierkv_common.h"

namespace tierkv {

constexpr int SP_THREADS = 1024;
constexpr int SP_WAVES = SP_THREADS / 64;
constexpr int SP_BINS = 256;
constexpr int SP_MAX_VOCAB = 1 << 20;
constexpr double SP_ONE = 4398046511104.0;   // 2^42

struct SampleParams {
  const void* logits;
  int64_t stride;
  int32_t batch, vocab;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int64_t* tokens;
  float* probs;
};

// The logit as an unsigned integer of the same order; -0 as +0, NaN lowest
// (a NaN logit is never drawn).
__device__ __forceinline__ uint32_t sp_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  if (x != x) return 0;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

struct SpRow {
  float top;      // the row's largest logit
  double rt;      // 1 / T
  double floor;   // weights below it (min-p) count as 0 in the draw
  __device__ __forceinline__ uint64_t weight(float x) const {
    if (x == top) return uint64_t(SP_ONE);
    const double d = double(x) - double(top);
    if (!(d > -1e300)) return 0;               // -inf, NaN
    return uint64_t(rint(exp(d * rt) * SP_ONE));
  }
};

template <typename T> __device__ __forceinline__ float sp_load(const T* x, int64_t i) { return to_f32<T>(x[i]); }
template <> __device__ __forceinline__ float sp_load<float>(const float* x, int64_t i) { return x[i]; }

__device__ __forceinline__ uint64_t sp_wave_sum(uint64_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

struct SpShared {
  uint64_t hist[SP_BINS];
  uint64_t wave[SP_WAVES];
  uint32_t key[SP_WAVES];
  int32_t index[SP_WAVES];
  uint64_t above;
  int32_t digit;
};

// The first digit from the top whose bins down to it add up to thr or more
// (sh.digit), and the sum of the bins above it (sh.above).  hist is complete
// and visible to the first wave.
__device__ __forceinline__ void sp_cross(SpShared& sh, uint64_t above, double thr) {
  const int lane = threadIdx.x;
  if (lane >= 64) return;
  uint64_t b[4], own = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    b[i] = sh.hist[SP_BINS - 1 - (lane * 4 + i)];
    own += b[i];
  }
  uint64_t incl = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t y = __shfl_up(incl, d, 64);
    if (lane >= d) incl += y;
  }
  const bool here = double(above + incl) >= thr;
  const uint64_t any = __ballot(here);
  const int first = any ? __ffsll((unsigned long long)any) - 1 : 63;
  if (lane == first) {
    uint64_t run = above + incl - own;
    int i = 0;
    while (i < 3 && double(run + b[i]) < thr) run += b[i++];
    sh.digit = SP_BINS - 1 - (lane * 4 + i);
    sh.above = run;
  }
}

// The key K with measure(> K) < thr <= measure(>= K); *above = measure(> K).
// measure(i, key) is the measure of element i; extra (key_x) is a measure
// added once at key_x.
template <typename T, typename M>
__device__ uint32_t sp_select(SpShared& sh, const T* x, int n, double thr, M measure, uint32_t key_x, uint64_t extra,
                              uint64_t* above) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0;
  uint64_t sum = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (tid < SP_BINS) sh.hist[tid] = 0;
    __syncthreads();
    const uint32_t high = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int i = tid; i < n; i += SP_THREADS) {
      const float v = sp_load(x, i);
      const uint32_t k = sp_key(v);
      if ((k & high) == prefix) {
        const uint64_t m = measure(v, k);
        if (m) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[(k >> shift) & 255]), (unsigned long long)m);
      }
    }
    if (tid == 0 && extra && (key_x & high) == prefix)
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[(key_x >> shift) & 255]), (unsigned long long)extra);
    __syncthreads();
    sp_cross(sh, sum, thr);
    __syncthreads();
    prefix |= uint32_t(sh.digit) << shift;
    sum = sh.above;
  }
  *above = sum;
  return prefix;
}

// Sum of measure(i) over [lo, hi) per wave segment; every thread gets the
// segments' sums in sh.wave.  Returns the segment length.
template <typename M>
__device__ int sp_segments(SpShared& sh, int lo, int hi, M measure) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int seg = (((hi - lo) + SP_WAVES * 64 - 1) / (SP_WAVES * 64)) * 64;
  uint64_t s = 0;
  for (int i = lo + w * seg + lane; i < min(lo + (w + 1) * seg, hi); i += 64) s += measure(i);
  s = sp_wave_sum(s);
  __syncthreads();
  if (lane == 0) sh.wave[w] = s;
  __syncthreads();
  return seg;
}

// The smallest index in [lo, hi) whose running sum of measure exceeds
// target, which is below the sum over [lo, hi).
template <typename M>
__device__ int sp_descend(SpShared& sh, int lo, int hi, uint64_t target, M measure) {
  while (hi - lo > 64) {
    const int seg = sp_segments(sh, lo, hi, measure);
    int w = 0;
    while (w < SP_WAVES - 1 && target >= sh.wave[w]) target -= sh.wave[w++];
    lo += w * seg;
    hi = min(lo + seg, hi);
  }
  const int lane = threadIdx.x & 63;
  uint64_t c = lo + lane < hi ? measure(lo + lane) : 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t y = __shfl_up(c, d, 64);
    if (lane >= d) c += y;
  }
  const uint64_t hit = __ballot(c > target);
  return hit ? lo + __ffsll((unsigned long long)hit) - 1 : hi - 1;
}

template <typename T>
__global__ __launch_bounds__(SP_THREADS) void sample_kernel(SampleParams p) {
  __shared__ SpShared sh;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int b = blockIdx.x, n = p.vocab;
  const T* x = reinterpret_cast<const T*>(p.logits) + int64_t(b) * p.stride;

  // The largest logit and its first index.
  uint32_t best = 0;
  int at = n;
  for (int i = tid; i < n; i += SP_THREADS) {
    const uint32_t k = sp_key(sp_load(x, i));
    if (k > best) {
      best = k;
      at = i;
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint32_t k = __shfl_xor(best, m, 64);
    const int i = __shfl_xor(at, m, 64);
    if (k > best || (k == best && i < at)) {
      best = k;
      at = i;
    }
  }
  if (lane == 0) {
    sh.key[w] = best;
    sh.index[w] = at;
  }
  __syncthreads();
  for (int i = 0; i < SP_WAVES; ++i)
    if (sh.key[i] > best || (sh.key[i] == best && sh.index[i] < at)) {
      best = sh.key[i];
      at = sh.index[i];
    }
  const float t = p.temperature ? p.temperature[b] : p.temperature_all;
  const uint32_t minus_inf = sp_key(-INFINITY);
  if (best <= minus_inf || !(t > 0.f)) {
    if (tid == 0) {
      const bool none = best <= minus_inf;
      p.tokens[b] = none ? -1 : at;
      if (p.probs) p.probs[b] = none ? 0.f : 1.f;
    }
    return;
  }
  SpRow row;
  row.top = sp_load(x, at);
  row.rt = 1.0 / double(t);
  const float mp = p.min_p ? p.min_p[b] : p.min_p_all;
  row.floor = mp > 0.f ? fmin(double(mp), 1.0) * SP_ONE : 0.0;

  // The prefix (cut, ties): every key above cut and the first `ties` equal
  // to it; ties < 0: all of them.
  uint32_t cut = 0;
  int64_t ties = -1;
  uint64_t above = 0;
  const int k = p.top_k ? p.top_k[b] : p.top_k_all;
  if (k > 0 && k < n) {
    cut = sp_select(sh, x, n, double(k), [](float, uint32_t) -> uint64_t { return 1; }, 0u, 0, &above);
    ties = k - int64_t(above);
  }
  auto key_value = [](uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); };
  const float tp = p.top_p ? p.top_p[b] : p.top_p_all;
  if (tp < 1.f) {
    const uint32_t cut_k = cut;
    const uint64_t at_cut = ties >= 0 ? uint64_t(ties) * row.weight(key_value(cut_k)) : 0;
    auto measure = [&](float v, uint32_t key) -> uint64_t { return key > cut_k || ties < 0 ? row.weight(v) : 0; };
    sp_segments(sh, 0, n, [&](int i) {
      const float v = sp_load(x, i);
      return measure(v, sp_key(v));
    });
    uint64_t total = at_cut;
    for (int i = 0; i < SP_WAVES; ++i) total += sh.wave[i];
    const double thr = fmax(double(tp) * double(total), 1.0);   // one token at least
    cut = sp_select(sh, x, n, thr, measure, cut_k, at_cut, &above);
    const uint64_t each = row.weight(key_value(cut));
    // The fewest ties that reach thr (one at least).
    int64_t m = 1;
    if (each > 0 && thr > double(above)) m = max(int64_t(1), int64_t((thr - double(above)) / double(each)) - 1);
    while (each > 0 && double(above + uint64_t(m) * each) < thr) ++m;
    ties = m;
  }
  // The index of the last tie kept.
  int last = n;
  if (ties >= 0) {
    auto tie = [&](int i) -> uint64_t { return sp_key(sp_load(x, i)) == cut ? 1 : 0; };
    sp_segments(sh, 0, n, tie);
    int64_t count = 0;
    for (int i = 0; i < SP_WAVES; ++i) count += int64_t(sh.wave[i]);
    if (ties < count) last = sp_descend(sh, 0, n, uint64_t(ties - 1), tie);
  }
  auto kept = [&](int i) -> uint64_t {
    const float v = sp_load(x, i);
    const uint32_t key = sp_key(v);
    if (key < cut || (key == cut && i > last)) return 0;
    const uint64_t weight = row.weight(v);
    return double(weight) >= row.floor ? weight : 0;
  };
  sp_segments(sh, 0, n, kept);
  uint64_t total = 0;
  for (int i = 0; i < SP_WAVES; ++i) total += sh.wave[i];
  const double u = double(p.u[b]);
  uint64_t target = u > 0.0 ? uint64_t(fmin(u, 1.0) * double(total)) : 0;
  target = min(target, total - 1);
  const int token = sp_descend(sh, 0, n, target, kept);
  if (tid == 0) {
    p.tokens[b] = token;
    if (p.probs) p.probs[b] = float(double(kept(token)) / double(total));
  }
}

}  // namespace tierkv

using namespace tierkv;

extern "C" int64_t tierkv_sample_workspace_bytes(int32_t batch, int32_t vocab) {
  if (batch <= 0 || vocab <= 0) return -1;
  return 256;
}

extern "C" int32_t tierkv_sample_tokens(
    const void* logits, int32_t dtype, int64_t row_stride, int32_t batch, int32_t vocab, const float* uniforms,
    const float* temperature, float temperature_all, const int32_t* top_k, int32_t top_k_all,
    const float* top_p, float top_p_all, const float* min_p, float min_p_all,
    int64_t* tokens, float* probs, void* workspace, int64_t workspace_bytes, void* stream_) {
  clear_error();
  if (!logits || !uniforms || !tokens || !workspace) return fail(TIERKV_ERR_INVALID, "null pointer");
  if (batch <= 0 || vocab <= 0) return fail(TIERKV_ERR_INVALID, "empty logits");
  if (vocab > SP_MAX_VOCAB) return fail(TIERKV_ERR_UNSUPPORTED, "vocabularies of more than 2^20 tokens");
  if (batch > 1 && row_stride < vocab) return fail(TIERKV_ERR_INVALID, "logit rows overlap");
  if (dtype != TIERKV_DTYPE_F16 && dtype != TIERKV_DTYPE_BF16 && dtype != TIERKV_DTYPE_F32)
    return fail(TIERKV_ERR_INVALID, "logits must be fp16, bf16 or fp32");
  if (workspace_bytes < tierkv_sample_workspace_bytes(batch, vocab))
    return fail(TIERKV_ERR_WORKSPACE, "workspace too small");
  SampleParams p{};
  p.logits = logits;
  p.stride = row_stride;
  p.batch = batch;
  p.vocab = vocab;
  p.u = uniforms;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.temperature_all = temperature_all;
  p.top_k_all = top_k_all;
  p.top_p_all = top_p_all;
  p.min_p_all = min_p_all;
  p.tokens = tokens;
  p.probs = probs;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (dtype == TIERKV_DTYPE_F32)
    hipLaunchKernelGGL(sample_kernel<float>, dim3(batch), dim3(SP_THREADS), 0, stream, p);
  else if (dtype == TIERKV_DTYPE_BF16)
    hipLaunchKernelGGL(sample_kernel<__hip_bfloat16>, dim3(batch), dim3(SP_THREADS), 0, stream, p);
  else
    hipLaunchKernelGGL(sample_kernel<__half>, dim3(batch), dim3(SP_THREADS), 0, stream, p);
  return check_launch("tierkv_sample_tokens");
}
