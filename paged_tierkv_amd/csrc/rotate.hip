// Per-head norms and rotation by position of packed query and key rows, with
// the keys and values written into their HOT slots, for gfx950 (CDNA4).
//
// Row r of request b stands at positions[r] of its context.  With R rotated
// dims and frequencies f_i (i < R / 2):
//   x' = x * rsqrt(mean(x^2) + eps) * w      (where a weight w is given)
//   y_a = c x'_a - s x'_b,  y_b = c x'_b + s x'_a,
//   c = A cos(position f_i),  s = A sin(position f_i)
// for the pair (a, b) = (i, i + R / 2), or (2 i, 2 i + 1) when interleaved;
// dims from R on pass.  The angle is formed in 64 bits and reduced to a
// fraction of a turn before it becomes 32 bits: position * f_i in 32 bits is
// off by up to 2^-24 of the angle, 0.007 at position 120000.  Everything else
// is 32-bit, rounded once when it is stored.

#include "tierkv_common.h"

#include <cmath>

namespace tierkv {

constexpr int ROT_THREADS = 256;

struct RotateParams {
  const void* src[3];       // q, k, v rows (v: NULL without pools)
  int64_t st_t[3], st_h[3];
  void* q_out;              // [rows, heads, D]
  void* k_out;              // [rows, kv_heads, D] or NULL
  const int32_t* positions;
  const float* inv_freq;
  const void* weight[2];    // of q and k, or NULL
  const int32_t* slots;     // or NULL
  __half* hot[2];
  int64_t pool_rows;        // hot_slots * block_size
  int32_t rows, heads, kv_heads, D, half, bs;   // half: pairs that are rotated
  int32_t weight_f32;
  float eps, amplitude;
};

// cos and sin of a position's angle, times the amplitude.
__device__ __forceinline__ float2 rot_turn(const RotateParams& p, int pos, int i) {
  constexpr double kTurn = 0.15915494309189533577;   // 1 / (2 pi)
  double x = double(pos) * double(p.inv_freq[i]) * kTurn;
  x -= rint(x);
  float s, c;
  sincospif(2.f * float(x), &s, &c);
  return make_float2(c * p.amplitude, s * p.amplitude);
}

// The pool row's start for (row's slot, kv head), or -1.
__device__ __forceinline__ int64_t rot_pool(const RotateParams& p, int slot_row, int h) {
  if (slot_row < 0 || slot_row >= p.pool_rows) return -1;
  const int64_t slot = slot_row / p.bs;
  return ((slot * p.kv_heads + h) * p.bs + (slot_row - slot * p.bs)) * p.D;
}

template <typename T>
__device__ __forceinline__ float rot_weight(const RotateParams& p, int which, int d) {
  return p.weight_f32 ? reinterpret_cast<const float*>(p.weight[which])[d]
                      : to_f32<T>(reinterpret_cast<const T*>(p.weight[which])[d]);
}

// Any head dim, strides and alignment: a wave per (row, head), a lane per
// pair or passed dim.
template <typename T>
__global__ __launch_bounds__(ROT_THREADS) void rotate_scalar_kernel(RotateParams p, int32_t interleaved) {
  const int lane = threadIdx.x & 63;
  const int units = p.heads + p.kv_heads * (p.src[2] ? 2 : 1);
  const int64_t u = int64_t(blockIdx.x) * (ROT_THREADS / 64) + (threadIdx.x >> 6);
  const int64_t r = u / units;
  if (r >= p.rows) return;
  const int x = int(u - r * units);
  const int kind = x < p.heads ? 0 : (x < p.heads + p.kv_heads ? 1 : 2);
  const int h = kind == 0 ? x : (x - p.heads) % p.kv_heads;
  const int pos = p.positions[r];
  if (pos < 0) return;
  const T* src = reinterpret_cast<const T*>(p.src[kind]) + r * p.st_t[kind] + h * p.st_h[kind];
  const int64_t pool = kind && p.slots ? rot_pool(p, p.slots[r], h) : -1;
  auto put = [&](int d, float y) {
    if (kind == 0) reinterpret_cast<T*>(p.q_out)[(r * p.heads + h) * p.D + d] = from_f32<T>(y);
    if (kind == 1 && p.k_out) reinterpret_cast<T*>(p.k_out)[(r * p.kv_heads + h) * p.D + d] = from_f32<T>(y);
    if (pool >= 0) p.hot[kind - 1][pool + d] = from_f32<__half>(y);
  };
  if (kind == 2) {
    for (int d = lane; d < p.D; d += 64) put(d, to_f32<T>(src[d]));
    return;
  }
  float factor = 1.f;
  const bool norm = p.weight[kind] != nullptr;
  if (norm) {
    float sum = 0.f;
    for (int d = lane; d < p.D; d += 64) {
      const float v = to_f32<T>(src[d]);
      sum += v * v;
    }
    factor = 1.f / sqrtf(wave_sum(sum) / float(p.D) + p.eps);
  }
  auto get = [&](int d) {
    const float v = to_f32<T>(src[d]) * factor;
    return norm ? v * rot_weight<T>(p, kind, d) : v;
  };
  for (int i = lane; i < p.half; i += 64) {
    const int a = interleaved ? 2 * i : i, b = interleaved ? 2 * i + 1 : i + p.half;
    const float2 t = rot_turn(p, pos, i);
    const float xa = get(a), xb = get(b);
    put(a, t.x * xa - t.y * xb);
    put(b, t.x * xb + t.y * xa);
  }
  for (int d = 2 * p.half + lane; d < p.D; d += 64) put(d, get(d));
}

template <typename T>
static void launch_rotate(const RotateParams& p, bool interleaved, hipStream_t stream) {
  const int units = p.heads + p.kv_heads * (p.src[2] ? 2 : 1);
  const int64_t waves = int64_t(p.rows) * units;
  hipLaunchKernelGGL(rotate_scalar_kernel<T>, dim3(uint32_t((waves + 3) / 4)), dim3(ROT_THREADS), 0, stream, p,
                     int32_t(interleaved));
}

}  // namespace tierkv

using namespace tierkv;

extern "C" int32_t tierkv_rotate_rows(
    const void* query, int64_t q_stride_t, int64_t q_stride_h, void* q_out,
    const void* key, int64_t k_stride_t, int64_t k_stride_h, void* k_out,
    const void* value, int64_t v_stride_t, int64_t v_stride_h, int32_t dtype,
    const int32_t* positions, int32_t num_rows,
    const float* inv_freq, int32_t rotary_dim, int32_t interleaved, float attention_scaling,
    const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps,
    const int32_t* slots, void* hot_k, void* hot_v, int64_t hot_slots,
    int32_t num_heads, int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream_) {
  clear_error();
  if (num_rows < 0) return fail(TIERKV_ERR_INVALID, "negative row count");
  if (dtype != TIERKV_DTYPE_F16 && dtype != TIERKV_DTYPE_BF16) return fail(TIERKV_ERR_INVALID, "rows must be fp16 or bf16");
  if (weight_dtype != dtype && weight_dtype != TIERKV_DTYPE_F32)
    return fail(TIERKV_ERR_INVALID, "norm weights must have the rows' dtype or be fp32");
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads > 65536 || num_kv_heads > 65536 || head_dim <= 0 || head_dim > 256)
    return fail(TIERKV_ERR_UNSUPPORTED, "1 to 65536 heads and a head_dim in [1, 256]");
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0)
    return fail(TIERKV_ERR_INVALID, "rotary_dim must be even and at most head_dim");
  if (!std::isfinite(attention_scaling) || !(eps >= 0.f) || !std::isfinite(eps))
    return fail(TIERKV_ERR_INVALID, "attention_scaling must be finite and eps finite and not negative");
  const bool pools = slots || hot_k || hot_v || value;
  if (pools) {
    if (!slots || !hot_k || !hot_v || !value) return fail(TIERKV_ERR_INVALID, "slots, value and both HOT pools go together");
    if (block_size <= 0 || block_size > 64) return fail(TIERKV_ERR_UNSUPPORTED, "block_size must be in [1, 64]");
    if (hot_slots <= 0 || hot_slots * block_size > 0x7fffffff)
      return fail(TIERKV_ERR_UNSUPPORTED, "pool rows must lie in (0, 2^31)");
  } else if (!k_out && num_rows > 0) {
    return fail(TIERKV_ERR_INVALID, "the keys need HOT pools or k_out");
  }
  if (num_rows == 0) return TIERKV_OK;
  if (!query || !q_out || !key || !positions || (rotary_dim > 0 && !inv_freq))
    return fail(TIERKV_ERR_INVALID, "null pointer");
  if (q_stride_t < 0 || q_stride_h < 0 || k_stride_t < 0 || k_stride_h < 0 || v_stride_t < 0 || v_stride_h < 0)
    return fail(TIERKV_ERR_INVALID, "strides must be non-negative");
  // A wave per (row, head) at most, and fewer than 2^32 threads in a launch.
  if (int64_t(num_rows) * (num_heads + 2 * int64_t(num_kv_heads)) > (0xffffffffll - 255) / 64)
    return fail(TIERKV_ERR_UNSUPPORTED, "rotation too large for one call");
  RotateParams p{};
  p.src[0] = query;
  p.src[1] = key;
  p.src[2] = value;
  p.st_t[0] = q_stride_t;
  p.st_h[0] = q_stride_h;
  p.st_t[1] = k_stride_t;
  p.st_h[1] = k_stride_h;
  p.st_t[2] = v_stride_t;
  p.st_h[2] = v_stride_h;
  p.q_out = q_out;
  p.k_out = k_out;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.weight[0] = q_weight;
  p.weight[1] = k_weight;
  p.weight_f32 = weight_dtype == TIERKV_DTYPE_F32;
  p.slots = slots;
  p.hot[0] = reinterpret_cast<__half*>(hot_k);
  p.hot[1] = reinterpret_cast<__half*>(hot_v);
  p.pool_rows = pools ? hot_slots * block_size : 0;
  p.rows = num_rows;
  p.heads = num_heads;
  p.kv_heads = num_kv_heads;
  p.D = head_dim;
  p.half = rotary_dim / 2;
  p.bs = pools ? block_size : 1;
  p.eps = eps;
  p.amplitude = attention_scaling;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (dtype == TIERKV_DTYPE_BF16) launch_rotate<__hip_bfloat16>(p, interleaved != 0, stream);
  else launch_rotate<__half>(p, interleaved != 0, stream);
  return check_launch("tierkv_rotate_rows");
}
