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
//
// Bound: memory.  16384 bf16 rows of 32 / 8 heads of 128 with both norms, 403
// MB read and written, take 84 us, 4.8 TB/s (a copy of 1 GiB reaches 5.14);
// with every head forming its own sines and cosines from one workgroup's
// table, and the weights read again for each, the instructions bounded it
// (22 per element, 105 us); a wave per (row, head) with a sine and a cosine
// for each pair took 507, and layouts off 16 bytes still take it (16384 rows with
// 120 of 128 dims turned and norms: 455 us).  A few rows take 6 us, the chain
// from a position to its sine and cosine to the first store.

#include "tierkv_common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace tierkv {

constexpr int ROT_THREADS = 256;
// Rows from which a workgroup takes four, a wave to each, instead of one.
// Launches of 32 / 8 heads of 128, four against one: 64 rows 7.9 / 6.2 us, 512
// 8.6 / 7.4, 1024 9.3 / 9.4, 2048 13.1 / 16.8, 16384 84 / 130; of 14 / 2 heads
// of 64: 512 7.5 / 6.7, 1024 7.5 / 7.3, 2048 7.6 / 11.7.
constexpr int ROT_MANY = 1024;
constexpr int64_t ROT_GRID = 0xffffffffll / ROT_THREADS;   // workgroups of a launch: fewer than 2^32 threads
constexpr int ROT_HEADS = 2;     // heads of a thread whose loads are in flight together (1: 87 us, 4: 89 us of 85)

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

// Two 16-bit values of a word as floats, and back in the type's rounding.
template <typename T>
__device__ __forceinline__ float2 rot_two(uint32_t w) {
  if constexpr (__is_same(T, __half)) return make_float2(half_lo(w), half_hi(w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

template <typename T>
__device__ __forceinline__ uint32_t rot_pack(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  if constexpr (__is_same(T, __half)) {
    return bits_of(__builtin_convertvector(f2{a, b}, f16x2));
  } else {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, bf2));
  }
}

template <typename T>
__device__ __forceinline__ uint4 rot_pack8(const float (&x)[8]) {
  return make_uint4(rot_pack<T>(x[0], x[1]), rot_pack<T>(x[2], x[3]), rot_pack<T>(x[4], x[5]), rot_pack<T>(x[6], x[7]));
}

template <typename T>
__device__ __forceinline__ void rot_unpack8(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = rot_two<T>(w[i]);
    x[2 * i] = t.x;
    x[2 * i + 1] = t.y;
  }
}

// Sum over the 2^lanes_log2 (at most 16) neighbouring lanes of a head, the
// same in all of them: each step pairs groups that already agree.
__device__ __forceinline__ float rot_sum(float v, int lanes_log2) {
  auto step = [&](auto ctrl) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  if (lanes_log2 >= 1) step(std::integral_constant<int, 0xB1>{});    // quad_perm [1, 0, 3, 2]
  if (lanes_log2 >= 2) step(std::integral_constant<int, 0x4E>{});    // quad_perm [2, 3, 0, 1]
  if (lanes_log2 >= 3) step(std::integral_constant<int, 0x141>{});   // row_half_mirror
  if (lanes_log2 >= 4) step(std::integral_constant<int, 0x140>{});   // row_mirror
  return v;
}

// Head dims of whole 16-byte chunks.  A thread takes two chunks of its row's
// heads, one head after another: those of eight pairs, chunk l and l + half /
// 8, or 2 l and 2 l + 1 when the pairs are adjacent, so that a pair never
// crosses threads; 2^lanes_log2 threads hold a head.  ROT_THREADS / R threads
// share a row: they form its sines and cosines together, one each, and a
// thread keeps its eight, times the norm's weights, in registers over all
// heads.  R = 4, a wave to each row, where there are many rows.
template <typename T, bool PAIRS, int R>
__global__ __launch_bounds__(ROT_THREADS) void rotate_kernel(RotateParams p, int32_t lanes_log2) {
  constexpr int PER_ROW = ROT_THREADS / R, MAX_HALF = 128;   // head_dim up to 256
  constexpr int NI = ROT_HEADS;
  __shared__ __attribute__((aligned(16))) float s_turn[2][R][MAX_HALF];
  const int x = threadIdx.x % PER_ROW, of = threadIdx.x / PER_ROW;
  const int64_t r = int64_t(blockIdx.x) * R + of;
  const int pos = r < p.rows ? p.positions[r] : -1;
  const int l = x & ((1 << lanes_log2) - 1), first = x >> lanes_log2, step = PER_ROW >> lanes_log2;
  const int chunks = p.D / 8, turning = p.half / 8;   // turning: threads of a head whose chunks turn
  const bool turns = l < turning;
  const int c0 = PAIRS ? 2 * l : (turns ? l : 2 * l);
  const int c1 = PAIRS ? 2 * l + 1 : (turns ? l + turning : 2 * l + 1);
  const bool has0 = c0 < chunks && pos >= 0, has1 = c1 < chunks && pos >= 0;
  if (pos >= 0) {
    for (int i = x; i < p.half; i += PER_ROW) {
      const float2 t = rot_turn(p, pos, i);
      s_turn[0][of][i] = t.x;
      s_turn[1][of][i] = t.y;
    }
  }
  __syncthreads();
  if (pos < 0) return;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = turns ? s_turn[0][of][8 * l + e] : 1.f;
    sn[e] = turns ? s_turn[1][of][8 * l + e] : 0.f;
  }
  // The pool row of head 0, and the next head's distance.
  const int64_t pool = p.slots ? rot_pool(p, p.slots[r], 0) : -1;
  const int64_t pool_step = int64_t(p.bs) * p.D;
#pragma unroll 1
  for (int kind = 0; kind < 2; ++kind) {
    const int heads = kind ? p.kv_heads : p.heads;
    const void* weight = kind ? p.weight[1] : p.weight[0];
    // y_a = (c w_a) x_a - (s w_b) x_b, y_b = (c w_b) x_b + (s w_a) x_a; the norm's factor comes last.
    float ca[8], sa[8], cb[8], sb[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ca[e] = cb[e] = cs[e];
      sa[e] = sb[e] = sn[e];
    }
    if (weight) {
      float w[16];
      if (p.weight_f32) {
        const float* src = reinterpret_cast<const float*>(weight);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = has0 ? src[8 * c0 + e] : 0.f;
          w[8 + e] = has1 ? src[8 * c1 + e] : 0.f;
        }
      } else {
        float t[8];
        const uint4* src = reinterpret_cast<const uint4*>(weight);
        rot_unpack8<T>(has0 ? src[c0] : make_uint4(0, 0, 0, 0), t);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = t[e];
        rot_unpack8<T>(has1 ? src[c1] : make_uint4(0, 0, 0, 0), t);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[8 + e] = t[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float wa = PAIRS ? w[2 * e] : w[e], wb = PAIRS ? w[2 * e + 1] : w[8 + e];
        ca[e] *= wa;
        sa[e] *= wa;
        cb[e] *= wb;
        sb[e] *= wb;
      }
    }
    const T* src = reinterpret_cast<const T*>(kind ? p.src[1] : p.src[0]) + r * (kind ? p.st_t[1] : p.st_t[0]);
    const int64_t src_step = kind ? p.st_h[1] : p.st_h[0];
    T* const out = reinterpret_cast<T*>(kind ? p.k_out : p.q_out);
#pragma unroll 1
    for (int h0 = first; h0 < heads; h0 += step * NI) {
      uint4 v0[NI], v1[NI];
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int h = h0 + i * step;
        const uint4* at = reinterpret_cast<const uint4*>(src + (h < heads ? h : h0) * src_step);
        v0[i] = has0 ? at[c0] : make_uint4(0, 0, 0, 0);
        v1[i] = has1 ? at[c1] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int h = h0 + i * step;
        float v[16], t[8];
        rot_unpack8<T>(v0[i], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = t[e];
        rot_unpack8<T>(v1[i], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 + e] = t[e];
        float factor = 1.f;
        if (weight) {
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) sum = fmaf(v[e], v[e], sum);
          factor = 1.f / sqrtf(rot_sum(sum, lanes_log2) / float(p.D) + p.eps);
        }
        if (h >= heads) break;   // (a head's lanes alike)
        float y[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int a = PAIRS ? 2 * e : e, b = PAIRS ? 2 * e + 1 : 8 + e;
          if (turns) {
            y[a] = ca[e] * v[a] - sb[e] * v[b];
            y[b] = cb[e] * v[b] + sa[e] * v[a];
          } else {
            y[a] = ca[e] * v[a];
            y[b] = cb[e] * v[b];
          }
        }
        if (weight) {
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] *= factor;
        }
        const float lo[8] = {y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]};
        const float hi[8] = {y[8], y[9], y[10], y[11], y[12], y[13], y[14], y[15]};
        if (out) {
          uint4* dst = reinterpret_cast<uint4*>(out + (r * heads + h) * p.D);
          if (has0) dst[c0] = rot_pack8<T>(lo);
          if (has1) dst[c1] = rot_pack8<T>(hi);
        }
        if (kind && pool >= 0) {
          uint4* dst = reinterpret_cast<uint4*>(p.hot[0] + pool + h * pool_step);
          if (has0) dst[c0] = rot_pack8<__half>(lo);
          if (has1) dst[c1] = rot_pack8<__half>(hi);
        }
      }
    }
  }
  if (pool < 0) return;
  const T* src = reinterpret_cast<const T*>(p.src[2]) + r * p.st_t[2];
  for (int h = first; h < p.kv_heads; h += step) {
    const uint4* at = reinterpret_cast<const uint4*>(src + h * p.st_h[2]);
    uint4* dst = reinterpret_cast<uint4*>(p.hot[1] + pool + h * pool_step);
    float t[8];
    if (has0) {
      rot_unpack8<T>(at[c0], t);
      dst[c0] = rot_pack8<__half>(t);
    }
    if (has1) {
      rot_unpack8<T>(at[c1], t);
      dst[c1] = rot_pack8<__half>(t);
    }
  }
}

template <typename T, bool PAIRS>
static void launch_rotate_wide(const RotateParams& p, hipStream_t stream) {
  int lanes_log2 = 0;
  while ((16 << lanes_log2) < p.D) ++lanes_log2;
  if (p.rows >= ROT_MANY)
    hipLaunchKernelGGL((rotate_kernel<T, PAIRS, 4>), dim3((p.rows + 3) / 4), dim3(ROT_THREADS), 0, stream, p, lanes_log2);
  else
    hipLaunchKernelGGL((rotate_kernel<T, PAIRS, 1>), dim3(p.rows), dim3(ROT_THREADS), 0, stream, p, lanes_log2);
}

template <typename T>
static void launch_rotate(const RotateParams& p, bool interleaved, bool wide, hipStream_t stream) {
  if (wide && interleaved) return launch_rotate_wide<T, true>(p, stream);
  if (wide) return launch_rotate_wide<T, false>(p, stream);
  // As many rows as a launch has waves for, and again.  (A loop over them in
  // the kernel: 16384 rows of 32 / 8 heads of 126 in 288 us, 261 without.)
  const int64_t units = p.heads + p.kv_heads * (p.src[2] ? 2 : 1), most = ROT_GRID * (ROT_THREADS / 64) / units;
  for (int64_t r0 = 0; r0 < p.rows; r0 += most) {
    RotateParams part = p;
    part.rows = int32_t(std::min(most, p.rows - r0));
    for (int i = 0; i < 3; ++i)
      if (p.src[i]) part.src[i] = reinterpret_cast<const T*>(p.src[i]) + r0 * p.st_t[i];
    part.q_out = reinterpret_cast<T*>(p.q_out) + r0 * p.heads * p.D;
    if (p.k_out) part.k_out = reinterpret_cast<T*>(p.k_out) + r0 * p.kv_heads * p.D;
    part.positions = p.positions + r0;
    if (p.slots) part.slots = p.slots + r0;
    hipLaunchKernelGGL(rotate_scalar_kernel<T>, dim3(uint32_t((part.rows * units + 3) / 4)), dim3(ROT_THREADS), 0, stream,
                       part, int32_t(interleaved));
  }
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
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads > 65535 || num_kv_heads > 65535 || head_dim <= 0 || head_dim > 256)
    return fail(TIERKV_ERR_UNSUPPORTED, "1 to 65535 heads and a head_dim in [1, 256]");
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0)
    return fail(TIERKV_ERR_INVALID, "rotary_dim must be even and at most head_dim");
  if (!std::isfinite(attention_scaling) || !(eps >= 0.f) || !std::isfinite(eps))
    return fail(TIERKV_ERR_INVALID, "attention_scaling must be finite and eps finite and not negative");
  const bool pools = slots || hot_k || hot_v || value;
  if (pools) {
    // (no rows: their tensors have no address)
    if (!hot_k || !hot_v || (num_rows > 0 && (!slots || !value)))
      return fail(TIERKV_ERR_INVALID, "slots, value and both HOT pools go together");
    if (block_size <= 0 || block_size > 64) return fail(TIERKV_ERR_UNSUPPORTED, "block_size must be in [1, 64]");
    if (hot_slots <= 0 || hot_slots > 0x7fffffff / block_size)
      return fail(TIERKV_ERR_UNSUPPORTED, "pool rows must lie in (0, 2^31)");
  } else if (!k_out && num_rows > 0) {
    return fail(TIERKV_ERR_INVALID, "the keys need HOT pools or k_out");
  }
  if (num_rows == 0) return TIERKV_OK;
  if (!query || !q_out || !key || !positions || (rotary_dim > 0 && !inv_freq))
    return fail(TIERKV_ERR_INVALID, "null pointer");
  if (q_stride_t < 0 || q_stride_h < 0 || k_stride_t < 0 || k_stride_h < 0 || v_stride_t < 0 || v_stride_h < 0)
    return fail(TIERKV_ERR_INVALID, "strides must be non-negative");
  // A wave per row.
  if ((int64_t(num_rows) + 3) / 4 > ROT_GRID) return fail(TIERKV_ERR_UNSUPPORTED, "rotation too large for one call");
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
  const bool pairs = interleaved != 0;
  // 16-byte chunks throughout, of dims that turn or pass, in pairs of chunks.
  const int64_t strides = q_stride_t | q_stride_h | k_stride_t | k_stride_h | v_stride_t | v_stride_h;
  const bool wide = head_dim % 8 == 0 && rotary_dim % 16 == 0 && strides % 8 == 0 && aligned16(query) &&
                    aligned16(key) && aligned16(value) && aligned16(q_out) && aligned16(k_out) && aligned16(hot_k) &&
                    aligned16(hot_v) && aligned16(q_weight) && aligned16(k_weight);
  if (dtype == TIERKV_DTYPE_BF16) launch_rotate<__hip_bfloat16>(p, pairs, wide, stream);
  else launch_rotate<__half>(p, pairs, wide, stream);
  return check_launch("tierkv_rotate_rows");
}
