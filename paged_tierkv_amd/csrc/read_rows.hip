// Tokens of a tiered cache read back as packed rows, for gfx950 (CDNA4).
//
// Request b's rows [cu[b], cu[b + 1]) are its tokens of ordinal start[b],
// start[b] + 1, ... (ordinals count the valid tokens of all blocks): HOT ones
// as they are, WARM ones as the values that their codes stand for, formed in
// 32 bits and rounded once, evicted ones and those past what the request
// holds as zeros.
//
// One launch, a workgroup per block and K or V: it sums the lengths of the
// blocks before its own (a long row's lengths are read by all of them, from
// the caches: a scan of its own would be a second launch, 3 us of a window's
// 7), and blocks that end before the first token asked for, even if full, end
// at once (64 windows of 64 tokens in 2000: 21 -> 14 us).
// Bound: memory.  32768 tokens of 8 heads of 128, a tenth HOT, six tenths WARM
// and the rest zeros, 188 MB, take 41 to 43 us where two contexts are read in
// turn and 35 where one is read again; with one element per thread 334.  Two
// blocks per workgroup take 11 us for 500 tokens where one takes 7, and four 36
// for 32768 (read again).
// The sums grow with the square of the context, the launch with the tables'
// width: 262144 tokens take 493 us (3.1 TB/s), 2^20 2775 (2.2), their last 300
// 23 and 72; 250 tokens of each of 32 requests 14 us in tables of 16 blocks, 24
// of 1024 and 118 of 8192.

#include "tierkv_common.h"

namespace tierkv {

constexpr int RR_THREADS = 256;
constexpr int RR_AHEAD = 4;     // tokens of a thread in flight

struct ReadParams {
  const int32_t* start;
  const int32_t* cu;
  const int32_t* table;
  const int32_t* states;
  const int32_t* lengths;
  int64_t stride;
  const int32_t* nblocks;       // or NULL
  const __half* hot[2];
  const uint8_t* warm[2];
  const void* scale[2];
  const void* zero[2];
  int64_t hot_slots, warm_slots;
  void* out[2];
  int32_t rows, num_blocks, kv_heads, bs, D;
};

template <typename T> __device__ __forceinline__ T rr_from(float v) { return from_f32<T>(v); }
template <> __device__ __forceinline__ float rr_from<float>(float v) { return v; }

// What block i of request b gives: the packed rows [lo, lo + n) of the
// request, and the row among them of the block's first token, negative before
// them.
struct ReadPart {
  int lo, n;
  int64_t at;
  bool last, any;   // the request's last block; whether there is such a block (a request may have none)
};

// (Uniform.)  n is 0 where there is nothing to do.
__device__ __forceinline__ ReadPart rr_part(const ReadParams& p, int b, int i, int (&sums)[RR_THREADS / 64]) {
  ReadPart o{};
  int nb = p.num_blocks;
  if (p.nblocks) nb = min(max(p.nblocks[b], 0), p.num_blocks);
  if (i >= nb && i > 0) return o;
  o.last = i + 1 >= nb;
  o.any = i < nb;
  o.lo = min(max(p.cu[b], 0), p.rows);
  o.n = min(max(p.cu[b + 1], o.lo), p.rows) - o.lo;
  if (o.n <= 0) return o;
  const int start = max(p.start[b], 0);
  if (!o.last && int64_t(i + 1) * p.bs <= start) {   // even full blocks end before the first token asked for
    o.n = 0;
    return o;
  }
  int sum = 0;
  for (int j = threadIdx.x; j < i; j += RR_THREADS) sum += min(max(p.lengths[int64_t(b) * p.stride + j], 0), p.bs);
  sum = wave_inclusive_scan(sum);
  if ((threadIdx.x & 63) == 63) sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  o.at = -int64_t(start);
#pragma unroll
  for (int w = 0; w < RR_THREADS / 64; ++w) o.at += sums[w];
  return o;
}

// Block i of request b: its tokens [first, end) that are asked for, its tier
// (COLD where its slot is out of range) and slot.
struct ReadBlock {
  int len, first, end, state;
  int64_t slot;
};
__device__ __forceinline__ ReadBlock rr_block(const ReadParams& p, int b, int i, int n, int64_t at) {
  const int64_t row = int64_t(b) * p.stride + i;
  ReadBlock o;
  o.len = min(max(p.lengths[row], 0), p.bs);
  o.first = int(max(-at, int64_t(0)));
  o.end = int(min(n - at, int64_t(o.len)));
  o.state = p.states[row];
  o.slot = p.table[row];
  if (o.slot < 0 || o.slot >= (o.state == HOT ? p.hot_slots : p.warm_slots)) o.state = COLD;
  return o;
}

// Any layout: one element per thread and step.
template <int WF, typename T>
__global__ __launch_bounds__(RR_THREADS) void read_rows_scalar_kernel(ReadParams p) {
  __shared__ int sums[RR_THREADS / 64];
  const int b = blockIdx.y, i = blockIdx.x;
  ReadPart part = rr_part(p, b, i, sums);
  const int lo = part.lo, n = part.n;
  if (n <= 0) return;
  const int width = p.kv_heads * p.D;
  if (part.any) {
    const ReadBlock k = rr_block(p, b, i, n, part.at);
    const int count = max(k.end - k.first, 0);   // (far behind the last token asked for, its product would pass 32 bits)
    for (int x = threadIdx.x; x < 2 * count * width; x += RR_THREADS) {
      const int kv = x >= count * width, y = x - kv * count * width;
      const int h = y / (count * p.D), z = y - h * count * p.D;
      const int t = k.first + z / p.D, d = z % p.D;
      const int64_t src = (k.slot * p.kv_heads + h) * p.bs + t;
      float v = 0.f;
      if (k.state == HOT) {
        v = __half2float(p.hot[kv][src * p.D + d]);
      } else if (k.state == WARM) {
        const uint8_t c = p.warm[kv][src * p.D + d];
        if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
          v = float(int8_t(c)) * reinterpret_cast<const float*>(p.scale[kv])[k.slot * p.kv_heads + h];
        } else {
          v = (float(c) - __half2float(reinterpret_cast<const __half*>(p.zero[kv])[src])) *
              __half2float(reinterpret_cast<const __half*>(p.scale[kv])[src]);
        }
      }
      reinterpret_cast<T*>(p.out[kv])[(lo + part.at + t) * width + h * p.D + d] = rr_from<T>(v);
    }
    part.at += k.len;
  }
  if (part.last) {      // what the request does not hold
    const int64_t from = min(max(part.at, int64_t(0)), int64_t(n)) * width;
    for (int64_t x = from + threadIdx.x; x < int64_t(n) * width; x += RR_THREADS)
      for (int kv = 0; kv < 2; ++kv) reinterpret_cast<T*>(p.out[kv])[int64_t(lo) * width + x] = rr_from<T>(0.f);
  }
}

// Eight values of a row, as stored.
template <typename T>
__device__ __forceinline__ void rr_put8(T* dst, const float (&v)[8]) {
  if constexpr (__is_same(T, float)) {
    *reinterpret_cast<f32x4*>(dst) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(dst + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T a = from_f32<T>(v[2 * i]), b = from_f32<T>(v[2 * i + 1]);
      w[i] = uint32_t(__builtin_bit_cast(uint16_t, a)) | (uint32_t(__builtin_bit_cast(uint16_t, b)) << 16);
    }
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Head dims of whole 8-element chunks: 2^r_log2 threads take a token of a
// head, a chunk each, and walk K or V (blockIdx.z) of the blocks tokens first,
// so that codes leave the pool in one piece, RR_AHEAD tokens in flight.
template <int WF, typename T>
__global__ __launch_bounds__(RR_THREADS) void read_rows_wide_kernel(ReadParams p, int32_t r_log2) {
  __shared__ int sums[RR_THREADS / 64];
  const int b = blockIdx.y, kv = blockIdx.z, i = blockIdx.x;
  ReadPart part = rr_part(p, b, i, sums);
  const int n = part.n;
  if (n <= 0) return;
  const int chunk = threadIdx.x & ((1 << r_log2) - 1), mine = threadIdx.x >> r_log2, step = RR_THREADS >> r_log2;
  const int D = p.D, c = 8 * min(chunk, D / 8 - 1);
  const bool live = 8 * chunk < D;
  const int width = p.kv_heads * D;
  T* const out = reinterpret_cast<T*>(kv ? p.out[1] : p.out[0]) + int64_t(part.lo) * width + c;
  const __half* const hot = kv ? p.hot[1] : p.hot[0];
  const uint8_t* const warm = kv ? p.warm[1] : p.warm[0];
  const void* const scales = kv ? p.scale[1] : p.scale[0];
  const void* const zeros = kv ? p.zero[1] : p.zero[0];
  if (part.any) {
    const ReadBlock k = rr_block(p, b, i, n, part.at);
    const int count = k.end - k.first, items = count > 0 ? count * p.kv_heads : 0;
    const int64_t tile = k.slot * p.kv_heads * int64_t(p.bs);
    // Item x is token t of head h; the thread's next is `step` further.
    const int div = max(count, 1), more_h = step / div, more_t = step - more_h * div;
    int h = mine / div, t = mine - h * div;
    for (int x0 = mine; x0 < items; x0 += step * RR_AHEAD) {
      uint4 raw[RR_AHEAD];
      float scale[RR_AHEAD], zero[RR_AHEAD];
      int to[RR_AHEAD];
#pragma unroll
      for (int j = 0; j < RR_AHEAD; ++j) {
        to[j] = x0 + j * step < items && live ? (k.first + t) * width + h * D : -1;
        raw[j] = make_uint4(0, 0, 0, 0);
        scale[j] = zero[j] = 0.f;
        const int64_t row = tile + h * p.bs + k.first + t, of = k.slot * p.kv_heads + h;
        t += more_t;
        h += more_h + (t >= div);
        t -= t >= div ? div : 0;
        if (to[j] < 0) continue;
        if (k.state == HOT) {
          raw[j] = *reinterpret_cast<const uint4*>(hot + row * D + c);
        } else if (k.state == WARM) {
          const uint2 w = *reinterpret_cast<const uint2*>(warm + row * D + c);
          raw[j].x = w.x;
          raw[j].y = w.y;
          if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
            scale[j] = reinterpret_cast<const float*>(scales)[of];
          } else {
            scale[j] = __half2float(reinterpret_cast<const __half*>(scales)[row]);
            zero[j] = __half2float(reinterpret_cast<const __half*>(zeros)[row]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < RR_AHEAD; ++j) {
        if (to[j] < 0) continue;
        float v[8];
        const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
        if (k.state == HOT) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[2 * e] = half_lo(w[e]);
            v[2 * e + 1] = half_hi(w[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t code = (w[e >> 2] >> (8 * (e & 3))) & 0xffu;
            v[e] = WF == TIERKV_WARM_ABSMAX_I8 ? float(int8_t(code)) * scale[j] : (float(code) - zero[j]) * scale[j];
          }
        }
        rr_put8<T>(out + part.at * width + to[j], v);
      }
    }
    part.at += k.len;
  }
  if (part.last && live) {      // what the request does not hold
    const float none[8] = {};
    const int64_t from = min(max(part.at, int64_t(0)), int64_t(n));
    for (int64_t x = mine; x < (n - from) * p.kv_heads; x += step) rr_put8<T>(out + from * width + x * D, none);
  }
}

template <int WF, typename T>
static void launch_read(const ReadParams& p, int batch, bool wide, hipStream_t stream) {
  dim3 grid(p.num_blocks, batch);
  if (!wide) {
    hipLaunchKernelGGL((read_rows_scalar_kernel<WF, T>), grid, dim3(RR_THREADS), 0, stream, p);
    return;
  }
  int r_log2 = 0;
  while ((8 << r_log2) < p.D) ++r_log2;
  grid.z = 2;
  hipLaunchKernelGGL((read_rows_wide_kernel<WF, T>), grid, dim3(RR_THREADS), 0, stream, p, r_log2);
}

template <int WF>
static void dispatch_read(const ReadParams& p, int batch, int dtype, bool wide, hipStream_t stream) {
  if (dtype == TIERKV_DTYPE_BF16) launch_read<WF, __hip_bfloat16>(p, batch, wide, stream);
  else if (dtype == TIERKV_DTYPE_F32) launch_read<WF, float>(p, batch, wide, stream);
  else launch_read<WF, __half>(p, batch, wide, stream);
}

}  // namespace tierkv

using namespace tierkv;

extern "C" int32_t tierkv_read_rows(
    const int32_t* start, const int32_t* cu_tokens, int32_t num_rows,
    const int32_t* block_table, const int32_t* block_states, const int32_t* block_lengths, int64_t table_stride,
    const int32_t* seq_num_blocks, int32_t num_blocks,
    const void* hot_k, const void* hot_v, int64_t hot_slots,
    const void* warm_k, const void* warm_v, int64_t warm_slots,
    const void* k_scale, const void* k_zero, const void* v_scale, const void* v_zero, int32_t warm_format,
    void* out_k, void* out_v, int32_t out_dtype,
    int32_t batch, int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream_) {
  clear_error();
  if (num_rows < 0) return fail(TIERKV_ERR_INVALID, "negative row count");
  if (!start || !cu_tokens || !block_table || !block_states || !block_lengths || (num_rows > 0 && (!out_k || !out_v)))
    return fail(TIERKV_ERR_INVALID, "null tensor pointer");
  if (batch <= 0) return fail(TIERKV_ERR_INVALID, "batch must be positive");
  if (num_blocks <= 0) return fail(TIERKV_ERR_INVALID, "num_blocks must be positive.");
  if (num_blocks > table_stride) return fail(TIERKV_ERR_INVALID, "num_blocks exceeds the provided block table length.");
  if (warm_format != TIERKV_WARM_REF_U8 && warm_format != TIERKV_WARM_ABSMAX_I8)
    return fail(TIERKV_ERR_INVALID, "unknown warm format");
  if (out_dtype != TIERKV_DTYPE_F16 && out_dtype != TIERKV_DTYPE_BF16 && out_dtype != TIERKV_DTYPE_F32)
    return fail(TIERKV_ERR_INVALID, "rows must be fp16, bf16 or fp32");
  if (num_kv_heads <= 0 || num_kv_heads > 65535 || block_size <= 0 || block_size > 64 || head_dim <= 0 || head_dim > 256)
    return fail(TIERKV_ERR_UNSUPPORTED, "1 to 65535 heads, block_size in [1, 64] and head_dim in [1, 256]");
  if (!hot_k || !hot_v || hot_slots <= 0) return fail(TIERKV_ERR_INVALID, "HOT pools are required");
  if (!warm_k || !warm_v || !k_scale || !v_scale || warm_slots <= 0)
    return fail(TIERKV_ERR_INVALID, "WARM pools and scales are required (pass 1-slot placeholders when empty)");
  if (warm_format == TIERKV_WARM_REF_U8 && (!k_zero || !v_zero))
    return fail(TIERKV_ERR_INVALID, "reference-format WARM pools need zero points");
  if (int64_t(num_blocks) * block_size > 0x7fffffff) return fail(TIERKV_ERR_UNSUPPORTED, "rows of 2^31 tokens or more");
  if (batch > 65535) return fail(TIERKV_ERR_UNSUPPORTED, "more than 65535 requests");
  if (int64_t(num_blocks) > 0xffffffffll / RR_THREADS) return fail(TIERKV_ERR_UNSUPPORTED, "grid too large");
  if (num_rows == 0) return TIERKV_OK;
  ReadParams p{};
  p.start = start;
  p.cu = cu_tokens;
  p.table = block_table;
  p.states = block_states;
  p.lengths = block_lengths;
  p.stride = table_stride;
  p.nblocks = seq_num_blocks;
  p.hot[0] = reinterpret_cast<const __half*>(hot_k);
  p.hot[1] = reinterpret_cast<const __half*>(hot_v);
  p.warm[0] = reinterpret_cast<const uint8_t*>(warm_k);
  p.warm[1] = reinterpret_cast<const uint8_t*>(warm_v);
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.zero[0] = k_zero;
  p.zero[1] = v_zero;
  p.hot_slots = hot_slots;
  p.warm_slots = warm_slots;
  p.out[0] = out_k;
  p.out[1] = out_v;
  p.rows = num_rows;
  p.num_blocks = num_blocks;
  p.kv_heads = num_kv_heads;
  p.bs = block_size;
  p.D = head_dim;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  // 16-byte loads and stores, 8 bytes of codes; a token's place in its block's rows fits 32 bits.
  const bool wide = head_dim % 8 == 0 && aligned16(hot_k) && aligned16(hot_v) && aligned16(out_k) && aligned16(out_v) &&
                    reinterpret_cast<uintptr_t>(warm_k) % 8 == 0 && reinterpret_cast<uintptr_t>(warm_v) % 8 == 0;
  if (warm_format == TIERKV_WARM_ABSMAX_I8) dispatch_read<TIERKV_WARM_ABSMAX_I8>(p, batch, out_dtype, wide, stream);
  else dispatch_read<TIERKV_WARM_REF_U8>(p, batch, out_dtype, wide, stream);
  return check_launch("tierkv_read_rows");
}
