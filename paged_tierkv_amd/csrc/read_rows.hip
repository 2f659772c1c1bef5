// Tokens of a tiered cache read back as packed rows, for gfx950 (CDNA4).
//
// Request b's rows [cu[b], cu[b + 1]) are its tokens of ordinal start[b],
// start[b] + 1, ... (ordinals count the valid tokens of all blocks): HOT ones
// as they are, WARM ones as the values that their codes stand for, formed in
// 32 bits and rounded once, evicted ones and those past what the request
// holds as zeros.

#include "tierkv_common.h"

namespace tierkv {

constexpr int RR_THREADS = 256;
constexpr int RR_BLOCKS = 4;    // blocks of a request per workgroup

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

// One element per thread and step.
template <int WF, typename T>
__global__ __launch_bounds__(RR_THREADS) void read_rows_scalar_kernel(ReadParams p) {
  __shared__ int sums[RR_THREADS / 64];
  const int b = blockIdx.y, i0 = int(blockIdx.x) * RR_BLOCKS;
  int nb = p.num_blocks;
  if (p.nblocks) nb = min(max(p.nblocks[b], 0), p.num_blocks);
  const bool last = i0 + RR_BLOCKS >= nb;
  if (i0 >= nb && i0 > 0) return;
  const int lo = min(max(p.cu[b], 0), p.rows), n = min(max(p.cu[b + 1], lo), p.rows) - lo;
  if (n <= 0) return;
  const int64_t row = int64_t(b) * p.stride;
  int sum = 0;
  for (int i = threadIdx.x; i < min(i0, nb); i += RR_THREADS) sum += min(max(p.lengths[row + i], 0), p.bs);
  sum = wave_inclusive_scan(sum);
  if ((threadIdx.x & 63) == 63) sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  int64_t at = -int64_t(max(p.start[b], 0));    // the next token's row among the request's
  for (int w = 0; w < RR_THREADS / 64; ++w) at += sums[w];
  const int width = p.kv_heads * p.D;
  for (int i = i0; i < min(i0 + RR_BLOCKS, nb); ++i) {
    const int len = min(max(p.lengths[row + i], 0), p.bs);
    const int first = int(max(-at, int64_t(0))), end = int(min(int64_t(n) - at, int64_t(len)));
    if (first < end) {
      int state = p.states[row + i];
      const int64_t slot = p.table[row + i];
      if (slot < 0 || slot >= (state == HOT ? p.hot_slots : p.warm_slots)) state = COLD;
      for (int kv = 0; kv < 2; ++kv) {
        for (int x = threadIdx.x; x < (end - first) * width; x += RR_THREADS) {
          const int h = x / ((end - first) * p.D), y = x - h * (end - first) * p.D;
          const int t = first + y / p.D, d = y % p.D;
          const int64_t src = (slot * p.kv_heads + h) * p.bs + t;
          float v = 0.f;
          if (state == HOT) {
            v = __half2float(p.hot[kv][src * p.D + d]);
          } else if (state == WARM) {
            const uint8_t c = p.warm[kv][src * p.D + d];
            if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
              v = float(int8_t(c)) * reinterpret_cast<const float*>(p.scale[kv])[slot * p.kv_heads + h];
            } else {
              v = (float(c) - __half2float(reinterpret_cast<const __half*>(p.zero[kv])[src])) *
                  __half2float(reinterpret_cast<const __half*>(p.scale[kv])[src]);
            }
          }
          reinterpret_cast<T*>(p.out[kv])[(lo + at + t) * width + h * p.D + d] = rr_from<T>(v);
        }
      }
    }
    at += len;
  }
  if (last) {      // what the request does not hold
    const int64_t from = min(max(at, int64_t(0)), int64_t(n)) * width;
    for (int64_t x = from + threadIdx.x; x < int64_t(n) * width; x += RR_THREADS)
      for (int kv = 0; kv < 2; ++kv) reinterpret_cast<T*>(p.out[kv])[int64_t(lo) * width + x] = rr_from<T>(0.f);
  }
}

template <int WF>
static void launch_read(const ReadParams& p, int batch, int dtype, hipStream_t stream) {
  const dim3 grid((p.num_blocks + RR_BLOCKS - 1) / RR_BLOCKS, batch);
  if (dtype == TIERKV_DTYPE_BF16)
    hipLaunchKernelGGL((read_rows_scalar_kernel<WF, __hip_bfloat16>), grid, dim3(RR_THREADS), 0, stream, p);
  else if (dtype == TIERKV_DTYPE_F32)
    hipLaunchKernelGGL((read_rows_scalar_kernel<WF, float>), grid, dim3(RR_THREADS), 0, stream, p);
  else
    hipLaunchKernelGGL((read_rows_scalar_kernel<WF, __half>), grid, dim3(RR_THREADS), 0, stream, p);
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
  if (num_kv_heads <= 0 || num_kv_heads > 65536 || block_size <= 0 || block_size > 64 || head_dim <= 0 || head_dim > 256)
    return fail(TIERKV_ERR_UNSUPPORTED, "1 to 65536 heads, block_size in [1, 64] and head_dim in [1, 256]");
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
  if (warm_format == TIERKV_WARM_ABSMAX_I8) launch_read<TIERKV_WARM_ABSMAX_I8>(p, batch, out_dtype, stream);
  else launch_read<TIERKV_WARM_REF_U8>(p, batch, out_dtype, stream);
  return check_launch("tierkv_read_rows");
}
