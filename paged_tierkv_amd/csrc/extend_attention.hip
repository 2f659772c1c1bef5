// Attention of several query tokens per request over the tiered cache: its C
// entry, launches and workspace.  The kernels are extend_tile.h's.

#include "extend_tile.h"

namespace tierkv {

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

struct ExLayout {
  int64_t arrived, head, seq, subtile, item, cut, part_o, part_ml, total;
  int32_t max_items, max_cut, max_part, part_rows;
  int64_t subs_per_seq;
};

// Tiles of a call are at most those of rows spread over the requests; the
// items are at most the tiles and EX_TARGET / kv_heads more, and as many more
// as the rounding of a request's works can add (one per tile, counted as the
// tiles themselves).  Every cut tile has two items or more.
static ExLayout ex_layout(int64_t batch, int64_t rows, int64_t max_tokens, int64_t groups, int64_t kv_heads,
                          int64_t num_blocks, int64_t bs, int64_t D) {
  ExLayout l{};
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  const int64_t longest = std::min(rows, max_tokens);
  const int64_t per = (longest * groups + EX_WIDE - 1) / EX_WIDE;
  const int64_t tiles = std::max<int64_t>(1, std::min(rows * groups / EX_WIDE + batch, batch * std::max<int64_t>(1, per)));
  const int64_t target = std::max<int64_t>(EX_TARGET / kv_heads, 1);
  l.max_items = int32_t(std::min<int64_t>(tiles + target, 1 << 26));
  l.max_cut = int32_t(std::min(tiles, target));
  l.part_rows = longest * groups <= EX_NARROW ? EX_NARROW : EX_WIDE;
  l.subs_per_seq = num_blocks * ((bs + EX_SUB - 1) / EX_SUB) + EX_PAD;
  const int64_t partials = l.max_cut + target;
  l.max_part = int32_t(partials);
  l.arrived = 128;
  l.head = EX_WS_HEAD;
  l.seq = l.head + 256;
  l.subtile = up(l.seq + batch * 16);
  l.item = up(l.subtile + batch * l.subs_per_seq * 16);
  l.cut = up(l.item + int64_t(l.max_items) * 16);
  l.part_ml = up(l.cut + int64_t(l.max_cut) * 8);
  l.part_o = up(l.part_ml + partials * kv_heads * l.part_rows * 8);
  l.total = up(l.part_o + partials * kv_heads * l.part_rows * D * 4);
  return l;
}

template <int DP, int WF, typename QT>
static void ex_launch(const ExtendParams& p, hipStream_t stream) {
  const int lds = ex_lds_bytes<DP>();
  hipLaunchKernelGGL(extend_plan_kernel<false>, dim3(p.batch), dim3(EX_PLAN), 0, stream, p);
  const dim3 grid(p.max_items * p.kv_heads);
  if (p.part_rows > EX_NARROW) hipLaunchKernelGGL((extend_kernel<DP, WF, QT, true, false>), grid, dim3(EX_THREADS), lds, stream, p);
  else hipLaunchKernelGGL((extend_kernel<DP, WF, QT, false, false>), grid, dim3(EX_THREADS), lds, stream, p);
  const int rows_per_wg = 4 * EX_THREADS / p.D;
  hipLaunchKernelGGL(extend_merge_kernel<QT>,
                     dim3(p.max_cut * p.kv_heads, (p.part_rows + rows_per_wg - 1) / rows_per_wg), dim3(EX_THREADS), 0,
                     stream, p, rows_per_wg);
}

template <int DP, int WF>
static void ex_dispatch_q(const ExtendParams& p, int dtype, hipStream_t stream) {
  if (dtype == TIERKV_DTYPE_BF16) ex_launch<DP, WF, __hip_bfloat16>(p, stream);
  else ex_launch<DP, WF, __half>(p, stream);
}

template <int DP>
static void ex_dispatch(const ExtendParams& p, int wf, int dtype, hipStream_t stream) {
  if (wf == TIERKV_WARM_ABSMAX_I8) ex_dispatch_q<DP, TIERKV_WARM_ABSMAX_I8>(p, dtype, stream);
  else ex_dispatch_q<DP, TIERKV_WARM_REF_U8>(p, dtype, stream);
}

}  // namespace tierkv

using namespace tierkv;

extern "C" int64_t tierkv_extend_workspace_bytes(int32_t batch, int32_t num_rows, int32_t max_tokens, int32_t num_heads,
                                                 int32_t num_kv_heads, int32_t num_blocks, int32_t block_size,
                                                 int32_t head_dim) {
  if (batch <= 0 || num_rows < 0 || max_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads != 0 || num_blocks <= 0 || block_size <= 0 || head_dim <= 0)
    return -1;
  return ex_layout(batch, num_rows, max_tokens, num_heads / num_kv_heads, num_kv_heads, num_blocks, block_size,
                   head_dim).total;
}

extern "C" int32_t tierkv_extend_attention(
    const void* query, int64_t q_stride_t, int64_t q_stride_h, int32_t query_dtype, void* out,
    const int32_t* cu_tokens, int32_t num_rows, int32_t max_tokens,
    const int32_t* block_table, const int32_t* block_states, const int32_t* block_lengths, int64_t table_stride,
    const int32_t* seq_num_blocks, int32_t num_blocks,
    const void* hot_k, const void* hot_v, int64_t hot_slots,
    const void* warm_k, const void* warm_v, int64_t warm_slots,
    const void* k_scale, const void* k_zero, const void* v_scale, const void* v_zero,
    int32_t warm_format, int32_t cold_mode,
    int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t block_size, int32_t head_dim, float scaling,
    void* workspace, int64_t workspace_bytes, void* stream_) {
  clear_error();
  ExtendParams p{};
  const int32_t rc = ex_arguments(
      p, query, q_stride_t, q_stride_h, query_dtype, out, cu_tokens, num_rows, max_tokens, block_table, block_states, block_lengths,
      table_stride, seq_num_blocks, num_blocks, hot_k, hot_v, hot_slots, warm_k, warm_v, warm_slots, k_scale, k_zero, v_scale,
      v_zero, warm_format, cold_mode, batch, num_heads, num_kv_heads, block_size, head_dim, scaling, workspace);
  if (rc != TIERKV_OK) return rc;
  const ExLayout l = ex_layout(batch, num_rows, max_tokens, p.groups, num_kv_heads, num_blocks, block_size, head_dim);
  // (a launch has fewer than 2^32 threads)
  if (int64_t(l.max_items) * num_kv_heads > 0xffffffffll / EX_THREADS) return fail(TIERKV_ERR_UNSUPPORTED, "grid too large");
  if (workspace_bytes < l.total) return fail(TIERKV_ERR_WORKSPACE, "workspace too small");
  if (num_rows == 0 || max_tokens == 0) return TIERKV_OK;
  char* ws = reinterpret_cast<char*>(workspace);
  p.err = reinterpret_cast<int32_t*>(ws);
  p.arrived = reinterpret_cast<uint32_t*>(ws + l.arrived);
  p.head = reinterpret_cast<int32_t*>(ws + l.head);
  p.seq = reinterpret_cast<int4*>(ws + l.seq);
  p.subtile = reinterpret_cast<int4*>(ws + l.subtile);
  p.item = reinterpret_cast<int4*>(ws + l.item);
  p.cut = reinterpret_cast<int2*>(ws + l.cut);
  p.part_o = reinterpret_cast<float*>(ws + l.part_o);
  p.part_ml = reinterpret_cast<float*>(ws + l.part_ml);
  p.max_items = l.max_items;
  p.max_cut = l.max_cut;
  p.max_part = l.max_part;
  p.part_rows = l.part_rows;
  p.subs_per_seq = l.subs_per_seq;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (head_dim <= 64) ex_dispatch<64>(p, warm_format, query_dtype, stream);
  else ex_dispatch<128>(p, warm_format, query_dtype, stream);
  return check_launch("tierkv_extend_attention");
}
