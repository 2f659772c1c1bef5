// Attention for requests that share long prefixes: a prefix's keys and values
// are read once for the rows of all its requests together.
//
// Row i of request b sees every token of its prefix, then its own as in
// extend attention (extend_tile.h, whose kernels these calls run):
//   o = sum_t p_t v_t,  p = softmax over both;
// with m, l and o of the two parts (running maximum, sum, unscaled output)
//   m = max(m_1, m_2),  o = (o_1 2^(m_1 - m) + o_2 2^(m_2 - m)) / (l_1 2^(m_1 - m) + l_2 2^(m_2 - m)),
// which is how parts of a cut tile are joined too.
//
// The prefixes are segments of the plan beside the requests: their rows are
// the packed rows of their requests, taken through a list, and none of their
// tokens is hidden.  A decode step of 64 requests with 4 heads per kv head is
// one tile of 256 rows per prefix and kv head, cut along the prefix.

#include "extend_tile.h"

namespace tierkv {

struct PrefixLayout {
  int64_t arrived, head, seq, seg, tile, row_list, row_home, subtile, item, part_o, part_ml, total;
  int64_t subs, pre_subs, tiles, items, units;
  bool wide;
};

// Tiles and items as ex_layout counts them, for the requests' rows and once
// more for the prefixes'.  Partials in units of 32 rows: a part of every tile
// and those that cutting adds, eight units each where tiles are wide.
static PrefixLayout prefix_layout(int64_t batch, int64_t prefixes, int64_t rows, int64_t max_tokens, int64_t groups,
                                  int64_t kv_heads, int64_t num_blocks, int64_t pre_blocks, int64_t bs, int64_t D) {
  PrefixLayout l{};
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  const int64_t all = rows * groups, each = EX_WIDE / EX_UNIT;
  const int64_t target = std::max<int64_t>(EX_TARGET / kv_heads, 1);
  l.wide = all > EX_NARROW;
  auto units = [&](int64_t segments, int64_t longest) {
    return longest <= EX_NARROW ? segments : segments + all / EX_UNIT + each * std::min(segments, all / EX_NARROW);
  };
  l.tiles = 2 * (all / EX_WIDE) + batch + prefixes;
  l.items = l.tiles + target;
  l.units = units(batch, std::min(rows, max_tokens) * groups) + units(prefixes, all) + target * (l.wide ? each : 1);
  l.subs = num_blocks * ((bs + EX_SUB - 1) / EX_SUB) + EX_PAD;
  l.pre_subs = pre_blocks * ((bs + EX_SUB - 1) / EX_SUB) + EX_PAD;
  l.arrived = 128;
  l.head = EX_WS_HEAD;
  l.seq = l.head + 256;
  l.seg = up(l.seq + (batch + prefixes) * 16);
  l.tile = up(l.seg + (batch + prefixes) * 8);
  l.row_list = up(l.tile + l.tiles * 8);
  l.row_home = up(l.row_list + rows * 4);
  l.subtile = up(l.row_home + rows * 8);
  l.item = up(l.subtile + (batch * l.subs + prefixes * l.pre_subs) * 16);
  l.part_ml = up(l.item + l.items * 16);
  l.part_o = up(l.part_ml + l.units * kv_heads * EX_UNIT * 8);
  l.total = up(l.part_o + l.units * kv_heads * EX_UNIT * D * 4);
  return l;
}

template <int DP, int WF, typename QT>
static void prefix_launch(const ExtendParams& p, bool wide, hipStream_t stream) {
  const int lds = ex_lds_bytes<DP>();
  hipLaunchKernelGGL(extend_plan_kernel<true>, dim3(p.batch + p.prefixes), dim3(EX_PLAN), 0, stream, p);
  const dim3 grid(p.max_items * p.kv_heads);
  if (wide) hipLaunchKernelGGL((extend_kernel<DP, WF, QT, true, true>), grid, dim3(EX_THREADS), lds, stream, p);
  else hipLaunchKernelGGL((extend_kernel<DP, WF, QT, false, true>), grid, dim3(EX_THREADS), lds, stream, p);
  const int64_t threads = int64_t(p.rows) * p.heads * (p.D / 4);
  hipLaunchKernelGGL(extend_join_kernel<QT>, dim3(uint32_t((threads + EX_THREADS - 1) / EX_THREADS)), dim3(EX_THREADS), 0,
                     stream, p);
}

template <int DP>
static void prefix_dispatch(const ExtendParams& p, bool wide, int wf, int dtype, hipStream_t stream) {
  const bool bf = dtype == TIERKV_DTYPE_BF16, i8 = wf == TIERKV_WARM_ABSMAX_I8;
  if (bf && i8) prefix_launch<DP, TIERKV_WARM_ABSMAX_I8, __hip_bfloat16>(p, wide, stream);
  else if (bf) prefix_launch<DP, TIERKV_WARM_REF_U8, __hip_bfloat16>(p, wide, stream);
  else if (i8) prefix_launch<DP, TIERKV_WARM_ABSMAX_I8, __half>(p, wide, stream);
  else prefix_launch<DP, TIERKV_WARM_REF_U8, __half>(p, wide, stream);
}

}  // namespace tierkv

using namespace tierkv;

extern "C" int64_t tierkv_prefix_workspace_bytes(int32_t batch, int32_t num_prefixes, int32_t num_rows,
                                                 int32_t max_tokens, int32_t num_heads, int32_t num_kv_heads,
                                                 int32_t num_blocks, int32_t num_prefix_blocks, int32_t block_size,
                                                 int32_t head_dim) {
  if (batch <= 0 || num_prefixes <= 0 || num_rows < 0 || max_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads != 0 || num_blocks <= 0 || num_prefix_blocks <= 0 || block_size <= 0 || head_dim <= 0)
    return -1;
  return prefix_layout(batch, num_prefixes, num_rows, max_tokens, num_heads / num_kv_heads, num_kv_heads, num_blocks,
                       num_prefix_blocks, block_size, head_dim).total;
}

extern "C" int32_t tierkv_prefix_attention(
    const void* query, int64_t q_stride_t, int64_t q_stride_h, int32_t query_dtype, void* out,
    const int32_t* cu_tokens, int32_t num_rows, int32_t max_tokens,
    const int32_t* block_table, const int32_t* block_states, const int32_t* block_lengths, int64_t table_stride,
    const int32_t* seq_num_blocks, int32_t num_blocks,
    const int32_t* prefix_of, const int32_t* prefix_table, const int32_t* prefix_states, const int32_t* prefix_lengths,
    int64_t prefix_stride, const int32_t* prefix_num_blocks, int32_t num_prefix_blocks, int32_t num_prefixes,
    const void* hot_k, const void* hot_v, int64_t hot_slots,
    const void* warm_k, const void* warm_v, int64_t warm_slots,
    const void* k_scale, const void* k_zero, const void* v_scale, const void* v_zero,
    int32_t warm_format, int32_t cold_mode,
    int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t block_size, int32_t head_dim, float scaling,
    void* workspace, int64_t workspace_bytes, void* stream_) {
  clear_error();
  ExtendParams p{};
  const int32_t rc = ex_arguments(
      p, query, q_stride_t, q_stride_h, query_dtype, out, cu_tokens, num_rows, max_tokens, block_table, block_states,
      block_lengths, table_stride, seq_num_blocks, num_blocks, hot_k, hot_v, hot_slots, warm_k, warm_v, warm_slots, k_scale,
      k_zero, v_scale, v_zero, warm_format, cold_mode, batch, num_heads, num_kv_heads, block_size, head_dim, scaling, workspace);
  if (rc != TIERKV_OK) return rc;
  if (!prefix_of || !prefix_table || !prefix_states || !prefix_lengths)
    return fail(TIERKV_ERR_INVALID, "null prefix tables");
  if (num_prefixes <= 0 || num_prefix_blocks <= 0 || num_prefix_blocks > prefix_stride)
    return fail(TIERKV_ERR_INVALID, "num_prefixes must be positive and num_prefix_blocks within the prefix tables");
  if (int64_t(batch) + num_prefixes > EX_MAX_BATCH)
    return fail(TIERKV_ERR_UNSUPPORTED, "more than 4096 requests and prefixes");
  if (int64_t(num_prefix_blocks) * block_size + num_rows > 0x7fffffff - EX_SUB)
    return fail(TIERKV_ERR_UNSUPPORTED, "prefixes of 2^31 tokens or more");
  const PrefixLayout l = prefix_layout(batch, num_prefixes, num_rows, max_tokens, p.groups, num_kv_heads, num_blocks,
                                       num_prefix_blocks, block_size, head_dim);
  // (a launch has fewer than 2^32 threads)
  if (l.items * num_kv_heads > 0xffffffffll / EX_THREADS ||
      int64_t(num_rows) * num_heads > (0xffffffffll - EX_THREADS) / (head_dim / 4) || l.units > 0x7fffffff)
    return fail(TIERKV_ERR_UNSUPPORTED, "grid too large");
  if (workspace_bytes < l.total) return fail(TIERKV_ERR_WORKSPACE, "workspace too small");
  if (num_rows == 0 || max_tokens == 0) return TIERKV_OK;
  char* ws = reinterpret_cast<char*>(workspace);
  p.err = reinterpret_cast<int32_t*>(ws);
  p.arrived = reinterpret_cast<uint32_t*>(ws + l.arrived);
  p.head = reinterpret_cast<int32_t*>(ws + l.head);
  p.seq = reinterpret_cast<int4*>(ws + l.seq);
  p.seg = reinterpret_cast<int2*>(ws + l.seg);
  p.tile = reinterpret_cast<int2*>(ws + l.tile);
  p.row_list = reinterpret_cast<int32_t*>(ws + l.row_list);
  p.row_home = reinterpret_cast<int2*>(ws + l.row_home);
  p.subtile = reinterpret_cast<int4*>(ws + l.subtile);
  p.item = reinterpret_cast<int4*>(ws + l.item);
  p.part_o = reinterpret_cast<float*>(ws + l.part_o);
  p.part_ml = reinterpret_cast<float*>(ws + l.part_ml);
  p.max_items = int32_t(l.items);
  p.max_tiles = int32_t(l.tiles);
  p.max_part = int32_t(l.units);
  p.subs_per_seq = l.subs;
  p.pre_subs = l.pre_subs;
  p.prefix_of = prefix_of;
  p.pre_table = prefix_table;
  p.pre_states = prefix_states;
  p.pre_lengths = prefix_lengths;
  p.pre_stride = prefix_stride;
  p.pre_nblocks = prefix_num_blocks;
  p.pre_blocks = num_prefix_blocks;
  p.prefixes = num_prefixes;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (head_dim <= 64) prefix_dispatch<64>(p, l.wide, warm_format, query_dtype, stream);
  else prefix_dispatch<128>(p, l.wide, warm_format, query_dtype, stream);
  return check_launch("tierkv_prefix_attention");
}
