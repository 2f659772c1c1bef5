// Attention of several query tokens per request over the tiered cache: its C
// entry, launches and workspace.  The kernels are extend_tile.h's.

#include "extend_tile.h"

namespace tierkv {

__global__ __launch_bounds__(EX_PLAN) void extend_plan_kernel(ExtendParams p) {
  __shared__ Ex3 sh[EX_PLAN / 64];
  __shared__ int s_last;
  __shared__ int2 s_tile[EX_MAX_BATCH];   // a request's first tile, its sub-tiles
  __shared__ int s_rows[EX_MAX_BATCH];    // its query rows per kv head
  __shared__ float s_work[EX_PLAN / 64];
  const int tid = threadIdx.x, b = blockIdx.x;
  int nb = p.num_blocks;
  if (p.seq_nblocks) nb = min(max(p.seq_nblocks[b], 0), p.num_blocks);
  const int64_t row = int64_t(b) * p.stride;
  int n_all;   // the request's new tokens, of which the first n are computed
  const int n = ex_rows(p, b, &n_all).y;
  int tokens = 0;
  Ex3 total;
  if (p.cold_zero) {   // COLD sub-tiles need the distance to the row's end
    int sum = 0;
    for (int i = tid; i < nb; i += EX_PLAN) sum += min(max(p.lengths[row + i], 0), p.bs);
    ex_scan3({sum, 0, 0}, sh, &total);
    tokens = total.a;
  }
  ExWalk list;
  ex_walk(p, p.table + row, p.states + row, p.lengths + row, nb, tokens - n_all + 1, p.subtile + int64_t(b) * p.subs_per_seq, sh, list);
  if (tid == 0) {
    // Agent-scope stores: the last workgroup may read them from another XCD.
    int32_t* s = reinterpret_cast<int32_t*>(p.seq + b);
    if (n < n_all) atomicOr(p.err, 4);
    const int v[4] = {list.at, list.ordinal - (n_all - n), list.cold, n};
    for (int k = 0; k < 4; ++k) __hip_atomic_store(s + k, v[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    s_last = __hip_atomic_fetch_add(p.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u == gridDim.x;
  }
  __syncthreads();
  if (!s_last) return;
  if (tid == 0) __hip_atomic_store(p.arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // The requests' tiles and an upper bound of the sum of the tiles' works:
  // each is at most g(t) = max(f(t), 1) with f linear, g is convex, and a
  // convex sum lies below its chord's.
  const int G = p.groups;
  float work = 0.f;
  int tiles_all = 0;
  for (int i0 = 0; i0 < p.batch; i0 += EX_PLAN) {
    const int i = i0 + tid;
    int rows = 0, subs = 0;
    if (i < p.batch) {
      int32_t* s = reinterpret_cast<int32_t*>(p.seq + i);
      subs = __hip_atomic_load(s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      rows = __hip_atomic_load(s + 3, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) * G;
    }
    const int tiles = ex_tiles(rows);
    const bool wide = rows > EX_NARROW;
    if (tiles > 0) {
      auto g = [&](int t) {
        const float last = wide ? float(t + 1) * EX_WIDE : float(rows);
        return fmaxf(float(subs) + 1.f - fmaxf((float(rows) - last) / float(G) - 1.f, 0.f) / EX_SUB, 1.f);
      };
      work += 0.5f * (g(0) + g(tiles - 1)) * float(tiles);
    }
    const Ex3 s = ex_scan3({tiles, 0, 0}, sh, &total);
    if (i < p.batch) {
      s_tile[i] = make_int2(tiles_all + s.a - tiles, subs);
      s_rows[i] = rows;
    }
    tiles_all += total.a;
  }
  work = wave_sum(work);
  if ((tid & 63) == 0) s_work[tid >> 6] = work;
  __syncthreads();
  work = 0.f;
  for (int i = 0; i < EX_PLAN / 64; ++i) work += s_work[i];
  work = work * 1.001f + 1.f;   // the rounding of these sums
  // Sub-tiles per item: each wave rates one choice.  P = longest / (w + 1) for
  // the first eight waves, a few sizes around an even share for the others;
  // with the items' count and the longest of them the time is the rounds over
  // the slots, or the even share and a quarter of an item where the items are
  // of mixed lengths and fill each other's gaps, and the cost of the partials.
  // Measured with the whole call: 2048 tokens on 32768, 32 tiles on as many
  // slots, are left whole, 973 us against 1221 cut in two (the tiles of a head
  // then also walk the same keys at the same time, in one L2); a single token
  // on 100000 in 32 parts 85 us, in 64 99; a cost of 24 per partial leaves 512
  // tokens beside 15 single ones whole, 98 us against 78 cut in four.
  __shared__ float s_time[EX_PLAN / 64];
  __shared__ int s_per[EX_PLAN / 64];
  const float slots = fmaxf(float(EX_SLOTS / p.kv_heads), 1.f);
  const int least = max(EX_MIN_SUBS, int(ceilf(work / fmaxf(float(EX_TARGET / p.kv_heads), 1.f))));
  {
    const int w = tid >> 6, lane = tid & 63;
    auto tile_work = [&](int f) {
      const ExTileId x = ex_tile_id(p.batch, f, s_tile, s_rows);
      return ex_work(s_tile[x.request].y, s_rows[x.request], x.tile, x.wide, G);
    };
    float longest = 0.f;
    for (int i = lane; i < p.batch; i += 64)
      if (s_rows[i] > 0) longest = fmaxf(longest, float(s_tile[i].y));
    longest = wave_max(longest);
    const float share = work / slots;
    const float f = w == 8 ? 0.34f : w == 9 ? 0.51f : w == 10 ? 0.68f : w == 11 ? 0.8f : w == 12 ? 1.02f
                  : w == 13 ? 1.25f : w == 14 ? 1.5f : 2.f;
    const int per = max(least, int(ceilf(w < 8 ? longest / float(w + 1) : share * f)));
    float items = 0.f, partials = 0.f, len = 0.f;
    for (int i = lane; i < tiles_all; i += 64) {
      const int v = tile_work(i), k = ex_parts(v, per);
      items += float(k);
      if (k > 1) partials += float(k);
      len = fmaxf(len, float(v) / float(k));
    }
    items = wave_sum(items);
    partials = wave_sum(partials);
    len = wave_max(len) + EX_ITEM_COST;
    const float even = (work + EX_ITEM_COST * items) / slots;
    const float time = fmaxf(len, fminf(ceilf(items / slots) * len, even + 0.25f * len)) + EX_PART_COST * partials / slots;
    if (lane == 0) {
      s_time[w] = time;
      s_per[w] = per;
    }
  }
  __syncthreads();
  int per_item = s_per[0];
  {
    float best = s_time[0];
    for (int i = 1; i < EX_PLAN / 64; ++i)
      if (s_time[i] < best) {
        best = s_time[i];
        per_item = s_per[i];
      }
  }
  // Items, tile by tile; each request's longest tiles first.
  int items = 0, cuts = 0, partials = 0;
  for (int f0 = 0; f0 < tiles_all; f0 += EX_PLAN) {
    const int f = f0 + tid;
    int i = 0, t = 0, parts = 0;
    bool wide = false;
    if (f < tiles_all) {
      const ExTileId x = ex_tile_id(p.batch, f, s_tile, s_rows);
      i = x.request;
      t = x.tile;
      wide = x.wide;
      parts = ex_parts(ex_work(s_tile[i].y, s_rows[i], t, wide, G), per_item);
    }
    const int cut = parts > 1 ? 1 : 0;
    const Ex3 s = ex_scan3({parts, cut, cut ? parts : 0}, sh, &total);
    const int at_item = items + s.a - parts, at_cut = cuts + s.b - cut, at_part = partials + s.c - (cut ? parts : 0);
    items += total.a;
    cuts += total.b;
    partials += total.c;
    if (parts > 0) {
      // The host's bounds hold for packed ranges that do not overlap; items of others may be left out (-1).
      const bool fits = at_item + parts <= p.max_items && (!cut || (at_cut < p.max_cut && at_part + parts <= p.max_part));
      if (!fits) atomicOr(p.err, 4);
      for (int k = 0; k < parts; ++k)
        if (at_item + k < p.max_items)
          p.item[at_item + k] = make_int4(fits ? i : -1, t | (wide ? 1 << 30 : 0), k | (parts << 16), cut ? at_part + k : -1);
      if (cut && at_cut < p.max_cut) p.cut[at_cut] = make_int2(at_part, fits ? at_item : -1);
    }
  }
  if (tid == 0) {
    p.head[0] = min(items, p.max_items);
    p.head[1] = min(cuts, p.max_cut);
  }
}

// An item of the plan.
template <int DP, int WF, typename QT, bool WIDE>
__device__ __forceinline__ void ex_item(const ExtendParams& p, char* lds, int h, const ex_int4 it) {
  const int b = it.x, q0 = ex_rows(p, b).x;
  const ExWorkspaceList list = {p.subtile + int64_t(b) * p.subs_per_seq};
  ex_tile_part<DP, WF, QT, WIDE, false, WIDE ? 1 : EX_WAVES>(p, lds, h, it.y & 0x3fffffff, it.z & 0xffff, it.z >> 16, p.seq[b],
                                                             list, [&](int t) { return q0 + t; }, it.w);
}

// MIXED: calls that may hold wide tiles; the others' kernel is without their code.
template <int DP, int WF, typename QT, bool MIXED>
__global__ __launch_bounds__(EX_THREADS, 2) void extend_kernel(ExtendParams p) {
  extern __shared__ __attribute__((aligned(16))) char ex_lds[];
  const int i = int(blockIdx.x) / p.kv_heads, h = int(blockIdx.x) - i * p.kv_heads;
  if (i >= p.head[0]) return;
  const ex_int4 it = ((ExList)(uintptr_t)p.item)[i];
  if (it.x < 0) return;
  if (MIXED && (it.y & (1 << 30))) ex_item<DP, WF, QT, true>(p, ex_lds, h, it);
  else ex_item<DP, WF, QT, false>(p, ex_lds, h, it);
}

// Join of a cut tile's partials, in part order: a workgroup per (cut tile, kv
// head, 4 EX_THREADS / D of its rows), four dims of one row per thread.
template <typename QT>
__global__ __launch_bounds__(EX_THREADS) void extend_merge_kernel(ExtendParams p, int32_t rows_per_wg) {
  const int c = int(blockIdx.x) / p.kv_heads, h = int(blockIdx.x) - c * p.kv_heads;
  if (c >= p.head[1]) return;
  const int2 cut = p.cut[c];
  if (cut.y < 0) return;
  const int4 it = p.item[cut.y];
  const int b = it.x, tile = it.y & 0x3fffffff, parts = it.z >> 16;
  const int G = p.groups, D = p.D, rows = p.seq[b].w * G;
  const int D4 = D / 4;
  const int rr = int(blockIdx.y) * rows_per_wg + int(threadIdx.x) / D4, d = 4 * (int(threadIdx.x) % D4);
  const int row = tile * EX_WIDE + rr;
  if (int(threadIdx.x) >= rows_per_wg * D4 || rr >= p.part_rows || row >= rows) return;
  constexpr int AHEAD = 8;   // partials loaded together
  const int64_t step = int64_t(p.kv_heads) * p.part_rows;
  const int64_t at = (int64_t(cut.x) * p.kv_heads + h) * p.part_rows + rr;
  ExJoin j;
  for (int k0 = 0; k0 < parts; k0 += AHEAD) j.take<AHEAD>(p, parts - k0, d, [&](int k) { return at + (k0 + k) * step; });
  const int tk = row / G;
  j.put<QT>(p, ex_rows(p, b).x + tk, h * G + row - tk * G, d);
}

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
  hipLaunchKernelGGL(extend_plan_kernel, dim3(p.batch), dim3(EX_PLAN), 0, stream, p);
  const dim3 grid(p.max_items * p.kv_heads);
  if (p.part_rows > EX_NARROW) hipLaunchKernelGGL((extend_kernel<DP, WF, QT, true>), grid, dim3(EX_THREADS), lds, stream, p);
  else hipLaunchKernelGGL((extend_kernel<DP, WF, QT, false>), grid, dim3(EX_THREADS), lds, stream, p);
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
