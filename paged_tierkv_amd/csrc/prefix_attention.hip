// Attention for requests that share long prefixes: a prefix's keys and values
// are read once for the rows of all its requests together.
//
// Row i of request b sees every token of its prefix, then its own as in
// extend attention (extend_tile.h, whose items these calls run):
//   o = sum_t p_t v_t,  p = softmax over both;
// with m, l and o of the two parts (running maximum, sum, unscaled output)
//   m = max(m_1, m_2),  o = (o_1 2^(m_1 - m) + o_2 2^(m_2 - m)) / (l_1 2^(m_1 - m) + l_2 2^(m_2 - m)),
// which is how parts of a cut tile are joined too.
//
// The prefixes are segments of the plan beside the requests: their rows are
// the packed rows of their requests, taken through a list, and none of their
// tokens is hidden.  A decode step of 64 requests with 4 heads per kv head is
// one tile of 256 rows per prefix and kv head, cut along the prefix.  A request
// that fills tiles of its own ("lone", PX_LONE rows and more) gains nothing from
// sharing: its tiles walk the prefix and then its own tokens, as if its table
// held both, and have no parts to join.
//
// Three launches:
//   * prefix_plan_kernel, a workgroup per segment, lists its sub-tiles and
//     enters its rows; the last to finish cuts the segments' tiles into items;
//   * prefix_kernel, up to one workgroup per CU, which take items until none is
//     left: wide ones (256 rows, eight waves together) first, then narrow ones
//     (up to 32 rows), four side by side with two waves each.  Single tokens on
//     short contexts are most of a decode step's items, and each is a chain
//     of reads; one at a time per workgroup took three times as long;
//   * prefix_join_kernel adds up the parts of rows that have several.

#include "extend_tile.h"

namespace tierkv {

#ifndef PX_LONE_
#define PX_LONE_ 512
#endif
#ifndef PX_KW_
#define PX_KW_ 2
#endif
constexpr int PX_LONE = PX_LONE_;       // rows (tokens times heads of a kv head) from which a request walks its prefix itself
constexpr int PX_KW = PX_KW_;           // waves of a narrow item
constexpr int PX_SIDE = EX_WAVES / PX_KW;   // narrow items side by side
constexpr int PX_MIN_NARROW = 8;        // sub-tiles of a narrow item, at least, when a tile is cut
constexpr float PX_NARROW_COST = 0.5f;  // a narrow item's sub-tile, in wide sub-tiles' time

// A request's prefix, -1 for none (also for a number that no prefix has).
__device__ __forceinline__ int px_prefix(const ExtendParams& p, int b) {
  const int g = p.prefix_of[b];
  return g >= 0 && g < p.prefixes ? g : -1;
}

__device__ __forceinline__ bool px_lone(const ExtendParams& p, int b) {
  return px_prefix(p, b) >= 0 && ex_rows(p, b).y * p.groups >= PX_LONE;
}

__global__ __launch_bounds__(EX_PLAN) void prefix_plan_kernel(ExtendParams p) {
  __shared__ Ex3 sh[EX_PLAN / 64];
  __shared__ int s_last;
  __shared__ int2 s_tile[EX_MAX_BATCH];   // a segment's first tile, its sub-tiles
  __shared__ int s_rows[EX_MAX_BATCH];    // its query rows per kv head
  __shared__ float s_sum[3][EX_PLAN / 64];
  const int tid = threadIdx.x, seg = blockIdx.x, segments = p.prefixes + p.batch;
  const bool pre = seg < p.prefixes;
  const int b = seg - p.prefixes, G = p.groups;
  const int g = pre ? seg : px_prefix(p, b);
  const bool lone = !pre && px_lone(p, b);
  Ex3 total;
  // Rows of prefixes before this one, of its requests before this, and of all
  // its requests; of a lone request, the lone ones before it.
  Ex3 sum = {0, 0, 0};
  if (g >= 0) {
    for (int i = tid; i < p.batch; i += EX_PLAN) {
      const int k = px_prefix(p, i), rows = ex_rows(p, i).y;
      const bool other = k >= 0 && rows * G >= PX_LONE;
      if (lone) {
        if (other && i < b) ++sum.a;
      } else if (!other) {
        if (k >= 0 && k < g) sum.a += rows;
        if (k == g && !pre && i < b) sum.b += rows;
        if (k == g) sum.c += rows;
      }
    }
  }
  ex_scan3(sum, sh, &total);
  int n, n_all, where = 0;
  bool fits = true;
  if (pre) {
    // (packed ranges that overlap have more rows than there are)
    where = min(total.a, p.rows);
    n = n_all = min(total.c, p.rows - where);
    fits = n == total.c;
  } else {
    const int2 r = ex_rows(p, b, &n_all);
    n = r.y;
    const int place = min(total.a, p.rows), end = min(n_all, p.rows - r.x);
    if (lone) {
      where = ~total.a;
      if (total.a >= p.max_lone) {   // (the same)
        fits = false;
        n = 0;
      }
    }
    for (int i = tid; i < end; i += EX_PLAN) {
      const int mine = g >= 0 && !lone ? total.b + i : -1;
      const bool in = i < n && mine < p.rows - place;
      if (in && mine >= 0) p.row_list[place + mine] = r.x + i;
      p.row_home[r.x + i] = make_int4(in ? b : -1, i, mine >= 0 ? g : -1, mine);
    }
  }
  // The segment's sub-tiles: a lone request's are its prefix's and its own.
  ExWalk list;
  const int own_blocks = pre ? 0 : (p.seq_nblocks ? min(max(p.seq_nblocks[b], 0), p.num_blocks) : p.num_blocks);
  const int pre_blocks = pre || lone ? (p.pre_nblocks ? min(max(p.pre_nblocks[g], 0), p.pre_blocks) : p.pre_blocks) : 0;
  const int64_t pre_row = g * p.pre_stride, row = b * p.stride;
  int tokens = 0;
  if (p.cold_zero && !pre) {   // COLD sub-tiles need the distance to the row's end
    int held = 0;
    for (int i = tid; i < own_blocks; i += EX_PLAN) held += min(max(p.lengths[row + i], 0), p.bs);
    for (int i = tid; i < pre_blocks; i += EX_PLAN) held += min(max(p.pre_lengths[pre_row + i], 0), p.bs);
    ex_scan3({held, 0, 0}, sh, &total);
    tokens = total.a;
  }
  const int all_see = pre ? 0x7fffffff : tokens - n_all + 1;
  int4* const out = p.subtile + (pre ? seg * p.pre_subs : ex_list_of(p, b, fits ? where : 0));
  if (pre_blocks && fits) ex_walk(p, p.pre_table + pre_row, p.pre_states + pre_row, p.pre_lengths + pre_row, pre_blocks, all_see, out, sh, list);
  if (own_blocks && fits) ex_walk(p, p.table + row, p.states + row, p.lengths + row, own_blocks, all_see, out, sh, list);
  if (tid == 0) {
    // Agent-scope stores: the last workgroup may read them from another XCD.
    int32_t* s = reinterpret_cast<int32_t*>(p.seq + seg);
    if (n < n_all || !fits) atomicOr(p.err, 4);
    // (every row of a prefix's sees all of it: a limit past its tokens)
    const int v[4] = {list.at, pre ? list.ordinal + n : list.ordinal - (n_all - n), list.cold, n};
    for (int k = 0; k < 4; ++k) __hip_atomic_store(s + k, v[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    p.seg[seg].y = where;
    __builtin_amdgcn_s_waitcnt(0);
    s_last = __hip_atomic_fetch_add(p.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u == gridDim.x;
  }
  __syncthreads();
  if (!s_last) return;
  if (tid == 0) __hip_atomic_store(p.arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // The segments' tiles, an upper bound of the sum of the wide ones' works
  // (extend_plan_kernel's), the narrow ones' sub-tiles and the longest of each.
  float wide_work = 0.f, narrow_work = 0.f, wide_longest = 0.f;
  int tiles_all = 0;
  for (int i0 = 0; i0 < segments; i0 += EX_PLAN) {
    const int i = i0 + tid;
    int rows = 0, subs = 0;
    if (i < segments) {
      int32_t* s = reinterpret_cast<int32_t*>(p.seq + i);
      subs = __hip_atomic_load(s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      rows = __hip_atomic_load(s + 3, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) * G;
    }
    const int tiles = ex_tiles(rows);
    if (rows > EX_NARROW) {
      auto work = [&](int t) {
        if (i < p.prefixes) return float(subs) + 1.f;
        return fmaxf(float(subs) + 1.f - fmaxf((float(rows) - float(t + 1) * EX_WIDE) / float(G) - 1.f, 0.f) / EX_SUB, 1.f);
      };
      wide_work += 0.5f * (work(0) + work(tiles - 1)) * float(tiles);
      wide_longest = fmaxf(wide_longest, float(subs));
    } else if (tiles) {
      narrow_work += float(max(subs, 1));
    }
    const Ex3 s = ex_scan3({tiles, 0, 0}, sh, &total);
    if (i < segments) {
      s_tile[i] = make_int2(tiles_all + s.a - tiles, subs);
      s_rows[i] = rows;
      p.seg[i].x = s_tile[i].x;
    }
    tiles_all += total.a;
  }
  {
    const float a = wave_sum(wide_work), c = wave_sum(narrow_work), d = wave_max(wide_longest);
    if ((tid & 63) == 0) {
      s_sum[0][tid >> 6] = a;
      s_sum[1][tid >> 6] = c;
      s_sum[2][tid >> 6] = d;
    }
  }
  __syncthreads();
  wide_work = narrow_work = wide_longest = 0.f;
  for (int i = 0; i < EX_PLAN / 64; ++i) {
    wide_work += s_sum[0][i];
    narrow_work += s_sum[1][i];
    wide_longest = fmaxf(wide_longest, s_sum[2][i]);
  }
  wide_work = wide_work * 1.001f + 1.f;   // the rounding of these sums
  narrow_work = narrow_work * 1.001f + 1.f;
  // Narrow items: no longer than an even share of the chip's places for them.
  const float slots = fmaxf(float(EX_SLOTS) / float(p.kv_heads), 1.f);
  const int per_narrow = max(PX_MIN_NARROW, int(ceilf(narrow_work / (slots * PX_SIDE))));
  auto tile_work = [&](const ExTileId& x) {
    const int subs = s_tile[x.request].y;
    return x.request < p.prefixes ? max(subs, 1) : ex_work(subs, s_rows[x.request], x.tile, x.wide, G);
  };
  // Sub-tiles per wide item: each wave rates one choice, as extend attention's
  // plan does; the narrow items fill what the wide ones leave.
  __shared__ float s_time[EX_PLAN / 64];
  __shared__ int s_per[EX_PLAN / 64];
  const int least = max(EX_MIN_SUBS, int(ceilf(wide_work / fmaxf(float(EX_TARGET / p.kv_heads), 1.f))));
  {
    const int w = tid >> 6, lane = tid & 63;
    const float share = wide_work / slots;
    const float f = w == 8 ? 0.34f : w == 9 ? 0.51f : w == 10 ? 0.68f : w == 11 ? 0.8f : w == 12 ? 1.02f
                  : w == 13 ? 1.25f : w == 14 ? 1.5f : 2.f;
    const int per = max(least, int(ceilf(w < 8 ? wide_longest / float(w + 1) : share * f)));
    float items = 0.f, narrow = 0.f, len = 0.f;
    for (int i = lane; i < tiles_all; i += 64) {
      const ExTileId x = ex_tile_id(segments, i, s_tile, s_rows);
      const int v = tile_work(x), k = ex_parts(v, x.wide ? per : per_narrow);
      if (x.wide) {
        items += float(k);
        len = fmaxf(len, float(v) / float(k));
      } else {
        narrow += float(k) * EX_ITEM_COST + PX_NARROW_COST * float(v);
      }
    }
    items = wave_sum(items);
    narrow = wave_sum(narrow) / PX_SIDE;
    len = wave_max(len) + EX_ITEM_COST;
    const float even = (wide_work + EX_ITEM_COST * items + narrow) / slots;
    const float time = fmaxf(len, fminf(ceilf(items / slots) * len + narrow / slots, even + 0.25f * len)) + EX_PART_COST * items / slots;
    if (lane == 0) {
      s_time[w] = time;
      s_per[w] = per;
    }
  }
  __syncthreads();
  int per_wide = s_per[0];
  {
    float best = s_time[0];
    for (int i = 1; i < EX_PLAN / 64; ++i)
      if (s_time[i] < best) {
        best = s_time[i];
        per_wide = s_per[i];
      }
  }
  // Items, tile by tile: wide ones from the front, narrow ones from the back.
  int wide_items = 0, narrow_items = 0, units = 0;
  for (int f0 = 0; f0 < tiles_all; f0 += EX_PLAN) {
    const int f = f0 + tid;
    ExTileId x = {0, 0, false};
    int parts = 0;
    if (f < tiles_all) {
      x = ex_tile_id(segments, f, s_tile, s_rows);
      parts = ex_parts(tile_work(x), x.wide ? per_wide : per_narrow);
    }
    // Rows that also have a prefix's part keep partials in any case.
    const int rb = x.request - p.prefixes;
    const bool joined = parts > 0 && (rb < 0 || (px_prefix(p, rb) >= 0 && s_rows[x.request] < PX_LONE));
    const bool kept = joined || parts > 1;
    const int each = x.wide ? EX_WIDE / EX_UNIT : 1;   // of a part
    const Ex3 s = ex_scan3({x.wide ? parts : 0, x.wide ? 0 : parts, kept ? parts * each : 0}, sh, &total);
    const int at = x.wide ? wide_items + s.a - parts : narrow_items + s.b - parts;
    const int unit = units + s.c - (kept ? parts * each : 0);
    wide_items += total.a;
    narrow_items += total.b;
    units += total.c;
    if (parts > 0) {
      // The host's bounds hold for packed ranges that do not overlap; items of others may be left out (-1).
      const int room = x.wide ? p.max_cut : p.max_items - p.max_cut;
      const bool ok = at + parts <= room && f < p.max_tiles && (!kept || unit + parts * each <= p.max_part);
      if (!ok) atomicOr(p.err, 4);
      for (int k = 0; k < parts; ++k)
        if (at + k < room)
          p.item[x.wide ? at + k : p.max_items - 1 - (at + k)] =
              make_int4(ok ? x.request : -1, x.tile, k | (parts << 16), kept ? unit + k * each : -1);
      if (f < p.max_tiles) p.tile[f] = make_int2(kept ? unit : -1, ok ? parts : 0);
    }
  }
  if (tid == 0) {
    p.head[0] = min(wide_items, p.max_cut);
    p.head[1] = min(narrow_items, p.max_items - p.max_cut);
    p.head[2] = 0;
  }
}

// Workgroups take wide items one by one, then narrow ones PX_SIDE at a time,
// until none is left: the first by their number, the others from a counter.
template <int DP, int WF, typename QT, bool MIXED>
__global__ __launch_bounds__(EX_THREADS, 2) void prefix_kernel(ExtendParams p) {
  extern __shared__ __attribute__((aligned(16))) char px_lds[];
  __shared__ int s_next;
  const int wide = p.head[0] * p.kv_heads, narrow = p.head[1] * p.kv_heads;
  const int all = wide + (narrow + PX_SIDE - 1) / PX_SIDE;
  int j = blockIdx.x;
  while (j < all) {
    int next = 0;
    if (threadIdx.x == 0) next = atomicAdd(p.head + 2, 1) + int(gridDim.x);
    if (MIXED && j < wide) {
      const int i = j / p.kv_heads, h = j - i * p.kv_heads;
      const ex_int4 it = ((ExList)(uintptr_t)p.item)[i];
      if (it.x >= 0) ex_item<DP, WF, QT, true, true, 1>(p, px_lds, h, it, it.w);
    } else {
      const int u = (j - wide) * PX_SIDE + ex_uniform(threadIdx.x >> 6) / PX_KW;
      const int x = min(u, narrow - 1), i = x / p.kv_heads, h = x - i * p.kv_heads;
      ex_int4 it = ((ExList)(uintptr_t)p.item)[p.max_items - 1 - i];
      const bool dead = u >= narrow || it.x < 0;
      if (it.x < 0) it.x = 0;
      ex_item<DP, WF, QT, false, true, PX_KW>(p, px_lds, h, it, it.w, dead);
    }
    if (threadIdx.x == 0) s_next = next;
    __syncthreads();
    j = ex_uniform(s_next);
    __syncthreads();
  }
}

// Four dims of one packed row and head per thread: the request's own partials,
// then those of its prefix.
template <typename QT>
__global__ __launch_bounds__(EX_THREADS) void prefix_join_kernel(ExtendParams p) {
  const int D4 = p.D / 4, G = p.groups;
  const int64_t x = int64_t(blockIdx.x) * EX_THREADS + threadIdx.x;
  const int64_t rh = x / D4;
  const int d = 4 * int(x - rh * D4);
  const int64_t r = rh / p.heads;
  if (r >= p.rows) return;
  const int hd = int(rh - r * p.heads), h = hd / G;
  const int4 home = p.row_home[r];
  // (a row of no request has whatever the workspace held)
  if (home.x < 0 || home.x >= p.batch || home.z >= p.prefixes) return;
  const int s = p.prefixes + home.x;
  const int2 rows_of = ex_rows(p, home.x);
  const int n = p.seq[s].w, all = home.z >= 0 ? p.seq[home.z].w : 0;
  const int first = p.seg[s].x, first_pre = home.z >= 0 ? p.seg[home.z].x : 0;
  if (home.y < 0 || home.y >= n || int(r) - rows_of.x != home.y) return;
  if (home.z >= 0 && (home.w < 0 || home.w >= all)) return;
  struct Part {
    int64_t at, step;
    int count;
  };
  auto find = [&](int from, int rows, int row) {
    const int t = row / EX_WIDE, f = from + ex_tiles(rows) - 1 - t;
    Part o = {0, 0, 0};
    if (f >= p.max_tiles) return o;
    const int2 tile = p.tile[f];
    if (tile.x < 0) return o;   // its item wrote the rows
    o.at = ex_unit_row(p, tile.x, h, row - t * EX_WIDE);
    o.step = int64_t(rows > EX_NARROW ? EX_WIDE / EX_UNIT : 1) * p.kv_heads * EX_UNIT;
    o.count = max(tile.y, 0);
    return o;
  };
  const Part own = find(first, n * G, home.y * G + hd - h * G);
  const Part pre = home.z >= 0 ? find(first_pre, all * G, home.w * G + hd - h * G) : Part{0, 0, 0};
  if (own.count == 0 || (home.z >= 0 && pre.count == 0)) return;   // (no room for them: an error of the plan's)
  const int count = own.count + pre.count;
  auto place = [&](int k) { return k < own.count ? own.at + k * own.step : pre.at + (k - own.count) * pre.step; };
  ExJoin j;
  int k0 = 0;
  for (; count - k0 > 4; k0 += 8) j.take<8>(p, count - k0, d, [&](int k) { return place(k0 + k); });
  if (count - k0 > 2) j.take<4>(p, count - k0, d, [&](int k) { return place(k0 + k); });
  else if (count - k0 > 0) j.take<2>(p, count - k0, d, [&](int k) { return place(k0 + k); });
  j.put<QT>(p, r, hd, d);
}

struct PrefixLayout {
  int64_t arrived, head, seq, seg, tile, row_list, row_home, subtile, item, part_o, part_ml, total;
  int64_t subs, pre_subs, lone, tiles, wide_items, items, units;
  bool wide;
};

// Tiles as ex_layout counts them, for the requests' rows and once more for the
// prefixes'.  An item is a tile or a part of one: wide tiles are cut into
// EX_TARGET / kv_heads more parts at most, narrow ones into as many as there are
// places for them.  Partials in units of 32 rows: eight for every wide item.
static PrefixLayout prefix_layout(int64_t batch, int64_t prefixes, int64_t rows, int64_t max_tokens, int64_t groups,
                                  int64_t kv_heads, int64_t num_blocks, int64_t pre_blocks, int64_t bs, int64_t D) {
  PrefixLayout l{};
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  const int64_t all = rows * groups, longest = std::min(rows, max_tokens) * groups;
  l.wide = all > EX_NARROW;
  // Segments of more than 32 rows, and their tiles of up to 256.
  auto wide_tiles = [&](int64_t segments, int64_t most) {
    return most <= EX_NARROW ? 0 : all / EX_WIDE + std::min(segments, all / (EX_NARROW + 1));
  };
  const int64_t wide = wide_tiles(batch, longest) + wide_tiles(prefixes, all), narrow = batch + prefixes;
  l.tiles = wide + narrow;
  l.wide_items = l.wide ? wide + std::max<int64_t>(EX_TARGET / kv_heads, 1) : 0;
  l.items = l.wide_items + narrow + (EX_SLOTS / kv_heads + 1) * PX_SIDE;
  l.units = l.wide_items * (EX_WIDE / EX_UNIT) + (l.items - l.wide_items);
  l.lone = longest >= PX_LONE ? std::min(batch, all / PX_LONE) : 0;
  l.subs = num_blocks * ((bs + EX_SUB - 1) / EX_SUB) + EX_PAD;
  l.pre_subs = pre_blocks * ((bs + EX_SUB - 1) / EX_SUB) + EX_PAD;
  l.arrived = 128;
  l.head = EX_WS_HEAD;
  l.seq = l.head + 256;
  l.seg = up(l.seq + (batch + prefixes) * 16);
  l.tile = up(l.seg + (batch + prefixes) * 8);
  l.row_list = up(l.tile + l.tiles * 8);
  l.row_home = up(l.row_list + rows * 4);
  l.subtile = up(l.row_home + rows * 16);
  l.item = up(l.subtile + (batch * l.subs + prefixes * l.pre_subs + l.lone * (l.subs + l.pre_subs)) * 16);
  l.part_ml = up(l.item + l.items * 16);
  l.part_o = up(l.part_ml + l.units * kv_heads * EX_UNIT * 8);
  l.total = up(l.part_o + l.units * kv_heads * EX_UNIT * D * 4);
  return l;
}

template <int DP, int WF, typename QT>
static void prefix_launch(const ExtendParams& p, bool wide, hipStream_t stream) {
  const int lds = ex_lds_bytes<DP>();
  hipLaunchKernelGGL(prefix_plan_kernel, dim3(p.batch + p.prefixes), dim3(EX_PLAN), 0, stream, p);
  const int64_t most = (int64_t(p.max_cut) + (p.max_items - p.max_cut + PX_SIDE - 1) / PX_SIDE) * p.kv_heads;
  const dim3 grid(uint32_t(std::min<int64_t>(most, EX_SLOTS)));
  if (wide) hipLaunchKernelGGL((prefix_kernel<DP, WF, QT, true>), grid, dim3(EX_THREADS), lds, stream, p);
  else hipLaunchKernelGGL((prefix_kernel<DP, WF, QT, false>), grid, dim3(EX_THREADS), lds, stream, p);
  const int64_t threads = int64_t(p.rows) * p.heads * (p.D / 4);
  hipLaunchKernelGGL(prefix_join_kernel<QT>, dim3(uint32_t((threads + EX_THREADS - 1) / EX_THREADS)), dim3(EX_THREADS), 0,
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
  if (l.items * num_kv_heads > 0x7fffffff ||
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
  p.row_home = reinterpret_cast<int4*>(ws + l.row_home);
  p.subtile = reinterpret_cast<int4*>(ws + l.subtile);
  p.item = reinterpret_cast<int4*>(ws + l.item);
  p.part_o = reinterpret_cast<float*>(ws + l.part_o);
  p.part_ml = reinterpret_cast<float*>(ws + l.part_ml);
  p.max_items = int32_t(l.items);
  p.max_cut = int32_t(l.wide_items);
  p.max_lone = int32_t(l.lone);
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
