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
// Steps of a few tokens per request are laid out by the host (below), unless
// their tables are very wide (prefix_call).  Others take three launches:
//   * prefix_plan_kernel, a workgroup per segment, lists its sub-tiles and
//     enters its rows; the last to finish cuts the segments' tiles into items;
//   * prefix_kernel, up to one workgroup per CU, which take items until none is
//     left: wide ones (256 rows, eight waves together) first, then narrow ones
//     (up to 32 rows), four side by side with two waves each, since each is a
//     chain of reads; one at a time per workgroup took three times as long;
//   * prefix_join_kernel adds up the parts of rows that have several.
//
// Bound: vector instructions beside the matrix products for prompts (16 of up
// to 512 tokens on a prefix of 16384, 32 heads on 8 kv heads of 128: 1937 us,
// 665 TFLOP/s; the reference format 2460); for steps the requests' own tokens
// at the memory rate, and 7 us that a workgroup takes to start and end, one at
// a time per CU (64 single tokens on a prefix of 8192: 44 us; 256 on 4 of 4096,
// reference format: 83; 24 x 5 on 1501: 27; 2 on 600: 17); between them the
// plan and wide tiles that are not full (32 requests of 100 tokens on 4096: 368
// us, 109 at the products' rate).  All of calls replayed from a graph.

#include "extend_tile.h"

namespace tierkv {

// Rows (tokens times heads of a kv head) from which a request walks its prefix
// itself (32 requests on a prefix of 4096, 4 heads per kv head: 127 tokens each,
// shared, 397 us; 128, by themselves, 343).
constexpr int PX_LONE = 512;
constexpr int PX_KW = 2;                // waves of a narrow item
constexpr int PX_SIDE = EX_WAVES / PX_KW;   // narrow items side by side
constexpr int PX_TAIL = 4;              // items that cutting the last tiles adds, at most, for each place
constexpr int PX_MIN_NARROW = 8;        // sub-tiles of a narrow item, at least, when a tile is cut
constexpr float PX_NARROW_COST = 0.5f;  // a narrow item's sub-tile, in wide sub-tiles' time
// A step's workgroup, in microseconds: its start and end, a wide sub-tile, a
// round of narrow ones (alone, and how much more beside others), and what each part
// adds to the join; and the bytes of partials per microsecond.
constexpr double PX_COST = 7., PX_COST_WIDE = 0.5, PX_COST_ROUND = 1.7, PX_COST_SIDE = 1.8, PX_COST_PART = 0.08, PX_COST_BYTES = 3e6;

// A request's prefix, -1 for none (also for a number that no prefix has).
__device__ __forceinline__ int px_prefix(const ExtendParams& p, int b) {
  const int g = p.prefix_of[b];
  return g >= 0 && g < p.prefixes ? g : -1;
}

__device__ __forceinline__ bool px_lone(const ExtendParams& p, int b) {
  return px_prefix(p, b) >= 0 && ex_rows(p, b).y * p.groups >= PX_LONE;
}

// Where the list of request b's sub-tiles is: behind the prefixes', or, for
// ~where >= 0, among those of requests that walk their prefix themselves.
__device__ __forceinline__ int64_t px_list_of(const ExtendParams& p, int b, int where) {
  const int64_t own = p.prefixes * p.pre_subs + b * p.subs_per_seq;
  return where >= 0 ? own : p.prefixes * p.pre_subs + p.batch * p.subs_per_seq + ~where * (p.pre_subs + p.subs_per_seq);
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
    // (packed ranges that overlap have more rows than there are, perhaps more than 2^31)
    where = min(max(total.a, 0), p.rows);
    n = n_all = min(max(total.c, 0), p.rows - where);
    fits = n == total.c;
  } else {
    const int2 r = ex_rows(p, b, &n_all);
    n = r.y;
    const int place = min(max(total.a, 0), p.rows), end = min(n_all, p.rows - r.x);
    if (lone) {
      where = ~total.a;
      if (total.a >= p.max_lone) {   // (the same)
        fits = false;
        n = 0;
      }
    }
    for (int i = tid; i < end; i += EX_PLAN) {
      const int mine = g >= 0 && !lone ? total.b + i : -1;
      const bool in = i < n && mine < p.rows - place;   // (mine: -1 or less for none)
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
  int4* const out = p.subtile + (pre ? seg * p.pre_subs : px_list_of(p, b, fits ? where : 0));
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
  __shared__ float s_time[EX_PLAN / 64], s_items[EX_PLAN / 64], s_len[EX_PLAN / 64];
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
      s_items[w] = items;
      s_len[w] = len;
    }
  }
  __syncthreads();
  int choice = 0;
  for (int i = 1; i < EX_PLAN / 64; ++i)
    if (s_time[i] < s_time[choice]) choice = i;
  const int per_wide = s_per[choice];
  // Whole tiles that would begin a last round of the slots, not full, are cut
  // by `tail`, so that the round is shorter (113 tiles on 32 places: 2147 us
  // with four rounds, 1920 with the last 17 tiles cut, before absmax values
  // entered the products exactly).
  int tail = 1, tail_from = 0x7fffffff;
  {
    const int places = int(slots), items = int(s_items[choice]);
    const int rest = places > 0 ? items % places : 0;
    if (items > places && rest > 0) {
      float best = 1.f;
      for (int k = 2; k <= 8; ++k) {
        const float t = ceilf(float(rest * k) / float(places)) / float(k) + float(k) * EX_ITEM_COST / s_len[choice];
        if (rest * (k - 1) <= places * PX_TAIL && t < best) {
          best = t;
          tail = k;
          tail_from = items - rest;
        }
      }
    }
  }
  // Items, tile by tile: wide ones from the front, narrow ones from the back.
  int wide_items = 0, narrow_items = 0, units = 0, before = 0;   // before: wide items without the tail's cuts
  for (int f0 = 0; f0 < tiles_all; f0 += EX_PLAN) {
    const int f = f0 + tid;
    ExTileId x = {0, 0, false};
    int parts = 0;
    if (f < tiles_all) {
      x = ex_tile_id(segments, f, s_tile, s_rows);
      parts = ex_parts(tile_work(x), x.wide ? per_wide : per_narrow);
    }
    if (tail > 1) {
      const Ex3 s = ex_scan3({x.wide ? parts : 0, 0, 0}, sh, &total);
      if (x.wide && parts == 1 && before + s.a - parts >= tail_from) parts = tail;
      before += total.a;
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

template <int DP, int WF, typename QT, bool WIDE>
__device__ __forceinline__ void px_item(const ExtendParams& p, char* lds, int h, const ex_int4 it, bool dead) {
  const int s = it.x, where = p.seg[s].y;
  const bool pre = s < p.prefixes;
  const int q0 = pre ? where : ex_rows(p, s - p.prefixes).x;
  const ExWorkspaceList list = {p.subtile + (pre ? s * p.pre_subs : px_list_of(p, s - p.prefixes, where))};
  ex_tile_part<DP, WF, QT, WIDE, true, WIDE ? 1 : PX_KW>(p, lds, h, it.y, it.z & 0xffff, it.z >> 16, p.seq[s], list,
                                                         [&](int t) { return pre ? p.row_list[q0 + t] : q0 + t; }, it.w, dead);
}

// Workgroups take wide items one by one, then narrow ones PX_SIDE at a time,
// until none is left: the first by their number, the others from a counter.
template <int DP, int WF, typename QT>
__global__ __launch_bounds__(EX_THREADS, 2) void prefix_kernel(ExtendParams p) {
  extern __shared__ __attribute__((aligned(16))) char px_lds[];
  __shared__ int s_next;
  const int wide = p.head[0] * p.kv_heads, narrow = p.head[1] * p.kv_heads;
  const int all = wide + (narrow + PX_SIDE - 1) / PX_SIDE;
  int j = blockIdx.x;
  while (j < all) {
    int next = 0;
    if (threadIdx.x == 0) next = atomicAdd(p.head + 2, 1) + int(gridDim.x);
    if (j < wide) {
      const int i = j / p.kv_heads, h = j - i * p.kv_heads;
      const ex_int4 it = ((ExList)(uintptr_t)p.item)[i];
      if (it.x >= 0) px_item<DP, WF, QT, true>(p, px_lds, h, it, false);
    } else {
      const int u = (j - wide) * PX_SIDE + ex_uniform(threadIdx.x >> 6) / PX_KW;
      const int x = min(u, narrow - 1), i = x / p.kv_heads, h = x - i * p.kv_heads;
      ex_int4 it = ((ExList)(uintptr_t)p.item)[p.max_items - 1 - i];
      const bool dead = u >= narrow || it.x < 0;
      if (it.x < 0) it.x = 0;
      px_item<DP, WF, QT, false>(p, px_lds, h, it, dead);
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

// ---------------------------------------------------------------------------
// Steps of a few tokens per request
// ---------------------------------------------------------------------------
// Where no request brings more than PX_STEP rows (single tokens, drafts), the plan
// would cost as much as the attention: a launch of its own, and five dependent
// reads between it and an item's first key.  These calls are laid out on the
// host, from sizes alone: a request's table row is cut into up to own_parts
// ranges of blocks, a prefix's into up to pre_parts, and a workgroup lists the
// sub-tiles of its range in LDS itself.  A prefix's rows fill tiles ("slots")
// of 256; how many there are follows from the requests' prefixes, which each
// workgroup of a slot reads.  Two launches: the parts, and their join.

// Rows of a request, at most: tiles of 32 (32 requests on a prefix of 4096, 4
// heads per kv head: 16 tokens each, a step, 74 us; 17, planned, 105), and what
// prefix_call says.
constexpr int PX_STEP = 64;
constexpr int PX_LIST = 416;       // sub-tiles that a workgroup lists
constexpr int PX_MOST = 8;         // requests' parts side by side in a workgroup, where it is not one

// What a workgroup of a step takes, or one of several side by side: parts of
// one slot's rows, for one kv head, or of a request's own.
struct PxWork {
  int h, tile, rows, n;    // rows: of the slot's prefix or of the request, n: their tokens
  int row, nb, per, used;  // of the tables: row, its blocks, how they are cut (used 0: nothing to do)
  int hidden;              // tokens of the request in all
  int first;               // packed row of token 0, or, of a slot, the token of its first entry
  int unit;                // of part 0
};

// A step's workgroup's LDS beside the tiles'.
struct PxShared {
  int4 list[PX_LIST + 4 * PX_MOST];   // (spare entries behind each part's, which may be read)
  int rows[EX_WIDE + 4];              // packed rows of a tile's tokens
  int2 scan[EX_WAVES];
  int found[4];
  int dead[EX_WAVES];
};
static_assert(ex_lds_bytes<128>() + sizeof(PxShared) + 256 <= 160 * 1024 && ex_lds_bytes<64>() <= ex_lds_bytes<128>(),
              "a CU's LDS, 256 bytes of it for a vote of the workgroup");

// Sub-tiles in LDS.
struct PxList {
  const int4* list;
  __device__ __forceinline__ int4 any(int i) const { return list[i]; }
  __device__ __forceinline__ ex_int4 one(int i) const {
    const int4 v = list[i];
    return ex_int4{ex_uniform(v.x), ex_uniform(v.y), ex_uniform(v.z), 0};
  }
};

struct PxBlock {
  int len, slot, state, keep, count;   // keep: 1 resident, 2 COLD that enters with logit 0; sub-tiles
};

// Block i of a table row, from `end` on an empty one.
__device__ __forceinline__ PxBlock px_block(const ExtendParams& p, const int32_t* table, const int32_t* states,
                                            const int32_t* lengths, int i, int end) {
  PxBlock o = {0, 0, COLD, 0, 0};
  if (i < end) {
    o.len = min(max(lengths[i], 0), p.bs);
    o.state = states[i];
    o.slot = table[i];
  }
  if (o.len > 0) {
    if (o.state == HOT || o.state == WARM) {
      const int64_t slots = o.state == HOT ? p.hot_slots : p.warm_slots;
      if (o.slot >= 0 && o.slot < slots) o.keep = 1;
      else atomicOr(p.err, 1);
    } else if (o.state != COLD) {
      atomicOr(p.err, 2);
    } else if (p.cold_zero) {
      o.keep = 2;
    }
  }
  o.count = o.keep ? (o.len + EX_SUB - 1) / EX_SUB : 0;
  return o;
}

__device__ __forceinline__ void px_enter(int4* list, const PxBlock& k, int count, int first) {
  const int code = k.state == COLD ? EX_STATE_ZERO : k.state;
  for (int j = 0; j < count; ++j)
    list[j] = make_int4(k.slot, min(k.len - j * EX_SUB, EX_SUB) | (code << 8) | (j << 16), first + j * EX_SUB, 0);
}

// Inclusive sums of two values over groups of W waves, and the groups' sums.
template <int W>
__device__ __forceinline__ int2 px_scan(int a, int b, int2 (&sh)[EX_WAVES], int2* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, w0 = w / W * W;
  int2 v = make_int2(wave_inclusive_scan(a), wave_inclusive_scan(b));
  __syncthreads();
  if (lane == 63) sh[w] = v;
  __syncthreads();
  int2 all = make_int2(0, 0);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int2 t = sh[w0 + i];
    if (w0 + i < w) {
      v.x += t.x;
      v.y += t.y;
    }
    all.x += t.x;
    all.y += t.y;
  }
  *total = all;
  return v;
}

// How a table row of nb blocks is cut: blocks of a part, and parts, at least
// one.  The host's parts are for rows of the table's width; shorter ones have
// fewer, and the workgroups of the others, last in the launch, end at once (64
// requests of 250 tokens in tables of 16384 blocks: 143 us, 611 with all parts).
__device__ __forceinline__ int2 px_cut(int nb, int parts, int least) {
  const int per = max((nb + parts - 1) / parts, least);
  return make_int2(per, max((nb + per - 1) / per, 1));
}

struct PxPart {
  int4 seq;
  const int4* list;
};

// A slot's.
__device__ __forceinline__ PxWork px_step_prefix(const ExtendParams& p, char* lds, PxShared& s, int h, int slot, bool enters, int each) {
  const int tid = threadIdx.x, G = p.groups;
  // The slot's prefix g, its tile of it, and the prefix's rows.
  int* const counts = reinterpret_cast<int*>(lds);
  for (int i = tid; i < p.prefixes; i += EX_THREADS) counts[i] = 0;
  if (tid == 0) s.found[0] = -1;
  __syncthreads();
  for (int i = tid; i < p.batch; i += EX_THREADS) {
    const int k = px_prefix(p, i);
    if (k >= 0) atomicAdd(counts + k, ex_rows(p, i).y);
  }
  __syncthreads();
  int2 total;
  int before = 0;
  for (int i0 = 0; i0 < p.prefixes; i0 += EX_THREADS) {
    const int i = i0 + tid, n = i < p.prefixes ? counts[i] : 0;
    const int tiles = (n * G + EX_WIDE - 1) / EX_WIDE;
    const int2 v = px_scan<EX_WAVES>(tiles, 0, s.scan, &total);
    const int first = before + v.x - tiles;
    if (slot >= first && slot < first + tiles) {
      s.found[0] = i;
      s.found[1] = slot - first;
      s.found[2] = n;
    }
    before += total.x;
  }
  if (before > p.pre_slots && tid == 0) atomicOr(p.err, 4);   // (packed ranges that overlap)
  __syncthreads();
  const int g = ex_uniform(s.found[0]), t = ex_uniform(s.found[1]), n = ex_uniform(s.found[2]);
  PxWork o{};
  if (g < 0) return o;
  o.nb = p.pre_nblocks ? min(max(p.pre_nblocks[g], 0), p.pre_blocks) : p.pre_blocks;
  const int2 cut = px_cut(o.nb, p.pre_parts, p.pre_least);
  // The tile's tokens, in the order of their requests.
  const int row0 = t * EX_WIDE, t0 = row0 / G, t1 = min((min(row0 + EX_WIDE, n * G) + G - 1) / G, n);
  before = 0;
  for (int i0 = 0; i0 < p.batch; i0 += EX_THREADS) {
    const int i = i0 + tid;
    int2 r = make_int2(0, 0);
    if (i < p.batch && px_prefix(p, i) == g) r = ex_rows(p, i);
    const int2 v = px_scan<EX_WAVES>(r.y, 0, s.scan, &total);
    const int place = before + v.x - r.y;
    for (int k = max(t0 - place, 0); k < min(t1 - place, r.y); ++k) {
      s.rows[place + k - t0] = r.x + k;
      // Where its rows are among the slots', by the tile that its first is in.
      if (enters && (place + k) * G >= row0) p.row_pre[r.x + k] = make_int4(i, (slot - t) * EX_WIDE + (place + k) * G, cut.y, 0);
    }
    before += total.x;
  }
  o.h = h;
  o.tile = t;
  o.rows = n * G;
  o.n = n;
  o.row = g;
  o.per = cut.x;
  o.used = cut.y;
  o.first = t0;
  o.unit = slot * p.pre_parts * each;
  return o;
}

__device__ __forceinline__ PxPart px_prefix_part(const ExtendParams& p, PxShared& s, const PxWork& o, int part) {
  const int k0 = min(part * o.per, o.nb), k1 = min(k0 + o.per, o.nb);
  const int64_t row = o.row * p.pre_stride;
  int2 total;
  int subs = 0, cold = 0;
  for (int i0 = k0; i0 < k1; i0 += EX_THREADS) {
    const PxBlock k = px_block(p, p.pre_table + row, p.pre_states + row, p.pre_lengths + row, i0 + int(threadIdx.x), k1);
    const int count = k.keep == 2 ? 0 : k.count;   // (every row sees them: a count)
    const int2 v = px_scan<EX_WAVES>(count, k.keep == 2 ? k.len : 0, s.scan, &total);
    px_enter(s.list + subs + v.x - count, k, count, 0);
    subs += total.x;
    cold += total.y;
  }
  __syncthreads();
  return {make_int4(subs, o.n + 64, cold, o.n), s.list};   // (every row sees every token: limits past a sub-tile's end)
}

// A request's, EX_WAVES / KW side by side: unit u of (request, tile, kv head).
template <int KW>
__device__ __forceinline__ PxWork px_step_own(const ExtendParams& p, int x, bool enters) {
  const int units = p.batch * p.own_tiles * p.kv_heads;
  const int u = x * (EX_WAVES / KW) + ex_uniform(threadIdx.x >> 6) / KW;
  const bool dead = u >= units;
  const int v0 = min(u, units - 1), v1 = v0 / p.kv_heads, tile = v1 % p.own_tiles, b = v1 / p.own_tiles;
  PxWork o{};
  const int2 rows = ex_rows(p, b, &o.hidden);
  o.h = v0 - v1 * p.kv_heads;
  o.tile = tile;
  o.n = rows.y;
  o.rows = o.n * p.groups;
  o.first = rows.x;
  o.nb = p.seq_nblocks ? min(max(p.seq_nblocks[b], 0), p.num_blocks) : p.num_blocks;
  const int2 cut = px_cut(o.nb, p.own_parts, p.own_least);
  if (enters && o.h == 0 && tile == 0 && !dead) {
    const int g = px_prefix(p, b);
    for (int i = threadIdx.x % (64 * KW); i < min(o.hidden, p.rows - rows.x); i += 64 * KW)
      p.row_home[rows.x + i] = make_int4(i < o.n ? b : -1, i, g, cut.y);
    if (o.n < o.hidden && threadIdx.x % (64 * KW) == 0) atomicOr(p.err, 4);
  }
  o.row = b;
  o.per = cut.x;
  o.used = dead || tile * EX_NARROW >= o.rows ? 0 : cut.y;
  o.unit = int(p.own_unit) + v1 * p.own_parts;
  return o;
}

template <int KW>
__device__ __forceinline__ PxPart px_own_part(const ExtendParams& p, PxShared& s, const PxWork& o, int part) {
  constexpr int SIDE = EX_WAVES / KW, THREADS = 64 * KW;
  const int mine = ex_uniform(threadIdx.x >> 6) / KW, tid = threadIdx.x % THREADS;
  const int k0 = min(part * o.per, o.nb), k1 = min(k0 + o.per, o.nb);
  const int64_t row = o.row * p.stride;
  const PxBlock k = px_block(p, p.table + row, p.states + row, p.lengths + row, k0 + tid, k1);   // (per <= THREADS)
  // Tokens before the part and in all.
  int2 total;
  int below = 0, held = 0;
  for (int i = tid; i < o.nb; i += THREADS) {
    const int len = min(max(p.lengths[row + i], 0), p.bs);
    held += len;
    if (i < k0) below += len;
  }
  px_scan<KW>(below, held, s.scan, &total);
  const int base = total.x, tokens = total.y;
  const int2 lens = px_scan<KW>(k.len, 0, s.scan, &total);
  const int first = base + lens.x - k.len;
  const bool all_see = k.keep == 2 && first + k.len <= tokens - o.hidden + 1;
  const int count = all_see ? 0 : k.count;
  const int2 v = px_scan<KW>(count, all_see ? k.len : 0, s.scan, &total);
  int4* const list = s.list + mine * (PX_LIST / SIDE + 4);
  px_enter(list + v.x - count, k, count, first);
  __syncthreads();
  return {make_int4(total.x, tokens - (o.hidden - o.n), total.y, o.n), list};
}

// MIXED: calls that may hold wide tiles; the others' kernel is without their code.
template <int DP, int WF, typename QT, bool MIXED>
__global__ __launch_bounds__(EX_THREADS, 2) void prefix_step_kernel(ExtendParams p) {
  extern __shared__ __attribute__((aligned(16))) char px_lds[];
  __shared__ PxShared s;
  constexpr int KW_SIDE = EX_WAVES / PX_MOST;
  const int pre = p.pre_slots * p.pre_parts * p.kv_heads, x = blockIdx.x, each = MIXED ? EX_WIDE / EX_UNIT : 1;
  const bool shared = x < pre;
  const int side = shared ? 1 : p.own_side;
  PxWork o;
  int part;
  if (shared) {
    const int v = x / p.kv_heads, h = x - v * p.kv_heads, slot = v / p.pre_parts;
    part = v - slot * p.pre_parts;
    o = px_step_prefix(p, px_lds, s, h, slot, h == 0 && part == 0, each);
  } else {   // (part by part: those that are not there come last)
    const int groups = (p.batch * p.own_tiles * p.kv_heads + side - 1) / side, y = x - pre;
    part = y / groups;
    if (side == 1) o = px_step_own<EX_WAVES>(p, y - part * groups, part == 0);
    else o = px_step_own<KW_SIDE>(p, y - part * groups, part == 0);
  }
  const bool dead = part >= o.used;
  if (side == 1) {
    if (dead) return;
  } else {
    if ((threadIdx.x & 63) == 0) s.dead[threadIdx.x >> 6] = dead;
    __syncthreads();
    int all = 1;
    for (int w = 0; w < EX_WAVES; ++w) all &= s.dead[w];
    if (all) return;
  }
  PxPart of;
  if (shared) of = px_prefix_part(p, s, o, part);
  else if (side == 1) of = px_own_part<EX_WAVES>(p, s, o, part);
  else of = px_own_part<KW_SIDE>(p, s, o, part);
  // (a wave's all alike: scalar registers)
  for (int* v : {&of.seq.x, &of.seq.y, &of.seq.z, &of.seq.w, &o.h, &o.tile, &o.rows, &o.first, &o.unit}) *v = ex_uniform(*v);
  const PxList list = {of.list};
  const int first = o.first;
  auto packed = [&](int t) { return shared ? s.rows[max(t - first, 0)] : first + t; };
  const int64_t unit = o.unit + part * (shared ? each : 1);
  if (MIXED && shared && o.rows > EX_NARROW) ex_tile_part<DP, WF, QT, true, true, 1>(p, px_lds, o.h, o.tile, 0, 1, of.seq, list, packed, unit);
  else if (side == 1) ex_tile_part<DP, WF, QT, false, true, EX_WAVES>(p, px_lds, o.h, o.tile, 0, 1, of.seq, list, packed, unit);
  else ex_tile_part<DP, WF, QT, false, true, KW_SIDE>(p, px_lds, o.h, o.tile, 0, 1, of.seq, list, packed, unit, dead);
}

template <typename QT>
__global__ __launch_bounds__(EX_THREADS) void prefix_step_join_kernel(ExtendParams p, int32_t each) {
  const int D4 = p.D / 4, G = p.groups;
  const int64_t x = int64_t(blockIdx.x) * EX_THREADS + threadIdx.x;
  const int64_t rh = x / D4;
  const int d = 4 * int(x - rh * D4);
  const int64_t r = rh / p.heads;
  if (r >= p.rows) return;
  const int hd = int(rh - r * p.heads), h = hd / G;
  const int4 home = p.row_home[r];
  const int4 of = p.row_pre[r];
  // (a row of no request has whatever the workspace held)
  if (home.x < 0 || home.x >= p.batch) return;
  const int2 rows_of = ex_rows(p, home.x);
  if (home.y < 0 || home.y >= rows_of.y || int(r) - rows_of.x != home.y) return;
  const int64_t step = int64_t(p.kv_heads) * EX_UNIT;
  const int mine = home.y * G + hd - h * G;   // (in tile mine / 32)
  const int64_t tile = int64_t(home.x) * p.own_tiles + mine / EX_NARROW;
  const int64_t at = ex_unit_row(p, p.own_unit + tile * p.own_parts, h, mine % EX_NARROW);
  int pre_count = 0;
  int64_t pre_at = 0;
  if (home.z >= 0) {
    const int64_t row = int64_t(of.y) + hd - h * G, slot = row / EX_WIDE;
    if (of.x != home.x || of.y < 0 || slot >= p.pre_slots) return;
    pre_count = min(max(of.z, 0), p.pre_parts);
    pre_at = ex_unit_row(p, slot * p.pre_parts * each, h, int(row - slot * EX_WIDE));
  }
  const int own_count = min(max(home.w, 0), p.own_parts), count = own_count + pre_count;
  auto place = [&](int k) { return k < own_count ? at + k * step : pre_at + (k - own_count) * each * step; };
  ExJoin j;
  int k0 = 0;
  for (; count - k0 > 4; k0 += 8) j.take<8>(p, count - k0, d, [&](int k) { return place(k0 + k); });
  if (count - k0 > 2) j.take<4>(p, count - k0, d, [&](int k) { return place(k0 + k); });
  else if (count - k0 > 0) j.take<2>(p, count - k0, d, [&](int k) { return place(k0 + k); });
  j.put<QT>(p, r, hd, d);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

struct PrefixLayout {
  int64_t arrived, head, seq, seg, tile, row_list, row_home, subtile, item, part_o, part_ml, total;
  int64_t subs, pre_subs, lone, tiles, wide_items, items, units;
};

// Tiles as ex_layout counts them, for the requests' rows and once more for the
// prefixes'.  An item is a tile or a part of one: wide tiles are cut into
// EX_TARGET / kv_heads more parts at most, and the last of them into PX_TAIL
// more for each place, narrow ones into as many as there are places for them.  Partials in units of 32 rows: eight for every wide item.
static PrefixLayout prefix_layout(int64_t batch, int64_t prefixes, int64_t rows, int64_t max_tokens, int64_t groups,
                                  int64_t kv_heads, int64_t num_blocks, int64_t pre_blocks, int64_t bs, int64_t D) {
  PrefixLayout l{};
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  const int64_t all = rows * groups, longest = std::min(rows, max_tokens) * groups;
  // Segments of more than 32 rows, and their tiles of up to 256.
  auto wide_tiles = [&](int64_t segments) { return all / EX_WIDE + std::min(segments, all / (EX_NARROW + 1)); };
  const int64_t wide = wide_tiles(batch) + wide_tiles(prefixes), narrow = batch + prefixes;
  l.tiles = wide + narrow;
  l.wide_items = wide + std::max<int64_t>(EX_TARGET / kv_heads, 1) + (EX_SLOTS / kv_heads + 1) * PX_TAIL;
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

// A step's layout: how many ranges the tables' rows are cut into, and where
// its workspace lies.  parts are rated by the time of their workgroups, one per
// CU at a time, in microseconds measured on steps of 1 to 256 requests.
struct StepLayout {
  int64_t row_home, row_pre, part_o, part_ml, total;
  int64_t slots, pre_parts, own_parts, own_tiles, side, each, own_unit, units, workgroups;
  int64_t pre_least, own_least;
  bool use;
  int64_t bytes() const { return std::max<int64_t>(total, EX_WS_HEAD); }
};

static StepLayout step_layout(int64_t batch, int64_t prefixes, int64_t rows, int64_t max_tokens, int64_t groups,
                              int64_t kv_heads, int64_t num_blocks, int64_t pre_blocks, int64_t bs, int64_t D) {
  StepLayout l{};
  const int64_t all = std::min(rows, batch * max_tokens) * groups, longest = std::min(rows, max_tokens) * groups;
  l.use = longest <= PX_STEP;
  if (!l.use || rows == 0) return l;
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  auto div = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t subs = div(bs, EX_SUB), fit = PX_LIST / subs;
  const bool wide = all > EX_NARROW;
  l.own_tiles = std::max<int64_t>(div(longest, EX_NARROW), 1);
  l.each = wide ? EX_WIDE / EX_UNIT : 1;
  const int64_t groups_n = std::min(prefixes, batch);
  l.slots = all / EX_WIDE + groups_n;
  // The slots there are when the requests are spread evenly over the prefixes.
  const int64_t live = groups_n * div(div(all, groups_n), EX_WIDE);
  const bool pre_wide = div(all, groups_n) > EX_NARROW;
  double best = 0;
  for (int64_t side : {1, PX_MOST}) {
    const int64_t own_fit = fit / side, least_own = div(num_blocks, own_fit), least_pre = div(pre_blocks, fit);
    const int64_t waves = EX_WAVES / side;
    for (int64_t own = least_own; own <= std::max<int64_t>(least_own, 8); own *= 2) {
      for (int64_t pre = least_pre, last = 0; last == 0; pre = pre < 4 ? pre + 1 : pre + pre * 2 / 5) {
        if (pre >= std::max<int64_t>(least_pre, 64)) last = 1;
        const double pre_subs = double(div(pre_blocks, pre) * subs), own_subs = double(div(num_blocks, own) * subs);
        const double c_pre = PX_COST + (pre_wide ? PX_COST_WIDE * pre_subs : PX_COST_ROUND * std::ceil(pre_subs / (2 * EX_WAVES)));
        const double c_own = PX_COST + PX_COST_ROUND * std::ceil(own_subs / (2 * waves)) * (side > 1 ? PX_COST_SIDE : 1.);
        const double n_pre = double(live * pre * kv_heads), n_own = double(div(batch * l.own_tiles * own * kv_heads, side));
        const double sum = (n_pre * c_pre + n_own * c_own) / EX_SLOTS, most = std::max(c_pre, c_own);
        const double makespan = n_pre + n_own <= EX_SLOTS ? most : std::max(most, sum + 0.5 * std::min(c_pre, c_own));
        const double bytes = (double(all) * pre + double(batch) * longest * own) * kv_heads * D * 4;
        const double time = makespan + PX_COST_PART * (pre + own) + 2 * bytes / PX_COST_BYTES;
        if (best == 0 || time < best) {
          best = time;
          l.side = side;
          l.own_parts = own;
          l.pre_parts = pre;
        }
      }
    }
  }
  l.own_unit = l.slots * l.pre_parts * l.each;
  l.units = l.own_unit + batch * l.own_tiles * l.own_parts;
  // Least parts: one round of narrow sub-tiles, and eight wide sub-tiles.
  l.own_least = std::max<int64_t>(2 * (EX_WAVES / l.side) / subs, 1);
  l.pre_least = std::max<int64_t>(8 / subs, 1);
  l.workgroups = l.slots * l.pre_parts * kv_heads + div(batch * l.own_tiles * kv_heads, l.side) * l.own_parts;
  l.row_home = EX_WS_HEAD;
  l.row_pre = up(l.row_home + rows * 16);
  l.part_ml = up(l.row_pre + rows * 16);
  l.part_o = up(l.part_ml + l.units * kv_heads * EX_UNIT * 8);
  l.total = up(l.part_o + l.units * kv_heads * EX_UNIT * D * 4);
  return l;
}

// The way that a call of these sizes takes, and its workspace.  A step's parts
// and partials follow the tables' width, the plan's the rows there are: past
// PX_STEP_MEMORY of the plan's workspace, or of a launch's 2^32 threads, calls
// of few tokens are planned too.  Around that size tables are mostly far wider
// than their rows, which a step's workgroups pay for and the plan's do not: 256
// single tokens with 256 of their own in tables of 16384 blocks, 1.4 GB, 501 us
// as a step and 131 planned; full rows lose by it (64 whose tables of 16384 are
// full, 1.4 times the plan's: 11.0 ms as a step, 20.9 planned).
constexpr int64_t PX_STEP_MEMORY = 2;
struct PrefixCall {
  StepLayout step;
  PrefixLayout plan;
  const char* refused;   // why no such call is taken, or NULL
  int64_t bytes() const { return step.use ? step.bytes() : plan.total; }
};

static PrefixCall prefix_call(int64_t batch, int64_t prefixes, int64_t rows, int64_t max_tokens, int64_t groups,
                              int64_t kv_heads, int64_t num_blocks, int64_t pre_blocks, int64_t bs, int64_t D) {
  PrefixCall c{};
  c.refused = ex_refused(batch, rows, groups, num_blocks, bs, D);
  if (!c.refused && batch + prefixes > EX_MAX_BATCH) c.refused = "more than 4096 requests and prefixes";
  if (!c.refused && pre_blocks * bs + rows > 0x7fffffff - EX_SUB) c.refused = "prefixes of 2^31 tokens or more";
  if (c.refused) return c;
  c.step = step_layout(batch, prefixes, rows, max_tokens, groups, kv_heads, num_blocks, pre_blocks, bs, D);
  c.plan = prefix_layout(batch, prefixes, rows, max_tokens, groups, kv_heads, num_blocks, pre_blocks, bs, D);
  c.step.use = c.step.use && c.step.workgroups <= 0xffffffffll / EX_THREADS && c.step.units <= 0x7fffffff &&
               batch * c.step.own_tiles * kv_heads <= 0x7fffff00 && c.step.bytes() <= PX_STEP_MEMORY * c.plan.total;
  // (a lone request's tokens are its prefix's and its own)
  if (!c.step.use && c.plan.lone > 0 && (pre_blocks + num_blocks) * bs + rows > 0x7fffffff - EX_SUB)
    c.refused = "prefixes and rows of 2^31 tokens or more together, walked by requests of 512 rows or more";
  // (a launch has fewer than 2^32 threads)
  if ((!c.step.use && (c.plan.items * kv_heads > 0x7fffffff || c.plan.units > 0x7fffffff)) ||
      rows * groups * kv_heads > (0xffffffffll - EX_THREADS) / (D / 4))
    c.refused = "grid too large";
  return c;
}

template <int DP, int WF, typename QT>
static void prefix_launch(const ExtendParams& p, hipStream_t stream) {
  const int lds = ex_lds_bytes<DP>();
  hipLaunchKernelGGL(prefix_plan_kernel, dim3(p.batch + p.prefixes), dim3(EX_PLAN), 0, stream, p);
  const int64_t most = (int64_t(p.max_cut) + (p.max_items - p.max_cut + PX_SIDE - 1) / PX_SIDE) * p.kv_heads;
  const dim3 grid(uint32_t(std::min<int64_t>(most, EX_SLOTS)));
  hipLaunchKernelGGL((prefix_kernel<DP, WF, QT>), grid, dim3(EX_THREADS), lds, stream, p);
  const int64_t threads = int64_t(p.rows) * p.heads * (p.D / 4);
  hipLaunchKernelGGL(prefix_join_kernel<QT>, dim3(uint32_t((threads + EX_THREADS - 1) / EX_THREADS)), dim3(EX_THREADS), 0,
                     stream, p);
}

template <int DP, int WF, typename QT>
static void step_launch(const ExtendParams& p, const StepLayout& l, hipStream_t stream) {
  const int lds = ex_lds_bytes<DP>();
  const dim3 grid(uint32_t(l.workgroups));
  if (l.each > 1) hipLaunchKernelGGL((prefix_step_kernel<DP, WF, QT, true>), grid, dim3(EX_THREADS), lds, stream, p);
  else hipLaunchKernelGGL((prefix_step_kernel<DP, WF, QT, false>), grid, dim3(EX_THREADS), lds, stream, p);
  const int64_t threads = int64_t(p.rows) * p.heads * (p.D / 4);
  hipLaunchKernelGGL(prefix_step_join_kernel<QT>, dim3(uint32_t((threads + EX_THREADS - 1) / EX_THREADS)), dim3(EX_THREADS), 0,
                     stream, p, int32_t(l.each));
}

// step: NULL for calls that are planned on the device.
template <int DP, int WF, typename QT>
static void prefix_start(const ExtendParams& p, const StepLayout* step, hipStream_t stream) {
  if (step) step_launch<DP, WF, QT>(p, *step, stream);
  else prefix_launch<DP, WF, QT>(p, stream);
}

template <int DP>
static void prefix_dispatch(const ExtendParams& p, const StepLayout* step, int wf, int dtype, hipStream_t stream) {
  const bool bf = dtype == TIERKV_DTYPE_BF16, i8 = wf == TIERKV_WARM_ABSMAX_I8;
  if (bf && i8) prefix_start<DP, TIERKV_WARM_ABSMAX_I8, __hip_bfloat16>(p, step, stream);
  else if (bf) prefix_start<DP, TIERKV_WARM_REF_U8, __hip_bfloat16>(p, step, stream);
  else if (i8) prefix_start<DP, TIERKV_WARM_ABSMAX_I8, __half>(p, step, stream);
  else prefix_start<DP, TIERKV_WARM_REF_U8, __half>(p, step, stream);
}

}  // namespace tierkv

using namespace tierkv;

extern "C" int64_t tierkv_prefix_workspace_bytes(int32_t batch, int32_t num_prefixes, int32_t num_rows,
                                                 int32_t max_tokens, int32_t num_heads, int32_t num_kv_heads,
                                                 int32_t num_blocks, int32_t num_prefix_blocks, int32_t block_size,
                                                 int32_t head_dim) {
  if (batch <= 0 || num_prefixes <= 0 || num_rows < 0 || max_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads != 0 || num_blocks <= 0 || num_prefix_blocks <= 0)
    return fail(-1, "sizes must be positive, and num_heads a multiple of num_kv_heads");
  const PrefixCall way = prefix_call(batch, num_prefixes, num_rows, max_tokens, num_heads / num_kv_heads, num_kv_heads,
                                     num_blocks, num_prefix_blocks, block_size, head_dim);
  return way.refused ? fail(-1, way.refused) : way.bytes();
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
  const PrefixCall way = prefix_call(batch, num_prefixes, num_rows, max_tokens, p.groups, num_kv_heads, num_blocks,
                                     num_prefix_blocks, block_size, head_dim);
  if (way.refused) return fail(TIERKV_ERR_UNSUPPORTED, way.refused);
  const StepLayout& step = way.step;
  const PrefixLayout& l = way.plan;
  if (workspace_bytes < way.bytes()) return fail(TIERKV_ERR_WORKSPACE, "workspace too small");
  if (num_rows == 0 || max_tokens == 0) return TIERKV_OK;
  char* ws = reinterpret_cast<char*>(workspace);
  p.err = reinterpret_cast<int32_t*>(ws);
  if (step.use) {
    p.row_home = reinterpret_cast<int4*>(ws + step.row_home);
    p.row_pre = reinterpret_cast<int4*>(ws + step.row_pre);
    p.part_o = reinterpret_cast<float*>(ws + step.part_o);
    p.part_ml = reinterpret_cast<float*>(ws + step.part_ml);
    p.pre_slots = int32_t(step.slots);
    p.pre_parts = int32_t(step.pre_parts);
    p.own_parts = int32_t(step.own_parts);
    p.own_tiles = int32_t(step.own_tiles);
    p.own_side = int32_t(step.side);
    p.own_unit = step.own_unit;
    p.pre_least = int32_t(step.pre_least);
    p.own_least = int32_t(step.own_least);
  } else {
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
  }
  p.prefix_of = prefix_of;
  p.pre_table = prefix_table;
  p.pre_states = prefix_states;
  p.pre_lengths = prefix_lengths;
  p.pre_stride = prefix_stride;
  p.pre_nblocks = prefix_num_blocks;
  p.pre_blocks = num_prefix_blocks;
  p.prefixes = num_prefixes;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const StepLayout* of = step.use ? &step : nullptr;
  if (head_dim <= 64) prefix_dispatch<64>(p, of, warm_format, query_dtype, stream);
  else prefix_dispatch<128>(p, of, warm_format, query_dtype, stream);
  return check_launch("tierkv_prefix_attention");
}
