// Attention of several query tokens per request over the tiered paged cache,
// for gfx950 (CDNA4): prompts in pieces, follow-up prompts, drafted tokens to
// verify, and single tokens beside them, packed as rows [N, heads, D].
//
// Request b's rows are the last n_b of its L_b cached tokens; row i sees the
// tokens of ordinal <= L_b - n_b + i (ordinals count the valid tokens of all
// blocks, evicted ones among them):
//   o = sum_t p_t v_t,  p = softmax(scaling * q . k_t) over what it sees.
// WARM tokens are code * scale (absmax: one scale per (slot, head)) or
// (code - zero) * scale per token; COLD ones are left out or enter with
// logit 0 and value 0, as in the single-token kernel.
//
// Three launches:
//   * extend_plan_kernel, a workgroup per request, lists the resident
//     16-token sub-tiles of its row (slot, state, first ordinal, valid
//     tokens); the last workgroup to finish turns the requests' query rows
//     into tiles and cuts the tiles' key ranges into items where that
//     shortens the whole;
//   * extend_kernel, a workgroup of eight waves per (item, kv head);
//   * extend_merge_kernel joins the items of tiles that were cut.
//
// Rows of a tile are (token, head of the GQA group) pairs of one kv head, so
// each K/V byte serves the whole group.  A wave holds 32 rows as the B operand
// of MFMA 32x32x16 f16:
//   S^T = K Q^T    (A = 32 keys of K from LDS)
//   O^T += V^T P^T (A = 32 dims of V^T from LDS; B = P^T is S^T's accumulator
//                   layout as it stands, once the keys of a 16-key step are
//                   numbered as the lanes hold them: slot 8h + 4a + j of the
//                   step is key 8a + 4h + j; V^T's rows are stored in that order)
// so probabilities never leave their registers, and a row's running maximum
// and sum live in the two lanes that own it.  Tiles of more than 32 rows
// ("wide") are 256 rows over eight waves that share 64 keys at a time, four
// waves half a tile ahead of the others so that one half's products run beside
// the other's exponentials; smaller ones ("narrow") give each wave its own 32
// keys of the same rows, merged in LDS.
//
// K goes to LDS as fp16 of the codes themselves (exact), and the scale is
// applied to the logits in 32 bits.  The reference format's zero point is the
// same for all dims of a token, q . (code - zero) = q . code - zero sum q: one
// more product step takes it off, with the zero point (fp16, exact) beside
// the token's row of K and the query's sum in three fp16 pieces beside the
// query, so that it is off by a 32-bit rounding.  (code - zero in fp16 was off
// by as much as the codes are where keys lie far from 0 against their spread,
// mean 10 and deviation 0.2, and infinite past 65504.  2048 tokens on 32768 of
// that format take 1178 us, with code - zero 1140, with the zero point taken
// off each logit by vector instructions 1239 to 1369.)
// V goes to LDS as fp16 of code * scale, one rounding of at most 2^-11 of the
// value, as the probabilities have one when they become fp16 operands: the
// matrix units take 16-bit operands at sixteen times the rate of 32-bit ones.
// (Values past fp16's range become infinite, as the format's own
// dequantization makes them, tierkv_policy.py:39-44.)
// Probabilities carry a factor 2^6 so that small ones stay normal fp16.
// bf16 queries become fp16 after division by a power of two near the row's
// largest value, which the logits get back in 32 bits.
//
// Bound: the matrix products and the exponentials between them for wide tiles
// (2048 tokens on 32768, 32 heads on 8 kv heads of 128: 977 us, 820 TFLOP/s of
// the 1100 that a large library product reaches here, 8.5 other vector
// instructions per product; with tiles still cut in
// two, 1165, where 128-row tiles of four waves took 1297, eight waves in step
// 1313 and one loop with branches for the two halves 1844); for narrow ones
// the reads of the cache and a chain of plan, attention and merge (8 x 5
// tokens on 4096, 53 MB: 11 + 24 + 4 us).

#include "tierkv_common.h"

#include <algorithm>
#include <cmath>

namespace tierkv {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int EX_THREADS = 512;
constexpr int EX_WAVES = EX_THREADS / 64;
constexpr int EX_PLAN = 1024;             // threads of a plan workgroup
constexpr int EX_MAX_BATCH = 4096;        // requests per call
constexpr int EX_SUB = 16;                // tokens per sub-tile
constexpr int EX_NARROW = 32;             // rows of a narrow tile
constexpr int EX_WIDE = 32 * EX_WAVES;   // rows of a wide tile
constexpr int EX_SLOTS = 256;             // workgroups that run at once: one per CU
constexpr int EX_TARGET = 512;            // workgroups that a cut adds, at most
constexpr int EX_MIN_SUBS = 16;           // sub-tiles per item, at least, when a tile is cut
constexpr float EX_ITEM_COST = 8.f;       // an item's start and end, in sub-tiles' time
constexpr float EX_PART_COST = 12.f;      // a partial's write and read, in sub-tiles' time
constexpr int EX_WS_HEAD = 256 + (1 << 16) * 4;   // the decode launches' error word and counters
constexpr float EX_LAZY = 8.f;            // log2 headroom of the running maximum
constexpr float EX_BOOST = 6.f;           // log2 of the probabilities' factor
constexpr float EX_NONE = -1e30f;         // running maximum before the first visible key
constexpr float EX_LOG2E = 1.4426950408889634f;
constexpr int EX_PAD = 16;                // spare entries behind a request's sub-tile list
constexpr int EX_STATE_ZERO = 3;          // sub-tile of COLD tokens that enter with logit 0

struct ExtendParams {
  const void* q;
  int64_t qs_t, qs_h;
  void* out;
  const int32_t* cu;
  int32_t rows, max_tokens;
  const int32_t* table;
  const int32_t* states;
  const int32_t* lengths;
  int64_t stride;
  const int32_t* seq_nblocks;
  int32_t num_blocks;
  const __half* hot_k;
  const __half* hot_v;
  int64_t hot_slots;
  const uint8_t* warm_k;
  const uint8_t* warm_v;
  int64_t warm_slots;
  const void* k_scale;
  const void* k_zero;
  const void* v_scale;
  const void* v_zero;
  int32_t batch, heads, kv_heads, bs, D, groups;
  int32_t cold_zero;
  float scale_log2;
  // Workspace.
  int32_t* err;
  uint32_t* arrived;   // zero between launches; in the workspace's first 256 bytes, which no launch uses otherwise
  int32_t* head;       // {items, cut tiles}
  int4* seq;           // [batch] {sub-tiles, tokens up to the last computed row, COLD tokens that every row sees, query rows n}
  int4* subtile;       // [batch][num_blocks * subs] {slot, valid | state << 8 | sub << 16, first ordinal, 0}
  int4* item;          // [max_items] {request, tile | wide << 30, part | parts << 16, partial or -1}
  int2* cut;           // [max_cut] {first partial, item}
  float* part_o;       // [partials][kv_heads][tile rows][D]
  float* part_ml;      // [partials][kv_heads][tile rows][2]
  int32_t max_items, max_cut, max_part, part_rows;
  int64_t subs_per_seq;
};

__device__ __forceinline__ int ex_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ---------------------------------------------------------------------------
// Plan
// ---------------------------------------------------------------------------

// Inclusive prefix sums of three values over a plan workgroup; total gets the
// three sums.
struct Ex3 {
  int a, b, c;
};
__device__ __forceinline__ Ex3 ex_scan3(Ex3 v, Ex3 (&sh)[EX_PLAN / 64], Ex3* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  Ex3 x = {wave_inclusive_scan(v.a), wave_inclusive_scan(v.b), wave_inclusive_scan(v.c)};
  __syncthreads();
  if (lane == 63) sh[w] = x;
  __syncthreads();
  Ex3 all = {0, 0, 0};
#pragma unroll
  for (int i = 0; i < EX_PLAN / 64; ++i) {
    const Ex3 t = sh[i];
    if (i < w) {
      x.a += t.a;
      x.b += t.b;
      x.c += t.c;
    }
    all.a += t.a;
    all.b += t.b;
    all.c += t.c;
  }
  *total = all;
  return x;
}

// Query rows of request b that are computed (first packed row, count): at
// most max_tokens of those that there are.  The limits of what they see come
// from the tokens that the request brings, `all`, computed or not.
__device__ __forceinline__ int2 ex_rows(const ExtendParams& p, int b, int* all = nullptr) {
  const int lo = min(max(p.cu[b], 0), p.rows), end = max(p.cu[b + 1], lo);
  if (all) *all = end - lo;
  return make_int2(lo, min(min(end, p.rows) - lo, p.max_tokens));
}

__device__ __forceinline__ int ex_tiles(int rows) { return rows <= EX_NARROW ? (rows > 0) : (rows + EX_WIDE - 1) / EX_WIDE; }

// Sub-tiles that a tile's last row sees (of `subs`), within one of each
// sub-tile behind it: exact when the tokens after it fill whole sub-tiles.
__device__ __forceinline__ int ex_work(int subs, int rows, int tile, bool wide, int groups) {
  const int last = wide ? min((tile + 1) * EX_WIDE, rows) - 1 : rows - 1;
  const int hidden = (rows - 1) / groups - last / groups;
  return max(subs - hidden / EX_SUB, 1);
}

// Items of one tile: its work in parts of at most per_item sub-tiles.
__device__ __forceinline__ int ex_parts(int work, int per_item) { return min((work + per_item - 1) / per_item, 32767); }

// Tile f of all: its request (the last one whose first tile is at most f, and
// that has tiles) and its place there, the longest first.
struct ExTileId {
  int request, tile;
  bool wide;
};
__device__ __forceinline__ ExTileId ex_tile_id(const ExtendParams& p, int f, const int2* first, const int* rows) {
  int lo = 0, hi = p.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid].x <= f) lo = mid;
    else hi = mid;
  }
  return {lo, ex_tiles(rows[lo]) - 1 - (f - first[lo].x), rows[lo] > EX_NARROW};
}

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
  int at = 0, ordinal = 0, cold = 0;   // sub-tiles, tokens and COLD tokens before this chunk
  int4* out = p.subtile + int64_t(b) * p.subs_per_seq;
  for (int i0 = 0; i0 < nb; i0 += EX_PLAN) {
    const int i = i0 + tid;
    int len = 0, state = COLD, slot = 0, keep = 0;
    if (i < nb) {
      len = min(max(p.lengths[row + i], 0), p.bs);
      state = p.states[row + i];
      slot = p.table[row + i];
    }
    if (len > 0) {
      if (state == HOT || state == WARM) {
        const int64_t slots = state == HOT ? p.hot_slots : p.warm_slots;
        if (slot >= 0 && slot < slots) keep = 1;
        else atomicOr(p.err, 1);
      } else if (state != COLD) {
        atomicOr(p.err, 2);
      } else if (p.cold_zero) {
        keep = 2;          // a count when every row sees it (known below), else a sub-tile of zeros
      }
    }
    int count = keep ? (len + EX_SUB - 1) / EX_SUB : 0;
    Ex3 s = ex_scan3({len, keep == 2 ? 0 : count, 0}, sh, &total);
    const int first = ordinal + s.a - len;
    int pos = at + s.b - (keep == 2 ? 0 : count);
    ordinal += total.a;
    if (p.cold_zero) {
      const bool all_see = keep == 2 && first + len <= tokens - n_all + 1;
      if (all_see) count = 0;
      const Ex3 z = ex_scan3({count, all_see ? len : 0, 0}, sh, &total);
      pos = at + z.a - count;
      at += total.a;
      cold += total.b;
    } else {
      at += total.b;
    }
    const int code = state == COLD ? EX_STATE_ZERO : state;
    for (int j = 0; j < count; ++j)
      out[pos + j] = make_int4(slot, min(len - j * EX_SUB, EX_SUB) | (code << 8) | (j << 16), first + j * EX_SUB, 0);
  }
  if (tid == 0) {
    // Agent-scope stores: the last workgroup may read them from another XCD.
    int32_t* s = reinterpret_cast<int32_t*>(p.seq + b);
    if (n < n_all) atomicOr(p.err, 4);
    const int v[4] = {at, ordinal - (n_all - n), cold, n};
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
      const ExTileId x = ex_tile_id(p, f, s_tile, s_rows);
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
      const ExTileId x = ex_tile_id(p, f, s_tile, s_rows);
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

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------

// Half a sub-tile, its K or its V, in registers as loaded.
//   K: r[i] is piece x = lane + 64 i of the 16 rows' 8-element pieces (row
//      x / (DP / 8)), i < NPK;
//   V: r[j] is key 4g + j (g = lane >> 4), dims DL n .. DL n + DL - 1 (n = lane & 15).
// WARM codes fill the front of each entry.  meta: the reference format's zero
// (low half) and scale of each entry's token, absmax: the scale (fp32) in [0].
template <int DP>
struct ExHalf {
  static constexpr int NPK = DP / 32;
  static constexpr int DL = DP / 16;
  uint4 r[4];
  uint32_t meta[4];
};

// The sub-tile list is read through the constant address space: uniform
// scalar loads, which do not wait behind the tile loads in flight.
typedef int ex_int4 __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(4))) ex_int4* ExList;

struct ExSub {
  int slot, valid, state, sub, ordinal;
};

// Sub-tile i of a list; from `end` on an empty one.  (Lists have EX_PAD spare
// entries behind them, which may be read.)
__device__ __forceinline__ ExSub ex_sub(ExList list, int i, int end) {
  const ex_int4 v = list[i];
  ExSub s;
  const bool in = i < end;
  s.slot = in ? v.x : 0;
  s.valid = in ? v.y & 0xff : 0;
  s.state = in ? (v.y >> 8) & 0xff : EX_STATE_ZERO;
  s.sub = in ? v.y >> 16 : 0;
  s.ordinal = in ? v.z : 0;
  return s;
}

// Keys of each sub-tile of a tile that a row with the given limit sees.
template <int TK>
__device__ __forceinline__ void ex_ends(ExList list, int at, int hi, int lim, int (&end)[TK / 16]) {
#pragma unroll
  for (int i = 0; i < TK / 16; ++i) {
    const ExSub s = ex_sub(list, at + i, hi);
    end[i] = min(s.valid, lim - s.ordinal + 1);
  }
}

// KV: 0 K, 1 V.
template <int DP, int WF, int KV>
__device__ __forceinline__ void ex_load(const ExtendParams& p, int h, const ExSub& s, ExHalf<DP>& st) {
  typedef ExHalf<DP> St;
  if (s.state == EX_STATE_ZERO) return;
  const int lane = threadIdx.x & 63;
  const int D = p.D, bs = p.bs;
  const int t0 = s.sub * EX_SUB;
  const int64_t tile = (int64_t(s.slot) * p.kv_heads + h) * bs;   // the block's first row of this head
  constexpr int N = KV ? 4 : St::NPK;
  // Uniform bases and 32-bit offsets within the block.
  const bool hot = s.state == HOT;
  const char* base = hot ? reinterpret_cast<const char*>((KV ? p.hot_v : p.hot_k) + tile * D)
                         : reinterpret_cast<const char*>((KV ? p.warm_v : p.warm_k) + tile * D);
  uint32_t row[N], off[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int x = lane + 64 * i;
    const int d = KV ? St::DL * (lane & 15) : 8 * (x % (DP / 8));
    row[i] = uint32_t(min(t0 + (KV ? 4 * (lane >> 4) + i : x / (DP / 8)), bs - 1));
    off[i] = row[i] * uint32_t(D) + uint32_t(d < D ? d : 0);
  }
  if (hot) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const char* src = base + off[i] * 2u;
      if (KV && St::DL < 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(src);
        st.r[i].x = w.x;
        st.r[i].y = w.y;
      } else {
        st.r[i] = *reinterpret_cast<const uint4*>(src);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const char* src = base + off[i];
    if (KV && St::DL < 8) {
      st.r[i].x = *reinterpret_cast<const uint32_t*>(src);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(src);
      st.r[i].x = w.x;
      st.r[i].y = w.y;
    }
  }
  const void* scale = KV ? p.v_scale : p.k_scale;
  if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
    st.meta[0] = reinterpret_cast<const uint32_t*>(scale)[int64_t(s.slot) * p.kv_heads + h];
  } else {
    const void* zero = KV ? p.v_zero : p.k_zero;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t z = (reinterpret_cast<const uint16_t*>(zero) + tile)[row[i]];
      st.meta[i] = z | uint32_t((reinterpret_cast<const uint16_t*>(scale) + tile)[row[i]]) << 16;
    }
  }
}

// LDS of one key tile of TK keys.  Rows are 16 bytes longer than their data:
// eight lanes that read one chunk column of neighbouring rows then touch 32
// banks in all (rows 4, 36 and 20 banks apart), and every access of a lane
// is one base address with a constant offset.  (With the chunks swizzled by
// exclusive-or each needs its own address register, 36 of them at D = 128, and
// the tile loop spilled.)  V^T has 16 bytes more per eight rows, since the
// lanes that store it are eight rows apart (without them 70 % of the LDS's
// active cycles were conflicts).
template <int DP, int TK>
struct ExTile {
  uint4 k[TK * (DP / 8 + 1)];   // K rows of DP halves
  uint4 v[DP * (TK / 8 + 1) + DP / 8];   // V^T rows of TK halves
  float kscale[TK];             // factor of each key's logits (REF_U8; absmax: one per sub-tile)
};

template <int DP>
__device__ __forceinline__ int ex_k_at(int r, int c) { return r * (DP / 8 + 1) + c; }

template <int TK>
__device__ __forceinline__ int ex_v_at(int d, int c) { return d * (TK / 8 + 1) + (d >> 3) + c; }

// Byte b of a word as a float (v_cvt_f32_ubyte).
template <int B>
__device__ __forceinline__ float ex_byte(uint32_t w) { return float((w >> (8 * B)) & 0xffu); }

__device__ __forceinline__ float ex_byte_at(uint32_t w, int i) {
  return i == 0 ? ex_byte<0>(w) : i == 1 ? ex_byte<1>(w) : i == 2 ? ex_byte<2>(w) : ex_byte<3>(w);
}

__device__ __forceinline__ uint32_t ex_pack(float a, float b) {
  const f16x2 v = {_Float16(a), _Float16(b)};
  return bits_of(v);
}

// Larger of two words' halves, as unsigned integers (v_pk_max_u16).
__device__ __forceinline__ uint32_t ex_max_u16(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// Write a loaded K half into sub-tile place `at` (0 .. TK / 16 - 1) of a tile.
template <int DP, int WF, int TK>
__device__ __forceinline__ void ex_store_k(const ExtendParams& p, const ExSub& s, const ExHalf<DP>& st, int at,
                                           ExTile<DP, TK>& t) {
  typedef ExHalf<DP> St;
  const int lane = threadIdx.x & 63, D = p.D;
  const bool zero = s.state == EX_STATE_ZERO, hot = s.state == HOT;
  // The first piece's place; the next is 64 / (DP / 8) rows further.
  uint4* const dst = t.k + ex_k_at<DP>(at * EX_SUB + lane / (DP / 8), lane % (DP / 8));
  constexpr int NEXT = 64 / (DP / 8) * (DP / 8 + 1);
  const bool clear = zero || (D != DP && (lane % (DP / 8)) * 8 >= D);
#pragma unroll
  for (int i = 0; i < St::NPK; ++i) {
    uint4 v = st.r[i];
    if (!zero && !hot) {
      f16x4 a, b;
      if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
        const f16x4 off = {1152, 1152, 1152, 1152};
        a = i8x4_plus1152(v.x) - off;
        b = i8x4_plus1152(v.y) - off;
      } else {
        const f16x4 off = {1024, 1024, 1024, 1024};
        a = u8x4_plus1024(v.x) - off;
        b = u8x4_plus1024(v.y) - off;
      }
      const uint2 lo = __builtin_bit_cast(uint2, a), hi = __builtin_bit_cast(uint2, b);
      v = make_uint4(lo.x, lo.y, hi.x, hi.y);
      if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {   // (see ex_softmax: the factors of the logits are not negative)
        const uint32_t sign = __uint_as_float(st.meta[0]) < 0.f ? 0x80008000u : 0u;
        v.x ^= sign;
        v.y ^= sign;
        v.z ^= sign;
        v.w ^= sign;
      }
    }
    if (clear) v = make_uint4(0, 0, 0, 0);
    dst[i * NEXT] = v;
    if constexpr (WF == TIERKV_WARM_REF_U8) {
      if (lane % (DP / 8) == 0) {
        t.kscale[at * EX_SUB + (lane + 64 * i) / (DP / 8)] = (zero || hot) ? 1.f : half_hi(st.meta[i]);
        const uint32_t z = (zero || hot) ? 0u : st.meta[i] & 0xffffu;
        dst[i * NEXT + DP / 8] = make_uint4(z | (z << 16), z, 0, 0);   // behind the row
      }
    }
  }
  if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
    if (lane == 0) t.kscale[at] = (zero || hot) ? 1.f : fabsf(__uint_as_float(st.meta[0]));
  }
}

// The same of a V half, transposed; returns, when asked to check, the largest
// magnitude bits of its values (two halves).
template <int DP, int WF, int TK>
__device__ __forceinline__ uint32_t ex_store_v(const ExtendParams& p, const ExSub& s, const ExHalf<DP>& st, int at,
                                               bool check, ExTile<DP, TK>& t) {
  typedef ExHalf<DP> St;
  const int lane = threadIdx.x & 63, D = p.D;
  const int n = lane & 15, g = lane >> 4;
  const bool zero = s.state == EX_STATE_ZERO, hot = s.state == HOT;
  const bool plain = s.valid == EX_SUB && D == DP;   // nothing to clear
  // The lane's four keys side by side, for each of its dims.
  uint2* const dst = reinterpret_cast<uint2*>(t.v + ex_v_at<TK>(St::DL * n, at * 2 + (g & 1))) + (g >> 1);
  constexpr int NEXT = 2 * (TK / 8 + 1);             // the next dim's row
  uint32_t largest = 0;
  auto put = [&](int i, uint2 o) {
    dst[i * NEXT] = o;
    if (check) largest = ex_max_u16(largest, ex_max_u16(o.x & 0x7fff7fffu, o.y & 0x7fff7fffu));
  };
  bool off[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) off[j] = !plain && (zero || 4 * g + j >= s.valid || St::DL * n >= D);
  if (zero || hot) {
    uint32_t w[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j][0] = st.r[j].x;
      w[j][1] = st.r[j].y;
      w[j][2] = st.r[j].z;
      w[j][3] = st.r[j].w;
      if (!plain || zero) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[j][i] = zero || off[j] ? 0u : w[j][i];
      }
    }
#pragma unroll
    for (int i = 0; i < St::DL; ++i) {
      const uint32_t sel = (i & 1) ? 0x07060302u : 0x05040100u;
      put(i, make_uint2(perm_b32(w[1][i / 2], w[0][i / 2], sel), perm_b32(w[3][i / 2], w[2][i / 2], sel)));
    }
    return largest;
  }
  float mul[4], add[4];   // value = code' * mul + add (absmax), (code - add) * mul (reference)
  uint32_t w[4][2];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
      mul[j] = off[j] ? 0.f : __uint_as_float(st.meta[0]);
      add[j] = -128.f * mul[j];
      w[j][0] = st.r[j].x ^ 0x80808080u;
      w[j][1] = st.r[j].y ^ 0x80808080u;
    } else {
      mul[j] = off[j] ? 0.f : half_hi(st.meta[j]);
      add[j] = off[j] ? 0.f : half_lo(st.meta[j]);
      w[j][0] = st.r[j].x;
      w[j][1] = st.r[j].y;
    }
  }
#pragma unroll
  for (int i = 0; i < St::DL; ++i) {
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float c = ex_byte_at(w[j][i / 4], i & 3);
      f[j] = WF == TIERKV_WARM_ABSMAX_I8 ? fmaf(c, mul[j], add[j]) : (c - add[j]) * mul[j];
    }
    put(i, make_uint2(ex_pack(f[0], f[1]), ex_pack(f[2], f[3])));
  }
  return largest;
}

// Whether a word of two magnitudes holds an infinity or NaN.
__device__ __forceinline__ bool ex_wild(uint32_t w) { return (w & 0xffffu) >= 0x7c00u || (w >> 16) >= 0x7c00u; }

// A hidden key's probability is 0, but 0 times an infinity or NaN is not: in
// tiles with hidden keys those V entries enter the product as 0 (this call,
// by the lanes that stored them) and reach the rows that see them at the end
// (ex_add_wild).  Both are rare and kept out of the tile loop's registers.
template <int DP, int TK>
__device__ __attribute__((noinline)) void ex_clear_wild(int at, ExTile<DP, TK>* t) {
  typedef ExHalf<DP> St;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int chunk = at * 2 + (g & 1), piece = g >> 1;
  uint2* const dst = reinterpret_cast<uint2*>(t->v);
#pragma unroll 1
  for (int i = 0; i < St::DL; ++i) {
    const int x = ex_v_at<TK>(St::DL * n + i, chunk) * 2 + piece;
    auto clear = [](uint32_t w) {
      if ((w & 0x7c00u) == 0x7c00u) w &= 0xffff0000u;
      if ((w & 0x7c000000u) == 0x7c000000u) w &= 0xffffu;
      return w;
    };
    const uint2 o = dst[x];
    dst[x] = make_uint2(clear(o.x), clear(o.y));
  }
}

// V of token t of a sub-tile (its row in the block), one dim, as the product
// takes it.
template <int WF>
__device__ __forceinline__ float ex_value(const ExtendParams& p, int h, const ExSub& s, int t, int d) {
  const int64_t row = (int64_t(s.slot) * p.kv_heads + h) * p.bs + s.sub * EX_SUB + t;
  if (s.state == HOT) return __half2float(p.hot_v[row * p.D + d]);
  if (s.state != WARM) return 0.f;
  const uint8_t c = p.warm_v[row * p.D + d];
  float f;
  if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
    f = float(int8_t(c)) * reinterpret_cast<const float*>(p.v_scale)[int64_t(s.slot) * p.kv_heads + h];
  } else {
    f = (float(c) - __half2float(reinterpret_cast<const __half*>(p.v_zero)[row])) *
        __half2float(reinterpret_cast<const __half*>(p.v_scale)[row]);
  }
  return __half2float(__float2half_rn(f));
}

// Sub-tiles of a list whose first ordinal is at most `limit` (ordinals grow):
// 64 samples at a time by one wave, all waves alike.
__device__ __forceinline__ int ex_visible(const int4* list, int count, int limit) {
  int lo = 0, hi = count;   // sub-tiles before lo are visible, from hi on hidden
  const int lane = threadIdx.x & 63;
  while (hi > lo) {
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const bool vis = i < hi && list[i].z <= limit;
    const int seen = __popcll(__ballot(vis));
    if (seen == 0) return lo;
    const int last = lo + (seen - 1) * step;   // visible
    hi = min(hi, last + step);
    lo = last + 1;
  }
  return lo;
}

// The first sub-tile of [lo, hi) that is not full, or not seen by every row
// (from the limit lim on): tiles before it need no masks.  By one wave.
__device__ __forceinline__ int ex_full_until(const int4* list, int lo, int hi, int lim) {
  const int lane = threadIdx.x & 63;
  for (int i0 = lo; i0 < hi; i0 += 256) {
    uint64_t odd[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = min(i0 + k * 64 + lane, hi - 1);
      const int4 v = list[i];
      odd[k] = __ballot((v.y & 0xff) != EX_SUB || v.z + EX_SUB - 1 > lim);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (odd[k]) return min(i0 + k * 64 + __ffsll((unsigned long long)odd[k]) - 1, hi);
  }
  return hi;
}

// The running state of 32 rows in a wave: lane (row = lane & 31, half = lane >> 5).
template <int DP>
struct ExAcc {
  f32x16 o[DP / 32];
  float m, l;
};

// Scheduling of a matrix product whose A operands come from LDS: AHEAD reads
// go first, then one read per product, so that no product waits for a read
// just issued (left to itself the compiler reads each operand when it is
// due: 16 LDS latencies per product chain).
template <int N, int AHEAD>
__device__ __forceinline__ void ex_pace() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);   // LDS reads
#pragma unroll
  for (int i = 0; i < N - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);     // MFMA
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// The sum of a row's query, negated, in three fp16 pieces (the sum is below
// 2^8, so what they miss is below 2^-26), by the lane's half 0.
__device__ __forceinline__ f16x8 ex_sum_pieces(float qsum) {
  asm volatile("" : "+v"(qsum));   // formed for each tile: kept over the loop they cost four registers, and it spilled
  const float v = (threadIdx.x & 32) ? 0.f : -qsum;
  const _Float16 a = _Float16(v), b = _Float16(v - float(a)), c = _Float16(v - float(a) - float(b));
  return f16x8{a, b, c, 0, 0, 0, 0, 0};
}

// Logits of one key tile, S^T = K Q^T, unscaled; reference format: with the
// zero points taken off, qsum is the sum of the row's query.
template <int DP, int WF, int TK>
__device__ __forceinline__ void ex_logits(const ExTile<DP, TK>& t, const f16x8 (&q)[DP / 16], float qsum,
                                          f32x16 (&s)[TK / 32]) {
  constexpr bool REF = WF == TIERKV_WARM_REF_U8;
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
#pragma unroll
  for (int kt = 0; kt < TK / 32; ++kt) s[kt] = f32x16{};
  const uint4* const kb = t.k + ex_k_at<DP>(col, h);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
    for (int kt = 0; kt < TK / 32; ++kt) {
      const f16x8 k = __builtin_bit_cast(f16x8, kb[kt * 32 * (DP / 8 + 1) + kk * 2]);
      s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[kk], s[kt], 0, 0, 0);
    }
  }
  if constexpr (REF) {
    const f16x8 qz = ex_sum_pieces(qsum);
#pragma unroll
    for (int kt = 0; kt < TK / 32; ++kt) {
      const f16x8 z = __builtin_bit_cast(f16x8, t.k[ex_k_at<DP>(kt * 32 + col, DP / 8)]);
      s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(z, qz, s[kt], 0, 0, 0);
    }
  }
  ex_pace<(DP / 16 + REF) * (TK / 32), 6>();
  __builtin_amdgcn_sched_barrier(0);
}

// Online softmax and output of one key tile.
//   end[i]  keys of sub-tile i that this lane's row sees (bounds on the key's
//           place in the sub-tile), used unless every row sees the whole tile
// The factor of a sub-tile's logits (K scale, softmax scale) is not negative,
// so the largest logit is the factor times the largest unscaled one and the
// factor's product joins the exponential's subtraction (absmax; the reference
// format has a factor per key and takes the product first, as masked tiles do).
template <int DP, int WF, int TK>
__device__ __forceinline__ void ex_softmax(const ExTile<DP, TK>& t, float qscale, const int (&end)[TK / 16], bool whole,
                                           f32x16 (&s)[TK / 32], ExAcc<DP>& a) {
  constexpr int KT = TK / 32;
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  float c[KT * 2];
  if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
#pragma unroll
    for (int sub = 0; sub < KT * 2; ++sub) c[sub] = t.kscale[sub] * qscale;
  } else {
#pragma unroll
    for (int sub = 0; sub < KT * 2; ++sub) {
#pragma unroll
      for (int r = 0; r < 8; ++r)
        s[sub / 2][(sub & 1) * 8 + r] *= t.kscale[sub * 16 + 8 * (r >> 2) + 4 * h + (r & 3)] * qscale;
      c[sub] = 1.f;
    }
  }
  if (!whole) {
#pragma unroll
    for (int sub = 0; sub < KT * 2; ++sub) {
      const int e = end[sub] - 4 * h;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int i = (sub & 1) * 8 + r;
        s[sub / 2][i] = (8 * (r >> 2) + (r & 3)) < e ? s[sub / 2][i] * c[sub] : -INFINITY;
      }
      c[sub] = 1.f;
    }
  }
  float mx = EX_NONE;
#pragma unroll
  for (int sub = 0; sub < KT * 2; ++sub) {
    float m = s[sub / 2][(sub & 1) * 8];
#pragma unroll
    for (int r = 1; r < 8; ++r) m = fmaxf(m, s[sub / 2][(sub & 1) * 8 + r]);
    mx = fmaxf(mx, m * c[sub]);
  }
  mx = fmaxf(mx, xor32_f(mx));
  // A row is re-based when its own maximum asks for it, so its bits do not
  // depend on the other rows of its wave.
  if (__any(mx > a.m + EX_LAZY)) {
    const float m = mx > a.m + EX_LAZY ? mx : a.m;
    const float alpha = __builtin_amdgcn_exp2f(a.m - m);
    a.m = m;
    a.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) a.o[dt][r] *= alpha;
  }
  // Probabilities of 16 keys, then their products with V^T while the next 16
  // keys' exponentials are taken and their V is read: each region below holds
  // DT products, DT reads and eight exponentials, and the schedule puts a
  // share of the others behind each product.
  const float base = EX_BOOST - a.m;
  constexpr int DT = DP / 32, SUBS = KT * 2;
  const uint4* const vb = t.v + ex_v_at<TK>(col, h);
  constexpr int VROW = 32 * (TK / 8 + 1) + 4;   // 32 rows of V^T
  f16x8 v[2][DT], pr[2];
  auto read = [&](int sub) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) v[sub & 1][dt] = __builtin_bit_cast(f16x8, vb[dt * VROW + sub * 2]);
  };
  auto probabilities = [&](int sub) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float e = __builtin_amdgcn_exp2f(fmaf(s[sub / 2][(sub & 1) * 8 + r], c[sub], base));
      a.l += e;
      pr[sub & 1][r] = _Float16(e);
    }
  };
  __builtin_amdgcn_sched_barrier(0);
  read(0);
  probabilities(0);
#pragma unroll
  for (int sub = 0; sub < SUBS; ++sub) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      a.o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[sub & 1][dt], pr[sub & 1], a.o[dt], 0, 0, 0);
    if (sub + 1 < SUBS) {
      read(sub + 1);
      probabilities(sub + 1);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 20 / DT, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, 8 / DT, 0);
      }
    }
  }
  __builtin_amdgcn_sched_barrier(0);
}

template <typename QT>
__device__ __forceinline__ uint32_t ex_out2(float a, float b) {
  const QT x = from_f32<QT>(a), y = from_f32<QT>(b);
  return uint32_t(__builtin_bit_cast(uint16_t, x)) | (uint32_t(__builtin_bit_cast(uint16_t, y)) << 16);
}

template <int DP>
constexpr int ex_lds_bytes() {
  const int wide = 2 * int(sizeof(ExTile<DP, 64>)), narrow = EX_WAVES * int(sizeof(ExTile<DP, 32>));
  const int merge = EX_WAVES * 32 * (DP + 4 + 2) * 4;
  return wide > narrow ? (wide > merge ? wide : merge) : (narrow > merge ? narrow : merge);
}

// An item: query rows of one tile, sub-tiles [part / parts) of what it sees.
//   WIDE  every wave holds 32 rows of its own and all share 64 keys at a time,
//         each wave staging the K or the V of one sub-tile; else all hold the
//         same 32 rows and each stages and takes 32 keys of its own
template <int DP, int WF, typename QT, bool WIDE>
__device__ __forceinline__ void ex_item(const ExtendParams& p, char* lds, int h, const ex_int4 it, int64_t partial) {
  constexpr int TK = WIDE ? 64 : 32;
  constexpr int NS = WIDE ? 1 : 4;          // halves a wave stages
  constexpr int KW = WIDE ? 1 : EX_WAVES;   // waves that split the keys
  const int tid = threadIdx.x, lane = tid & 63, w = ex_uniform(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int b = it.x, tile = it.y & 0x3fffffff;
  const int part = it.z & 0xffff, parts = it.z >> 16;
  const int4 seq = p.seq[b];
  const int q0 = ex_rows(p, b).x, n = seq.w, G = p.groups, D = p.D;
  const int rows = n * G;
  const int row_first = tile * EX_WIDE, row_last = min(row_first + (WIDE ? EX_WIDE : 32), rows) - 1;
  const int lim_min = seq.y - n + row_first / G, lim_max = seq.y - n + row_last / G;
  const int4* raw_list = p.subtile + int64_t(b) * p.subs_per_seq;
  const ExList list = (ExList)(uintptr_t)raw_list;

  // This lane's row.
  const int r = row_first + (WIDE ? w * 32 : 0) + col;
  const bool live = r < rows;
  const int tok = live ? r / G : 0, head = h * G + (live ? r - tok * G : 0);
  const int lim = live ? seq.y - n + tok : -1;
  f16x8 q[DP / 16];
  float qscale = fabsf(p.scale_log2);       // (its sign goes to the query)
  {
    const QT* src = reinterpret_cast<const QT*>(p.q) + int64_t(q0 + tok) * p.qs_t + int64_t(head) * p.qs_h;
    uint4 raw[DP / 16];
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const int d = kk * 16 + half * 8;
      raw[kk] = (live && d < D) ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
    }
    // bf16 rows become fp16, and the reference format needs their sum to fit it.
    constexpr bool BF = !__is_same(QT, __half);
    if constexpr (BF || WF == TIERKV_WARM_REF_U8) {
      auto lo = [](uint32_t w) { return BF ? __uint_as_float(w << 16) : half_lo(w); };
      auto hi = [](uint32_t w) { return BF ? __uint_as_float(w & 0xffff0000u) : half_hi(w); };
      float mx = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const uint32_t x[4] = {raw[kk].x, raw[kk].y, raw[kk].z, raw[kk].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mx = fmaxf(mx, fmaxf(fabsf(lo(x[i])), fabsf(hi(x[i]))));
      }
      mx = fmaxf(mx, xor32_f(mx));
      // 2^-e with mx in [2^e, 2^(e + 1)), by the exponent bits; rows of
      // zeros, infinities and the smallest normals keep their values.
      int e = int((__float_as_uint(mx) >> 23) & 0xff);
      if (e < 2 || e > 252) e = 127;
      const float inv = __uint_as_float(uint32_t(254 - e) << 23);
      qscale *= __uint_as_float(uint32_t(e) << 23);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const uint32_t x[4] = {raw[kk].x, raw[kk].y, raw[kk].z, raw[kk].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          q[kk][2 * i] = _Float16(lo(x[i]) * inv);
          q[kk][2 * i + 1] = _Float16(hi(x[i]) * inv);
        }
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) q[kk] = __builtin_bit_cast(f16x8, raw[kk]);
    }
  }
  if (p.scale_log2 < 0.f) {
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) q[kk] = -q[kk];
  }
  float qsum = 0.f;
  if constexpr (WF == TIERKV_WARM_REF_U8) {
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
      for (int i = 0; i < 8; ++i) qsum += float(q[kk][i]);
    qsum += xor32_f(qsum);
  }
  ExAcc<DP> a;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) a.o[dt] = f32x16{};
  a.m = EX_NONE;
  a.l = 0.f;
  if (part == 0 && seq.z > 0 && (KW == 1 || w == 0)) {   // COLD tokens with logit 0 that every row sees
    a.m = 0.f;
    a.l = half == 0 ? float(seq.z) * exp2f(EX_BOOST) : 0.f;
  }

  const int visible = ex_uniform(ex_visible(raw_list, seq.x, lim_max));
  constexpr int ROUND = TK / 16 * KW;       // sub-tiles per round of the workgroup
  const int chunk = ((visible + parts - 1) / parts + ROUND - 1) & ~(ROUND - 1);
  const int lo = min(part * chunk, visible), hi = min(lo + chunk, visible);

  // Wide: two tiles in LDS; the next tile is stored while this one is taken,
  // and the one after it loads.  Narrow: a tile per wave, stored between its
  // steps in the wave's own order.
  ExTile<DP, TK>* tiles = reinterpret_cast<ExTile<DP, TK>*>(lds);
  const int first = WIDE ? lo : lo + w * (TK / 16);
  ExHalf<DP> st[NS];
  ExSub sub[WIDE ? 1 : 2];
  bool wild = false;
  auto find = [&](int at) {
    if constexpr (WIDE) {
      sub[0] = ex_sub(list, min(at, hi) + (w & 3), hi);
    } else {
      sub[0] = ex_sub(list, min(at, hi), hi);
      sub[1] = ex_sub(list, min(at, hi) + 1, hi);
    }
  };
  auto load = [&]() {
    if constexpr (WIDE) {
      if (w < 4) ex_load<DP, WF, 0>(p, h, sub[0], st[0]);
      else ex_load<DP, WF, 1>(p, h, sub[0], st[0]);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ex_load<DP, WF, 0>(p, h, sub[i], st[2 * i]);
        ex_load<DP, WF, 1>(p, h, sub[i], st[2 * i + 1]);
      }
    }
  };
  auto store_v = [&](ExTile<DP, TK>& t, const ExSub& of, const ExHalf<DP>& v, int place, bool whole) {
    const uint32_t largest = ex_store_v<DP, WF, TK>(p, of, v, place, !whole, t);
    if (!whole && __any(ex_wild(largest))) {
      ex_clear_wild<DP, TK>(place, &t);
      wild = true;
    }
  };
  auto store = [&](ExTile<DP, TK>& t, const auto& of, bool whole) {
    if constexpr (WIDE) {
      if (w < 4) ex_store_k<DP, WF, TK>(p, of[0], st[0], w, t);
      else store_v(t, of[0], st[0], w - 4, whole);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ex_store_k<DP, WF, TK>(p, of[i], st[2 * i], i, t);
        store_v(t, of[i], st[2 * i + 1], i, whole);
      }
    }
  };
  if constexpr (WIDE) {
    // The two waves of a SIMD work half a tile apart: while waves 0-3 form a
    // tile's logits, waves 4-7 take the softmax and the output of the tile
    // before, so one's matrix products run beside the other's exponentials
    // (in step, the products and the exponentials of all waves came one after
    // the other: 1313 us at 2048 tokens on 32768). Waves 0-3 stage K, 4-7 V.
    const bool idle = row_first + w * 32 >= rows;   // a wave without rows only stages
    const int tiles_n = (hi - lo + 3) / 4;
    int full = 0;
    if (tiles_n > 0) {
      full = ex_uniform(ex_full_until(raw_list, lo, hi, lim_min));
      find(lo);
      load();
      store(tiles[0], sub, lo + 4 <= full);
      find(lo + 4);
      load();
      __syncthreads();
    }
    auto output = [&](int at, f32x16 (&s)[TK / 32], const ExTile<DP, TK>& t) {
      const bool whole = at + 4 <= full;
      int end[TK / 16] = {};
      if (!whole) ex_ends<TK>(list, at, hi, lim, end);
      ex_softmax<DP, WF, TK>(t, qscale, end, whole, s, a);
    };
    // Two barriers per tile; every wave meets 2 tiles_n + 1 of them.
    int buf = 0;
    if (w < 4) {
      for (int at = lo; at < hi; at += 4, buf ^= 1) {
        f32x16 s[TK / 32];
        if (!idle) ex_logits<DP, WF, TK>(tiles[buf], q, qsum, s);
        __syncthreads();
        if (at + 4 < hi) {
          ex_store_k<DP, WF, TK>(p, sub[0], st[0], w, tiles[buf ^ 1]);
          find(at + 8);
          ex_load<DP, WF, 0>(p, h, sub[0], st[0]);
        }
        if (!idle) output(at, s, tiles[buf]);
        __syncthreads();
      }
      __syncthreads();
    } else {
      __syncthreads();
      for (int at = lo; at < hi; at += 4, buf ^= 1) {
        f32x16 s[TK / 32];
        if (!idle) ex_logits<DP, WF, TK>(tiles[buf], q, qsum, s);
        if (at + 4 < hi) {
          store_v(tiles[buf ^ 1], sub[0], st[0], w - 4, at + 8 <= full);
          find(at + 8);
          ex_load<DP, WF, 1>(p, h, sub[0], st[0]);
        }
        __syncthreads();
        if (!idle) output(at, s, tiles[buf]);
        __syncthreads();
      }
    }
  } else if (first < hi) {
    const int full = ex_uniform(ex_full_until(raw_list, lo, hi, lim_min));
    find(first);
    load();
    store(tiles[w], sub, first + TK / 16 <= full);
    find(first + ROUND);
    load();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int at = first; at < hi; at += ROUND) {
      const bool whole = at + TK / 16 <= full;
      ExSub held[2];
      held[0] = sub[0];
      held[1] = sub[WIDE ? 0 : 1];
      find(at + 2 * ROUND);
      f32x16 s[TK / 32];
      ex_logits<DP, WF, TK>(tiles[w], q, qsum, s);
      int end[TK / 16] = {};
      if (!whole) ex_ends<TK>(list, at, hi, lim, end);
      ex_softmax<DP, WF, TK>(tiles[w], qscale, end, whole, s, a);
      if (at + ROUND < hi) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        store(tiles[w], held, at + ROUND + TK / 16 <= full);
        load();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    }
  }
  // Infinities and NaN of the tiles with hidden keys, for the rows that see them.
  if constexpr (WIDE) wild = __syncthreads_or(wild);
  if (wild) {
    const int full = ex_full_until(raw_list, lo, hi, lim_min);
#pragma unroll 1
    for (int at = first; at < hi; at += ROUND) {
      if (at + TK / 16 <= full) continue;
#pragma unroll 1
      for (int k = 0; k < TK / 16; ++k) {
        const ExSub sb = ex_sub(list, at + k, hi);
#pragma unroll 1
        for (int x = 0; x < min(sb.valid, lim - sb.ordinal + 1); ++x) {
#pragma unroll
          for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int d = dt * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
              const float v = d < D ? ex_value<WF>(p, h, sb, x, d) : 0.f;
              if (!(fabsf(v) < INFINITY)) a.o[dt][i] += v;
            }
        }
      }
    }
  }

  a.l += xor32_f(a.l);
  if constexpr (KW > 1) {
    // The waves' states of the same rows meet in LDS: 32 rows of DP sums each.
    __syncthreads();
    float* so = reinterpret_cast<float*>(lds);
    float* sml = so + KW * 32 * (DP + 4);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 v = {a.o[dt][4 * i], a.o[dt][4 * i + 1], a.o[dt][4 * i + 2], a.o[dt][4 * i + 3]};
        *reinterpret_cast<f32x4*>(so + (w * 32 + col) * (DP + 4) + dt * 32 + 8 * i + 4 * half) = v;
      }
    if (half == 0) {
      sml[(w * 32 + col) * 2] = a.m;
      sml[(w * 32 + col) * 2 + 1] = a.l;
    }
    __syncthreads();
    // Row x / (DP / 4), dims 4 (x % (DP / 4)) ..
    for (int x = tid; x < 32 * (DP / 4); x += EX_THREADS) {
      const int rr = x / (DP / 4), d = 4 * (x % (DP / 4));
      float m = EX_NONE;
#pragma unroll
      for (int k = 0; k < KW; ++k) m = fmaxf(m, sml[(k * 32 + rr) * 2]);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const float c = __builtin_amdgcn_exp2f(sml[(k * 32 + rr) * 2] - m);
        if (c > 0.f) {   // (a state of no weight may hold an infinity's product)
          l += sml[(k * 32 + rr) * 2 + 1] * c;
          o += *reinterpret_cast<const f32x4*>(so + (k * 32 + rr) * (DP + 4) + d) * c;
        }
      }
      const int row = row_first + rr;
      if (row >= rows || d >= D) continue;
      if (partial >= 0) {
        const int64_t at = (partial * p.kv_heads + h) * p.part_rows + rr;
        *reinterpret_cast<f32x4*>(p.part_o + at * D + d) = o;
        if (d == 0) {
          p.part_ml[at * 2] = m;
          p.part_ml[at * 2 + 1] = l;
        }
      } else {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        const int tk = row / G, hd = h * G + row - tk * G;
        QT* dst = reinterpret_cast<QT*>(p.out) + (int64_t(q0 + tk) * p.heads + hd) * D + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(ex_out2<QT>(o[0] * inv, o[1] * inv), ex_out2<QT>(o[2] * inv, o[3] * inv));
      }
    }
  } else {
    if (!live) return;
    if (partial >= 0) {
      const int64_t at = (partial * p.kv_heads + h) * p.part_rows + (r - row_first);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = dt * 32 + 8 * i + 4 * half;
          const f32x4 v = {a.o[dt][4 * i], a.o[dt][4 * i + 1], a.o[dt][4 * i + 2], a.o[dt][4 * i + 3]};
          if (d < D) *reinterpret_cast<f32x4*>(p.part_o + at * D + d) = v;
        }
      if (half == 0) {
        p.part_ml[at * 2] = a.m;
        p.part_ml[at * 2 + 1] = a.l;
      }
    } else {
      const float inv = a.l > 0.f ? 1.f / a.l : (a.l == 0.f ? 0.f : a.l);
      QT* dst = reinterpret_cast<QT*>(p.out) + (int64_t(q0 + tok) * p.heads + head) * D;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = dt * 32 + 8 * i + 4 * half;
          if (d < D)
            *reinterpret_cast<uint2*>(dst + d) =
                make_uint2(ex_out2<QT>(a.o[dt][4 * i] * inv, a.o[dt][4 * i + 1] * inv),
                           ex_out2<QT>(a.o[dt][4 * i + 2] * inv, a.o[dt][4 * i + 3] * inv));
        }
    }
  }
}

// MIXED: calls that may hold wide tiles; the others' kernel is without their code.
template <int DP, int WF, typename QT, bool MIXED>
__global__ __launch_bounds__(EX_THREADS, 2) void extend_kernel(ExtendParams p) {
  extern __shared__ __attribute__((aligned(16))) char ex_lds[];
  const int i = int(blockIdx.x) / p.kv_heads, h = int(blockIdx.x) - i * p.kv_heads;
  if (i >= p.head[0]) return;
  const ex_int4 it = ((ExList)(uintptr_t)p.item)[i];
  if (it.x < 0) return;
  if (MIXED && (it.y & (1 << 30))) ex_item<DP, WF, QT, true>(p, ex_lds, h, it, it.w);
  else ex_item<DP, WF, QT, false>(p, ex_lds, h, it, it.w);
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
  float m = EX_NONE, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < parts; k0 += AHEAD) {
    float2 ml[AHEAD];
    f32x4 v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t x = at + min(k0 + k, parts - 1) * step;
      ml[k] = reinterpret_cast<const float2*>(p.part_ml)[x];
      v[k] = *reinterpret_cast<const f32x4*>(p.part_o + x * D + d);
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) top = fmaxf(top, ml[k].x);
    const float f0 = __builtin_amdgcn_exp2f(m - top);
    m = top;
    l *= f0;
    o *= f0;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const float f = k0 + k < parts ? __builtin_amdgcn_exp2f(ml[k].x - m) : 0.f;
      if (f > 0.f) {   // (a partial of no weight may hold an infinity's product)
        l += ml[k].y * f;
        o += v[k] * f;
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const int tk = row / G, hd = h * G + row - tk * G;
  QT* dst = reinterpret_cast<QT*>(p.out) + (int64_t(ex_rows(p, b).x + tk) * p.heads + hd) * D + d;
  *reinterpret_cast<uint2*>(dst) = make_uint2(ex_out2<QT>(o[0] * inv, o[1] * inv), ex_out2<QT>(o[2] * inv, o[3] * inv));
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
  if (num_rows < 0 || max_tokens < 0) return fail(TIERKV_ERR_INVALID, "negative row counts");
  if (!cu_tokens || !block_table || !block_states || !block_lengths || !workspace ||
      (num_rows > 0 && (!query || !out)))
    return fail(TIERKV_ERR_INVALID, "null tensor pointer");
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(TIERKV_ERR_INVALID, "num_heads must be a positive multiple of num_kv_heads");
  if (num_blocks <= 0) return fail(TIERKV_ERR_INVALID, "num_blocks must be positive.");
  if (num_blocks > table_stride) return fail(TIERKV_ERR_INVALID, "num_blocks exceeds the provided block table length.");
  if (query_dtype != TIERKV_DTYPE_F16 && query_dtype != TIERKV_DTYPE_BF16)
    return fail(TIERKV_ERR_INVALID, "query dtype must be fp16 or bf16");
  if (warm_format != TIERKV_WARM_REF_U8 && warm_format != TIERKV_WARM_ABSMAX_I8)
    return fail(TIERKV_ERR_INVALID, "unknown warm format");
  if (cold_mode != TIERKV_COLD_ZERO_LOGIT && cold_mode != TIERKV_COLD_MASKED)
    return fail(TIERKV_ERR_INVALID, "unknown cold mode");
  if (block_size <= 0 || block_size > 64 || head_dim <= 0 || head_dim > 128 || head_dim % 8 != 0)
    return fail(TIERKV_ERR_UNSUPPORTED, "block_size must be in [1, 64] and head_dim a multiple of 8 up to 128");
  if (!hot_k || !hot_v || hot_slots <= 0) return fail(TIERKV_ERR_INVALID, "HOT pools are required");
  if (!warm_k || !warm_v || !k_scale || !v_scale || warm_slots <= 0)
    return fail(TIERKV_ERR_INVALID, "WARM pools and scales are required (pass 1-slot placeholders when empty)");
  if (warm_format == TIERKV_WARM_REF_U8 && (!k_zero || !v_zero))
    return fail(TIERKV_ERR_INVALID, "reference-format WARM pools need zero points");
  if (!std::isfinite(scaling)) return fail(TIERKV_ERR_INVALID, "scaling must be finite");
  if (q_stride_t < 0 || q_stride_h < 0 || q_stride_t % 8 != 0 || q_stride_h % 8 != 0)
    return fail(TIERKV_ERR_INVALID, "query strides must be non-negative multiples of 8 elements");
  if (!aligned16(query) || !aligned16(out) || !aligned16(hot_k) || !aligned16(hot_v) || !aligned16(warm_k) ||
      !aligned16(warm_v) || !aligned16(workspace))
    return fail(TIERKV_ERR_INVALID, "query, out, pools and workspace must be 16-byte aligned");
  if (int64_t(num_blocks) * block_size > 0x7fffffff - EX_SUB)
    return fail(TIERKV_ERR_UNSUPPORTED, "rows of 2^31 tokens or more");
  if (batch > EX_MAX_BATCH) return fail(TIERKV_ERR_UNSUPPORTED, "more than 4096 requests");
  const int groups = num_heads / num_kv_heads;
  if (int64_t(num_rows) * groups > (int64_t(1) << 29))
    return fail(TIERKV_ERR_UNSUPPORTED, "more than 2^29 query rows per kv head");
  const ExLayout l = ex_layout(batch, num_rows, max_tokens, groups, num_kv_heads, num_blocks, block_size, head_dim);
  // (a launch has fewer than 2^32 threads)
  if (int64_t(l.max_items) * num_kv_heads > 0xffffffffll / EX_THREADS) return fail(TIERKV_ERR_UNSUPPORTED, "grid too large");
  if (workspace_bytes < l.total) return fail(TIERKV_ERR_WORKSPACE, "workspace too small");
  if (num_rows == 0 || max_tokens == 0) return TIERKV_OK;
  char* ws = reinterpret_cast<char*>(workspace);
  ExtendParams p{};
  p.q = query;
  p.qs_t = q_stride_t;
  p.qs_h = q_stride_h;
  p.out = out;
  p.cu = cu_tokens;
  p.rows = num_rows;
  p.max_tokens = max_tokens;
  p.table = block_table;
  p.states = block_states;
  p.lengths = block_lengths;
  p.stride = table_stride;
  p.seq_nblocks = seq_num_blocks;
  p.num_blocks = num_blocks;
  p.hot_k = reinterpret_cast<const __half*>(hot_k);
  p.hot_v = reinterpret_cast<const __half*>(hot_v);
  p.hot_slots = hot_slots;
  p.warm_k = reinterpret_cast<const uint8_t*>(warm_k);
  p.warm_v = reinterpret_cast<const uint8_t*>(warm_v);
  p.warm_slots = warm_slots;
  p.k_scale = k_scale;
  p.k_zero = k_zero;
  p.v_scale = v_scale;
  p.v_zero = v_zero;
  p.batch = batch;
  p.heads = num_heads;
  p.kv_heads = num_kv_heads;
  p.bs = block_size;
  p.D = head_dim;
  p.groups = groups;
  p.cold_zero = cold_mode == TIERKV_COLD_ZERO_LOGIT;
  p.scale_log2 = scaling * EX_LOG2E;
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
