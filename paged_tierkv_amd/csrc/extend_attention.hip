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
//     into tiles and cuts the tiles' key ranges into items of about equal
//     work, about as many as the chip runs at once;
//   * extend_kernel, a workgroup of four waves per (item, kv head);
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
// ("wide") are 128 rows over four waves that share 64 keys at a time; smaller
// ones ("narrow") give each wave its own 32 keys of the same rows, merged in LDS.
//
// K goes to LDS as fp16 of the codes themselves (exact: |code| <= 127, or
// code - zero, an integer below 2048 for any row whose values are not far
// from 0 against their spread), and the scale is applied to the logits in 32 bits.
// V goes to LDS as fp16 of code * scale, one rounding of at most 2^-11 of the
// value, as the probabilities have one when they become fp16 operands.
// Probabilities carry a factor 2^6 so that small ones stay normal fp16.
// bf16 queries become fp16 after division by a power of two near the row's
// largest value, which the logits get back in 32 bits.

#include "tierkv_common.h"

#include <algorithm>
#include <cmath>

namespace tierkv {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int EX_THREADS = 256;
constexpr int EX_PLAN = 512;              // threads of a plan workgroup
constexpr int EX_SUB = 16;                // tokens per sub-tile
constexpr int EX_NARROW = 32;             // rows of a narrow tile
constexpr int EX_WIDE = 128;              // rows of a wide tile
constexpr int EX_TARGET = 1024;           // workgroups that the cut aims at
constexpr int EX_MIN_SUBS = 8;            // sub-tiles per item, at least, when a tile is cut
constexpr int EX_WS_HEAD = 256 + (1 << 16) * 4;   // the decode launches' error word and counters
constexpr float EX_LAZY = 8.f;            // log2 headroom of the running maximum
constexpr float EX_BOOST = 6.f;           // log2 of the probabilities' factor
constexpr float EX_NONE = -1e30f;         // running maximum before the first visible key
constexpr float EX_LOG2E = 1.4426950408889634f;
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
  int4* seq;           // [batch] {sub-tiles, tokens L, COLD tokens that every row sees, query rows n}
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

template <int NW>
__device__ __forceinline__ int ex_scan(int v, int* sh, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int x = wave_inclusive_scan(v);
  if (lane == 63) sh[w] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int t = sh[i];
    before += i < w ? t : 0;
    all += t;
  }
  __syncthreads();
  *total = all;
  return x + before;
}

// Query rows of request b: its packed range, clamped to the rows there are.
__device__ __forceinline__ int2 ex_rows(const ExtendParams& p, int b) {
  const int lo = min(max(p.cu[b], 0), p.rows), hi = min(max(p.cu[b + 1], lo), p.rows);
  return make_int2(lo, min(hi - lo, p.max_tokens));
}

__device__ __forceinline__ int ex_tiles(int rows) { return rows <= EX_NARROW ? (rows > 0) : (rows + EX_WIDE - 1) / EX_WIDE; }

// Sub-tiles that a tile's last row sees, within one of each sub-tile
// behind it: exact when the tokens after it fill whole sub-tiles.
__device__ __forceinline__ int ex_work(const int4 s, int tile, bool wide, int groups) {
  if (s.x == 0) return 1;
  const int rows = s.w * groups;
  const int last = wide ? min((tile + 1) * EX_WIDE, rows) - 1 : rows - 1;
  const int hidden = s.w - 1 - last / groups;
  return max(s.x - hidden / EX_SUB, 1);
}

__global__ __launch_bounds__(EX_PLAN) void extend_plan_kernel(ExtendParams p) {
  constexpr int NW = EX_PLAN / 64;
  __shared__ int sh[NW];
  __shared__ int s_last;
  const int tid = threadIdx.x, b = blockIdx.x;
  int nb = p.num_blocks;
  if (p.seq_nblocks) nb = min(max(p.seq_nblocks[b], 0), p.num_blocks);
  const int64_t row = int64_t(b) * p.stride;
  const int n = ex_rows(p, b).y;
  // Tokens of the row first: COLD sub-tiles need the distance to its end.
  int len_sum = 0;
  for (int i = tid; i < nb; i += EX_PLAN) len_sum += min(max(p.lengths[row + i], 0), p.bs);
  int tokens;
  ex_scan<NW>(len_sum, sh, &tokens);
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
    int total;
    const int first = ordinal + ex_scan<NW>(len, sh, &total) - len;
    ordinal += total;
    int mine_cold = 0;
    if (len > 0) {
      if (state == HOT || state == WARM) {
        const int64_t slots = state == HOT ? p.hot_slots : p.warm_slots;
        if (slot >= 0 && slot < slots) keep = 1;
        else atomicOr(p.err, 1);
      } else if (state != COLD) {
        atomicOr(p.err, 2);
      } else if (p.cold_zero) {
        // Seen by every row: a count.  Else a sub-tile of zeros, masked like others.
        if (first + len <= tokens - n + 1) mine_cold = len;
        else keep = 1;
      }
    }
    const int count = keep ? (len + EX_SUB - 1) / EX_SUB : 0;
    const int pos = at + ex_scan<NW>(count, sh, &total) - count;
    at += total;
    ex_scan<NW>(mine_cold, sh, &total);
    cold += total;
    const int code = state == COLD ? EX_STATE_ZERO : state;
    for (int j = 0; j < count; ++j)
      out[pos + j] = make_int4(slot, min(len - j * EX_SUB, EX_SUB) | (code << 8) | (j << 16), first + j * EX_SUB, 0);
  }
  if (tid == 0) {
    // Relaxed agent-scope stores: the last workgroup reads them from another XCD's cache.
    int32_t* s = reinterpret_cast<int32_t*>(p.seq + b);
    const int v[4] = {at, tokens, cold, n};
    for (int k = 0; k < 4; ++k) __hip_atomic_store(s + k, v[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    s_last = __hip_atomic_fetch_add(p.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u == gridDim.x;
  }
  __syncthreads();
  if (!s_last) return;
  if (tid == 0) __hip_atomic_store(p.arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  auto seq_of = [&](int i) -> int4 {
    int32_t* s = reinterpret_cast<int32_t*>(p.seq + i);
    int4 v;
    v.x = __hip_atomic_load(s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    v.y = 0;
    v.z = 0;
    v.w = __hip_atomic_load(s + 3, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return v;
  };
  // Total work, then sub-tiles per item.
  float work = 0.f;
  for (int i = tid; i < p.batch; i += EX_PLAN) {
    const int4 s = seq_of(i);
    const int tiles = ex_tiles(s.w * p.groups);
    const bool wide = s.w * p.groups > EX_NARROW;
    // At least the sum of the tiles' works: each is at most g(t) = max(f(t), 1)
    // with f linear, g is convex, and a convex sum lies below its chord's.
    if (tiles > 0) {
      auto g = [&](int t) {
        const float last = wide ? float(t + 1) * EX_WIDE : float(s.w * p.groups);
        return fmaxf(float(s.x) + 1.f - fmaxf(float(s.w) - 1.f - last / float(p.groups), 0.f) / EX_SUB, 1.f);
      };
      work += 0.5f * (g(0) + g(tiles - 1)) * float(tiles);
    }
  }
  __shared__ float s_work[NW];
  work = wave_sum(work);
  if ((tid & 63) == 0) s_work[tid >> 6] = work;
  __syncthreads();
  work = 0.f;
  for (int i = 0; i < NW; ++i) work += s_work[i];
  work = work * 1.001f + 1.f;   // the rounding of these sums
  const int target = max(EX_TARGET / p.kv_heads, 1);
  const int per_item = max(EX_MIN_SUBS, (int(ceilf(work / float(target))) + 3) & ~3);
  // Items, request by request; each request's longest tiles first.
  int items = 0, cuts = 0, partials = 0;
  for (int i0 = 0; i0 < p.batch; i0 += EX_PLAN) {
    const int i = i0 + tid;
    int4 s = make_int4(0, 0, 0, 0);
    if (i < p.batch) s = seq_of(i);
    const int tiles = ex_tiles(s.w * p.groups);
    const bool wide = s.w * p.groups > EX_NARROW;
    int mine = 0, mine_cut = 0, mine_part = 0;
    for (int t = 0; t < tiles; ++t) {
      const int parts = min((ex_work(s, t, wide, p.groups) + per_item - 1) / per_item, 32767);
      mine += parts;
      if (parts > 1) {
        ++mine_cut;
        mine_part += parts;
      }
    }
    int total;
    int at_item = items + ex_scan<NW>(mine, sh, &total) - mine;
    items += total;
    int at_cut = cuts + ex_scan<NW>(mine_cut, sh, &total) - mine_cut;
    cuts += total;
    int at_part = partials + ex_scan<NW>(mine_part, sh, &total) - mine_part;
    partials += total;
    for (int t = tiles - 1; t >= 0; --t) {
      const int parts = min((ex_work(s, t, wide, p.groups) + per_item - 1) / per_item, 32767);
      // The host's bounds hold for packed ranges that do not overlap; items of others may be left out (-1).
      const bool fits = at_item + parts <= p.max_items &&
                        (parts == 1 || (at_cut < p.max_cut && at_part + parts <= p.max_part));
      for (int k = 0; k < parts; ++k)
        if (at_item + k < p.max_items)
          p.item[at_item + k] = make_int4(fits ? i : -1, t | (wide ? 1 << 30 : 0), k | (parts << 16),
                                          parts > 1 ? at_part + k : -1);
      if (parts > 1) {
        if (at_cut < p.max_cut) p.cut[at_cut] = make_int2(at_part, fits ? at_item : -1);
        ++at_cut;
        at_part += parts;
      }
      at_item += parts;
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

// A sub-tile's K and V in registers, as loaded.
//   k: piece x = lane + 64 i of the 16 rows' 8-element pieces (row x / (DP / 8));
//   v: keys 4g + j (g = lane >> 4, j = 0..3), dims DL n .. DL n + DL - 1 (n = lane & 15),
//      in units of up to 8 dims.
template <int DP>
struct ExStage {
  static constexpr int NPK = DP / 32;            // K pieces per lane
  static constexpr int DL = DP / 16;             // V dims per lane
  static constexpr int U = DL / 8 > 0 ? DL / 8 : 1;   // V units per row
  static constexpr int UD = DL < 8 ? DL : 8;     // dims per unit
  uint4 k[NPK];
  uint4 v[4][U];
  float kmeta[NPK][2];    // REF_U8: zero and scale of the piece's token; absmax: scale in [0][0]
  float vmeta[4][2];      // REF_U8: of key 4g + j; absmax: scale in [0][0]
};

struct ExSub {
  int slot, valid, state, sub, ordinal;
};

__device__ __forceinline__ ExSub ex_sub(const int4* list, int i, int end) {
  ExSub s;
  s.valid = 0;
  s.state = EX_STATE_ZERO;
  s.slot = s.sub = 0;
  s.ordinal = 0;
  if (i < end) {
    const int4 v = list[i];
    s.slot = ex_uniform(v.x);
    const int y = ex_uniform(v.y);
    s.valid = y & 0xff;
    s.state = (y >> 8) & 0xff;
    s.sub = y >> 16;
    s.ordinal = ex_uniform(v.z);
  }
  return s;
}

// Whether every row of an item sees every key of the TK keys from sub-tile `at` on.
template <int TK>
__device__ __forceinline__ bool ex_whole(const int4* list, int at, int end, int lim_min) {
  bool whole = true;
#pragma unroll
  for (int i = 0; i < TK / 16; ++i) {
    const ExSub s = ex_sub(list, at + i, end);
    whole = whole && s.valid == EX_SUB && s.ordinal + EX_SUB - 1 <= lim_min;
  }
  return whole;
}

template <int DP, int WF>
__device__ __forceinline__ void ex_load(const ExtendParams& p, int h, const ExSub& s, ExStage<DP>& st) {
  typedef ExStage<DP> St;
  if (s.state == EX_STATE_ZERO) return;
  const int lane = threadIdx.x & 63;
  const int D = p.D, bs = p.bs;
  const int t0 = s.sub * EX_SUB;
  const int64_t tile = (int64_t(s.slot) * p.kv_heads + h) * bs;   // the block's first row of this head
  const int n = lane & 15, g = lane >> 4;
  if (s.state == HOT) {
#pragma unroll
    for (int i = 0; i < St::NPK; ++i) {
      const int x = lane + 64 * i, r = min(t0 + x / (DP / 8), bs - 1);
      const int c = x % (DP / 8);
      st.k[i] = *reinterpret_cast<const uint4*>(p.hot_k + (tile + r) * D + (c * 8 < D ? c * 8 : 0));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = min(t0 + 4 * g + j, bs - 1);
#pragma unroll
      for (int u = 0; u < St::U; ++u) {
        const int d = St::DL * n + 8 * u;
        const __half* src = p.hot_v + (tile + r) * D + (d < D ? d : 0);
        if constexpr (St::UD == 8) st.v[j][u] = *reinterpret_cast<const uint4*>(src);
        else {
          const uint2 w = *reinterpret_cast<const uint2*>(src);
          st.v[j][u].x = w.x;
          st.v[j][u].y = w.y;
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < St::NPK; ++i) {
    const int x = lane + 64 * i, r = min(t0 + x / (DP / 8), bs - 1);
    const int c = x % (DP / 8);
    const uint2 w = *reinterpret_cast<const uint2*>(p.warm_k + (tile + r) * D + (c * 8 < D ? c * 8 : 0));
    st.k[i].x = w.x;
    st.k[i].y = w.y;
    if constexpr (WF == TIERKV_WARM_REF_U8) {
      st.kmeta[i][0] = __half2float(reinterpret_cast<const __half*>(p.k_zero)[tile + r]);
      st.kmeta[i][1] = __half2float(reinterpret_cast<const __half*>(p.k_scale)[tile + r]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = min(t0 + 4 * g + j, bs - 1);
#pragma unroll
    for (int u = 0; u < St::U; ++u) {
      const int d = St::DL * n + 8 * u;
      const uint8_t* src = p.warm_v + (tile + r) * D + (d < D ? d : 0);
      if constexpr (St::UD == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(src);
        st.v[j][u].x = w.x;
        st.v[j][u].y = w.y;
      } else {
        st.v[j][u].x = *reinterpret_cast<const uint32_t*>(src);
      }
    }
    if constexpr (WF == TIERKV_WARM_REF_U8) {
      st.vmeta[j][0] = __half2float(reinterpret_cast<const __half*>(p.v_zero)[tile + r]);
      st.vmeta[j][1] = __half2float(reinterpret_cast<const __half*>(p.v_scale)[tile + r]);
    }
  }
  if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
    const int64_t m = int64_t(s.slot) * p.kv_heads + h;
    st.kmeta[0][0] = reinterpret_cast<const float*>(p.k_scale)[m];
    st.vmeta[0][0] = reinterpret_cast<const float*>(p.v_scale)[m];
  }
}

// LDS of one key tile of TK keys.
template <int DP, int TK>
struct ExTile {
  // K rows of DP halves; 16-byte chunk c of row r at chunk c ^ swizzle(r): the
  // 16 lanes that read one chunk column of 16 rows touch all 64 banks.
  uint4 k[TK * DP / 8];
  // V^T rows of TK halves; chunk c of row d at c ^ swizzle(d).
  uint4 v[DP * TK / 8];
  float kscale[TK];       // factor of each key's logits (REF_U8; absmax: one per sub-tile)
};

template <int DP>
__device__ __forceinline__ int ex_k_at(int r, int c) {
  constexpr int C = DP / 8;
  const int s = C >= 16 ? (r & 15) : ((r >> 1) & 7);
  return r * C + (c ^ s);
}

template <int TK>
__device__ __forceinline__ int ex_v_at(int d, int c) {
  constexpr int C = TK / 8;
  const int s = C == 8 ? (((d >> 1) ^ (d >> 4)) & 7) : (((d >> 2) ^ (d >> 4)) & 3);
  return d * C + (c ^ s);
}

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

// Write a loaded sub-tile into sub-tile place `at` (0 .. TK / 16 - 1) of a
// tile; returns the largest magnitude bits of its V (two halves).
template <int DP, int WF, int TK>
__device__ __forceinline__ uint32_t ex_store(const ExtendParams& p, const ExSub& s, const ExStage<DP>& st, int at,
                                         ExTile<DP, TK>& t) {
  typedef ExStage<DP> St;
  const int lane = threadIdx.x & 63, D = p.D;
  const int n = lane & 15, g = lane >> 4;
  const bool zero = s.state == EX_STATE_ZERO, hot = s.state == HOT;
#pragma unroll
  for (int i = 0; i < St::NPK; ++i) {
    const int x = lane + 64 * i, r = x / (DP / 8), c = x % (DP / 8);
    uint4 v = st.k[i];
    if (zero || c * 8 >= D) {
      v = make_uint4(0, 0, 0, 0);
    } else if (!hot) {
      f16x4 a, b;
      f16x4 off;
      if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
        a = i8x4_plus1152(v.x);
        b = i8x4_plus1152(v.y);
        off = f16x4{1152, 1152, 1152, 1152};
        a -= off;
        b -= off;
      } else {
        off = f16x4{1024, 1024, 1024, 1024};
        const _Float16 z = _Float16(st.kmeta[i][0]);
        a = u8x4_plus1024(v.x) - off;
        b = u8x4_plus1024(v.y) - off;
        a -= f16x4{z, z, z, z};
        b -= f16x4{z, z, z, z};
      }
      const uint2 lo = __builtin_bit_cast(uint2, a), hi = __builtin_bit_cast(uint2, b);
      v = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    t.k[ex_k_at<DP>(at * EX_SUB + r, c)] = v;
    if constexpr (WF == TIERKV_WARM_REF_U8) {
      if (c == 0) t.kscale[at * EX_SUB + r] = (zero || hot) ? 1.f : st.kmeta[i][1];
    }
  }
  if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
    if (lane == 0) t.kscale[at] = (zero || hot) ? 1.f : st.kmeta[0][0];
  }
  // V^T: the lane's four keys side by side, for each of its dims.
  uint2* const dst = reinterpret_cast<uint2*>(t.v);
  const int chunk = at * 2 + (g & 1), piece = g >> 1;
  uint32_t largest = 0;
  auto put = [&](int d, uint2 o) {
    dst[ex_v_at<TK>(d, chunk) * 2 + piece] = o;
    largest = ex_max_u16(largest, ex_max_u16(o.x & 0x7fff7fffu, o.y & 0x7fff7fffu));
  };
#pragma unroll
  for (int u = 0; u < St::U; ++u) {
    uint32_t w[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool off = zero || 4 * g + j >= s.valid || St::DL * n + 8 * u >= D;
      w[j][0] = off ? 0u : st.v[j][u].x;
      w[j][1] = off ? 0u : st.v[j][u].y;
      w[j][2] = off ? 0u : st.v[j][u].z;
      w[j][3] = off ? 0u : st.v[j][u].w;
    }
    if (zero || hot) {
#pragma unroll
      for (int i = 0; i < St::UD; ++i) {
        const uint32_t sel = (i & 1) ? 0x07060302u : 0x05040100u;
        put(St::DL * n + 8 * u + i,
            make_uint2(perm_b32(w[1][i / 2], w[0][i / 2], sel), perm_b32(w[3][i / 2], w[2][i / 2], sel)));
      }
    } else {
      float mul[4], add[4];   // value = code' * mul + add (absmax), (code - add) * mul (reference)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool off = 4 * g + j >= s.valid || St::DL * n + 8 * u >= D;
        if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
          mul[j] = off ? 0.f : st.vmeta[0][0];
          add[j] = -128.f * mul[j];
        } else {
          mul[j] = off ? 0.f : st.vmeta[j][1];
          add[j] = off ? 0.f : st.vmeta[j][0];
        }
      }
#pragma unroll
      for (int i = 0; i < St::UD; ++i) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (WF == TIERKV_WARM_ABSMAX_I8)
            f[j] = fmaf(ex_byte_at(w[j][i / 4] ^ 0x80808080u, i & 3), mul[j], add[j]);
          else
            f[j] = (ex_byte_at(w[j][i / 4], i & 3) - add[j]) * mul[j];
        }
        put(St::DL * n + 8 * u + i, make_uint2(ex_pack(f[0], f[1]), ex_pack(f[2], f[3])));
      }
    }
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
  typedef ExStage<DP> St;
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

// The running state of 32 rows in a wave: lane (row = lane & 31, half = lane >> 5).
template <int DP>
struct ExAcc {
  f32x16 o[DP / 32];
  float m, l;
};

// One key tile: logits, online softmax, output.
//   end[i]  keys of sub-tile i that this lane's row sees (bounds on the key's
//           place in the sub-tile), used unless every row sees the whole tile
template <int DP, int WF, int TK>
__device__ __forceinline__ void ex_step(const ExTile<DP, TK>& t, const f16x8 (&q)[DP / 16], float qscale,
                                        const int (&end)[TK / 16], bool whole, ExAcc<DP>& a) {
  constexpr int KT = TK / 32;
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  f32x16 s[KT];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    s[kt] = f32x16{};
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const f16x8 k = __builtin_bit_cast(f16x8, t.k[ex_k_at<DP>(kt * 32 + col, kk * 2 + h)]);
      s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[kk], s[kt], 0, 0, 0);
    }
  }
  // Logits in units of log 2.
  float mx = EX_NONE;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int sub = kt * 2 + half;
      if constexpr (WF == TIERKV_WARM_ABSMAX_I8) {
        const float c = t.kscale[sub] * qscale;
#pragma unroll
        for (int r = 0; r < 8; ++r) s[kt][half * 8 + r] *= c;
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          s[kt][half * 8 + r] *= t.kscale[sub * 16 + 8 * (r >> 2) + 4 * h + (r & 3)] * qscale;
      }
      if (!whole) {
        const int e = end[sub] - 4 * h;
#pragma unroll
        for (int r = 0; r < 8; ++r)
          s[kt][half * 8 + r] = (8 * (r >> 2) + (r & 3)) < e ? s[kt][half * 8 + r] : -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) mx = fmaxf(mx, s[kt][half * 8 + r]);
    }
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
  const float base = a.m - EX_BOOST;
  f16x8 pr[KT * 2];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float e = __builtin_amdgcn_exp2f(s[kt][half * 8 + r] - base);
        a.l += e;
        pr[kt * 2 + half][r] = _Float16(e);
      }
    }
  }
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) {
#pragma unroll
    for (int sub = 0; sub < TK / 16; ++sub) {
      const f16x8 v = __builtin_bit_cast(f16x8, t.v[ex_v_at<TK>(dt * 32 + col, sub * 2 + h)]);
      a.o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pr[sub], a.o[dt], 0, 0, 0);
    }
  }
}

template <typename QT>
__device__ __forceinline__ uint32_t ex_out2(float a, float b) {
  const QT x = from_f32<QT>(a), y = from_f32<QT>(b);
  return uint32_t(__builtin_bit_cast(uint16_t, x)) | (uint32_t(__builtin_bit_cast(uint16_t, y)) << 16);
}

template <int DP>
constexpr int ex_lds_bytes() {
  return int(sizeof(ExTile<DP, 64>)) > 4 * int(sizeof(ExTile<DP, 32>)) ? int(sizeof(ExTile<DP, 64>))
                                                                       : 4 * int(sizeof(ExTile<DP, 32>));
}

// An item: query rows of one tile, sub-tiles [part / parts) of what it sees.
//   RW  waves that hold different rows (4: wide, 1: narrow); 4 / RW waves
//       share the rows and split the keys
template <int DP, int WF, typename QT, int RW>
__device__ void ex_item(const ExtendParams& p, char* lds, int h, const int4 it, int64_t partial) {
  constexpr int TK = RW == 4 ? 64 : 32;
  constexpr int NS = TK / 16 / RW;          // sub-tiles a wave stages
  constexpr int KW = 4 / RW;
  const int tid = threadIdx.x, lane = tid & 63, w = ex_uniform(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int b = it.x, tile = it.y & 0x3fffffff;
  const int part = it.z & 0xffff, parts = it.z >> 16;
  const int4 seq = p.seq[b];
  const int q0 = ex_rows(p, b).x, n = seq.w, G = p.groups, D = p.D;
  const int rows = n * G;
  const int row_first = tile * EX_WIDE, row_last = min(row_first + RW * 32, rows) - 1;
  const int lim_min = seq.y - n + row_first / G, lim_max = seq.y - n + row_last / G;
  const int4* list = p.subtile + int64_t(b) * p.subs_per_seq;

  // This lane's row.
  const int r = row_first + (RW == 4 ? w * 32 : 0) + col;
  const bool live = r < rows;
  const int tok = live ? r / G : 0, head = h * G + (live ? r - tok * G : 0);
  const int lim = live ? seq.y - n + tok : -1;
  f16x8 q[DP / 16];
  float qscale = p.scale_log2;
  {
    const QT* src = reinterpret_cast<const QT*>(p.q) + int64_t(q0 + tok) * p.qs_t + int64_t(head) * p.qs_h;
    uint4 raw[DP / 16];
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const int d = kk * 16 + half * 8;
      raw[kk] = (live && d < D) ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
    }
    if constexpr (sizeof(QT) == 2 && !__is_same(QT, __half)) {
      float mx = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const uint32_t x[4] = {raw[kk].x, raw[kk].y, raw[kk].z, raw[kk].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(x[i] << 16)), fabsf(__uint_as_float(x[i] & 0xffff0000u))));
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
          q[kk][2 * i] = _Float16(__uint_as_float(x[i] << 16) * inv);
          q[kk][2 * i + 1] = _Float16(__uint_as_float(x[i] & 0xffff0000u) * inv);
        }
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) q[kk] = __builtin_bit_cast(f16x8, raw[kk]);
    }
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

  const int visible = ex_uniform(ex_visible(list, seq.x, lim_max));
  const int chunk = ((visible + parts - 1) / parts + 3) & ~3;
  const int lo = min(part * chunk, visible), hi = min(lo + chunk, visible);

  ExTile<DP, TK>* tiles = reinterpret_cast<ExTile<DP, TK>*>(lds);
  ExTile<DP, TK>& mine = tiles[RW == 4 ? 0 : w];
  constexpr int STEP = TK / 16 * KW;        // sub-tiles per round of the workgroup
  const int first = RW == 4 ? lo : lo + w * (TK / 16);
  ExStage<DP> st[NS];
  ExSub sub[NS];
  int wild = 0;
  auto load = [&](int at) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      sub[i] = ex_sub(list, at + (RW == 4 ? w : i), hi);
      ex_load<DP, WF>(p, h, sub[i], st[i]);
    }
  };
  if (first < hi) load(first);
  for (int at = first; at < hi; at += STEP) {
    const bool whole = ex_whole<TK>(list, at, hi, lim_min);
    int end[TK / 16];
#pragma unroll
    for (int i = 0; i < TK / 16; ++i) {
      const ExSub s = ex_sub(list, at + i, hi);
      end[i] = min(s.valid, lim - s.ordinal + 1);
    }
    if constexpr (RW == 4) __syncthreads();           // every wave has read the tile before
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const uint32_t largest = ex_store<DP, WF, TK>(p, sub[i], st[i], RW == 4 ? w : i, mine);
      if (!whole && __any(ex_wild(largest))) {
        ex_clear_wild<DP, TK>(RW == 4 ? w : i, &mine);
        wild = 1;
      }
    }
    if constexpr (RW == 4) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (at + STEP < hi) load(at + STEP);
    ex_step<DP, WF, TK>(mine, q, qscale, end, whole, a);
  }
  // Infinities and NaN of the tiles with hidden keys, for the rows that see them.
  if constexpr (RW == 4) wild = __syncthreads_or(wild);
  if (wild) {
#pragma unroll 1
    for (int at = first; at < hi; at += STEP) {
      if (ex_whole<TK>(list, at, hi, lim_min)) continue;
#pragma unroll 1
      for (int k = 0; k < TK / 16; ++k) {
        const ExSub s = ex_sub(list, at + k, hi);
#pragma unroll 1
        for (int t = 0; t < min(s.valid, lim - s.ordinal + 1); ++t) {
#pragma unroll
          for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int d = dt * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
              const float v = d < D ? ex_value<WF>(p, h, s, t, d) : 0.f;
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
        l += sml[(k * 32 + rr) * 2 + 1] * c;
        o += *reinterpret_cast<const f32x4*>(so + (k * 32 + rr) * (DP + 4) + d) * c;
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

template <int DP, int WF, typename QT>
__global__ __launch_bounds__(EX_THREADS, 2) void extend_kernel(ExtendParams p) {
  extern __shared__ __attribute__((aligned(16))) char ex_lds[];
  const int i = int(blockIdx.x) / p.kv_heads, h = int(blockIdx.x) - i * p.kv_heads;
  if (i >= p.head[0]) return;
  int4 it = p.item[i];
  it.x = ex_uniform(it.x);
  it.y = ex_uniform(it.y);
  it.z = ex_uniform(it.z);
  it.w = ex_uniform(it.w);
  if (it.x < 0) return;
  if (it.y & (1 << 30)) ex_item<DP, WF, QT, 4>(p, ex_lds, h, it, it.w);
  else ex_item<DP, WF, QT, 1>(p, ex_lds, h, it, it.w);
}

// Join of a cut tile's partials, in part order: a workgroup per (cut tile, kv
// head, 32 of its rows).
template <typename QT>
__global__ __launch_bounds__(EX_THREADS) void extend_merge_kernel(ExtendParams p) {
  const int c = int(blockIdx.x) / p.kv_heads, h = int(blockIdx.x) - c * p.kv_heads;
  if (c >= p.head[1]) return;
  const int2 cut = p.cut[c];
  if (cut.y < 0) return;
  const int4 it = p.item[cut.y];
  const int b = it.x, tile = it.y & 0x3fffffff, parts = it.z >> 16;
  const int n = p.seq[b].w, G = p.groups, D = p.D;
  const int row_first = tile * EX_WIDE, row_base = int(blockIdx.y) * 32;
  const int q0 = ex_rows(p, b).x;
  const int D4 = D / 4;
  for (int x = threadIdx.x; x < 32 * D4; x += EX_THREADS) {
    const int rr = row_base + x / D4, d = 4 * (x % D4);
    const int row = row_first + rr;
    if (row >= n * G || rr >= p.part_rows) continue;
    float m = EX_NONE;
    for (int k = 0; k < parts; ++k)
      m = fmaxf(m, p.part_ml[((int64_t(cut.x + k) * p.kv_heads + h) * p.part_rows + rr) * 2]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int k = 0; k < parts; ++k) {
      const int64_t at = (int64_t(cut.x + k) * p.kv_heads + h) * p.part_rows + rr;
      const float f = __builtin_amdgcn_exp2f(p.part_ml[at * 2] - m);
      l += p.part_ml[at * 2 + 1] * f;
      o += *reinterpret_cast<const f32x4*>(p.part_o + at * D + d) * f;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const int tk = row / G, hd = h * G + row - tk * G;
    QT* dst = reinterpret_cast<QT*>(p.out) + (int64_t(q0 + tk) * p.heads + hd) * D + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(ex_out2<QT>(o[0] * inv, o[1] * inv), ex_out2<QT>(o[2] * inv, o[3] * inv));
  }
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
  l.subs_per_seq = num_blocks * ((bs + EX_SUB - 1) / EX_SUB);
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
  const int lds = std::max(ex_lds_bytes<DP>(), 4 * 32 * (DP + 4 + 2) * 4);
  hipLaunchKernelGGL(extend_plan_kernel, dim3(p.batch), dim3(EX_PLAN), 0, stream, p);
  hipLaunchKernelGGL((extend_kernel<DP, WF, QT>), dim3(p.max_items * p.kv_heads), dim3(EX_THREADS), lds, stream, p);
  hipLaunchKernelGGL(extend_merge_kernel<QT>, dim3(p.max_cut * p.kv_heads, p.part_rows / 32), dim3(EX_THREADS), 0,
                     stream, p);
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
  const int groups = num_heads / num_kv_heads;
  if (int64_t(num_rows) * groups > (int64_t(1) << 29))
    return fail(TIERKV_ERR_UNSUPPORTED, "more than 2^29 query rows per kv head");
  const ExLayout l = ex_layout(batch, num_rows, max_tokens, groups, num_kv_heads, num_blocks, block_size, head_dim);
  if (int64_t(l.max_items) * num_kv_heads > 0x7fffffff) return fail(TIERKV_ERR_UNSUPPORTED, "grid too large");
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
