// Next tokens from logits on gfx950: temperature, top-k, top-p, min-p and the
// draw from a given random number.
//
// A row's weights are whole numbers,
//   W_i = rint(2^42 exp((x_i - max x) / T)),
// so that every sum of them is exact, whatever its order and however it is
// split over workgroups, and one rule decides what a border falls on.  The
// tokens in the order (logit descending, index ascending) are cut to a
// prefix three times: the first k; of these the tokens whose sum of weights
// before them lies below p times their total; of these the tokens with
// W_i >= 2^42 min_p.  The token is the smallest index whose running sum of
// the remaining weights, in index order, exceeds u times their total.
// A vocabulary of up to 2^20 keeps sums within 2^62; tokens below 2^-43 of
// the likeliest have weight 0.
//
// Bound: memory, one read of the logits, and below a few megabytes the
// latency of the dependent steps.  No row is sorted.  A first launch reads
// every row with up to 16 workgroups for its largest logit; then
//   top-k     Launch 1 also keeps the largest logit of every group (the
//             elements of a thread).  The k-th largest of the groups' maxima
//             is at most the k-th largest logit, so the first k tokens lie in
//             the groups whose maximum reaches it: a second launch, one
//             workgroup per row, reads those alone again, a few thousand
//             elements, and lists and ranks the tokens in LDS.  (With this in
//             launch 1, by each row's last workgroup, 256 x 128256 fp32 took
//             77 us where the read alone takes 26: the dependent steps held
//             back the reads of other rows.)
//   top-p     needs every weight: a second launch adds counts and weights to
//             2048 bins of the distance to the maximum, and the row's last
//             workgroup to arrive (a counter per row) finds the bin where p is
//             crossed.  When the bins down to it hold up to 512 tokens, a
//             third launch lists and draws from them; else it lists that
//             bin's alone, which settles the border, and a fourth adds up
//             what is kept and draws.
//   neither   the second launch adds up each part of the row and its last
//             workgroup draws in the part that holds the token.
// Measured (us per launch; maxima, top-k, sums, list, draw): 1 x 32000 fp16
// with top-k 3.6 + 13.6; 16 x 128256 bf16 with top-p 4.8, -, 14.2, 14.8, 20.6;
// 256 x 128256 fp32, limits of each row, 23.1 (5.7 TB/s), 19.5, 16.4, 20.9,
// 29.7 (the later launches read a row again only where its limits need it).
// Rows that fit none of these (a thousand equal logits at the border, k from
// about a thousand on) take a radix select over the row by one workgroup (64 x
// 128256 fp32 of whole numbers: 344 us with top-k 3000, 1019 with top-p 0.9).

#include "tierkv_common.h"

#include <algorithm>

namespace tierkv {

constexpr int SP_THREADS = 512;
constexpr int SP_WAVES = SP_THREADS / 64;
constexpr int SP_DIGITS = 256;               // digits of the radix select
constexpr int SP_BINS = 2048;                // bins of the distance to the maximum
constexpr int SP_LIST = 1024;                // tokens listed, at most
constexpr int SP_FEW = SP_THREADS;           // lists of one token per thread
constexpr int SP_PARTS = 16;                 // workgroups per row, at most
constexpr int SP_GROUPS = SP_PARTS * SP_THREADS;
constexpr int SP_MAX_VOCAB = 1 << 20;
constexpr int SP_MAX_BATCH = 1 << 16;
constexpr double SP_ONE = 4398046511104.0;   // 2^42
constexpr float SP_REACH = 30.f;             // weights are 0 from exp(-29.81) on

enum SpMode { SP_DONE = 0, SP_SHORT, SP_BORDER, SP_DRAW, SP_SLOW };

// A row's state between the launches.
struct SpState {
  int32_t mode;
  int32_t bin;          // the crossing bin
  uint32_t cut;         // the prefix: keys above cut, and those equal to it up to index last
  int32_t last;
  uint64_t above;       // weight in the bins above the crossing one
  uint64_t total;       // weight of the row
};

struct SampleParams {
  const void* logits;
  int64_t stride;
  int32_t batch, vocab;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int64_t* tokens;
  float* probs;
  int32_t parts, steps;   // workgroups per row; vectors per thread
  // Workspace.
  uint32_t* counter;      // [SP_MAX_BATCH][2] arrivals and list entries of a row, zero between launches
  SpState* state;         // [batch]
  uint64_t* part;         // [batch][parts] the parts' maxima (key, ~index)
  uint64_t* weight;       // [batch][parts] the parts' weights
  uint32_t* group;        // [batch][parts * SP_THREADS] the groups' largest keys
  uint32_t* count;        // [batch][SP_BINS]
  uint64_t* mass;         // [batch][SP_BINS]
  uint64_t* list;         // [batch][SP_LIST] (key, ~index)
};

// The logit as an unsigned integer of the same order; -0 as +0, NaN lowest
// (a NaN logit is never drawn).
__device__ __forceinline__ uint32_t sp_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  if (x != x) return 0;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float sp_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
constexpr uint32_t SP_MINUS_INF = 0x007fffffu;   // the key of -infinity

// (key, index) as one integer in the tokens' order.
__device__ __forceinline__ uint64_t sp_entry(uint32_t key, int i) { return (uint64_t(key) << 32) | uint32_t(~i); }

// Agent-scope accesses for what workgroups of one launch exchange.
template <typename V>
__device__ __forceinline__ void sp_put(V* p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename V>
__device__ __forceinline__ V sp_get(V* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

struct SpRow {
  float top;      // the row's largest logit
  double rt;      // 1 / T
  double floor;   // weights below it (min-p) count as 0 in the draw
  float reach;    // logits further below the largest have weight 0
  float bins;     // bins per unit of distance
  __device__ __forceinline__ uint64_t weight(float x) const {
    if (x == top) return uint64_t(SP_ONE);
    const double d = double(x) - double(top);
    if (!(d > -1e300)) return 0;               // -inf, NaN
    return uint64_t(rint(exp(d * rt) * SP_ONE));
  }
  __device__ __forceinline__ bool kept_by_min_p(uint64_t w) const { return double(w) >= floor; }
  // Bin of a logit: monotone in it (each step's rounding is).
  __device__ __forceinline__ int bin(float x) const {
    if (x == top) return 0;
    return int(fminf((top - x) * bins, float(SP_BINS - 1)));
  }
};

struct SpLimits {
  float t, top_p;
  int top_k;      // 0: off
  bool greedy;
};

__device__ __forceinline__ SpLimits sp_limits(const SampleParams& p, int b) {
  SpLimits l;
  l.t = p.temperature ? p.temperature[b] : p.temperature_all;
  l.greedy = !(l.t > 0.f);
  l.top_p = p.top_p ? p.top_p[b] : p.top_p_all;
  const int k = p.top_k ? p.top_k[b] : p.top_k_all;
  l.top_k = k > 0 && k < p.vocab ? k : 0;
  return l;
}

__device__ __forceinline__ SpRow sp_row(const SampleParams& p, int b, float top, float t) {
  SpRow r;
  r.top = top;
  r.rt = 1.0 / double(t);
  const float m = p.min_p ? p.min_p[b] : p.min_p_all;
  r.floor = m > 0.f ? fmin(double(m), 1.0) * SP_ONE : 0.0;
  r.reach = SP_REACH * t;
  r.bins = float(SP_BINS) / r.reach;
  return r;
}

template <typename T> __device__ __forceinline__ float sp_load(const T* x, int64_t i) { return to_f32<T>(x[i]); }
template <> __device__ __forceinline__ float sp_load<float>(const float* x, int64_t i) { return x[i]; }

// Elements [i, i + VL) of a row of n, NaN past its end: one 16-byte load
// where rows are aligned (WIDE).
template <typename T, bool WIDE>
__device__ __forceinline__ void sp_load_vector(const T* x, int i, int n, float (&v)[16 / sizeof(T)]) {
  constexpr int VL = 16 / sizeof(T);
  if (WIDE && i + VL <= n) {
    const uint4 w = *reinterpret_cast<const uint4*>(x + i);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int j = 0; j < VL; ++j) v[j] = sp_load(e, j);
  } else {
#pragma unroll
    for (int j = 0; j < VL; ++j) v[j] = i + j < n ? sp_load(x, i + j) : __uint_as_float(0x7fc00000u);
  }
}

__device__ __forceinline__ uint64_t sp_wave_sum(uint64_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

struct SpShared {
  uint64_t wave[SP_WAVES + 1];
  uint64_t above;
  int32_t digit, flag;
  uint32_t n;
  union {
    uint64_t hist[SP_DIGITS];
    struct {
      uint64_t mass[SP_BINS];
      uint32_t count[SP_BINS];
    };
    struct {
      alignas(16) uint64_t list[SP_LIST];
      uint64_t sum[SP_LIST];
      uint64_t other[SP_LIST];
    };
  };
  uint16_t pick[SP_LIST];         // groups to read again
};

// Inclusive prefix sum over the workgroup; *total gets the sum.
__device__ __forceinline__ uint64_t sp_scan(SpShared& sh, uint64_t v, uint64_t* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint64_t x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) sh.wave[w] = x;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < SP_WAVES; ++i) {
    const uint64_t t = sh.wave[i];
    before += i < w ? t : 0;
    all += t;
  }
  *total = all;
  return x + before;
}

// Running sums of f(i) for i < n into sh.sum (n <= SP_LIST); returns the total.
template <typename F>
__device__ __forceinline__ uint64_t sp_running(SpShared& sh, int n, F f) {
  constexpr int PER = SP_LIST / SP_THREADS;
  uint64_t v[PER], own = 0, total;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = int(threadIdx.x) * PER + i;
    v[i] = at < n ? f(at) : 0;
    own += v[i];
  }
  uint64_t run = sp_scan(sh, own, &total) - own;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    run += v[i];
    if (int(threadIdx.x) * PER + i < n) sh.sum[threadIdx.x * PER + i] = run;
  }
  __syncthreads();
  return total;
}

// Bitonic sort of a[0, n), descending, n <= SP_LIST; a has room for the next
// power of two (filled with 0, which no entry is).  The pairs of a wave's
// threads lie in 128 neighbouring entries while their distance is at most 64:
// such steps need no barrier, only the wave's own order of LDS accesses (1024
// entries: 10 barriers for 55 steps).
__device__ __forceinline__ void sp_sort(uint64_t* a, int n) {
  int size = 2;
  while (size < n) size *= 2;
  for (int i = n + int(threadIdx.x); i < size; i += SP_THREADS) a[i] = 0;
  int before = SP_LIST;
  for (int k = 2; k <= size; k *= 2) {
    for (int j = k / 2; j > 0; j /= 2) {
      if (j > 64 || before > 64) __syncthreads();
      else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      before = j;
      for (int x = threadIdx.x; x < size / 2; x += SP_THREADS) {
        const int i = 2 * x - (x & (j - 1)), l = i + j;
        const uint64_t u = a[i], v = a[l];
        if ((u < v) == ((i & k) == 0)) {
          a[i] = v;
          a[l] = u;
        }
      }
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void sp_write(const SampleParams& p, int b, int token, double prob) {
  if (threadIdx.x == 0) {
    p.tokens[b] = token;
    if (p.probs) p.probs[b] = float(prob);
  }
}

__device__ __forceinline__ uint64_t sp_target(const SampleParams& p, int b, uint64_t total) {
  const double u = double(p.u[b]);
  const uint64_t t = u > 0.0 ? uint64_t(fmin(u, 1.0) * double(total)) : 0;
  return min(t, total - 1);
}

// Place of this thread's entry among the n of a (n <= SP_FEW, distinct, one
// per thread) in descending order: every thread reads all of them, two per
// access and all lanes the same (200 entries: 0.6 us, where the 36 dependent
// steps of a bitonic sort take 10).  a has a spare entry behind the last.
__device__ __forceinline__ int sp_rank(const uint64_t* a, int n, uint64_t mine) {
  int r = 0;
#pragma unroll 4
  for (int j = 0; j < n; j += 2) {
    const ulonglong2 e = *reinterpret_cast<const ulonglong2*>(a + j);
    r += (e.x > mine ? 1 : 0) + (j + 1 < n && e.y > mine ? 1 : 0);
  }
  return r;
}

// The draw from sh.list, the n first tokens of the row or more (n <= SP_FEW):
// the first k of them (k > 0), top-p of their weight or of `total` (k == 0),
// min-p.  One token per thread.
__device__ __forceinline__ void sp_draw_few(SpShared& sh, const SampleParams& p, int b, const SpRow& row, int n, int k,
                                            float top_p, uint64_t total) {
  const int tid = threadIdx.x;
  uint64_t e = tid < n ? sh.list[tid] : 0;
  const int place = tid < n ? sp_rank(sh.list, n, e) : 0;
  if (tid < n) sh.other[place] = e;
  if (k > 0) n = min(n, k);
  __syncthreads();
  e = tid < n ? sh.other[tid] : 0;
  const uint64_t w = tid < n ? row.weight(sp_value(uint32_t(e >> 32))) : 0;
  uint64_t sum;
  const uint64_t before = sp_scan(sh, w, &sum) - w;
  if (k > 0) total = sum;
  const double thr = top_p < 1.f ? fmax(double(top_p) * double(total), 1.0) : 1e300;
  // Tokens kept: a prefix of m.
  const bool kept = tid < n && double(before) < thr && row.kept_by_min_p(w);
  const int m = __syncthreads_count(kept);
  const uint32_t index = ~uint32_t(e);
  if (kept) sh.list[tid] = sp_entry(uint32_t(e), int(tid));   // (~index descending is index ascending)
  __syncthreads();
  if (kept) {
    const int at = sp_rank(sh.list, m, sp_entry(uint32_t(e), int(tid)));
    sh.other[at] = w;
    sh.sum[at] = index;
  }
  __syncthreads();
  uint64_t all;
  const uint64_t v = tid < m ? sh.other[tid] : 0;
  const uint64_t run = sp_scan(sh, v, &all);
  const uint64_t target = sp_target(p, b, all);
  if (tid < m && target < run && target >= run - v) {
    p.tokens[b] = int64_t(sh.sum[tid]);
    if (p.probs) p.probs[b] = float(double(v) / double(all));
  }
}

// The same for up to SP_LIST tokens.
__device__ __forceinline__ void sp_draw_list(SpShared& sh, const SampleParams& p, int b, const SpRow& row, int n, int k,
                                             float top_p, uint64_t total) {
  if (n <= SP_FEW) {
    sp_draw_few(sh, p, b, row, n, k, top_p, total);
    return;
  }
  sp_sort(sh.list, n);
  if (k > 0) n = min(n, k);
  const uint64_t sum = sp_running(sh, n, [&](int i) { return row.weight(sp_value(uint32_t(sh.list[i] >> 32))); });
  if (k > 0) total = sum;
  const double thr = top_p < 1.f ? fmax(double(top_p) * double(total), 1.0) : 1e300;
  uint64_t kept = 0, m;
  for (int i = threadIdx.x; i < n; i += SP_THREADS) {
    const uint64_t before = i ? sh.sum[i - 1] : 0, w = sh.sum[i] - before;
    kept += (double(before) < thr && row.kept_by_min_p(w)) ? 1 : 0;
  }
  sp_scan(sh, kept, &m);
  const uint64_t all = sh.sum[m - 1];
  const uint64_t target = sp_target(p, b, all);
  // In index order: (~index, place), sorted.
  for (int i = threadIdx.x; i < int(m); i += SP_THREADS)
    sh.other[i] = (uint64_t(uint32_t(sh.list[i])) << 32) | uint32_t(i);
  sp_sort(sh.other, int(m));
  sp_running(sh, int(m), [&](int i) { return row.weight(sp_value(uint32_t(sh.list[uint32_t(sh.other[i])] >> 32))); });
  for (int i = threadIdx.x; i < int(m); i += SP_THREADS) {
    const uint64_t before = i ? sh.sum[i - 1] : 0;
    if (target >= before && target < sh.sum[i]) {
      p.tokens[b] = int64_t(uint32_t(~uint32_t(sh.other[i] >> 32)));
      if (p.probs) p.probs[b] = float(double(sh.sum[i] - before) / double(all));
    }
  }
}

// ---- any row, by one workgroup --------------------------------------------

// The first digit from the top whose bins down to it add up to thr or more
// (sh.digit), and the sum of the bins above it (sh.above).
__device__ __forceinline__ void sp_cross(SpShared& sh, uint64_t above, double thr) {
  const int lane = threadIdx.x;
  if (lane >= 64) return;
  uint64_t b[4], own = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    b[i] = sh.hist[SP_DIGITS - 1 - (lane * 4 + i)];
    own += b[i];
  }
  uint64_t incl = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t y = __shfl_up(incl, d, 64);
    if (lane >= d) incl += y;
  }
  const bool here = double(above + incl) >= thr;
  const uint64_t any = __ballot(here);
  const int first = any ? __ffsll((unsigned long long)any) - 1 : 63;
  if (lane == first) {
    uint64_t run = above + incl - own;
    int i = 0;
    while (i < 3 && double(run + b[i]) < thr) run += b[i++];
    sh.digit = SP_DIGITS - 1 - (lane * 4 + i);
    sh.above = run;
  }
}

// The key K with measure(> K) < thr <= measure(>= K); *above = measure(> K).
// measure(x, key) is the measure of an element; extra is one added at key_x.
template <typename T, typename M>
__device__ __forceinline__ uint32_t sp_select(SpShared& sh, const T* x, int n, double thr, M measure, uint32_t key_x, uint64_t extra,
                              uint64_t* above) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0;
  uint64_t sum = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (tid < SP_DIGITS) sh.hist[tid] = 0;
    __syncthreads();
    const uint32_t high = shift == 24 ? 0u : ~0u << (shift + 8);
    constexpr int AHEAD = 16;   // loads in flight
    for (int i0 = tid; i0 < n; i0 += SP_THREADS * AHEAD) {
      float v[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) v[j] = sp_load(x, min(i0 + SP_THREADS * j, n - 1));
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const uint32_t k = sp_key(v[j]);
        if (i0 + SP_THREADS * j < n && (k & high) == prefix) {
          const uint64_t m = measure(v[j], k);
          if (m) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[(k >> shift) & 255]), (unsigned long long)m);
        }
      }
    }
    if (tid == 0 && extra && (key_x & high) == prefix)
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[(key_x >> shift) & 255]), (unsigned long long)extra);
    __syncthreads();
    sp_cross(sh, sum, thr);
    __syncthreads();
    prefix |= uint32_t(sh.digit) << shift;
    sum = sh.above;
  }
  *above = sum;
  return prefix;
}

// Sum of measure(i) over [lo, hi) by wave segments; every thread finds the
// segments' sums in sh.wave.  Returns the segment length.
template <typename T, typename M>
__device__ __forceinline__ int sp_segments(SpShared& sh, const T* x, int lo, int hi, M measure) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int seg = (((hi - lo) + SP_WAVES * 64 - 1) / (SP_WAVES * 64)) * 64;
  uint64_t s = 0;
  const int first = lo + w * seg, end = min(first + seg, hi);
  constexpr int AHEAD = 16;   // loads in flight (one at a time, a part of 8016 took 16 round trips)
  for (int i0 = first + lane; i0 < end; i0 += 64 * AHEAD) {
    float v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) v[k] = sp_load(x, min(i0 + 64 * k, end - 1));
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i0 + 64 * k < end) s += measure(v[k], i0 + 64 * k);
  }
  s = sp_wave_sum(s);
  __syncthreads();
  if (lane == 0) sh.wave[w] = s;
  __syncthreads();
  return seg;
}

// The smallest index in [lo, hi) whose running sum of measure exceeds
// target, which is below the sum over [lo, hi).
template <typename T, typename M>
__device__ __forceinline__ int sp_descend(SpShared& sh, const T* x, int lo, int hi, uint64_t target, M measure) {
  while (hi - lo > 64) {
    const int seg = sp_segments(sh, x, lo, hi, measure);
    int w = 0;
    while (w < SP_WAVES - 1 && target >= sh.wave[w]) target -= sh.wave[w++];
    lo += w * seg;
    hi = min(lo + seg, hi);
  }
  const int lane = threadIdx.x & 63;
  uint64_t c = lo + lane < hi ? measure(sp_load(x, lo + lane), lo + lane) : 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t y = __shfl_up(c, d, 64);
    if (lane >= d) c += y;
  }
  const uint64_t hit = __ballot(c > target);
  return hit ? lo + __ffsll((unsigned long long)hit) - 1 : hi - 1;
}

// Weight of element i in the draw under the prefix (cut, last).
template <typename T>
__device__ __forceinline__ uint64_t sp_kept(const SpRow& row, float v, int i, uint32_t cut, int last) {
  const uint32_t key = sp_key(v);
  if (key < cut || (key == cut && i > last)) return 0;
  const uint64_t w = row.weight(v);
  return row.kept_by_min_p(w) ? w : 0;
}

template <typename T>
__device__ __forceinline__ void sp_slow(SpShared& sh, const SampleParams& p, int b, const T* x, SpRow row,
                                                  int k, float top_p) {
  const int n = p.vocab;
  // The prefix (cut, ties): every key above cut and the first `ties` equal
  // to it; ties < 0: all of them.
  uint32_t cut = 0;
  int64_t ties = -1;
  uint64_t above = 0;
  if (k > 0) {
    cut = sp_select(sh, x, n, double(k), [](float, uint32_t) -> uint64_t { return 1; }, 0u, 0, &above);
    ties = k - int64_t(above);
  }
  if (top_p < 1.f) {
    const uint32_t cut_k = cut;
    const uint64_t at_cut = ties >= 0 ? uint64_t(ties) * row.weight(sp_value(cut_k)) : 0;
    auto measure = [&](float v, uint32_t key) -> uint64_t { return key > cut_k || ties < 0 ? row.weight(v) : 0; };
    sp_segments(sh, x, 0, n, [&](float v, int) { return measure(v, sp_key(v)); });
    uint64_t total = at_cut;
    for (int i = 0; i < SP_WAVES; ++i) total += sh.wave[i];
    const double thr = fmax(double(top_p) * double(total), 1.0);   // one token at least
    cut = sp_select(sh, x, n, thr, measure, cut_k, at_cut, &above);
    const uint64_t each = row.weight(sp_value(cut));
    // The fewest ties that reach thr.
    int64_t m = 1;
    if (each > 0 && thr > double(above)) m = max(int64_t(1), int64_t((thr - double(above)) / double(each)) - 1);
    while (each > 0 && double(above + uint64_t(m) * each) < thr) ++m;
    ties = m;
  }
  // The index of the last tie kept.
  int last = n;
  if (ties >= 0) {
    auto tie = [&](float v, int) -> uint64_t { return sp_key(v) == cut ? 1 : 0; };
    sp_segments(sh, x, 0, n, tie);
    int64_t count = 0;
    for (int i = 0; i < SP_WAVES; ++i) count += int64_t(sh.wave[i]);
    if (ties < count) last = sp_descend(sh, x, 0, n, uint64_t(ties - 1), tie);
  }
  auto kept = [&](float v, int i) -> uint64_t { return sp_kept<T>(row, v, i, cut, last); };
  sp_segments(sh, x, 0, n, kept);
  uint64_t total = 0;
  for (int i = 0; i < SP_WAVES; ++i) total += sh.wave[i];
  const int token = sp_descend(sh, x, 0, n, sp_target(p, b, total), kept);
  sp_write(p, b, token, double(kept(sp_load(x, token), token)) / double(total));
}

// ---- the launches ----------------------------------------------------------

// Whether this workgroup is the last of its row to get here; what the others
// stored with sp_put before it (written through to what all XCDs share, and
// waited for) is visible to sp_get after it.
__device__ __forceinline__ bool sp_last(SpShared& sh, uint32_t* arrived, int parts) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t before = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh.flag = before + 1 == uint32_t(parts);
    if (sh.flag) sp_put(arrived, 0u);
  }
  __syncthreads();
  return sh.flag != 0;
}

// The element range of a part.
template <typename T>
__device__ __forceinline__ int sp_part_size(const SampleParams& p) { return p.steps * SP_THREADS * int(16 / sizeof(T)); }

// f(x_i, i) for this thread's elements of part c, in index order (elements
// past the row are NaN), four vectors in flight.
template <typename T, bool WIDE, typename F>
__device__ __forceinline__ void sp_sweep(const SampleParams& p, int c, const T* x, F f) {
  constexpr int VL = 16 / sizeof(T), AHEAD = 4;
  const int base = (c * p.steps * SP_THREADS + int(threadIdx.x)) * VL;
  for (int s = 0; s < p.steps; s += AHEAD) {
    float v[AHEAD][VL];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int i = base + (s + a) * SP_THREADS * VL;
      if (s + a < p.steps && i < p.vocab) sp_load_vector<T, WIDE>(x, i, p.vocab, v[a]);
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int i = base + (s + a) * SP_THREADS * VL;
      if (s + a < p.steps && i < p.vocab) {
#pragma unroll
        for (int j = 0; j < VL; ++j) f(v[a][j], i + j);
      }
    }
  }
}

// The first k tokens' groups, listed and drawn from; false: not this way.
template <typename T, bool WIDE>
__device__ __forceinline__ bool sp_top_k(SpShared& sh, const SampleParams& p, int b, const T* x, SpRow row, int k, float top_p) {
  constexpr int VL = 16 / sizeof(T), PER = SP_GROUPS / SP_THREADS;
  const int tid = threadIdx.x, groups = p.parts * SP_THREADS;
  const uint32_t* group = p.group + int64_t(b) * groups;
  uint32_t key[PER], low = ~0u;
  uint64_t filled = 0, total;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    key[i] = i * SP_THREADS + tid < groups ? group[i * SP_THREADS + tid] : 0;
    if (key[i] > SP_MINUS_INF && !(row.top - sp_value(key[i]) <= row.reach)) key[i] = 0;   // its tokens have weight 0
    if (key[i] > SP_MINUS_INF) {
      ++filled;
      low = min(low, key[i]);
    }
  }
  // The smallest maximum, and how many there are.
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) low = min(low, uint32_t(__shfl_xor(low, m, 64)));
  sp_scan(sh, filled, &total);
  __syncthreads();
  if ((tid & 63) == 0) sh.wave[tid >> 6] = low;
  for (int i = tid; i < SP_BINS; i += SP_THREADS) sh.count[i] = 0;
  if (tid == 0) sh.n = 0;
  __syncthreads();
  for (int i = 0; i < SP_WAVES; ++i) low = min(low, uint32_t(sh.wave[i]));
  // With fewer such groups than k, all of their tokens that have a weight are listed.
  const bool every = int64_t(total) < k;
  const float span = row.top - sp_value(low);
  if (!(span < INFINITY)) return false;
  row.bins = span > 0.f ? float(SP_BINS) / span : 0.f;
  if (!(row.bins < INFINITY)) return false;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (key[i] > SP_MINUS_INF) atomicAdd(&sh.count[row.bin(sp_value(key[i]))], 1u);
  __syncthreads();
  // The bin with the k-th largest maximum.
  {
    constexpr int C = SP_BINS / SP_THREADS;
    uint64_t own = 0, all;
    for (int i = 0; i < C; ++i) own += sh.count[tid * C + i];
    uint64_t run = sp_scan(sh, own, &all) - own;
    if (every) {
      if (tid == 0) {
        sh.digit = SP_BINS - 1;
        sh.above = total;
      }
    } else if (run < uint64_t(k) && run + own >= uint64_t(k)) {
      int i = 0;
      while (run + sh.count[tid * C + i] < uint64_t(k)) run += sh.count[tid * C + i++];
      sh.digit = tid * C + i;
      sh.above = run + sh.count[tid * C + i];
    }
    __syncthreads();
  }
  const int border = sh.digit;
  if (sh.above > uint64_t(SP_LIST)) return false;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (key[i] > SP_MINUS_INF && row.bin(sp_value(key[i])) <= border)
      sh.pick[atomicAdd(&sh.n, 1u)] = uint16_t(i * SP_THREADS + tid);
  __syncthreads();
  const int picked = int(sh.n);
  __syncthreads();
  if (tid == 0) sh.n = 0;
  __syncthreads();
  for (int e = tid; e < picked * p.steps; e += SP_THREADS) {
    const int g = sh.pick[e / p.steps], step = e % p.steps;
    const int i0 = (((g / SP_THREADS) * p.steps + step) * SP_THREADS + g % SP_THREADS) * VL;
    float v[VL];
    sp_load_vector<T, WIDE>(x, i0, p.vocab, v);
#pragma unroll
    for (int j = 0; j < VL; ++j) {
      const uint32_t kk = sp_key(v[j]);
      if (kk > SP_MINUS_INF && row.top - v[j] <= row.reach && row.bin(v[j]) <= border) {
        const uint32_t at = atomicAdd(&sh.n, 1u);
        if (at < uint32_t(SP_LIST)) sh.list[at] = sp_entry(kk, i0 + j);
      }
    }
  }
  __syncthreads();
  const int n = int(sh.n);
  if (n > SP_LIST) return false;
  sp_draw_list(sh, p, b, row, n, k, top_p, 0);
  return true;
}

// The row's largest logit and its first index, from the parts' (every wave).
struct SpTop {
  uint32_t key;
  int at;
};
__device__ __forceinline__ SpTop sp_top(const SampleParams& p, int b) {
  const int lane = threadIdx.x & 63;
  uint64_t e = lane < p.parts ? p.part[int64_t(b) * p.parts + lane] : 0;
#pragma unroll
  for (int m = SP_PARTS / 2; m >= 1; m >>= 1) {
    const uint64_t o = __shfl_xor(e, m, 64);
    e = o > e ? o : e;
  }
  e = __shfl(e, 0, 64);
  return SpTop{uint32_t(e >> 32), int(~uint32_t(e))};
}

// Rows that their largest logit decides; whether b is one.
__device__ __forceinline__ bool sp_decided(const SampleParams& p, int b, const SpTop& top, const SpLimits& lim) {
  const bool none = top.key <= SP_MINUS_INF;
  if (none) sp_write(p, b, -1, 0.0);
  else if (lim.greedy) sp_write(p, b, top.at, 1.0);
  return none || lim.greedy;
}

// Launch 1: the parts' and the groups' largest logits.
template <typename T, bool WIDE>
__global__ __launch_bounds__(SP_THREADS) void sample_max_kernel(SampleParams p) {
  __shared__ uint64_t s_wave[SP_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int b = int(blockIdx.x) / p.parts, c = int(blockIdx.x) - b * p.parts;
  const T* x = reinterpret_cast<const T*>(p.logits) + int64_t(b) * p.stride;
  const SpLimits lim = sp_limits(p, b);
  uint32_t best = 0;
  int at = 0x7fffffff;
  sp_sweep<T, WIDE>(p, c, x, [&](float v, int i) {
    const uint32_t k = sp_key(v);
    if (k > best) {
      best = k;
      at = i;
    }
  });
  if (lim.top_k && !lim.greedy) {
    p.group[(int64_t(b) * p.parts + c) * SP_THREADS + tid] = best;
  } else if (lim.top_p < 1.f && !lim.greedy) {   // this part's share of the next launch's bins
    for (int i = c * SP_THREADS + tid; i < SP_BINS; i += p.parts * SP_THREADS) {
      p.mass[int64_t(b) * SP_BINS + i] = 0;
      p.count[int64_t(b) * SP_BINS + i] = 0;
    }
  }
  uint64_t e = sp_entry(best, at);
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = __shfl_xor(e, m, 64);
    e = o > e ? o : e;
  }
  if (lane == 0) s_wave[w] = e;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < SP_WAVES; ++i) e = s_wave[i] > e ? s_wave[i] : e;
    p.part[int64_t(b) * p.parts + c] = e;
  }
}

// Rows with a top-k, a workgroup each.
template <typename T, bool WIDE>
__global__ __launch_bounds__(SP_THREADS) void sample_top_k_kernel(SampleParams p) {
  __shared__ SpShared sh;
  const int b = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.logits) + int64_t(b) * p.stride;
  const SpLimits lim = sp_limits(p, b);
  const SpTop top = sp_top(p, b);
  if (sp_decided(p, b, top, lim) || !lim.top_k) return;
  const SpRow row = sp_row(p, b, sp_value(top.key), lim.t);
  if (!sp_top_k<T, WIDE>(sh, p, b, x, row, lim.top_k, lim.top_p)) sp_slow<T>(sh, p, b, x, row, lim.top_k, lim.top_p);
}

// This part's weight under the prefix (cut, last) to p.weight; the last part's
// workgroup draws.
template <typename T, bool WIDE>
__device__ __forceinline__ void sp_draw_parts(SpShared& sh, const SampleParams& p, int b, int c, const T* x, const SpRow& row,
                              uint32_t cut, int last) {
  const int tid = threadIdx.x, n = p.vocab;
  uint64_t sum = 0;
  sp_sweep<T, WIDE>(p, c, x, [&](float v, int i) { sum += sp_kept<T>(row, v, i, cut, last); });
  uint64_t total;
  sp_scan(sh, sum, &total);
  uint64_t* part = p.weight + int64_t(b) * p.parts;
  if (tid == 0) sp_put(part + c, total);
  if (!sp_last(sh, p.counter + 2 * b, p.parts)) return;
  const int lane = tid & 63;
  const uint64_t own = lane < p.parts ? sp_get(part + lane) : 0;
  uint64_t run = own;
#pragma unroll
  for (int d = 1; d < SP_PARTS; d <<= 1) {
    const uint64_t y = __shfl_up(run, d, 64);
    if (lane >= d) run += y;
  }
  const uint64_t all = __shfl(run, SP_PARTS - 1, 64);
  uint64_t target = sp_target(p, b, all);
  const uint64_t past = __ballot(lane < p.parts && run > target);
  const int i = past ? __ffsll((unsigned long long)past) - 1 : p.parts - 1;
  target -= __shfl(run - own, i, 64);
  const int size = sp_part_size<T>(p);
  auto kept = [&](float v, int e) -> uint64_t { return sp_kept<T>(row, v, e, cut, last); };
  const int token = sp_descend(sh, x, i * size, min((i + 1) * size, n), target, kept);
  sp_write(p, b, token, double(kept(sp_load(x, token), token)) / double(all));
}

// Launch 2: rows without a top-k.  With a top-p the bins of the distance to
// the maximum and the bin where p is crossed; without one the draw.
template <typename T, bool WIDE>
__global__ __launch_bounds__(SP_THREADS) void sample_sum_kernel(SampleParams p) {
  __shared__ SpShared sh;
  const int tid = threadIdx.x;
  const int b = int(blockIdx.x) / p.parts, c = int(blockIdx.x) - b * p.parts, n = p.vocab;
  SpState* st = p.state + b;
  const T* x = reinterpret_cast<const T*>(p.logits) + int64_t(b) * p.stride;
  const SpLimits lim = sp_limits(p, b);
  const SpTop top = sp_top(p, b);
  if (lim.top_k || top.key <= SP_MINUS_INF || lim.greedy) {
    if (c == 0) {
      sp_decided(p, b, top, lim);
      if (tid == 0) st->mode = SP_DONE;
    }
    return;
  }
  const SpRow row = sp_row(p, b, sp_value(top.key), lim.t);
  if (!(lim.top_p < 1.f)) {
    if (c == 0 && tid == 0) st->mode = SP_DONE;
    sp_draw_parts<T, WIDE>(sh, p, b, c, x, row, 0, n);
    return;
  }
  for (int i = tid; i < SP_BINS; i += SP_THREADS) {
    sh.mass[i] = 0;
    sh.count[i] = 0;
  }
  __syncthreads();
  sp_sweep<T, WIDE>(p, c, x, [&](float v, int) {
    const uint64_t wt = row.weight(v);
    if (wt) {
      const int bin = row.bin(v);
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[bin]), (unsigned long long)wt);
      atomicAdd(&sh.count[bin], 1u);
    }
  });
  __syncthreads();
  uint64_t* mass = p.mass + int64_t(b) * SP_BINS;
  uint32_t* count = p.count + int64_t(b) * SP_BINS;
  for (int i = tid; i < SP_BINS; i += SP_THREADS)
    if (sh.count[i]) {
      __hip_atomic_fetch_add(mass + i, sh.mass[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_fetch_add(count + i, sh.count[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  if (!sp_last(sh, p.counter + 2 * b, p.parts)) return;
  constexpr int C = SP_BINS / SP_THREADS;
  uint64_t m[C], own = 0, total, own_n = 0, all_n;
  uint32_t k[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    m[i] = sp_get(mass + tid * C + i);
    k[i] = sp_get(count + tid * C + i);
    own += m[i];
    own_n += k[i];
  }
  uint64_t run = sp_scan(sh, own, &total) - own;
  uint64_t run_n = sp_scan(sh, own_n, &all_n) - own_n;
  const double thr = fmax(double(lim.top_p) * double(total), 1.0);
  if (double(run) < thr && double(run + own) >= thr) {
    int i = 0;
#pragma unroll
    for (int j = 0; j < C - 1; ++j)
      if (i == j && double(run + m[j]) < thr) {
        run += m[j];
        run_n += k[j];
        ++i;
      }
    uint32_t here = k[0];
#pragma unroll
    for (int j = 1; j < C; ++j) here = i == j ? k[j] : here;
    st->bin = tid * C + i;
    st->above = run;
    st->total = total;
    st->mode = run_n + here <= uint64_t(SP_FEW) ? SP_SHORT : (here <= uint32_t(SP_LIST) ? SP_BORDER : SP_SLOW);
  }
}

// Launch 3: the tokens down to the crossing bin, or that bin's.
template <typename T, bool WIDE>
__global__ __launch_bounds__(SP_THREADS) void sample_list_kernel(SampleParams p) {
  __shared__ SpShared sh;
  const int tid = threadIdx.x;
  const int b = int(blockIdx.x) / p.parts, c = int(blockIdx.x) - b * p.parts;
  SpState* st = p.state + b;
  const int mode = st->mode;
  if (mode == SP_DONE) return;
  const T* x = reinterpret_cast<const T*>(p.logits) + int64_t(b) * p.stride;
  const SpLimits lim = sp_limits(p, b);
  const SpRow row = sp_row(p, b, sp_value(sp_top(p, b).key), lim.t);
  if (mode == SP_SLOW) {
    if (c == 0) sp_slow<T>(sh, p, b, x, row, 0, lim.top_p);   // (the draw's launch passes such rows by)
    return;
  }
  const int hi = st->bin, lo = mode == SP_BORDER ? hi : 0;
  if (tid == 0) sh.n = 0;
  __syncthreads();
  sp_sweep<T, WIDE>(p, c, x, [&](float v, int i) {
    const uint32_t key = sp_key(v);
    if (key > SP_MINUS_INF) {
      const int bin = row.bin(v);
      // (tokens of weight 0 lie in the last bins, uncounted)
      if (bin >= lo && bin <= hi && row.weight(v) > 0) {
        const uint32_t at = atomicAdd(&sh.n, 1u);
        if (at < uint32_t(SP_LIST)) sh.list[at] = sp_entry(key, i);
      }
    }
  });
  __syncthreads();
  uint64_t* list = p.list + int64_t(b) * SP_LIST;
  uint32_t* listed = p.counter + 2 * b + 1;
  const int mine = min(int(sh.n), SP_LIST);
  if (tid == 0) sh.digit = int(__hip_atomic_fetch_add(listed, uint32_t(mine), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  __syncthreads();
  for (int i = tid; i < mine; i += SP_THREADS)
    if (sh.digit + i < SP_LIST) sp_put(list + sh.digit + i, sh.list[i]);
  if (!sp_last(sh, p.counter + 2 * b, p.parts)) return;
  const int total_n = min(int(sp_get(listed)), SP_LIST);
  __syncthreads();
  if (tid == 0) sp_put(listed, 0u);
  for (int i = tid; i < total_n; i += SP_THREADS) sh.list[i] = sp_get(list + i);
  __syncthreads();
  if (mode == SP_SHORT) {
    sp_draw_list(sh, p, b, row, total_n, 0, lim.top_p, st->total);
    if (tid == 0) st->mode = SP_DONE;
    return;
  }
  const double thr = fmax(double(lim.top_p) * double(st->total), 1.0);
  if (total_n <= SP_FEW) {
    uint64_t e = tid < total_n ? sh.list[tid] : 0;
    if (tid < total_n) sh.other[sp_rank(sh.list, total_n, e)] = e;
    __syncthreads();
    e = tid < total_n ? sh.other[tid] : 0;
    const uint64_t w = tid < total_n ? row.weight(sp_value(uint32_t(e >> 32))) : 0;
    uint64_t all;
    const uint64_t before = st->above + sp_scan(sh, w, &all) - w;
    const int m = __syncthreads_count(tid < total_n && double(before) < thr);
    if (tid == m - 1) {
      st->cut = uint32_t(e >> 32);
      st->last = int(~uint32_t(e));
      st->mode = SP_DRAW;
    }
    return;
  }
  sp_sort(sh.list, total_n);
  sp_running(sh, total_n, [&](int i) { return row.weight(sp_value(uint32_t(sh.list[i] >> 32))); });
  uint64_t kept = 0, m;
  for (int i = tid; i < total_n; i += SP_THREADS) kept += double(st->above + (i ? sh.sum[i - 1] : 0)) < thr ? 1 : 0;
  sp_scan(sh, kept, &m);
  if (tid == 0) {
    st->cut = uint32_t(sh.list[m - 1] >> 32);
    st->last = int(~uint32_t(sh.list[m - 1]));
    st->mode = SP_DRAW;
  }
}

// Launch 4: the draw of rows with a settled border.
template <typename T, bool WIDE>
__global__ __launch_bounds__(SP_THREADS) void sample_draw_kernel(SampleParams p) {
  __shared__ SpShared sh;
  const int b = int(blockIdx.x) / p.parts, c = int(blockIdx.x) - b * p.parts;
  const SpState* st = p.state + b;
  if (st->mode != SP_DRAW) return;
  const T* x = reinterpret_cast<const T*>(p.logits) + int64_t(b) * p.stride;
  const SpLimits lim = sp_limits(p, b);
  const SpRow row = sp_row(p, b, sp_value(sp_top(p, b).key), lim.t);
  sp_draw_parts<T, WIDE>(sh, p, b, c, x, row, st->cut, st->last);
}

// ---- host --------------------------------------------------------------------

struct SpLayout {
  int64_t state, part, weight, group, count, mass, list, total;
};

static SpLayout sp_layout(int64_t batch) {
  SpLayout l{};
  auto up = [](int64_t v) { return (v + 255) & ~int64_t(255); };
  // The counters have the same place and size for every call, so a call of
  // any shape finds them zero.
  l.state = int64_t(SP_MAX_BATCH) * 8;
  l.count = up(l.state + batch * int64_t(sizeof(SpState)));
  l.mass = up(l.count + batch * SP_BINS * 4);
  l.part = up(l.mass + batch * SP_BINS * 8);
  l.weight = up(l.part + batch * SP_PARTS * 8);
  l.group = up(l.weight + batch * SP_PARTS * 8);
  l.list = up(l.group + batch * SP_GROUPS * 4);
  l.total = up(l.list + batch * SP_LIST * 8);
  return l;
}

template <typename T, bool WIDE>
static void sp_launch(const SampleParams& p, hipStream_t stream) {
  const dim3 grid(uint32_t(p.batch) * uint32_t(p.parts)), block(SP_THREADS);
  hipLaunchKernelGGL((sample_max_kernel<T, WIDE>), grid, block, 0, stream, p);
  // One value for all rows says which launches none of them needs.
  const bool all_top_k = !p.top_k && p.top_k_all > 0 && p.top_k_all < p.vocab;
  const bool all_greedy = !p.temperature && !(p.temperature_all > 0.f);
  if (p.top_k || all_top_k || all_greedy)
    hipLaunchKernelGGL((sample_top_k_kernel<T, WIDE>), dim3(p.batch), block, 0, stream, p);
  if (all_top_k || all_greedy) return;
  hipLaunchKernelGGL((sample_sum_kernel<T, WIDE>), grid, block, 0, stream, p);
  if (!p.top_p && !(p.top_p_all < 1.f)) return;
  hipLaunchKernelGGL((sample_list_kernel<T, WIDE>), grid, block, 0, stream, p);
  hipLaunchKernelGGL((sample_draw_kernel<T, WIDE>), grid, block, 0, stream, p);
}

template <typename T>
static void sp_dispatch(SampleParams& p, hipStream_t stream) {
  constexpr int VL = 16 / sizeof(T);
  // Parts per row, up to 16: as many as put 512 workgroups (two per CU) on the
  // chip, and as give a thread no more than eight vectors (fp32 rows of up to
  // 262144 tokens, 16-bit ones of 524288; longer rows up to 32), so that single
  // rows of a large batch that need the later launches are not read by one or
  // two workgroups.
  const int steps = (p.vocab + SP_THREADS * VL - 1) / (SP_THREADS * VL);
  const int want = std::min({steps, SP_PARTS, std::max((steps + 7) / 8, (512 + p.batch - 1) / p.batch)});
  p.steps = (steps + want - 1) / want;
  p.parts = (steps + p.steps - 1) / p.steps;
  const bool wide = aligned16(p.logits) && (p.batch == 1 || p.stride % VL == 0);
  if (wide) sp_launch<T, true>(p, stream);
  else sp_launch<T, false>(p, stream);
}

}  // namespace tierkv

using namespace tierkv;

extern "C" int64_t tierkv_sample_workspace_bytes(int32_t batch, int32_t vocab) {
  if (batch <= 0 || vocab <= 0) return -1;
  return sp_layout(batch).total;
}

extern "C" int32_t tierkv_sample_tokens(
    const void* logits, int32_t dtype, int64_t row_stride, int32_t batch, int32_t vocab, const float* uniforms,
    const float* temperature, float temperature_all, const int32_t* top_k, int32_t top_k_all,
    const float* top_p, float top_p_all, const float* min_p, float min_p_all,
    int64_t* tokens, float* probs, void* workspace, int64_t workspace_bytes, void* stream_) {
  clear_error();
  if (!logits || !uniforms || !tokens || !workspace) return fail(TIERKV_ERR_INVALID, "null pointer");
  if (batch <= 0 || vocab <= 0) return fail(TIERKV_ERR_INVALID, "empty logits");
  if (vocab > SP_MAX_VOCAB) return fail(TIERKV_ERR_UNSUPPORTED, "vocabularies of more than 2^20 tokens");
  if (batch > 1 && row_stride < vocab) return fail(TIERKV_ERR_INVALID, "logit rows overlap");
  if (dtype != TIERKV_DTYPE_F16 && dtype != TIERKV_DTYPE_BF16 && dtype != TIERKV_DTYPE_F32)
    return fail(TIERKV_ERR_INVALID, "logits must be fp16, bf16 or fp32");
  if (batch > SP_MAX_BATCH) return fail(TIERKV_ERR_UNSUPPORTED, "more than 65536 rows");
  if (!aligned16(workspace)) return fail(TIERKV_ERR_INVALID, "the workspace must be 16-byte aligned");
  if (workspace_bytes < tierkv_sample_workspace_bytes(batch, vocab))
    return fail(TIERKV_ERR_WORKSPACE, "workspace too small");
  SampleParams p{};
  p.logits = logits;
  p.stride = row_stride;
  p.batch = batch;
  p.vocab = vocab;
  p.u = uniforms;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.temperature_all = temperature_all;
  p.top_k_all = top_k_all;
  p.top_p_all = top_p_all;
  p.min_p_all = min_p_all;
  p.tokens = tokens;
  p.probs = probs;
  const SpLayout l = sp_layout(batch);
  char* ws = reinterpret_cast<char*>(workspace);
  p.counter = reinterpret_cast<uint32_t*>(ws);
  p.state = reinterpret_cast<SpState*>(ws + l.state);
  p.part = reinterpret_cast<uint64_t*>(ws + l.part);
  p.weight = reinterpret_cast<uint64_t*>(ws + l.weight);
  p.group = reinterpret_cast<uint32_t*>(ws + l.group);
  p.count = reinterpret_cast<uint32_t*>(ws + l.count);
  p.mass = reinterpret_cast<uint64_t*>(ws + l.mass);
  p.list = reinterpret_cast<uint64_t*>(ws + l.list);
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (dtype == TIERKV_DTYPE_F32) sp_dispatch<float>(p, stream);
  else if (dtype == TIERKV_DTYPE_BF16) sp_dispatch<__hip_bfloat16>(p, stream);
  else sp_dispatch<__half>(p, stream);
  return check_launch("tierkv_sample_tokens");
}
