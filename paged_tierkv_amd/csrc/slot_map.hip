// Slot maps of a serving step over requests of different lengths, and the
// write of the step's packed K/V rows, on gfx950.
//
// tierkv_build_slot_map: request b brings n_b tokens.  Its open block (the
// last one, when open[b] is set, it is HOT and not full) takes
//   room_b = block_size - length  tokens first, then
//   need_b = ceil(max(n_b - room_b, 0) / block_size)  new HOT blocks, popped
// from the free stack in (request, block) order: block j of request b is
// free[top - 1 - (e_b + j)] with e the exclusive prefix sum of need.  The
// packed row r = cu[b] + i of token i gets its HOT pool row slot * block_size
// + position and the token's position in its request (tokens held + i).  All
// or nothing, as tierkv_runtime_append.
//
// Bound: latency, a chain of dependent reads (counts, then the last blocks'
// entries and the rows of lengths, then the stack) around two prefix sums.
// Small steps run in one workgroup (nothing but LDS between the phases);
// larger ones in two launches: the prefix sums in one workgroup beside the
// sums of the rows of lengths in others, then the rows, four per thread.
// Nothing is written to the tables before every read of them is done: the
// first launch (or phase) only reads.  Measured: 10.3 us in one workgroup (64
// requests, tables of 256 blocks), 6.0 + 5.6 us in two launches (256 requests,
// 26 700 packed rows).

#include "tierkv_common.h"

namespace tierkv {

constexpr int SM_THREADS = 1024;
constexpr int SM_WAVES = SM_THREADS / 64;
constexpr int SM_MAX_BATCH = 4096;              // as tierkv_runtime_append
constexpr int SM_NIT = SM_MAX_BATCH / SM_THREADS;
// One workgroup holds a step of at most SM_ONE_BATCH requests (four per wave,
// all lengths read at once), SM_ONE_ROWS packed rows (four per thread) and
// tables of SM_ONE_BLOCKS blocks.  Measured with one workgroup against two
// launches, replayed from a graph behind a 2 us copy of the tables (us):
//   requests x new tokens x blocks   one    two
//    1 x  1 x   16                   6.9   10.9
//    8 x 16 x  256                  10.1   11.8
//   64 x  1 x   16                   9.5   12.4
//   64 x 60 x  256                  12.4   13.0
//   64 x 16 x 1024                  14.1   14.4
// (level at tables of 512 to 1024 blocks, half a microsecond either way:
// 64 x 1 x 1024 14.4 and 13.9, 64 x 16 x 512 13.0 and 12.7), and with a workgroup that took several passes beyond these limits:
//   64 x 700 x 16                   27.6   12.9
//  256 x   1 x 64                   18.1   14.0
constexpr int SM_ONE_BATCH = 64;
constexpr int SM_ONE_ROWS = 4 * SM_THREADS;
constexpr int SM_ONE_BLOCKS = 1024;
constexpr int SM_FILL = 256;                    // threads of a fill workgroup
constexpr int SM_ROWS = SM_FILL * 4;            // packed rows per fill workgroup

constexpr int SM_ERR_HOT_EMPTY = 1;
constexpr int SM_ERR_TABLE_FULL = 4;
constexpr int SM_ERR_OPEN_STATE = 8;
constexpr int SM_ERR_ROWS = 16;                 // negative lengths, or more tokens than packed rows

struct SlotMapParams {
  const int32_t* new_tokens;
  int32_t batch, rows;
  int32_t* table;
  int32_t* states;
  int32_t* lengths;
  int64_t stride;
  int32_t* nblocks;
  int32_t* open;
  const int32_t* hot_free;
  int32_t hot_slots;
  int32_t* ctl;
  int32_t bs;
  int32_t* slots;
  int32_t* positions;
  int32_t* cu;
  int32_t* context;
  int4* seq;        // [batch] {first stack index, room, blocks before, new tokens}
  int32_t* held;    // [batch] tokens before
  int32_t* head;    // {ok, stack top, error bits, new blocks}
};

// Inclusive prefix sums of two 64-bit values over the workgroup.
struct Sm2 {
  int64_t n, need;
};
__device__ __forceinline__ Sm2 sm_scan(Sm2 v, Sm2* sh, Sm2* total) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  Sm2 x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t a = __shfl_up(x.n, d, 64), b = __shfl_up(x.need, d, 64);
    if (lane >= d) {
      x.n += a;
      x.need += b;
    }
  }
  __syncthreads();
  if (lane == 63) sh[w] = x;
  __syncthreads();
  Sm2 all = {0, 0};
#pragma unroll
  for (int i = 0; i < SM_WAVES; ++i) {
    const Sm2 t = sh[i];
    if (i < w) {
      x.n += t.n;
      x.need += t.need;
    }
    all.n += t.n;
    all.need += t.need;
  }
  *total = all;
  return x;
}

// Tokens that each request of [b0, b0 + 4) holds, the sums of their blocks'
// lengths, by the 16-lane rows of one wave (four requests of 256 blocks: two
// memory round trips, where a wave per request in turn took eight).
__device__ __forceinline__ void tokens_held(const SlotMapParams& p, int b0, int32_t* held) {
  const int lane = threadIdx.x & 63, c = lane & 15, b = b0 + (lane >> 4);
  int sum = 0;
  if (b < p.batch) {
    const int nb = min(max(p.nblocks[b], 0), int(min(p.stride, int64_t(0x7fffffff))));
    const int32_t* row = p.lengths + int64_t(b) * p.stride;
    int i = c;
    for (; i + 7 * 16 < nb; i += 8 * 16) {
      int v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = row[i + k * 16];
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += min(max(v[k], 0), p.bs);
    }
    for (; i < nb; i += 16) sum += min(max(row[i], 0), p.bs);
  }
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, 64);
  if (c == 0 && b < p.batch) held[b] = sum;
}

// The prefix sums (one workgroup of SM_THREADS): writes cu, the requests'
// plan entries (seq) and the head; cu also to where the caller keeps it.
template <int NIT>
__device__ __forceinline__ void sm_plan(const SlotMapParams& p, Sm2* sh, int* s_err, int4* seq, int32_t* head,
                                        int32_t* cu) {
  const int tid = threadIdx.x, B = p.batch, bs = p.bs;
  const int nit = (B + SM_THREADS - 1) / SM_THREADS;   // at most NIT
  int n[NIT], room[NIT], nb[NIT];
  int64_t need[NIT], cu_end[NIT], first[NIT];
  const int top = min(max(p.ctl[0], 0), p.hot_slots);
  if (tid == 0) *s_err = 0;
  __syncthreads();
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    n[it] = room[it] = nb[it] = 0;
    need[it] = 0;
    const int b = it * SM_THREADS + tid;
    if (it < nit && b < B) {
      n[it] = p.new_tokens[b];
      nb[it] = p.nblocks[b];
      const int opn = p.open[b];
      if (n[it] < 0) atomicOr(s_err, SM_ERR_ROWS);
      n[it] = max(n[it], 0);
      if (nb[it] < 0 || nb[it] > p.stride) {
        if (n[it] > 0) atomicOr(s_err, SM_ERR_TABLE_FULL);
        nb[it] = 0;
      } else if (n[it] > 0 && nb[it] > 0 && opn != 0) {
        const int64_t o = int64_t(b) * p.stride + nb[it] - 1;
        const int len = min(max(p.lengths[o], 0), bs);
        if (p.states[o] == HOT) room[it] = bs - len;
        else if (len < bs) atomicOr(p.ctl + 2, SM_ERR_OPEN_STATE);
      }
      need[it] = n[it] > room[it] ? (int64_t(n[it]) - room[it] + bs - 1) / bs : 0;
      if (nb[it] + need[it] > p.stride) atomicOr(s_err, SM_ERR_TABLE_FULL);
    }
  }
  int64_t tokens = 0, blocks = 0;
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    if (it < nit) {
      Sm2 total;
      const Sm2 x = sm_scan({n[it], need[it]}, sh, &total);
      cu_end[it] = tokens + x.n;
      first[it] = blocks + x.need - need[it];
      tokens += total.n;
      blocks += total.need;
    }
  }
  if (tid == 0) {
    if (tokens > p.rows) atomicOr(s_err, SM_ERR_ROWS);
    else if (blocks > top && *s_err == 0) atomicOr(s_err, SM_ERR_HOT_EMPTY);
  }
  __syncthreads();
  const bool ok = *s_err == 0;
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    const int b = it * SM_THREADS + tid;
    if (it < nit && b < B) {
      p.cu[b + 1] = ok ? int32_t(cu_end[it]) : 0;
      if (cu) cu[b + 1] = ok ? int32_t(cu_end[it]) : 0;
      seq[b] = make_int4(ok ? int32_t(first[it]) : 0, room[it], nb[it], ok ? n[it] : 0);
    }
  }
  if (tid == 0) {
    p.cu[0] = 0;
    if (cu) cu[0] = 0;
    head[0] = ok;
    head[1] = top;
    head[2] = *s_err;
    head[3] = ok ? int32_t(blocks) : 0;
  }
}

// Counts, open flags, the open blocks' lengths and the tokens held after the
// step, of request b.
__device__ __forceinline__ void sm_update(const SlotMapParams& p, int b, const int4 s, int held) {
  const int n = s.w, bs = p.bs;
  p.context[b] = held + n;
  if (n == 0) return;
  const int taken = min(s.y, n);
  const int need = (n - taken + bs - 1) / bs;
  if (taken > 0) p.lengths[int64_t(b) * p.stride + s.z - 1] = bs - s.y + taken;
  p.nblocks[b] = s.z + need;
  const int last = need > 0 ? n - taken - (need - 1) * bs : bs - s.y + taken;
  p.open[b] = last < bs ? 1 : 0;
}

__device__ __forceinline__ void sm_finish(const SlotMapParams& p, const int32_t* head) {
  if (head[2]) atomicOr(p.ctl + 2, head[2]);
  if (head[0]) p.ctl[0] = head[1] - head[3];
  p.ctl[3] = head[0];
}

// Rows [r0, r0 + 4) of the packed step: their slots and positions, and the
// table entries of the blocks whose first token is among them.  cu is in LDS.
__device__ __forceinline__ void sm_rows(const SlotMapParams& p, const int32_t* cu, const int4* seq, const int32_t* held,
                                        int top, int r0) {
  const int B = p.batch, bs = p.bs;
  const int total = cu[B];
  int lo = 0, hi = B;                       // cu[lo] <= r0 < cu[hi] (when r0 < total)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= r0) lo = mid;
    else hi = mid;
  }
  int b = lo, slot[4], pos[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + k;
    slot[k] = pos[k] = -1;
    if (r < total) {
      while (cu[b + 1] <= r) ++b;
      const int4 s = seq[b];
      const int i = r - cu[b];
      pos[k] = held[b] + i;
      const int64_t row = int64_t(b) * p.stride;
      if (i < s.y) {
        slot[k] = p.table[row + s.z - 1] * bs + (bs - s.y) + i;
      } else {
        const int j = (i - s.y) / bs, q = (i - s.y) - j * bs;
        const int id = p.hot_free[top - 1 - (s.x + j)];
        slot[k] = id * bs + q;
        if (q == 0) {
          p.table[row + s.z + j] = id;
          p.states[row + s.z + j] = HOT;
          p.lengths[row + s.z + j] = min(s.w - i, bs);
        }
      }
    }
  }
  if (r0 + 4 <= p.rows) {
    reinterpret_cast<int4*>(p.slots)[r0 >> 2] = make_int4(slot[0], slot[1], slot[2], slot[3]);
    reinterpret_cast<int4*>(p.positions)[r0 >> 2] = make_int4(pos[0], pos[1], pos[2], pos[3]);
  } else {
    for (int k = 0; k < 4; ++k)
      if (r0 + k < p.rows) {
        p.slots[r0 + k] = slot[k];
        p.positions[r0 + k] = pos[k];
      }
  }
}

// The whole step in one workgroup; what passes between the phases is in LDS.
__global__ __launch_bounds__(SM_THREADS) void slot_map_kernel(SlotMapParams p) {
  __shared__ Sm2 sh[SM_WAVES];
  __shared__ int s_err;
  __shared__ int32_t s_head[4];
  __shared__ int32_t s_cu[SM_ONE_BATCH + 1];
  __shared__ int32_t s_held[SM_ONE_BATCH];
  __shared__ int4 s_seq[SM_ONE_BATCH];
  static_assert(SM_ONE_BATCH == SM_WAVES * 4 && SM_ONE_ROWS == SM_THREADS * 4, "one pass each");
  const int tid = threadIdx.x;
  tokens_held(p, (tid >> 6) * 4, s_held);
  sm_plan<1>(p, sh, &s_err, s_seq, s_head, s_cu);
  __syncthreads();
  if (tid * 4 < p.rows) sm_rows(p, s_cu, s_seq, s_held, s_head[1], tid * 4);
  if (tid < p.batch) sm_update(p, tid, s_seq[tid], s_held[tid]);
  if (tid == 0) sm_finish(p, s_head);
}

// First launch of a large step: workgroup 0 forms the prefix sums, the
// others the tokens held, four requests per wave.
__global__ __launch_bounds__(SM_THREADS) void slot_plan_kernel(SlotMapParams p) {
  __shared__ Sm2 sh[SM_WAVES];
  __shared__ int s_err;
  if (blockIdx.x == 0) {
    sm_plan<SM_NIT>(p, sh, &s_err, p.seq, p.head, nullptr);
    return;
  }
  tokens_held(p, ((int(blockIdx.x) - 1) * SM_WAVES + (int(threadIdx.x) >> 6)) * 4, p.held);
}

// Second launch: the packed rows, and the requests' own words.
__global__ __launch_bounds__(SM_FILL) void slot_fill_kernel(SlotMapParams p) {
  __shared__ int32_t s_cu[SM_MAX_BATCH + 1];
  const int tid = threadIdx.x;
  for (int b = tid; b <= p.batch; b += SM_FILL) s_cu[b] = p.cu[b];
  __syncthreads();
  const int64_t r = int64_t(blockIdx.x) * SM_ROWS + tid * 4;
  if (r < p.rows) sm_rows(p, s_cu, p.seq, p.held, p.head[1], int(r));
  for (int b = int(blockIdx.x) * SM_FILL + tid; b < p.batch; b += int(gridDim.x) * SM_FILL)
    sm_update(p, b, p.seq[b], p.held[b]);
  if (blockIdx.x == 0 && tid == 0) sm_finish(p, p.head);
}

// ---------------------------------------------------------------------------
// tierkv_write_slots: row r of k / v [rows, kv_heads, D] into HOT pool row
// slots[r] = slot * block_size + position.  A copy: bound by memory.  One
// thread per 16 bytes of output (eight elements), so a row's reads and each
// head's writes are whole segments.  Measured: 16384 bf16 rows of 8 heads of
// 128, read and written 134 MB, 21.9 us, 6.1 TB/s; 64 rows 2.8 us.
// ---------------------------------------------------------------------------
struct WriteSlotsParams {
  const void* src[2];
  int64_t st_t[2], st_h[2];
  const int32_t* slots;
  int32_t rows, kv_heads, bs, D;
  int64_t pool_rows;      // hot_slots * block_size
  __half* hot[2];
};

template <typename T>
__device__ __forceinline__ uint4 to_half8(uint4 v);
template <>
__device__ __forceinline__ uint4 to_half8<__half>(uint4 v) { return v; }
template <>
__device__ __forceinline__ uint4 to_half8<__hip_bfloat16>(uint4 v) {
  auto two = [](uint32_t w) { return pack_f16x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); };
  return make_uint4(two(v.x), two(v.y), two(v.z), two(v.w));
}

template <typename T>
__global__ __launch_bounds__(256) void write_slots_kernel(WriteSlotsParams p, int32_t per_row) {
  const int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int kv = blockIdx.y;
  const int64_t r = e / per_row;
  if (r >= p.rows) return;
  const int x = int(e - r * per_row);
  const int C = p.D >> 3;
  const int h = x / C, c = x - h * C;
  const int row = p.slots[r];
  const T* src = reinterpret_cast<const T*>(p.src[kv]) + r * p.st_t[kv] + h * p.st_h[kv];
  const uint4 v = reinterpret_cast<const uint4*>(src)[c];
  if (row < 0 || row >= p.pool_rows) return;
  const int64_t slot = row / p.bs;
  const int pos = row - int(slot) * p.bs;
  reinterpret_cast<uint4*>(p.hot[kv] + ((slot * p.kv_heads + h) * p.bs + pos) * p.D)[c] = to_half8<T>(v);
}

// Any strides, alignment and head dim: one element per thread.
template <typename T>
__global__ __launch_bounds__(256) void write_slots_scalar_kernel(WriteSlotsParams p, int32_t per_row) {
  const int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int kv = blockIdx.y;
  const int64_t r = e / per_row;
  if (r >= p.rows) return;
  const int x = int(e - r * per_row);
  const int h = x / p.D, d = x - h * p.D;
  const int row = p.slots[r];
  if (row < 0 || row >= p.pool_rows) return;
  const int64_t slot = row / p.bs;
  const int pos = row - int(slot) * p.bs;
  const T* src = reinterpret_cast<const T*>(p.src[kv]) + r * p.st_t[kv] + h * p.st_h[kv];
  p.hot[kv][((slot * p.kv_heads + h) * p.bs + pos) * p.D + d] = from_f32<__half>(to_f32<T>(src[d]));
}

template <typename T>
static void launch_write(const WriteSlotsParams& p, bool wide, hipStream_t stream) {
  const int per_row = p.kv_heads * (wide ? p.D / 8 : p.D);
  const dim3 grid(uint32_t((int64_t(p.rows) * per_row + 255) / 256), 2);
  if (wide) hipLaunchKernelGGL(write_slots_kernel<T>, grid, dim3(256), 0, stream, p, per_row);
  else hipLaunchKernelGGL(write_slots_scalar_kernel<T>, grid, dim3(256), 0, stream, p, per_row);
}

}  // namespace tierkv

using namespace tierkv;

extern "C" int64_t tierkv_slot_map_workspace_bytes(int32_t batch) {
  if (batch <= 0) return -1;
  return 256 + int64_t(batch) * 20;
}

extern "C" int32_t tierkv_build_slot_map(
    const int32_t* new_tokens, int32_t batch, int32_t num_rows,
    int32_t* block_table, int32_t* block_states, int32_t* block_lengths, int64_t table_stride,
    int32_t* seq_num_blocks, int32_t* open_blocks, const int32_t* hot_free, int64_t hot_slots, int32_t* ctl,
    int32_t block_size, int32_t* slots, int32_t* positions, int32_t* cu_tokens, int32_t* context,
    void* workspace, int64_t workspace_bytes, void* stream_) {
  clear_error();
  if (!new_tokens || !block_table || !block_states || !block_lengths || !seq_num_blocks || !open_blocks || !hot_free ||
      !ctl || !cu_tokens || !context || !workspace || (num_rows > 0 && (!slots || !positions)))
    return fail(TIERKV_ERR_INVALID, "null pointer");
  if (batch <= 0 || num_rows < 0 || table_stride <= 0 || hot_slots <= 0)
    return fail(TIERKV_ERR_INVALID, "empty slot map");
  if (num_rows > (1 << 30)) return fail(TIERKV_ERR_UNSUPPORTED, "a slot map takes at most 2^30 packed rows");
  if (batch > SM_MAX_BATCH) return fail(TIERKV_ERR_UNSUPPORTED, "a slot map takes at most 4096 requests per call");
  if (block_size <= 0 || block_size > 64) return fail(TIERKV_ERR_UNSUPPORTED, "block_size must be in [1, 64]");
  if (hot_slots * block_size > 0x7fffffff || table_stride * block_size > 0x7fffffff)
    return fail(TIERKV_ERR_UNSUPPORTED, "pool rows or positions past 32 bits");
  if (!aligned16(workspace) || (num_rows > 0 && (!aligned16(slots) || !aligned16(positions))))
    return fail(TIERKV_ERR_INVALID, "slots, positions and the workspace must be 16-byte aligned");
  if (workspace_bytes < tierkv_slot_map_workspace_bytes(batch)) return fail(TIERKV_ERR_WORKSPACE, "workspace too small");
  char* ws = reinterpret_cast<char*>(workspace);
  SlotMapParams p{};
  p.new_tokens = new_tokens;
  p.batch = batch;
  p.rows = num_rows;
  p.table = block_table;
  p.states = block_states;
  p.lengths = block_lengths;
  p.stride = table_stride;
  p.nblocks = seq_num_blocks;
  p.open = open_blocks;
  p.hot_free = hot_free;
  p.hot_slots = int32_t(hot_slots);
  p.ctl = ctl;
  p.bs = block_size;
  p.slots = slots;
  p.positions = positions;
  p.cu = cu_tokens;
  p.context = context;
  p.head = reinterpret_cast<int32_t*>(ws);
  p.seq = reinterpret_cast<int4*>(ws + 256);
  p.held = reinterpret_cast<int32_t*>(ws + 256 + int64_t(batch) * 16);
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (batch <= SM_ONE_BATCH && num_rows <= SM_ONE_ROWS && table_stride <= SM_ONE_BLOCKS) {
    hipLaunchKernelGGL(slot_map_kernel, dim3(1), dim3(SM_THREADS), 0, stream, p);
  } else {
    hipLaunchKernelGGL(slot_plan_kernel, dim3(1 + (batch + SM_WAVES * 4 - 1) / (SM_WAVES * 4)), dim3(SM_THREADS), 0, stream, p);
    const int wgs = int((int64_t(num_rows) + SM_ROWS - 1) / SM_ROWS);
    hipLaunchKernelGGL(slot_fill_kernel, dim3(wgs > 0 ? wgs : 1), dim3(SM_FILL), 0, stream, p);
  }
  return check_launch("tierkv_build_slot_map");
}

extern "C" int32_t tierkv_write_slots(
    const void* key, int64_t k_stride_t, int64_t k_stride_h, const void* value, int64_t v_stride_t, int64_t v_stride_h,
    int32_t dtype, const int32_t* slots, int32_t num_rows, void* hot_k, void* hot_v, int64_t hot_slots,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream_) {
  clear_error();
  if (num_rows < 0) return fail(TIERKV_ERR_INVALID, "negative row count");
  if (dtype != TIERKV_DTYPE_F16 && dtype != TIERKV_DTYPE_BF16)
    return fail(TIERKV_ERR_INVALID, "K/V rows must be fp16 or bf16");
  if (num_kv_heads <= 0 || block_size <= 0 || block_size > 64 || head_dim <= 0 || head_dim > 256)
    return fail(TIERKV_ERR_UNSUPPORTED, "block_size must be in [1, 64] and head_dim in [1, 256]");
  if (hot_slots <= 0 || hot_slots * block_size > 0x7fffffff)
    return fail(TIERKV_ERR_UNSUPPORTED, "pool rows must lie in (0, 2^31)");
  if (num_rows == 0) return TIERKV_OK;
  if (!key || !value || !slots || !hot_k || !hot_v) return fail(TIERKV_ERR_INVALID, "null pointer");
  if (k_stride_t < 0 || k_stride_h < 0 || v_stride_t < 0 || v_stride_h < 0)
    return fail(TIERKV_ERR_INVALID, "strides must be non-negative");
  WriteSlotsParams p{};
  p.src[0] = key;
  p.src[1] = value;
  p.st_t[0] = k_stride_t;
  p.st_h[0] = k_stride_h;
  p.st_t[1] = v_stride_t;
  p.st_h[1] = v_stride_h;
  p.slots = slots;
  p.rows = num_rows;
  p.kv_heads = num_kv_heads;
  p.bs = block_size;
  p.D = head_dim;
  p.pool_rows = hot_slots * block_size;
  p.hot[0] = reinterpret_cast<__half*>(hot_k);
  p.hot[1] = reinterpret_cast<__half*>(hot_v);
  const bool wide = head_dim % 8 == 0 && ((k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 7) == 0 &&
                    aligned16(key) && aligned16(value) && aligned16(hot_k) && aligned16(hot_v);
  // One thread per vector or element, and fewer than 2^32 threads in a launch.
  if (int64_t(num_rows) * num_kv_heads > (0xffffffffll - 255) / (wide ? head_dim / 8 : head_dim))
    return fail(TIERKV_ERR_UNSUPPORTED, "write too large for one call");
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (dtype == TIERKV_DTYPE_BF16) launch_write<__hip_bfloat16>(p, wide, stream);
  else launch_write<__half>(p, wide, stream);
  return check_launch("tierkv_write_slots");
}
