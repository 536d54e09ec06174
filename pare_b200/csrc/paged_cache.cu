// Paged KV cache held in 8 bits, sm_100a: the step's tables, the append and the dense reconstruction (attention over it:
// paged_attn.cu).  The reference keeps one dense batch per cache (pare/kv_cache.py:163-288); a server's requests come and go and
// have lengths of their own, so here a pool of blocks of `bs` tokens is shared by R requests through a block table.
//
// A block is quantized once, when its last token arrives, with one scale per (block, head) for keys and one for values:
//   s = max |x| / 127 over the block's bs x D values of a head,   c = round_half_even(x / s) in [-127, 127].
// Until then its tokens stay in the input type in the request's open rows (tail_k / tail_v), so every code is the result of one
// rounding and tokens fed in pieces give what the same tokens fed at once give (the property of the reference's residual window,
// pare/kv_cache.py:231-244).
#include "paged.cuh"
#include "quant8.cuh"

namespace pare {
namespace {

using namespace paged;

// ---- tables -----------------------------------------------------------------------------------------------------------------------
// One prefix sum over the requests gives everything: first row of a request's new tokens, blocks taken from the free stack before
// it, touched blocks before it.  A thread block holds the sums of all requests in shared memory (every thread block computes them
// for itself: no order between thread blocks), then tokens, fresh blocks and touched blocks are spread over all threads, each
// finding its request by bisection.  Bound by latency: two dependent reads and a scan; 16 bytes are written per token.
constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;

struct PlanParams {
  const int* seq_lens;
  const int* new_lens;
  int* table;
  int64_t ld_table;
  const int* free_blocks;
  const int* free_count;
  int* step;
  int64_t o_query_start, o_seq_lens, o_context, o_slots, o_request, o_positions, o_units, o_info, o_items;
  int R, T, bs_log2, max_blocks, free_capacity, n_items, units;
};

// Exclusive prefix sum of one value per thread, and the total.  All threads call it.
__device__ __forceinline__ long long block_scan(long long v, long long* sums, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanWarps; ++w) {
    const long long s = sums[w];
    if (w < warp) before += s;
    all += s;
  }
  total = all;
  return before + x - v;
}

// Largest i in [0, n) with start[i] <= x (start[0] = 0 <= x, not decreasing).
__device__ __forceinline__ int last_at_most(const int* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanParams p) {
  extern __shared__ int s_mem[];
  __shared__ long long s_sums[kPlanWarps];
  int* s_start = s_mem;              // [R] first row of the new tokens
  int* s_len = s_start + p.R;        // [R] tokens before the step
  int* s_take = s_len + p.R;         // [R] blocks taken from the stack by the requests before
  int* s_item = s_take + p.R;        // [R] blocks touched by the requests before
  const int R = p.R, bs = 1 << p.bs_log2, per = (R + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
  const bool lead = blockIdx.x == 0;
  const int64_t max_len = (int64_t)p.max_blocks << p.bs_log2;

  int bad = 0;
  long long n_new = 0, n_take = 0, n_item = 0, n_ctx = 0;
  for (int r = r0; r < r1; ++r) {
    const int len = p.seq_lens[r], add = p.new_lens[r];
    if (len < 0 || add < 0) bad |= PARE_PAGED_NEGATIVE;
    else if (add > p.T) bad |= PARE_PAGED_ROWS;
    else if ((int64_t)len + add > max_len) bad |= PARE_PAGED_TABLE;
    else {
      const int end = len + add;
      s_start[r] = (int)n_new;
      s_len[r] = len;
      s_take[r] = (int)n_take;
      s_item[r] = (int)n_item;
      n_new += add;
      n_take += ((end + bs - 1) >> p.bs_log2) - ((len + bs - 1) >> p.bs_log2);
      if (add) {
        n_item += ((end - 1) >> p.bs_log2) - (len >> p.bs_log2) + 1;
        n_ctx += end;
      }
    }
  }
  const int count = *p.free_count;
  if (count < 0 || count > p.free_capacity) bad |= PARE_PAGED_BLOCKS;
  long long t_new, t_take, t_item, t_ctx;
  const long long b_new = block_scan(n_new, s_sums, t_new), b_take = block_scan(n_take, s_sums, t_take);
  const long long b_item = block_scan(n_item, s_sums, t_item), b_ctx = block_scan(n_ctx, s_sums, t_ctx);
  if (t_new > p.T) bad |= PARE_PAGED_ROWS;
  if (t_take > count) bad |= PARE_PAGED_BLOCKS;
  __shared__ int s_bad;
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  if (bad) atomicOr(&s_bad, bad);
  __syncthreads();
  bad = s_bad;                       // the step is done or refused as a whole
  if (bad) t_new = t_take = t_item = 0;
  long long ctx = b_ctx;
  for (int r = r0; r < r1; ++r) {
    if (!bad) {
      s_start[r] += (int)b_new;
      s_take[r] += (int)b_take;
      s_item[r] += (int)b_item;
    }
    if (lead) {
      const int len = p.seq_lens[r], add = bad ? 0 : p.new_lens[r];
      p.step[p.o_query_start + r] = bad ? 0 : s_start[r];
      p.step[p.o_seq_lens + r] = len + add;
      reinterpret_cast<long long*>(p.step + p.o_context)[r] = bad ? 0 : ctx;
      if (add) ctx += len + add;
    }
  }
  if (lead && threadIdx.x == 0) {
    p.step[0] = bad;
    p.step[1] = (int)t_new;
    p.step[2] = (int)t_item;
    p.step[3] = 0;
    p.step[p.o_query_start + R] = (int)t_new;
    p.step[p.o_seq_lens + R] = count - (int)t_take;
    reinterpret_cast<long long*>(p.step + p.o_context)[R] = bad ? 0 : t_ctx;
  }
  __syncthreads();

  const int g = blockIdx.x * kPlanThreads + threadIdx.x, stride = gridDim.x * kPlanThreads;
  // block `blk` of request r, taken in this step or before
  auto block_id = [&](int r, int blk) {
    const int have = (s_len[r] + bs - 1) >> p.bs_log2;
    return blk < have ? p.table[r * p.ld_table + blk] : p.free_blocks[count - 1 - (s_take[r] + blk - have)];
  };
  long long* slots = reinterpret_cast<long long*>(p.step + p.o_slots);
  for (int i = g; i < p.T; i += stride) {
    int r = -1, pos = -1;
    long long slot = -1;
    if (i < t_new) {
      r = last_at_most(s_start, R, i);
      pos = s_len[r] + i - s_start[r];
      slot = ((long long)block_id(r, pos >> p.bs_log2) << p.bs_log2) + (pos & (bs - 1));
    }
    if (p.units) {
      const int end = r < 0 ? 0 : s_len[r] + (r + 1 < R ? s_start[r + 1] : (int)t_new) - s_start[r];
      *reinterpret_cast<int4*>(p.step + p.o_info + 4 * (int64_t)i) = make_int4(r, pos, end, 0);
    }
    p.step[p.o_request + i] = r;
    p.step[p.o_positions + i] = pos;
    slots[i] = slot;
  }
  for (int i = g; i < p.n_items; i += stride) {
    int4 a = make_int4(-1, -1, 0, 0), b = make_int4(0, 0, 0, 0);
    if (i < t_item) {
      const int r = last_at_most(s_item, R, i), len = s_len[r];
      const int end = len + (r + 1 < R ? s_start[r + 1] : (int)t_new) - s_start[r];
      const int blk = (len >> p.bs_log2) + i - s_item[r], p0 = max(len, blk << p.bs_log2), p1 = min(end, (blk + 1) << p.bs_log2);
      a = make_int4(r, block_id(r, blk), s_start[r] + p0 - len, p0 & (bs - 1));
      b = make_int4(p1 - p0, blk, len, end);
    }
    int4* at = reinterpret_cast<int4*>(p.step + p.o_items + (int64_t)i * kItemInts);
    at[0] = a;
    at[1] = b;
  }
  for (int i = g; i < t_take; i += stride) {   // fresh blocks into the table: entries that nobody reads above
    const int r = last_at_most(s_take, R, i);
    p.table[r * p.ld_table + ((s_len[r] + bs - 1) >> p.bs_log2) + i - s_take[r]] = p.free_blocks[count - 1 - i];
  }
  if (lead && p.units) {   // units of attention work before each token: quantized tokens, then open rows, in pieces of kUnit
    const int each = (p.T + kPlanThreads - 1) / kPlanThreads;
    const int t0 = min(p.T, (int)threadIdx.x * each), t1 = min(p.T, t0 + each);
    auto units_of = [&](int t) {
      if (t >= t_new) return 0;
      const int r = last_at_most(s_start, R, t), seen = s_len[r] + t - s_start[r] + 1;
      const int end = s_len[r] + (r + 1 < R ? s_start[r + 1] : (int)t_new) - s_start[r];
      const int held = end >> p.bs_log2 << p.bs_log2, nq = min(seen, held);
      return (nq + kUnit - 1) / kUnit + (seen - nq + kUnit - 1) / kUnit;
    };
    long long n = 0, all;
    for (int t = t0; t < t1; ++t) n += units_of(t);
    int at = (int)block_scan(n, s_sums, all);
    for (int t = t0; t < t1; ++t) {
      p.step[p.o_units + t] = at;
      at += units_of(t);
    }
    if (threadIdx.x == 0) p.step[p.o_units + p.T] = (int)all;
  }
}

// Blocks of the requests marked in `release` go back to the stack, in request order, oldest block first; their lengths become 0.
__global__ void __launch_bounds__(kPlanThreads) paged_release_kernel(const int* release, int* seq_lens, const int* table, int64_t ld_table,
                                                                     int* free_blocks, int free_capacity, int* free_count, int R, int bs_log2,
                                                                     int max_blocks) {
  __shared__ long long s_sums[kPlanWarps];
  const int per = (R + kPlanThreads - 1) / kPlanThreads, r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
  auto blocks_of = [&](int r) {
    const int len = seq_lens[r];
    return release[r] == 0 || len <= 0 ? 0 : min(max_blocks, (int)(((int64_t)len + (1 << bs_log2) - 1) >> bs_log2));
  };
  long long n = 0, all;
  for (int r = r0; r < r1; ++r) n += blocks_of(r);
  const int count = max(0, *free_count);
  long long at = count + block_scan(n, s_sums, all);
  for (int r = r0; r < r1; ++r) {
    const int nb = blocks_of(r);
    for (int b = 0; b < nb; ++b, ++at)
      if (at < free_capacity) free_blocks[at] = table[r * ld_table + b];
    if (release[r] != 0) seq_lens[r] = 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) *free_count = (int)min((long long)free_capacity, count + all);
}

// ---- append -----------------------------------------------------------------------------------------------------------------------
// One thread block per (touched block of tokens, head); half the threads take the keys, half the values.  A block that fills up is
// held in registers (at most 64 values a thread) between the maximum and the codes, so its tokens are read once.
constexpr int kAppendThreads = 256;

struct AppendParams {
  const void* k;
  const void* v;
  int64_t k_st, k_sh, v_st, v_sh;
  const int* items;
  int8_t* k_codes;
  int8_t* v_codes;
  float* k_scale;
  float* v_scale;
  void* tail_k;
  void* tail_v;
  int H, num_blocks, R, T;
};

template <typename T, int D, int BS>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendParams p) {
  pdl_launch_dependents();
  constexpr int kChunks = D / 8, kHalf = kAppendThreads / 2, kEach = BS * kChunks / kHalf > 0 ? BS * kChunks / kHalf : 1;
  static_assert(BS * kChunks % kHalf == 0, "whole rounds");
  __shared__ uint32_t s_max[2][kHalf / 32];
  const int4* item = reinterpret_cast<const int4*>(p.items + (int64_t)blockIdx.x * kItemInts);
  const int4 a = item[0], b = item[1];
  const int r = a.x, id = a.y, row0 = a.z, off = a.w, n = b.x, blk = b.y, len = b.z, end = b.w, h = blockIdx.y;
  if (r < 0 || r >= p.R || row0 < 0 || row0 + n > p.T) return;
  const int half = threadIdx.x / kHalf, tid = threadIdx.x % kHalf;
  const T* src = reinterpret_cast<const T*>(half ? p.v : p.k) + h * (half ? p.v_sh : p.k_sh);
  const int64_t st = half ? p.v_st : p.k_st;
  T* tail = reinterpret_cast<T*>(half ? p.tail_v : p.tail_k) + ((int64_t)r * p.H + h) * BS * D;
  auto new_rows_to_tail = [&](int row, int to, int count) {
    for (int i = tid; i < count * kChunks; i += kHalf) {
      const int t = i / kChunks, c = i % kChunks * 8;
      *reinterpret_cast<uint4*>(tail + (to + t) * D + c) = *reinterpret_cast<const uint4*>(src + (row + t) * st + c);
    }
  };
  const bool starts_behind = len % BS != 0;     // the request's first touched block has rows in the tail already
  if (off + n < BS) {
    // stays open; behind a block that filled up from the same rows, that block's threads do this once they have read them
    if (!(off == 0 && starts_behind && blk > len / BS)) new_rows_to_tail(row0, off, n);
    return;
  }
  uint4 x[kEach];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int at = i * kHalf + tid, t = at / kChunks, c = at % kChunks * 8;
    x[i] = t < off ? *reinterpret_cast<const uint4*>(tail + t * D + c) : *reinterpret_cast<const uint4*>(src + (row0 + t - off) * st + c);
    top = __vmaxu2(top, q8::magnitudes(x[i]));
  }
  top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
  if ((threadIdx.x & 31) == 0) s_max[half][tid / 32] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kHalf / 32; ++w) top = max(top, s_max[half][w]);
  const uint16_t bits = (uint16_t)top;
  const q8::Grid grid(to_float<T>(*reinterpret_cast<const T*>(&bits)));
  if (id >= 0 && id < p.num_blocks) {
    int8_t* codes = (half ? p.v_codes : p.k_codes) + ((int64_t)id * p.H + h) * BS * D;
#pragma unroll
    for (int i = 0; i < kEach; ++i) *reinterpret_cast<uint2*>(codes + (i * kHalf + tid) * 8) = grid.codes<T>(x[i]);
    if (tid == 0) (half ? p.v_scale : p.k_scale)[(int64_t)id * p.H + h] = grid.step;
  }
  if (off > 0 && end % BS != 0 && end / BS > blk) {   // the open block behind it: its rows are free only now
    asm volatile("bar.sync %0, %1;" ::"r"(1 + half), "n"(kHalf) : "memory");
    new_rows_to_tail(row0 + end / BS * BS - (blk * BS + off), 0, end % BS);
  }
}

// ---- dense ------------------------------------------------------------------------------------------------------------------------
// Keys and values of every request with new tokens, one request after the other: [total][H][D].  A warp takes a token with all its
// heads: 16 codes (or 8 open values twice) per lane and round.
constexpr int kDenseTokens = 32, kDenseThreads = 256;

struct DenseParams {
  const long long* context_start;
  const int* seq_lens;
  const int* table;
  int64_t ld_table;
  const int8_t* k_codes;
  const int8_t* v_codes;
  const float* k_scale;
  const float* v_scale;
  const void* tail_k;
  const void* tail_v;
  void* out_k;
  void* out_v;
  int64_t total;
  int R, H, bs_log2, num_blocks, max_blocks;
};

template <typename T, int D>
__global__ void __launch_bounds__(kDenseThreads) paged_dense_kernel(const DenseParams p) {
  const int64_t first = (int64_t)blockIdx.x * kDenseTokens;
  __shared__ int s_r;
  if (threadIdx.x == 0) s_r = 0;
  __syncthreads();
  int before = 0;   // requests that begin at or before the first token
  for (int r = threadIdx.x; r < p.R; r += kDenseThreads) before += p.context_start[r] <= first;
  before = __reduce_add_sync(0xffffffffu, before);
  if ((threadIdx.x & 31) == 0) atomicAdd(&s_r, before);
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bs = 1 << p.bs_log2;
  int r = s_r - 1;
  for (int i = warp; i < kDenseTokens; i += kDenseThreads / 32) {
    const int64_t t = first + i;
    if (t >= p.total) return;
    while (r < p.R && p.context_start[r + 1] <= t) ++r;
    T* ok = reinterpret_cast<T*>(p.out_k) + t * p.H * D;
    T* ov = reinterpret_cast<T*>(p.out_v) + t * p.H * D;
    const bool real = r >= 0 && r < p.R;
    const int pos = real ? (int)(t - p.context_start[r]) : 0, end = real ? p.seq_lens[r] : 0;
    const bool held = pos < (end >> p.bs_log2 << p.bs_log2);
    int id = 0;
    if (real && held) id = (pos >> p.bs_log2) < p.max_blocks ? p.table[r * p.ld_table + (pos >> p.bs_log2)] : -1;
    const bool good = id >= 0 && id < p.num_blocks;
    for (int c = lane * 16; c < p.H * D; c += 32 * 16) {
      const int h = c / D, ch = c % D;
      uint4 wk[2], wv[2];
      if (real && held && good) {
        const int64_t row = (((int64_t)id * p.H + h) << p.bs_log2) + (pos & (bs - 1));
        const uint4 ck = ld_stream_v4(p.k_codes + row * D + ch), cv = ld_stream_v4(p.v_codes + row * D + ch);
        const float sk = p.k_scale[(int64_t)id * p.H + h], sv = p.v_scale[(int64_t)id * p.H + h];
        const int8_t* qk = reinterpret_cast<const int8_t*>(&ck);
        const int8_t* qv = reinterpret_cast<const int8_t*>(&cv);
        T* ek = reinterpret_cast<T*>(wk);
        T* ev = reinterpret_cast<T*>(wv);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          ek[j] = from_float<T>((float)qk[j] * sk);
          ev[j] = from_float<T>((float)qv[j] * sv);
        }
      } else if (real && !held) {
        const int64_t at = ((((int64_t)r * p.H + h) << p.bs_log2) + (pos & (bs - 1))) * D + ch;
        const uint4* tk = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.tail_k) + at);
        const uint4* tv = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.tail_v) + at);
        wk[0] = tk[0], wk[1] = tk[1], wv[0] = tv[0], wv[1] = tv[1];
      } else {   // behind the last request: zeros; a block that is not in the pool: NaN
        const uint32_t w = real ? 0x7fff7fffu : 0u;
        wk[0] = wk[1] = wv[0] = wv[1] = make_uint4(w, w, w, w);
      }
      reinterpret_cast<uint4*>(ok + c)[0] = wk[0], reinterpret_cast<uint4*>(ok + c)[1] = wk[1];
      reinterpret_cast<uint4*>(ov + c)[0] = wv[0], reinterpret_cast<uint4*>(ov + c)[1] = wv[1];
    }
  }
}

int log2_of(int bs) { return bs == 16 ? 4 : bs == 32 ? 5 : 6; }

}  // namespace
}  // namespace pare

extern "C" {

using namespace pare;
using namespace pare::paged;

size_t pare_paged_step_bytes(int R, int T, int block_size) {
  if (R <= 0 || R > kMaxRequests || T < 0 || T > kMaxTokens || !block_size_ok(block_size)) return 0;
  return (size_t)StepLayout(R, T, block_size).words * 4;
}

int64_t pare_paged_step_offset(int field, int R, int T, int block_size) {
  if (R <= 0 || R > kMaxRequests || T < 0 || T > kMaxTokens || !block_size_ok(block_size)) return -1;
  const StepLayout s(R, T, block_size);
  const int64_t at[] = {s.status, s.query_start, s.seq_lens, s.context_start, s.slots, s.token_request, s.positions};
  return field < 0 || field >= (int)(sizeof(at) / sizeof(at[0])) ? -1 : at[field] * 4;
}

int pare_paged_plan(const int32_t* seq_lens, const int32_t* new_lens, int R, int32_t* block_table, int64_t ld_table, int max_blocks,
                    const int32_t* free_blocks, int free_capacity, const int32_t* free_count, int block_size, int T, void* step,
                    size_t step_bytes, void* stream) {
  PARE_REQUIRE(seq_lens && new_lens && block_table && free_blocks && free_count && step, PARE_ERR_SHAPE);
  PARE_REQUIRE(R > 0 && R <= kMaxRequests && T >= 0 && T <= kMaxTokens && max_blocks > 0 && ld_table >= max_blocks && free_capacity >= 0,
               PARE_ERR_SHAPE);
  PARE_REQUIRE(block_size_ok(block_size), PARE_ERR_UNSUPPORTED);
  PARE_REQUIRE(((int64_t)max_blocks * block_size) < (int64_t)1 << 31, PARE_ERR_SHAPE);
  const StepLayout s(R, T, block_size);
  PARE_REQUIRE(step_bytes >= (size_t)s.words * 4, PARE_ERR_WORKSPACE);
  PARE_REQUIRE(aligned16(step), PARE_ERR_ALIGN);
  PlanParams p{seq_lens, new_lens, block_table, ld_table, free_blocks, free_count, reinterpret_cast<int*>(step),
               s.query_start, s.seq_lens, s.context_start, s.slots, s.token_request, s.positions, s.unit_start, s.info, s.items,
               R, T, log2_of(block_size), max_blocks, free_capacity, s.n_items, s.units ? 1 : 0};
  const size_t smem = (size_t)R * 4 * sizeof(int);
  if (!ensure_smem_attr(reinterpret_cast<const void*>(paged_plan_kernel), kMaxRequests * 4 * (int)sizeof(int))) return PARE_ERR_CUDA;
  int blocks = (T + kPlanThreads - 1) / kPlanThreads;
  blocks = blocks < 1 ? 1 : blocks > sm_count() ? sm_count() : blocks;
  paged_plan_kernel<<<blocks, kPlanThreads, smem, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return launch_status();
}

int pare_paged_release(const int32_t* release, int32_t* seq_lens, int R, const int32_t* block_table, int64_t ld_table, int max_blocks,
                       int32_t* free_blocks, int free_capacity, int32_t* free_count, int block_size, void* stream) {
  PARE_REQUIRE(release && seq_lens && block_table && free_blocks && free_count, PARE_ERR_SHAPE);
  PARE_REQUIRE(R > 0 && R <= kMaxRequests && max_blocks > 0 && ld_table >= max_blocks && free_capacity >= 0, PARE_ERR_SHAPE);
  PARE_REQUIRE(block_size_ok(block_size), PARE_ERR_UNSUPPORTED);
  paged_release_kernel<<<1, kPlanThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      release, seq_lens, block_table, ld_table, free_blocks, free_capacity, free_count, R, log2_of(block_size), max_blocks);
  return launch_status();
}

int pare_paged_append(const void* k, const void* v, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                      const pare_paged_layer* l, const pare_paged_tables* t, void* stream) {
  const int rc = check(l, t);
  if (rc != PARE_OK || t->T == 0) return rc;
  PARE_REQUIRE(k && v, PARE_ERR_SHAPE);
  PARE_REQUIRE(aligned16(k) && aligned16(v) && (k_stride_t | k_stride_h | v_stride_t | v_stride_h) % 8 == 0, PARE_ERR_ALIGN);
  const StepLayout s(t->R, t->T, t->block_size);
  const AppendParams p{k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, reinterpret_cast<const int*>(t->step) + s.items,
                       l->k_codes, l->v_codes, l->k_scale, l->v_scale, l->tail_k, l->tail_v, l->H, l->num_blocks, l->R, t->T};
  const dim3 grid(s.n_items, l->H);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) {
    kern<<<grid, kAppendThreads, 0, st>>>(p);
    return launch_status();
  };
  auto by_size = [&](auto tag) {
    using E = decltype(tag);
    const int bs = l->block_size;
    if (l->D == 64) return bs == 16 ? go(paged_append_kernel<E, 64, 16>) : bs == 32 ? go(paged_append_kernel<E, 64, 32>) : go(paged_append_kernel<E, 64, 64>);
    return bs == 16 ? go(paged_append_kernel<E, 128, 16>) : bs == 32 ? go(paged_append_kernel<E, 128, 32>) : go(paged_append_kernel<E, 128, 64>);
  };
  return l->dtype == PARE_F16 ? by_size(__half()) : by_size(__nv_bfloat16());
}

int pare_paged_dense(const pare_paged_layer* l, const pare_paged_tables* t, void* out_k, void* out_v, int64_t total, void* stream) {
  const int rc = check(l, t);
  if (rc != PARE_OK) return rc;
  PARE_REQUIRE(total >= 0 && total < (int64_t)1 << 35, PARE_ERR_SHAPE);
  if (total == 0) return PARE_OK;
  PARE_REQUIRE(out_k && out_v, PARE_ERR_SHAPE);
  PARE_REQUIRE(aligned16(out_k) && aligned16(out_v), PARE_ERR_ALIGN);
  const StepLayout s(t->R, t->T, t->block_size);
  const int* w = reinterpret_cast<const int*>(t->step);
  const DenseParams p{reinterpret_cast<const long long*>(w + s.context_start), w + s.seq_lens, t->block_table, t->ld_table, l->k_codes,
                      l->v_codes, l->k_scale, l->v_scale, l->tail_k, l->tail_v, out_k, out_v, total, t->R, l->H, log2_of(l->block_size),
                      l->num_blocks, t->max_blocks};
  const unsigned grid = (unsigned)((total + kDenseTokens - 1) / kDenseTokens);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) {
    kern<<<grid, kDenseThreads, 0, st>>>(p);
    return launch_status();
  };
  if (l->dtype == PARE_F16) return l->D == 64 ? go(paged_dense_kernel<__half, 64>) : go(paged_dense_kernel<__half, 128>);
  return l->D == 64 ? go(paged_dense_kernel<__nv_bfloat16, 64>) : go(paged_dense_kernel<__nv_bfloat16, 128>);
}

}  // extern "C"
