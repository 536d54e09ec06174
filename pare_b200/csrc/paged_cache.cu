// Paged KV cache held in 8 bits, sm_100a: the step's tables, the append and the dense reconstruction (attention over it:
// paged_attn.cu).  The reference keeps one dense batch per cache (pare/kv_cache.py:163-288); a server's requests come and go and
// have lengths of their own, so here a pool of blocks of `bs` tokens is shared by R requests through a block table.
//
// A block is quantized once, when its last token arrives, with one scale per (block, head) for keys and one for values:
//   s = max |x| / 127 over the block's bs x D values of a head,   c = round_half_even(x / s) in [-127, 127].
// Until then its tokens stay in the input type in the request's open rows (tail_k / tail_v), so every code is the result of one
// rounding and tokens fed in pieces give what the same tokens fed at once give (the property of the reference's residual window,
// pare/kv_cache.py:231-244).
#include <climits>
#include <type_traits>

#include "paged.cuh"
#include "quant8.cuh"

namespace pare {
namespace {

using namespace paged;

// ---- tables -----------------------------------------------------------------------------------------------------------------------
// One prefix sum over the requests gives everything: first row of a request's new tokens, blocks taken from the free stack before
// it, touched blocks before it.  A thread block holds the sums of all requests in shared memory (every thread block computes them
// for itself: no order between thread blocks), then tokens, fresh blocks and touched blocks are spread over all threads, each
// finding its request by bisection; one thread block does nothing but count attention's units.  Bound by latency (two dependent reads and
// a scan or two): one request 3.3 us, 64 requests with a token each 4.1, 256 prompts of 64000 tokens 5.5, 2056 tokens in chunks 7.6;
// bytes would take 0.2.
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
  int64_t o_query_start, o_seq_lens, o_context, o_slots, o_request, o_positions, o_units, unit_stride, o_info, o_items;
  int R, T, bs_log2, max_blocks, free_capacity, n_items, units;
};

// Exclusive prefix sums of N values per thread, and their totals.  All threads call it.
template <int N, typename V>
__device__ __forceinline__ void block_scan(const V (&v)[N], V (&before)[N], V (&total)[N], long long (*sums)[kPlanWarps]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = v[i];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const V y = __shfl_up_sync(0xffffffffu, x[i], o);
      if (lane >= o) x[i] += y;
    }
  }
  __syncthreads();
  if (lane == 31) {
#pragma unroll
    for (int i = 0; i < N; ++i) sums[i][warp] = x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    // the warps' sums, one per lane
    V s = lane < kPlanWarps ? (V)sums[i][lane] : 0, mine = lane < warp ? s : 0;
#pragma unroll
    for (int o = kPlanWarps / 2; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      mine += __shfl_xor_sync(0xffffffffu, mine, o);
    }
    total[i] = __shfl_sync(0xffffffffu, s, 0);
    before[i] = __shfl_sync(0xffffffffu, mine, 0) + x[i] - v[i];
  }
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
  pdl_launch_dependents();
  pdl_wait();
  __shared__ long long s_sums[4][kPlanWarps];
  __shared__ int s_bad;
  if (threadIdx.x == 0) s_bad = 0;
  int* s_start = s_mem;              // [R] first row of the new tokens
  int* s_len = s_start + p.R;        // [R] tokens before the step
  int* s_take = s_len + p.R;         // [R] blocks taken from the stack by the requests before
  int* s_item = s_take + p.R;        // [R] blocks touched by the requests before
  const int R = p.R, bs = 1 << p.bs_log2, per = (R + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
  const bool lead = blockIdx.x == 0;
  const int64_t max_len = (int64_t)p.max_blocks << p.bs_log2;

  int bad = 0;
  const int count = *p.free_count;
  long long sum[4] = {0, 0, 0, 0}, before[4], total[4];      // new tokens, blocks taken, blocks touched, tokens of requests with new ones
  for (int r = r0; r < r1; ++r) {
    const int len = p.seq_lens[r], add = p.new_lens[r];
    if (len < 0 || add < 0) bad |= PARE_PAGED_NEGATIVE;
    else if (add > p.T) bad |= PARE_PAGED_ROWS;
    else if ((int64_t)len + add > max_len) bad |= PARE_PAGED_TABLE;
    else {
      const int end = len + add;
      s_start[r] = (int)sum[0];
      s_len[r] = len;
      s_take[r] = (int)sum[1];
      s_item[r] = (int)sum[2];
      sum[0] += add;
      sum[1] += ((end + bs - 1) >> p.bs_log2) - ((len + bs - 1) >> p.bs_log2);
      if (add) {
        sum[2] += ((end - 1) >> p.bs_log2) - (len >> p.bs_log2) + 1;
        sum[3] += end;
      }
    }
  }
  if (count < 0 || count > p.free_capacity) bad |= PARE_PAGED_BLOCKS;
  block_scan(sum, before, total, s_sums);
  if (total[0] > p.T) bad |= PARE_PAGED_ROWS;
  if (total[1] > count) bad |= PARE_PAGED_BLOCKS;
  if (bad) atomicOr(&s_bad, bad);
  __syncthreads();
  bad = s_bad;                       // the step is done or refused as a whole
  const long long t_new = bad ? 0 : total[0], t_take = bad ? 0 : total[1], t_item = bad ? 0 : total[2];
  long long ctx = before[3];
  for (int r = r0; r < r1; ++r) {
    if (!bad) {
      s_start[r] += (int)before[0];
      s_take[r] += (int)before[1];
      s_item[r] += (int)before[2];
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
    reinterpret_cast<long long*>(p.step + p.o_context)[R] = bad ? 0 : total[3];
  }
  __syncthreads();

  // the last thread block counts units of attention, the others share what else there is
  const bool counts = p.units && blockIdx.x == gridDim.x - 1;
  const int g = counts ? INT_MAX : blockIdx.x * kPlanThreads + threadIdx.x, stride = (gridDim.x - (p.units ? 1 : 0)) * kPlanThreads;
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
      *reinterpret_cast<int4*>(p.step + p.o_info + 4 * (int64_t)i) = make_int4(r, pos, end, r < 0 ? 0 : i - s_start[r]);
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
  if (counts) {
    // Units of attention work before each token: quantized tokens, then open rows, in pieces of kUnit.  Where 2^i tokens of a request
    // share a tile, its last token has its units and the others have none.
    const int each = (p.T + kPlanThreads - 1) / kPlanThreads;
    const int t0 = min(p.T, (int)threadIdx.x * each), t1 = min(p.T, t0 + each);
    constexpr int kEach = kMaxQueryTokens / kPlanThreads;
    int units[kEach], pack[kEach];      // of tokens t0 ..; bit i of pack: the last one of a tile of 2^i
    int r = t0 < t_new ? last_at_most(s_start, R, t0) : 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int t = t0 + e;
      units[e] = pack[e] = 0;
      if (t >= t1 || t >= t_new) continue;
      while (r + 1 < R && s_start[r + 1] <= t) ++r;
      const int mine = t - s_start[r], seen = s_len[r] + mine + 1, end = s_len[r] + (r + 1 < R ? s_start[r + 1] : (int)t_new) - s_start[r];
      const int held = end >> p.bs_log2 << p.bs_log2, nq = min(seen, held);
      units[e] = (nq + kUnit - 1) / kUnit + (seen - nq + kUnit - 1) / kUnit;
#pragma unroll
      for (int i = 0; i < kPacks; ++i) pack[e] |= seen == end || (mine + 1) % (1 << i) == 0 ? 1 << i : 0;
    }
    auto tables = [&](auto packs) {
      constexpr int kN = decltype(packs)::value;
      int sums[kN] = {}, first[kN], all[kN];
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
#pragma unroll
        for (int i = 0; i < kN; ++i) sums[i] += pack[e] >> i & 1 ? units[e] : 0;
      }
      block_scan(sums, first, all, s_sums);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (t0 + e >= t1) break;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          p.step[p.o_units + i * p.unit_stride + t0 + e] = first[i];
          first[i] += pack[e] >> i & 1 ? units[e] : 0;
        }
      }
      if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < kN; ++i) p.step[p.o_units + i * p.unit_stride + p.T] = all[i];
      }
    };
    if (packs_tokens(p.R, p.T)) tables(std::integral_constant<int, kPacks>());
    else tables(std::integral_constant<int, 1>());
  }
}

// Blocks of the requests marked in `release` go back to the stack, in request order, oldest block first; their lengths become 0.
// One thread block: blocks before a request by a prefix sum, then the blocks of all requests are spread over the threads.
__global__ void __launch_bounds__(kPlanThreads) paged_release_kernel(const int* release, int* seq_lens, const int* table, int64_t ld_table,
                                                                     int* free_blocks, int free_capacity, int* free_count, int R, int bs_log2,
                                                                     int max_blocks) {
  extern __shared__ int s_start[];      // [R] blocks given back by the requests before
  __shared__ long long s_sums[1][kPlanWarps];
  const int per = (R + kPlanThreads - 1) / kPlanThreads, r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
  auto blocks_of = [&](int r) {
    const int len = seq_lens[r];
    return release[r] == 0 || len <= 0 ? 0 : min(max_blocks, (int)(((int64_t)len + (1 << bs_log2) - 1) >> bs_log2));
  };
  long long n[1] = {0}, before[1], all[1];
  for (int r = r0; r < r1; ++r) n[0] += blocks_of(r);
  const int count = max(0, *free_count);
  block_scan(n, before, all, s_sums);
  const int room = max(0, free_capacity - count), given = (int)min((long long)room, all[0]);      // a pool has no more blocks than its stack
  long long at = before[0];
  for (int r = r0; r < r1; ++r) {
    s_start[r] = (int)min(at, (long long)INT_MAX);
    at += blocks_of(r);
  }
  __syncthreads();
  for (int r = r0; r < r1; ++r)
    if (release[r] != 0) seq_lens[r] = 0;
  for (int i = threadIdx.x; i < given; i += kPlanThreads) {
    const int r = last_at_most(s_start, R, i);
    free_blocks[count + i] = table[r * ld_table + i - s_start[r]];
  }
  if (threadIdx.x == 0) *free_count = count + given;
}

// ---- append -----------------------------------------------------------------------------------------------------------------------
// A team of threads takes one (touched block of tokens, head) of the keys or of the values.  A block that fills up is held in registers
// between the maximum and the codes, so its tokens are read once.  Four threads per token (32 values each, all loads in flight at
// once) where eight per token would take several rounds of the SMs, else eight: 32768 tokens of 4 heads 25.6 us against 34, but 2056 tokens of 8
// heads 8.7 against 6.2 (two threads per token: 26.7; with cheaper codes since then 23.0 and 5.1).  Bytes would take 15.4 us for the
// first; it fills 55 % of the issue slots and 32 % of DRAM's rate with 44 % of the warps an SM holds (62 registers hold the block).  A decode step
// of one request 1.3 us.
__host__ __device__ constexpr int append_threads(int team) { return team > 256 ? team : 256; }

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

template <typename T, int D, int BS, int PER_TOKEN>
__global__ void __launch_bounds__(append_threads(BS * PER_TOKEN)) paged_append_kernel(const AppendParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kChunks = D / 8, kTeam = BS * PER_TOKEN, kThreads = append_threads(kTeam), kEach = BS * kChunks / kTeam;      // threads of a team, vectors of eight per thread
  __shared__ uint32_t s_max[kThreads / 32];
  const int4* item = reinterpret_cast<const int4*>(p.items + (int64_t)blockIdx.x * kItemInts);
  const int4 a = item[0], b = item[1];
  const int r = a.x, id = a.y, row0 = a.z, off = a.w, n = b.x, blk = b.y, len = b.z, end = b.w;
  const int team = threadIdx.x / kTeam, tid = threadIdx.x % kTeam, job = blockIdx.y * (kThreads / kTeam) + team;      // heads' keys, then heads' values
  if (r < 0 || r >= p.R || row0 < 0 || row0 + n > p.T || job >= 2 * p.H) return;
  const int half = job >= p.H, h = job - half * p.H;
  auto team_sync = [&] {
    if (kTeam == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(kTeam) : "memory");
  };
  const T* src = reinterpret_cast<const T*>(half ? p.v : p.k) + h * (half ? p.v_sh : p.k_sh);
  const int64_t st = half ? p.v_st : p.k_st;
  T* tail = reinterpret_cast<T*>(half ? p.tail_v : p.tail_k) + ((int64_t)r * p.H + h) * BS * D;
  auto new_rows_to_tail = [&](int row, int to, int count) {
    for (int i = tid; i < count * kChunks; i += kTeam) {
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
    const int at = i * kTeam + tid, t = at / kChunks, c = at % kChunks * 8;
    x[i] = t < off ? *reinterpret_cast<const uint4*>(tail + t * D + c) : *reinterpret_cast<const uint4*>(src + (row0 + t - off) * st + c);
    top = __vmaxu2(top, q8::magnitudes(x[i]));
  }
  top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
  if (kTeam > 32) {
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x / 32] = top;
    team_sync();
#pragma unroll
    for (int w = 0; w < kTeam / 32; ++w) top = max(top, s_max[team * (kTeam / 32) + w]);
  }
  const uint16_t bits = (uint16_t)top;
  const q8::Grid grid(to_float<T>(*reinterpret_cast<const T*>(&bits)));
  if (id >= 0 && id < p.num_blocks) {
    int8_t* codes = (half ? p.v_codes : p.k_codes) + ((int64_t)id * p.H + h) * BS * D;
#pragma unroll
    for (int i = 0; i < kEach; ++i) *reinterpret_cast<uint2*>(codes + (i * kTeam + tid) * 8) = grid.codes<T>(x[i]);
    if (tid == 0) (half ? p.v_scale : p.k_scale)[(int64_t)id * p.H + h] = grid.step;
  }
  if (off > 0 && end % BS != 0 && end / BS > blk) {   // the open block behind it: its rows are free only now
    team_sync();
    new_rows_to_tail(row0 + end / BS * BS - (blk * BS + off), 0, end % BS);
  }
}

// ---- dense ------------------------------------------------------------------------------------------------------------------------
// Keys and values of every request with new tokens, one request after the other: [total][H][D].  A warp takes two tokens with all
// their heads, 16 channels per lane and round (one token: 24.4 us for 32768 of 4 heads, two 20.3, four 20.7, eight 20.7).
constexpr int kDenseThreads = 256, kDenseEach = 2, kDenseTokens = kDenseThreads / 32 * kDenseEach;

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

// Sixteen codes.  Not the read-only path (.nc): that asks for data which nobody writes while the kernel lives, and this one is launched
// while the append before it still writes codes.
__device__ __forceinline__ uint4 ld_codes16(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// sixteen codes times their scale, rounded
template <typename T>
__device__ __forceinline__ void scaled16(const uint4& c, float s, uint4 (&out)[2]) {
  const int8_t* q = reinterpret_cast<const int8_t*>(&c);
  T* e = reinterpret_cast<T*>(out);
#pragma unroll
  for (int j = 0; j < 16; ++j) e[j] = from_float<T>((float)q[j] * s);
}

template <typename T, int D>
__global__ void __launch_bounds__(kDenseThreads) paged_dense_kernel(const DenseParams p) {
  pdl_launch_dependents();
  pdl_wait();
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
  const int64_t t0 = first + warp * kDenseEach;
  // lane i finds out about token i: its row of codes (>= 0), of open tokens (-1 - row), or what else it is
  constexpr long long kNothing = (1ll << 62), kBad = kNothing + 1;      // behind the last request; a block that is not in the pool
  long long where = kNothing;
  int id = 0;
  if (lane < kDenseEach) {
    const int64_t t = t0 + lane;
    int r = s_r - 1;
    while (r < p.R && p.context_start[r + 1] <= t) ++r;
    if (r < p.R) {
      const int pos = (int)(t - p.context_start[r]), blk = pos >> p.bs_log2, off = pos & (bs - 1);
      if (blk < p.seq_lens[r] >> p.bs_log2) {
        id = blk < p.max_blocks ? p.table[r * p.ld_table + blk] : -1;
        where = id >= 0 && id < p.num_blocks ? ((((long long)id * p.H) << p.bs_log2) + off) : kBad;
      } else {
        where = -1 - ((((long long)r * p.H) << p.bs_log2) + off);
      }
    }
  }
  const int tokens = (int)min((int64_t)kDenseEach, p.total - t0);
  for (int base = 0; base < p.H * D; base += 32 * 16) {
    const int c = base + lane * 16, h = c / D, ch = c % D;
    const bool inside = c < p.H * D;
    const int64_t skip = ((int64_t)h << p.bs_log2) * D + ch;       // from head 0 to this lane's channels
    uint4 ck[kDenseEach], cv[kDenseEach];
    float sk[kDenseEach], sv[kDenseEach];
#pragma unroll
    for (int i = 0; i < kDenseEach; ++i) {
      const long long w = __shfl_sync(0xffffffffu, where, i);
      const int block = __shfl_sync(0xffffffffu, id, i);
      if (inside && i < tokens && w >= 0 && w < kNothing) {
        ck[i] = ld_codes16(p.k_codes + w * D + skip);
        cv[i] = ld_codes16(p.v_codes + w * D + skip);
        sk[i] = p.k_scale[(int64_t)block * p.H + h];
        sv[i] = p.v_scale[(int64_t)block * p.H + h];
      }
    }
#pragma unroll
    for (int i = 0; i < kDenseEach; ++i) {
      const long long w = __shfl_sync(0xffffffffu, where, i);
      if (!inside || i >= tokens) continue;
      uint4 wk[2], wv[2];
      if (w >= 0 && w < kNothing) {
        scaled16<T>(ck[i], sk[i], wk);
        scaled16<T>(cv[i], sv[i], wv);
      } else if (w < 0) {
        const uint4* tk = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.tail_k) + (-1 - w) * D + skip);
        const uint4* tv = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.tail_v) + (-1 - w) * D + skip);
        wk[0] = tk[0], wk[1] = tk[1], wv[0] = tv[0], wv[1] = tv[1];
      } else {   // behind the last request: zeros; a block that is not in the pool: NaN
        const uint32_t x = w == kBad ? 0x7fff7fffu : 0u;
        wk[0] = wk[1] = wv[0] = wv[1] = make_uint4(x, x, x, x);
      }
      uint4* ok = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out_k) + (t0 + i) * p.H * D + c);
      uint4* ov = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out_v) + (t0 + i) * p.H * D + c);
      ok[0] = wk[0], ok[1] = wk[1], ov[0] = wv[0], ov[1] = wv[1];
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
               s.query_start, s.seq_lens, s.context_start, s.slots, s.token_request, s.positions, s.unit_start, s.unit_stride, s.info, s.items,
               R, T, log2_of(block_size), max_blocks, free_capacity, s.n_items, s.units ? 1 : 0};
  const size_t smem = (size_t)R * 4 * sizeof(int);
  if (!ensure_smem_attr(reinterpret_cast<const void*>(paged_plan_kernel), kMaxRequests * 4 * (int)sizeof(int))) return PARE_ERR_CUDA;
  int blocks = (T + kPlanThreads - 1) / kPlanThreads;
  blocks = blocks < 1 ? 1 : blocks > sm_count() ? sm_count() : blocks;
  const int rc = launch_pdl(paged_plan_kernel, dim3(blocks + (s.units ? 1 : 0)), dim3(kPlanThreads), smem, reinterpret_cast<cudaStream_t>(stream), p);
  return rc != PARE_OK ? rc : launch_status();
}

int pare_paged_release(const int32_t* release, int32_t* seq_lens, int R, const int32_t* block_table, int64_t ld_table, int max_blocks,
                       int32_t* free_blocks, int free_capacity, int32_t* free_count, int block_size, void* stream) {
  PARE_REQUIRE(release && seq_lens && block_table && free_blocks && free_count, PARE_ERR_SHAPE);
  PARE_REQUIRE(R > 0 && R <= kMaxRequests && max_blocks > 0 && ld_table >= max_blocks && free_capacity >= 0, PARE_ERR_SHAPE);
  PARE_REQUIRE(block_size_ok(block_size), PARE_ERR_UNSUPPORTED);
  paged_release_kernel<<<1, kPlanThreads, R * sizeof(int), reinterpret_cast<cudaStream_t>(stream)>>>(
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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int bs = l->block_size;
  const bool many = (int64_t)s.n_items * 2 * l->H * 8 * bs > (int64_t)sm_count() * 8192;
  auto go = [&](auto kern, int team) -> int {
    const int threads = append_threads(team), teams = threads / team, groups = (2 * l->H + teams - 1) / teams;
    PARE_REQUIRE(groups <= 65535, PARE_ERR_UNSUPPORTED);      // a grid's second dimension
    const int rc = launch_pdl(kern, dim3(s.n_items, groups), dim3(threads), 0, st, p);
    return rc != PARE_OK ? rc : launch_status();
  };
  auto by_size = [&](auto tag, auto dim) {
    using E = decltype(tag);
    constexpr int kD = decltype(dim)::value;
    if (bs == 16) return many ? go(paged_append_kernel<E, kD, 16, 4>, 64) : go(paged_append_kernel<E, kD, 16, 8>, 128);
    if (bs == 32) return many ? go(paged_append_kernel<E, kD, 32, 4>, 128) : go(paged_append_kernel<E, kD, 32, 8>, 256);
    return many ? go(paged_append_kernel<E, kD, 64, 4>, 256) : go(paged_append_kernel<E, kD, 64, 8>, 512);
  };
  auto by_type = [&](auto dim) { return l->dtype == PARE_F16 ? by_size(__half(), dim) : by_size(__nv_bfloat16(), dim); };
  return l->D == 64 ? by_type(std::integral_constant<int, 64>()) : by_type(std::integral_constant<int, 128>());
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
    const int rc = launch_pdl(kern, dim3(grid), dim3(kDenseThreads), 0, st, p);
    return rc != PARE_OK ? rc : launch_status();
  };
  if (l->dtype == PARE_F16) return l->D == 64 ? go(paged_dense_kernel<__half, 64>) : go(paged_dense_kernel<__half, 128>);
  return l->D == 64 ? go(paged_dense_kernel<__nv_bfloat16, 64>) : go(paged_dense_kernel<__nv_bfloat16, 128>);
}

}  // extern "C"
