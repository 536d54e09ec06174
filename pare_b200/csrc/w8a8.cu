// W8A8 linear, sm_100a: tokens quantized to int8 with a scale each, int8 weights with a scale (and zero-point) per output channel,
// integer products on tcgen05.mma kind::i8, everything else in the epilogue.  What the reference has as an eager
// fake-quantization (quantize_inputs, SmoothQuant W8A8: pare/layers/linear.py:121-138) in real integers:
//   x~ = x, or dtype(x / input_scale)      step_m = max(max_k |x~_mk|, 1e-6) / 127      c_mk = round_half_even(x~_mk / step_m)
//   y_mn = dtype((sum_k c_mk q_nk - z_n sum_k c_mk) * step_m s_n + b_n)
// The sums are exact 32-bit integers, so neither tiles nor splits of K nor their order change a bit of the result.
//
// Two launches: the tokens' codes (one thread block per row), then the product.  The second starts while the first runs and fills
// its ring with weights, which the first does not write (and what came before the first has ended); it waits before it touches
// anything else.  A few rows take one launch (w8a8_few_kernel below).
//
// The product: as in w4a16_gemm.cu the rows of a weight tile sit on the MMA's M axis (the TMEM lanes), activation rows on its N axis.
// Both operands come by TMA (128-byte rows, 128B swizzle) and are multiplied where they land; the accumulator is double-buffered in
// tensor memory so a tile's epilogue overlaps the next tile's products.
//   warp 0     TMA of both operands      warp 1  tcgen05.mma      warp 2  tensor memory      warps 4-11  epilogue
// All waits are bounded; when one runs out the thread block stops waiting and loading, lets its copies and products in flight
// end, and its outputs become NaN.
#include <algorithm>
#include <type_traits>

#include "quant8.cuh"
#include "tcgen05.cuh"

namespace pare {
namespace {

using namespace tc;

constexpr int kRows = 128;               // weight rows per tile (UMMA M)
constexpr int kUnitK = 128;              // columns per unit: one 128-byte swizzle row, four MMAs
constexpr int kWBytes = kRows * kUnitK;
constexpr int kMaxStages = 12;
constexpr int kThreads = 384;
constexpr int kEpiThreads = 256;         // eight warps: two per quarter of the tensor memory's lanes, every other 16 activation rows each
constexpr uint32_t kTmemCols = 512;      // two accumulators of up to 256 columns
constexpr int kMaxSmem = 214 * 1024;    // beside 12.1 KB of static shared memory
constexpr int kRingBytes = kMaxSmem - 1024 - 512;
constexpr int kMaxK = 65536;             // 65536 * 127 * (128 + 128) < 2^31

// ---- tokens -> codes ----------------------------------------------------------------------------------------------------------------
struct QuantParams {
  const void* x;
  int64_t ldx;
  const float* input_scale;
  int8_t* codes;
  int64_t ldc;
  float* step;
  int* sums;        // NULL: nobody asks for them
  int K;
};

template <typename T>
__device__ __forceinline__ T smoothed(T v, const float* input_scale, int k) {
  return input_scale ? from_float<T>(__fdiv_rn(to_float<T>(v), __ldg(input_scale + k))) : v;
}
template <typename T>
__device__ __forceinline__ uint32_t magnitude(T v) {   // orders like |v|, infinities and NaN above all numbers
  return *reinterpret_cast<const uint16_t*>(&v) & 0x7fffu;
}

// A row per thread block; where rows allow 16-byte pieces (VEC) it waits in shared memory between the maximum and the codes (and is divided
// by input_scale once: SCALED), all of it on its way at the same time and no registers held, so that as many rows as possible are
// resident (32 registers, without smoothing 16 bytes of them in local memory).  Others are read twice.  Neither DRAM (20 %) nor the issue
// slots (40 %) are full; the codes' arithmetic counts most (cheaper codes halved the time).  2048 rows of 4096 6.8 us (bytes: 3.8), 1024 of
// 14336 9.1 (6.7), 333 of 18944 5.9 and with input_scale 10.4 (2.9; rows held in registers, fewer of them at once: 12 and 18).
template <typename T, int THREADS, bool VEC, bool SCALED>
__global__ void __launch_bounds__(THREADS, (SCALED ? 1536 : 2048) / THREADS) w8a8_quantize_kernel(const QuantParams p) {
  pdl_wait();
  pdl_launch_dependents();      // only now: the product reads weights before it waits
  constexpr int kW = THREADS / 32;
  extern __shared__ uint4 s_row[];
  __shared__ uint32_t s_top[kW];
  __shared__ int s_sum[kW];
  const int m = blockIdx.x, tid = threadIdx.x, n8 = p.K / 8;
  const T* row = reinterpret_cast<const T*>(p.x) + m * p.ldx;
  int8_t* out = p.codes + m * p.ldc;
  uint32_t top = 0;
  if constexpr (VEC) {
    const uint32_t at = s_u32(s_row);
    for (int i = tid; i < n8; i += THREADS)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + i * 16), "l"(row + i * 8) : "memory");
    if constexpr (SCALED) {
      const float4* d = reinterpret_cast<const float4*>(p.input_scale);
      float4 a, b, a2, b2;      // of this vector and of the next
      if (tid < n8) a = __ldg(d + 2 * tid), b = __ldg(d + 2 * tid + 1);
      asm volatile("cp.async.wait_all;" ::: "memory");       // a thread reads what it loaded itself
#pragma unroll 1
      for (int i = tid; i < n8; i += THREADS, a = a2, b = b2) {
        if (i + THREADS < n8) a2 = __ldg(d + 2 * (i + THREADS)), b2 = __ldg(d + 2 * (i + THREADS) + 1);
        uint4 x = s_row[i];
        const float by[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        T* v = reinterpret_cast<T*>(&x);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = from_float<T>(__fdiv_rn(to_float<T>(v[j]), by[j]));
        s_row[i] = x;
        top = __vmaxu2(top, q8::magnitudes(x));
      }
    } else {
      asm volatile("cp.async.wait_all;" ::: "memory");
      for (int i = tid; i < n8; i += THREADS) top = __vmaxu2(top, q8::magnitudes(s_row[i]));
    }
    top = max(top & 0xffffu, top >> 16);
  } else {
    for (int k = tid; k < p.K; k += THREADS) top = max(top, magnitude(smoothed<T>(row[k], p.input_scale, k)));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) s_top[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kW; ++w) top = max(top, s_top[w]);
  const uint16_t bits = (uint16_t)top;
  const float amax = to_float<T>(*reinterpret_cast<const T*>(&bits));
  // a row with an infinity or NaN has a step that is not finite, so its outputs are NaN
  const q8::Grid grid(amax < 1e-6f ? 1e-6f : amax);
  int sum = 0;
  if constexpr (VEC) {
#pragma unroll 1
    for (int i = tid; i < n8; i += THREADS) {
      const uint2 o = grid.codes<T>(s_row[i]);
      sum = __dp4a((int)o.y, 0x01010101, __dp4a((int)o.x, 0x01010101, sum));
      *reinterpret_cast<uint2*>(out + i * 8) = o;
    }
  } else {
    for (int k = tid; k < p.K; k += THREADS) {
      const int c = grid.code(to_float<T>(smoothed<T>(row[k], p.input_scale, k)));
      sum += c;
      out[k] = (int8_t)c;
    }
  }
  if (tid == 0) p.step[m] = grid.finite ? grid.step : __int_as_float(0x7fffffff);
  if (!p.sums) return;
  sum = __reduce_add_sync(0xffffffffu, sum);
  if ((tid & 31) == 0) s_sum[tid >> 5] = sum;
  __syncthreads();
  if (tid == 0) {
    int all = 0;
#pragma unroll
    for (int w = 0; w < kW; ++w) all += s_sum[w];
    p.sums[m] = all;
  }
}

// ---- product --------------------------------------------------------------------------------------------------------------------------
struct W8Params {
  const float* step;     // [M]
  const int* sums;       // [M]
  const float* scale;    // [N]
  const float* zero;     // [N] or NULL
  const void* bias;
  void* y;
  int64_t ldy;
  int M, N;
  int mt;                // activation rows per tile (UMMA N), a multiple of 32
  int mtiles;
  int ku;                // units per tile
  int stages;
};

// bar_wait for arrivals from another thread block of the cluster
__device__ __forceinline__ bool bar_test_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void bar_wait_cluster(uint32_t bar, uint32_t parity, int* status, bool& dead) {
  if (dead || bar_test_cluster(bar, parity)) return;
  bar_wait(bar, parity, status, dead);
  if (!dead) bar_test_cluster(bar, parity);      // the same phase again, for its order with the other thread block's accesses
}

// both operands in shared memory, 8-bit integers
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}

// A thread's sums of one output column (weight row) and sixteen activation rows -> outputs.
template <typename T>
struct Epilogue {
  T* y;
  int64_t ldy;
  int M, N, n, zi;
  float bias, scale, zf;
  bool has_zero, pair_out, wide_out, bad;
  int row_sum = 0;       // where no array of sums is given: of row `lane`

  __device__ __forceinline__ Epilogue(const W8Params& p)
      : y(reinterpret_cast<T*>(p.y)), ldy(p.ldy), M(p.M), N(p.N), has_zero(p.zero != nullptr),
        pair_out((reinterpret_cast<uintptr_t>(p.y) & 3u) == 0 && (p.ldy & 1) == 0 && (p.N & 1) == 0),
        wide_out((reinterpret_cast<uintptr_t>(p.y) & 15u) == 0 && (p.ldy & 7) == 0 && (p.N & 7) == 0), bad(false) {}
  // The zero-point's whole part is taken off in integers, exactly; what is left (0 for the zero-points of quantizers, or a value
  // beyond any code) in fp32.
  __device__ __forceinline__ void column(const W8Params& p, int col) { column(col, fetch(p, col)); }
  // its scale, zero-point and bias
  __device__ __forceinline__ float3 fetch(const W8Params& p, int col) const {
    const bool there = col < N;
    return make_float3(there ? p.scale[col] : 0.f, p.zero && there ? p.zero[col] : 0.f,
                       p.bias && there ? to_float<T>(reinterpret_cast<const T*>(p.bias)[col]) : 0.f);
  }
  __device__ __forceinline__ void column(int col, const float3& of) {
    n = col;
    scale = of.x;
    bias = of.z;
    const float z = of.y;
    zi = fabsf(z) <= 128.f ? __float2int_rn(z) : 0;
    zf = z - (float)zi;
  }
  // rows m0 .. m0 + 15 (those below `end`); steps, sums: of these rows, in shared memory
  __device__ __forceinline__ void store16(const int (&a)[16], int m0, int end, const float* steps, const int* sums = nullptr) const {
    const int odd = threadIdx.x & 1;
    float f[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int xs = sums ? sums[i] : __shfl_sync(0xffffffffu, row_sum, i);
      float v = (float)(a[i] - zi * xs);
      if (has_zero) v = fmaf(-zf, (float)xs, v);
      f[i] = bad ? __int_as_float(0x7fffffff) : fmaf(v, steps[i] * scale, bias);
    }
    if (pair_out) {   // neighbouring lanes swap so that each stores two columns of every other row
      T* at = y + (int64_t)(m0 + odd) * ldy + (n & ~1);
#pragma unroll
      for (int i = 0; i < 16; i += 2, at += 2 * ldy) {
        const float mine = odd ? f[i + 1] : f[i], got = __shfl_xor_sync(0xffffffffu, odd ? f[i] : f[i + 1], 1);
        const uint32_t w = odd ? Pair<T>::pack(got, mine) : Pair<T>::pack(mine, got);
        if (m0 + i + odd < end && n < N) *reinterpret_cast<uint32_t*>(at) = w;
      }
    } else if (n < N) {
      T* at = y + (int64_t)m0 * ldy + n;
#pragma unroll
      for (int i = 0; i < 16; ++i, at += ldy)
        if (m0 + i < end) *at = from_float<T>(f[i]);
    }
  }
};

// The same where rows allow 16-byte pieces: through `stage`, 1 KB of shared memory of this warp's own, a word for two rows of a column.
// (2048 rows of 28672 x 256, bound by this: 53 us; with a 16-bit store per output there 57, with shuffles and 4-byte pieces 63.)
template <typename T>
__device__ __forceinline__ void store16_wide(const Epilogue<T>& e, const int (&a)[16], int m0, int end, const float* steps, const int* sums, uint4* stage) {
  const int lane = threadIdx.x & 31;
  uint32_t* to = reinterpret_cast<uint32_t*>(stage) + lane;
  const float scale = e.bad ? __int_as_float(0x7fffffff) : e.scale;
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 s4 = *reinterpret_cast<const float4*>(steps + i);
    const float s[4] = {s4.x, s4.y, s4.z, s4.w};
    float f[4];
    if (e.has_zero) {
      const int4 x4 = *reinterpret_cast<const int4*>(sums + i);
      const int xs[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = fmaf(fmaf(-e.zf, (float)xs[j], (float)(a[i + j] - e.zi * xs[j])), s[j] * scale, e.bias);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = fmaf((float)a[i + j], s[j] * scale, e.bias);
    }
    to[(i / 2) * 32] = Pair<T>::pack(f[0], f[1]);
    to[(i / 2 + 1) * 32] = Pair<T>::pack(f[2], f[3]);
  }
  __syncwarp();
  // rows 2 r, 2 r + 1 of eight columns, the halves in an order that spreads the lanes over the banks
  const int r = lane / 4, first = r & 1, m = m0 + 2 * r, n = e.n - lane + lane % 4 * 8;
  const uint4* from = stage + r * 8 + lane % 4 * 2;
  const uint4 p = from[first], q = from[first ^ 1], lo = first ? q : p, hi = first ? p : q;
  const uint4 even = make_uint4(__byte_perm(lo.x, lo.y, 0x5410), __byte_perm(lo.z, lo.w, 0x5410), __byte_perm(hi.x, hi.y, 0x5410), __byte_perm(hi.z, hi.w, 0x5410));
  const uint4 odd = make_uint4(__byte_perm(lo.x, lo.y, 0x7632), __byte_perm(lo.z, lo.w, 0x7632), __byte_perm(hi.x, hi.y, 0x7632), __byte_perm(hi.z, hi.w, 0x7632));
  if (n < e.N) {
    T* at = e.y + (int64_t)m * e.ldy + n;
    if (m < end) *reinterpret_cast<uint4*>(at) = even;
    if (m + 1 < end) *reinterpret_cast<uint4*>(at + e.ldy) = odd;
  }
  __syncwarp();
}

__device__ __forceinline__ void load16(uint32_t taddr, int (&a)[16]) {
  uint32_t v[16];
  tmem_ld16(taddr, v);
#pragma unroll
  for (int i = 0; i < 16; ++i) a[i] = (int)v[i];
}

// ---- product, two SMs on a tile -------------------------------------------------------------------------------------------------------
// cta_group::2: two SMs on a tile of 256 weight rows x mt activation rows.  Each loads its own 128 weight rows and half of the
// activation rows, the MMA reads both halves: 32 KB per SM and unit at mt = 256, where one SM alone with a 128 x 256 tile needs 48 KB, and
// that set its pace (half the MMAs took the same time: 87 GB/s and SM from L2; 28672 x 4096, 2048 rows 260 us against 158 - 164, 2930 - 3040 Top/s).  The
// even thread block of a pair issues the MMAs; its `full` barrier counts the bytes of both; commits arrive in both.
//
// A cluster is one pair, walking over tiles, or (few tiles, long K) two or four pairs that split K of one tile: then each of them adds up
// its share of the activation rows, which the others send to its shared memory.
struct PairParams {
  W8Params w;
  int tiles, splits;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_block(uint32_t addr, uint32_t rank) {     // the same place in another thread block of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tma_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint32_t bar, uint32_t mask, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b16 m;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "cvt.u16.u32 m, %1;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(bar), "r"(mask), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) w8a8_pair_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                                                                const PairParams pp) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ int s_failed;
  __shared__ __align__(16) float s_step[2][256];
  __shared__ __align__(16) int s_sums[2][256];
  __shared__ uint4 s_stage[kEpiThreads / 32][64];
  const W8Params& p = pp.w;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int ku = p.ku, stages = p.stages;
  const uint32_t half = (uint32_t)p.mt / 2, x_bytes = half * kUnitK, w_ring = s_u32(smem), x_ring = w_ring + stages * kWBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + stages * (kWBytes + x_bytes));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 5);
  const uint32_t full = s_u32(bars), empty = full + kMaxStages * 8, acc_full = empty + kMaxStages * 8, acc_empty = acc_full + 16,
                 mma_done = acc_empty + 16;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), odd = rank & 1, leader = rank & ~1u, pair_mask = 3u << leader;
  const int split = (int)rank >> 1, splits = pp.splits;
  // units of K that this pair takes; clusters of one pair walk over tiles, others have one
  const int k0 = (int)((int64_t)ku * split / splits), k1 = (int)((int64_t)ku * (split + 1) / splits), n_k = k1 - k0;
  const int first = (int)blockIdx.x / (2 * splits), step = (int)gridDim.x / (2 * splits);
  bool dead = false;
  int* status = &s_failed;

  if (threadIdx.x == 0) {
    s_failed = 0;
    for (int i = 0; i < kMaxStages; ++i) {
      bar_init(full + i * 8, 1);
      bar_init(empty + i * 8, 1);
    }
    bar_init(mma_done, 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(acc_full + i * 8, 1);
      bar_init(acc_empty + i * 8, 2 * kEpiThreads / 32);       // the epilogue warps of both thread blocks
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();         // barriers of the others are ready
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 0) {
    // ================= operands: own weight rows, own half of the activation rows =================
    if (lane == 0) {
      const uint32_t full_at = in_block(full, leader);
      const int mine = first < pp.tiles ? (pp.tiles - first + step - 1) / step * n_k : 0;      // units of all tiles
      struct Place {      // of a unit, kept by counting
        int t, k, row, m0;
      };
      auto at_tile = [&](int t) { return Place{t, k0, t / p.mtiles * 2 * kRows + (int)(odd * kRows), t % p.mtiles * p.mt + (int)(odd * half)}; };
      auto next = [&](Place& a) {
        if (++a.k == k1) a = at_tile(a.t + step);
      };
      auto load_w = [&](const Place& a, int s) {
        if (!odd) bar_expect(full + s * 8, 2 * (kWBytes + x_bytes));
        tma_pair(w_ring + s * kWBytes, &tm_w, a.k * kUnitK, a.row, full_at + s * 8);
      };
      auto load_x = [&](const Place& a, int s) { tma_pair(x_ring + s * x_bytes, &tm_x, a.k * kUnitK, a.m0, full_at + s * 8); };
      Place at = at_tile(first), x_at = at;
      int i = 0;
      for (; i < min(mine, stages); ++i, next(at)) load_w(at, i);      // weights: nothing that this launch may overlap writes them
      pdl_wait();
      for (int j = 0; j < i; ++j, next(x_at)) load_x(x_at, j);
      int s = 0;
      uint32_t par = 0;
      for (; i < mine; ++i, next(at)) {
        bar_wait(empty + s * 8, par, status, dead);
        if (dead) break;
        load_w(at, s);
        load_x(at, s);
        if (++s == stages) s = 0, par ^= 1;
      }
      bool late = false;
      if (!odd)       // the copies of both thread blocks end here
        for (int j = max(0, i - stages); j < i; ++j) bar_wait(full + (j % stages) * 8, (j / stages) & 1, status, late);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ================= products =================
    if (!odd) {
      const uint32_t me = elect_one();
      const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.mt >> 3) << 17) | ((uint32_t)(2 * kRows >> 4) << 24);
      const uint64_t w_desc0 = umma_desc(w_ring), x_desc0 = umma_desc(x_ring);
      int s = 0, seg = 0;
      uint32_t par = 0;
      for (int t = first; t < pp.tiles; t += step, ++seg) {
        const int buf = seg & 1;
        const uint32_t acc = tmem + buf * 256;
        bar_wait_cluster(acc_empty + buf * 8, ((seg >> 1) & 1) ^ 1, status, dead);
        for (int i = 0; i < n_k; ++i) {
          bar_wait(full + s * 8, par, status, dead);
          __syncwarp();
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t dw = w_desc0 + (uint64_t)(s * (kWBytes >> 4)), dx = x_desc0 + (uint64_t)(s * (x_bytes >> 4));
#pragma unroll
          for (int j = 0; j < 4; ++j) umma_i8_pair(acc, dw + 2 * j, dx + 2 * j, idesc, (i | j) != 0, me);
          umma_commit_pair(empty + s * 8, pair_mask, me);
          if (++s == stages) s = 0, par ^= 1;
        }
        if (dead)       // the other thread block's outputs are no good either
          asm volatile("st.shared::cluster.s32 [%0], %1;\n\tfence.acq_rel.cluster;" ::"r"(in_block(s_u32(&s_failed), leader + 1)), "r"((int)PARE_ERR_TIMEOUT) : "memory");
        umma_commit_pair(acc_full + buf * 8, pair_mask, me);
      }
      umma_commit_pair(mma_done, 1u << leader, me);
      bool late = false;
      bar_wait(mma_done, 0, status, late);
    }
    __syncwarp();
  } else if (warp >= 4 && splits == 1) {
    // ================= epilogue: tensor memory -> registers -> global =================
    pdl_wait();
    const int q4 = warp & 3, c0 = (warp - 4) / 4 * 16, te = threadIdx.x - 4 * 32;
    const uint32_t empty_at = in_block(acc_empty, leader);
    Epilogue<T> epi(p);
    // A tile's scales and steps are read while the tile before it is stored.
    static_assert(kEpiThreads >= 256, "a thread per activation row of a tile");
    float3 of, of_next;
    float mine = 0.f;
    int mine_sum = 0;
    auto column_of = [&](int t) { return t / p.mtiles * 2 * kRows + (int)(odd * kRows) + q4 * 32 + lane; };
    auto ahead = [&](int t) {
      const int m = t % p.mtiles * p.mt + te;
      of_next = epi.fetch(p, column_of(t));
      if (te < p.mt && m < p.M) {
        mine = p.step[m];
        mine_sum = p.zero ? p.sums[m] : 0;
      }
    };
    if (first < pp.tiles) ahead(first);
    int seg = 0;
    for (int t = first; t < pp.tiles; t += step, ++seg) {
      const int m0 = t % p.mtiles * p.mt, mrows = min(p.mt, p.M - m0), buf = seg & 1;
      const uint32_t acc = tmem + buf * 256 + ((uint32_t)(q4 * 32) << 16);
      of = of_next;
      epi.column(column_of(t), of);
      s_step[buf][te] = mine;
      s_sums[buf][te] = mine_sum;
      asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory");
      if (t + step < pp.tiles) ahead(t + step);
      bar_wait(acc_full + buf * 8, (seg >> 1) & 1, status, dead);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      epi.bad = __any_sync(0xffffffffu, dead || *const_cast<volatile int*>(&s_failed) != 0);
      for (int c = c0; c < mrows; c += 32) {
        int a[16];
        load16(acc + c, a);
        if (epi.wide_out) store16_wide<T>(epi, a, m0 + c, m0 + mrows, s_step[buf] + c, s_sums[buf] + c, s_stage[warp - 4]);
        else epi.store16(a, m0 + c, m0 + mrows, s_step[buf] + c, s_sums[buf] + c);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive_at(empty_at + buf * 8);
    }
  }

  if (splits > 1) {
    // ================= one tile: its sums meet in the cluster =================
    const int q4 = warp & 3, c0 = (warp - 4) / 4 * 16, te = threadIdx.x - 4 * 32;
    const int m0 = first % p.mtiles * p.mt, mrows = min(p.mt, p.M - m0), share = p.mt / splits;
    const uint32_t acc = tmem + ((uint32_t)(q4 * 32) << 16), row = (uint32_t)(q4 * 32 + lane);
    if (warp >= 4) {
      bar_wait(acc_full, 0, status, dead);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    __syncthreads();
    cluster_sync();       // everybody's products are done: the rings are free
    // [sender's number without the receiver][share / 4][128 weight rows][4 activation rows]
    const uint32_t slot_bytes = (uint32_t)share * kRows * 4;
    if (warp >= 4) {
      for (int q = 0; q < splits; ++q) {
        if (q == split || q * share >= mrows) continue;
        const uint32_t to = in_block(w_ring + (split < q ? split : split - 1) * slot_bytes, 2 * q + odd);
        for (int c = c0; c < share; c += 32) {
          int a[16];
          load16(acc + q * share + c, a);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            asm volatile("st.shared::cluster.v4.s32 [%0], {%1, %2, %3, %4};" ::"r"(to + ((c / 4 + i) * kRows + row) * 16), "r"(a[4 * i]),
                         "r"(a[4 * i + 1]), "r"(a[4 * i + 2]), "r"(a[4 * i + 3])
                         : "memory");
        }
      }
      if (*const_cast<volatile int*>(&s_failed) != 0 && te == 0) {     // a failure of one is a failure of the tile
        for (int q = 0; q < 2 * splits; ++q)
          asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(in_block(s_u32(&s_failed), q)), "r"((int)PARE_ERR_TIMEOUT) : "memory");
      }
    }
    __syncthreads();
    cluster_sync();
    if (warp >= 4) {
      pdl_wait();
      const int from = split * share, to = min(from + share, mrows);
      Epilogue<T> epi(p);
      epi.column(p, first / p.mtiles * 2 * kRows + odd * kRows + (int)row);
      epi.bad = *const_cast<volatile int*>(&s_failed) != 0;
      for (int i = te; i < to - from; i += kEpiThreads) {
        s_step[0][i] = p.step[m0 + from + i];
        s_sums[0][i] = p.zero ? p.sums[m0 + from + i] : 0;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory");
      for (int c = c0; c < to - from; c += 32) {
        int a[16];
        load16(acc + from + c, a);
        for (int e = 0; e < splits - 1; ++e) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 v = ld_s128(w_ring + e * slot_bytes + ((c / 4 + i) * kRows + row) * 16);
            a[4 * i] += (int)v.x;
            a[4 * i + 1] += (int)v.y;
            a[4 * i + 2] += (int)v.z;
            a[4 * i + 3] += (int)v.w;
          }
        }
        if (epi.wide_out) store16_wide<T>(epi, a, m0 + from + c, m0 + to, s_step[0] + c, s_sums[0] + c, s_stage[warp - 4]);
        else epi.store16(a, m0 + from + c, m0 + to, s_step[0] + c, s_sums[0] + c);
      }
    }
  }

  // ---- teardown: both thread blocks done with tensor memory and each other's shared memory, then free it ----
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ---- product of up to 16 rows, tokens quantized on the way ---------------------------------------------------------------------------------
// Streams the weights once, and what counts besides is the number of steps that wait for one another: so one launch, in which the
// weights are on their way while the tokens become codes.  `splits` thread blocks (a cluster of 1, 2, 4) share a
// weight tile's K; each quantizes its own columns (and looks at all of them for the rows' maxima), keeps their codes in shared memory in
// the order of the MMA's operand for all its tiles, and finishes the sums of its share of the 128 weight rows with what the others send.
//   warp 0  TMA of weights     warp 1  tcgen05.mma     warp 2  tensor memory     warps 4-11  tokens, then (4-7) the epilogue
// CODED: the tokens were quantized by a launch before this one (where that is too much to do beside the weights) and their codes
// come by TMA; what is left is the sums' short way through the cluster.
constexpr int kFewRows = 16;
constexpr int kFewThreads = 384;
constexpr int kFewCodes = 256;                        // threads that quantize
constexpr int kFewUnitBytes = kFewRows * kUnitK;      // codes of a unit
constexpr int kFewVecs = 8;                           // vectors of eight columns per thread: they stay in registers
constexpr int kFewMaxUnits = 60;                      // units of K per thread block: 120 KB of codes
constexpr uint32_t kFewTmem = 32;                     // two accumulators of 16 columns

struct FewParams {
  W8Params w;
  const void* x;
  int64_t ldx;
  const float* input_scale;
  int K, tiles, splits, stages;
};

template <typename T, bool CODED>
__global__ void __launch_bounds__(kFewThreads, 1) w8a8_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                                                                  const FewParams fp) {
  extern __shared__ unsigned char smem_raw[];
  pdl_launch_dependents();
  __shared__ int s_failed;
  __shared__ uint32_t s_top[kFewRows];                // row maxima
  __shared__ int s_sum[4][kFewRows];                  // sums of codes, from each thread block of the cluster
  __shared__ float s_step[kFewRows];
  __shared__ int4 s_in[3 * 128 / 4 * 4];              // sums from the others: [sender][4][rows of this share] of four activation rows
  __shared__ uint64_t s_bars[2 * kMaxStages + 8];
  __shared__ uint32_t s_tmem;
  const W8Params& p = fp.w;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int ku = p.ku, stages = fp.stages, M = p.M, splits = fp.splits;
  const uint32_t w_ring = s_u32(smem), codes = w_ring + stages * kWBytes;
  const uint32_t full = s_u32(s_bars), empty = full + kMaxStages * 8, acc_full = empty + kMaxStages * 8, acc_empty = acc_full + 16,
                 mma_done = acc_empty + 16, x_ready = mma_done + 8, sums_in = x_ready + 8;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = splits > 1 ? (int)cluster_rank() : 0;
  const int k0 = ku * rank / splits, k1 = ku * (rank + 1) / splits, n_k = k1 - k0;
  const int first = (int)blockIdx.x / splits, step = (int)gridDim.x / splits;
  bool dead = false;
  int* status = &s_failed;

  if (threadIdx.x == 0) {
    s_failed = 0;
    for (int i = 0; i < kMaxStages; ++i) {
      bar_init(full + i * 8, 1);
      bar_init(empty + i * 8, 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(acc_full + i * 8, 1);
      bar_init(acc_empty + i * 8, 4);
    }
    bar_init(mma_done, 1);
    bar_init(x_ready, CODED ? 1 : kFewCodes / 32);
    bar_init(sums_in, splits > 1 ? (splits - 1) * (4 / splits) : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < kFewRows) s_top[threadIdx.x] = 0;
  if (threadIdx.x < 4 * kFewRows) (&s_sum[0][0])[threadIdx.x] = 0;
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(&s_tmem)), "r"(kFewTmem) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  if (splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");    // the others' barriers: waited for below

  if (warp == 0) {
    // ================= weights =================
    if (lane == 0) {
      if (!CODED) pdl_wait();      // whoever made the weights may be the kernel before
      const int mine = first < fp.tiles ? (fp.tiles - first + step - 1) / step * n_k : 0;
      int t = first, k = k0, s = 0, i = 0;
      uint32_t par = 1;
      for (; i < mine; ++i) {
        bar_wait(empty + s * 8, par, status, dead);
        if (dead) break;
        bar_expect(full + s * 8, kWBytes);
        tma_tile(w_ring + s * kWBytes, &tm_w, k * kUnitK, t * kRows, full + s * 8);
        if (++s == stages) s = 0, par ^= 1;
        if (++k == k1) k = k0, t += step;
      }
      bool late = false;
      for (int j = max(0, i - stages); j < i; ++j) bar_wait(full + (j % stages) * 8, (j / stages) & 1, status, late);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ================= products =================
    const uint32_t me = elect_one();
    const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kFewRows >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
    const uint64_t w_desc0 = umma_desc(w_ring), x_desc0 = umma_desc(codes);
    bar_wait(x_ready, 0, status, dead);
    int s = 0, seg = 0;
    uint32_t par = 0;
    for (int t = first; t < fp.tiles; t += step, ++seg) {
      const int buf = seg & 1;
      bar_wait(acc_empty + buf * 8, ((seg >> 1) & 1) ^ 1, status, dead);
      for (int i = 0; i < n_k; ++i) {
        bar_wait(full + s * 8, par, status, dead);
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t dw = w_desc0 + (uint64_t)(s * (kWBytes >> 4)), dx = x_desc0 + (uint64_t)(i * (kFewUnitBytes >> 4));
#pragma unroll
        for (int j = 0; j < 4; ++j) umma_i8(tmem + buf * kFewRows, dw + 2 * j, dx + 2 * j, idesc, (i | j) != 0, me);
        umma_commit(empty + s * 8, me);
        if (++s == stages) s = 0, par ^= 1;
      }
      umma_commit(acc_full + buf * 8, me);
    }
    umma_commit(mma_done, me);
    bool late = false;
    bar_wait(mma_done, 0, status, late);
    __syncwarp();
  } else if (warp >= 4) {
    // ================= tokens =================
    pdl_wait();
    const int tid = threadIdx.x - 4 * 32;
    if constexpr (CODED) {
      if (tid == 0) {
        bar_expect(x_ready, n_k * kFewUnitBytes);
        for (int u = 0; u < n_k; ++u) tma_tile(codes + u * kFewUnitBytes, &tm_x, (k0 + u) * kUnitK, 0, x_ready);
      }
      if (tid < M) s_step[tid] = p.step[tid];
      asm volatile("bar.sync 2, 256;" ::: "memory");
      if (splits > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    } else {
      int per = kFewCodes;                              // threads per row, at least sixteen
      for (int r = 1; r < M; r <<= 1) per >>= 1;
      const int m = tid / per, at = tid % per, c0 = k0 * kUnitK, c1 = min(k1 * kUnitK, fp.K);
      const T* row = reinterpret_cast<const T*>(fp.x) + m * fp.ldx;
      uint4 v[kFewVecs];
      uint32_t top = 0;
      if (m < M) {
#pragma unroll
        for (int i = 0; i < kFewVecs; ++i) {
          const int c = (i * per + at) * 8;
          v[i] = c < fp.K ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
        }
        if (fp.input_scale) {
#pragma unroll
          for (int i = 0; i < kFewVecs; ++i) {
            const int c = (i * per + at) * 8;
            T* e = reinterpret_cast<T*>(&v[i]);
            if (c < fp.K) {
#pragma unroll
              for (int j = 0; j < 8; ++j) e[j] = smoothed<T>(e[j], fp.input_scale, c + j);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kFewVecs; ++i) top = __vmaxu2(top, q8::magnitudes(v[i]));
        top = max(top & 0xffffu, top >> 16);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));      // at least sixteen threads share a row
      if (m < M && (lane & 15) == 0) atomicMax(&s_top[m], top);
      asm volatile("bar.sync 2, 256;" ::: "memory");
      if (splits > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
      if (m < M) {
        top = s_top[m];
        const uint16_t bits = (uint16_t)top;
        const float amax = to_float<T>(*reinterpret_cast<const T*>(&bits));
        const q8::Grid grid(amax < 1e-6f ? 1e-6f : amax);
        if (at == 0) s_step[m] = grid.finite ? grid.step : __int_as_float(0x7fffffff);
        int sum = 0;
#pragma unroll
        for (int i = 0; i < kFewVecs; ++i) {
          const int c = (i * per + at) * 8;
          if (c < c0 || c >= c1) continue;
          const uint2 o = grid.codes<T>(v[i]);
          sum = __dp4a((int)o.y, 0x01010101, __dp4a((int)o.x, 0x01010101, sum));
          const int u = (c - c0) / kUnitK, chunk = (c % kUnitK) / 16;
          asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(codes + u * kFewUnitBytes + m * kUnitK + ((chunk ^ (m & 7)) << 4) + (c & 8)), "r"(o.x), "r"(o.y)
                       : "memory");
        }
        if (p.zero) atomicAdd(&s_sum[rank][m], sum);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("bar.sync 2, 256;" ::: "memory");    // steps and sums are there for the epilogue
      if (lane == 0) bar_arrive(x_ready);
    }

    if (warp < 8) {
      // ================= epilogue =================
      const int q4 = warp & 3, share = 4 / splits, owner = q4 / share;      // which thread block finishes this warp's 32 weight rows
      Epilogue<T> epi(p);
      int seg = 0;
      for (int t = first; t < fp.tiles; t += step, ++seg) {
        const int buf = seg & 1;
        const uint32_t acc = tmem + buf * kFewRows + ((uint32_t)(q4 * 32) << 16);
        epi.column(p, t * kRows + q4 * 32 + lane);
        bar_wait(acc_full + buf * 8, (seg >> 1) & 1, status, dead);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        int a[16];
        load16(acc, a);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(acc_empty + buf * 8);
        bool bad = __any_sync(0xffffffffu, dead || *const_cast<volatile int*>(&s_failed) != 0);
        if (splits > 1) {      // one tile
          // slot of the sender among the others; [4][rows of the share]
          auto slot = [&](int sender, int receiver) { return (sender < receiver ? sender : sender - 1) * 4 * share * 32 + (q4 % share) * 32 + lane; };
          if (owner != rank) {
            const uint32_t to = in_block(s_u32(s_in), owner);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              asm volatile("st.shared::cluster.v4.s32 [%0], {%1, %2, %3, %4};" ::"r"(to + (slot(rank, owner) + i * share * 32) * 16), "r"(a[4 * i]),
                           "r"(a[4 * i + 1]), "r"(a[4 * i + 2]), "r"(a[4 * i + 3])
                           : "memory");
            if (!CODED && p.zero && q4 % share == 0 && lane < kFewRows)
              asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(in_block(s_u32(&s_sum[rank][lane]), owner)), "r"(s_sum[rank][lane]) : "memory");
            if (bad && lane == 0)
              asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(in_block(s_u32(&s_failed), owner)), "r"((int)PARE_ERR_TIMEOUT) : "memory");
            asm volatile("fence.acq_rel.cluster;" ::: "memory");
            __syncwarp();
            if (lane == 0) arrive_at(in_block(sums_in, owner));
            continue;
          }
          bar_wait_cluster(sums_in, 0, status, dead);
          bad = __any_sync(0xffffffffu, dead || *const_cast<volatile int*>(&s_failed) != 0);
          for (int q = 0; q < splits; ++q) {
            if (q == rank) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int4 v = s_in[slot(q, rank) + i * share * 32];
              a[4 * i] += v.x;
              a[4 * i + 1] += v.y;
              a[4 * i + 2] += v.z;
              a[4 * i + 3] += v.w;
            }
          }
          if (!CODED && p.zero) {        // sums over all of K in this warp's own copy
            int all = 0;
            if (lane < kFewRows)
              for (int q = 0; q < splits; ++q) all += s_sum[q][lane];
            epi.row_sum = all;
          }
        } else if (!CODED && p.zero) {
          epi.row_sum = lane < kFewRows ? s_sum[0][lane] : 0;
        }
        if (CODED && p.zero) epi.row_sum = lane < M ? p.sums[lane] : 0;
        epi.bad = bad;
        epi.store16(a, 0, M, s_step);
      }
    }
  }
  if (splits > 1 && warp < 4) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");

  // ---- teardown ----
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (splits > 1) cluster_sync();      // nobody writes here any more
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kFewTmem) : "memory");
  }
}

// ---- host side --------------------------------------------------------------------------------------------------------------------------
// How many clusters of `size` thread blocks of a kernel fit the device at once (cached per device by the caller).
int resident_clusters(const void* kern, int size, int threads, int smem, int (&cached)[64]) {
  static std::mutex mu;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> lock(mu);
  if (cached[dev] == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)size, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    cached[dev] = n + 1;
  }
  return cached[dev] - 1;
}

// Up to 16 rows, if a thread block's codes fit beside a ring of weights.  The tokens are quantized on the way where a thread has at most
// eight vectors of eight columns to look at (4 rows of 4096): one launch, 1 / 2 / 4 rows of 4096 x 4096 7.4 / 7.5 / 8.1 us, 28672 x 4096 20.7 /
// 20.6 / 21.9 (0.86 of the copy rate); more rows in a launch of their own, 8 / 16 rows 8.4 / 8.4 and 23.0 / 23.4 (on the way 8 rows of 4096 x 4096
// cost 2.9 us more).  K is shared by as many thread blocks (4, 2) as keep every SM to one tile.
struct FewPlan {
  int splits, tiles, blocks, stages, units;      // splits 0: not this kernel
  bool coded;                                    // tokens are quantized by a launch of their own
};
constexpr int kFewSmem = 216 * 1024;

FewPlan few_plan(int M, int N, int K) {
  FewPlan f{};
  if (M > kFewRows) return f;
  const int ku = (K + kUnitK - 1) / kUnitK;
  f.tiles = (N + kRows - 1) / kRows;
  const void* kern = reinterpret_cast<const void*>(w8a8_few_kernel<__half, false>);
  static int cached4[64] = {}, cached2[64] = {};
  int splits = 1;
  if (ku >= 8 && f.tiles <= sm_count() / 2 && ensure_smem_attr(kern, kFewSmem)) {
    if (f.tiles <= resident_clusters(kern, 4, kFewThreads, kFewSmem, cached4)) splits = 4;
    else if (f.tiles <= resident_clusters(kern, 2, kFewThreads, kFewSmem, cached2)) splits = 2;
  }
  f.units = (ku + splits - 1) / splits;
  int per = kFewCodes;      // threads per row
  for (int r = 1; r < M; r <<= 1) per >>= 1;
  if (f.units > kFewMaxUnits) return f;
  f.coded = K % 8 || (K / 8 + per - 1) / per > kFewVecs;
  f.splits = splits;
  f.blocks = splits > 1 ? f.tiles * splits : f.tiles < sm_count() ? f.tiles : sm_count();
  f.stages = (kFewSmem - 1024 - f.units * kFewUnitBytes) / kWBytes;
  if (f.stages > kMaxStages) f.stages = kMaxStages;
  return f;
}

struct W8Plan {
  int mt, mtiles, ku, blocks, stages, splits;
  int tiles;         // weight tiles x activation tiles
  int64_t units;
};

// Height of the activation tiles (equal, a multiple of 32) and whether two or four pairs of SMs split K, by an estimate in microseconds: rounds of
// all pairs x units x what a unit of that height takes (0.21 at 32 rows, 0.36 at 256), the weights' way from memory as a lower
// bound, and what a split adds.  Within a few per cent of the best of 8 heights x 2 splits for 23 shapes of 17 - 3000 rows; four pairs, where
// all their clusters fit the device at once (not 16 of them): 17 rows of 512 x 18944 15.5 us against 22.7, of 3584 x 18944 18.9 against 24.1.
W8Plan w8_plan(int M, int N, int K) {
  W8Plan best{};
  double least = 1e30;
  const int sms = sm_count(), ku = (K + kUnitK - 1) / kUnitK;
  const double stream_us = (double)N * K / 6.0e6;
  const void* kern = reinterpret_cast<const void*>(w8a8_pair_kernel<__half>);
  static int cached[64] = {};
  const int eights = ku >= 8 && ensure_smem_attr(kern, kMaxSmem) ? resident_clusters(kern, 8, kThreads, kMaxSmem, cached) : 0;
  for (int target : {256, 192, 160, 128, 96, 64, 32}) {
    for (int splits : {1, 2, 4}) {
      W8Plan g{};
      const int step = splits == 4 ? 64 : 32;        // a pair's share of a split tile is a multiple of 16
      g.mtiles = (M + target - 1) / target;
      g.mt = ((M + g.mtiles - 1) / g.mtiles + step - 1) / step * step;
      g.mtiles = (M + g.mt - 1) / g.mt;
      g.ku = ku;
      g.splits = splits;
      g.units = (int64_t)((N + 2 * kRows - 1) / (2 * kRows)) * g.mtiles;
      if (g.mt > 256 || splits > ku || g.units * ku >= (int64_t)1 << 31) continue;
      g.tiles = (int)g.units;
      g.units *= ku;
      const int clusters = splits == 4 ? eights : sms / (2 * splits), rounds = splits > 1 ? 1 : (g.tiles + clusters - 1) / clusters;
      if (splits > 1 && g.tiles > clusters) continue;
      const double cost = std::max((double)rounds * ((ku + splits - 1) / splits) * (0.2 + 0.00055 * g.mt), stream_us) + 0.01 * g.mt +
                          (splits == 4 ? 2.4 + 0.02 * g.mt : splits == 2 ? 2.0 + 0.015 * g.mt : 0.0);
      if (cost < least - 1e-9) {
        least = cost;
        best = g;
      }
    }
  }
  if (best.splits == 0) return best;
  const int clusters = sms / (2 * best.splits);
  best.blocks = 2 * best.splits * (best.splits > 1 || best.tiles < clusters ? best.tiles : clusters);
  best.stages = std::min(kRingBytes / (kWBytes + best.mt / 2 * kUnitK), kMaxStages);
  return best;
}

struct W8Space {
  size_t codes, step, sums, bytes;
  int64_t ldc;
  W8Space(int M, int K) {
    auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    ldc = (K + 15) / 16 * 16;
    codes = 0;
    step = up((size_t)M * ldc);
    sums = step + up((size_t)M * 4);
    bytes = sums + up((size_t)M * 4);
  }
};

}  // namespace
}  // namespace pare

extern "C" {

using namespace pare;

size_t pare_w8a8_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > kMaxK) return 0;
  const FewPlan f = few_plan(M, N, K);
  if (f.splits && !f.coded) return 0;
  return f.splits || w8_plan(M, N, K).splits ? W8Space(M, K).bytes : 0;
}

int pare_w8a8_forward(const void* x, int x_dtype, int64_t ldx, const int8_t* weight, int64_t ldw, const float* scale, const float* zero,
                      const float* input_scale, const void* bias, void* y, int64_t ldy, int M, int N, int K, void* workspace,
                      size_t workspace_bytes, void* stream) {
  PARE_REQUIRE(M > 0 && N > 0 && K > 0 && ldw >= K && ldy >= N && (M == 1 || ldx >= K), PARE_ERR_SHAPE);
  PARE_REQUIRE(x_dtype == PARE_F16 || x_dtype == PARE_BF16, PARE_ERR_DTYPE);
  PARE_REQUIRE(x && weight && scale && y, PARE_ERR_SHAPE);
  PARE_REQUIRE(K <= kMaxK, PARE_ERR_UNSUPPORTED);
  PARE_REQUIRE(aligned16(weight) && ldw % 16 == 0 && aligned16(workspace), PARE_ERR_ALIGN);
  const FewPlan f = few_plan(M, N, K);
  const W8Plan g = f.splits ? W8Plan{} : w8_plan(M, N, K);
  const W8Space sp(M, K);
  if (f.splits && !f.coded) {
    PARE_REQUIRE(aligned16(x) && (M == 1 || ldx % 8 == 0), PARE_ERR_ALIGN);
  } else {
    PARE_REQUIRE(f.splits || g.splits, PARE_ERR_UNSUPPORTED);
    PARE_REQUIRE(workspace && workspace_bytes >= sp.bytes, PARE_ERR_WORKSPACE);
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  EncodeTiledFn enc = encode_fn();
  PARE_REQUIRE(enc != nullptr, PARE_ERR_CUDA);
  // tensor maps: operands in rows of K bytes, boxes of 128 bytes, 128B swizzle; rows and columns beyond the end read as zeros
  auto map = [&](CUtensorMap* tm, const void* base, int rows, int64_t pitch, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {(cuuint32_t)kUnitK, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  CUtensorMap tw, tx;
  PARE_REQUIRE(map(&tw, weight, N, ldw, kRows), PARE_ERR_CUDA);
  // with programmatic launch, and in clusters
  auto launch = [&](auto kern, int blocks, int threads, int most_smem, size_t smem, int cluster, auto... args) -> int {
    if (!ensure_smem_attr(reinterpret_cast<const void*>(kern), most_smem)) return PARE_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)cluster, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? launch_status() : (int)PARE_ERR_CUDA;
  };
  W8Params p{};
  p.scale = scale;
  p.zero = zero;
  p.bias = bias;
  p.y = y;
  p.ldy = ldy;
  p.M = M;
  p.N = N;
  p.ku = (K + kUnitK - 1) / kUnitK;

  const bool half = x_dtype == PARE_F16;
  const FewParams fp{p, x, ldx, input_scale, K, f.tiles, f.splits, f.stages};
  const size_t few_smem = 1024 + (size_t)f.stages * kWBytes + (size_t)f.units * kFewUnitBytes;
  if (f.splits && !f.coded)
    return half ? launch(w8a8_few_kernel<__half, false>, f.blocks, kFewThreads, kFewSmem, few_smem, f.splits, tw, tw, fp)
                : launch(w8a8_few_kernel<__nv_bfloat16, false>, f.blocks, kFewThreads, kFewSmem, few_smem, f.splits, tw, tw, fp);

  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  PARE_REQUIRE(map(&tx, ws + sp.codes, M, sp.ldc, f.splits ? kFewRows : g.mt / 2), PARE_ERR_CUDA);

  const QuantParams q{x, ldx, input_scale, reinterpret_cast<int8_t*>(ws + sp.codes), sp.ldc, reinterpret_cast<float*>(ws + sp.step),
                      zero ? reinterpret_cast<int*>(ws + sp.sums) : nullptr, K};
  const bool vec = aligned16(x) && (M == 1 || ldx % 8 == 0) && K % 8 == 0 && (!input_scale || aligned16(input_scale));
  // As many threads per row as still leave all rows resident at once.
  auto quantize = [&](auto tag, auto scaled) -> int {
    using E = decltype(tag);
    constexpr bool kS = decltype(scaled)::value;
    auto go = [&](auto kern, int threads) -> int {
      const size_t row = vec ? (size_t)K * 2 : 0;
      // 48 KB without asking, static shared memory (256 bytes at most) among them
      if (row > 47 * 1024 && !ensure_smem_attr(reinterpret_cast<const void*>(kern), kMaxK * 2)) return PARE_ERR_CUDA;
      return launch_pdl(kern, dim3(M), dim3(threads), row, st, q);
    };
    if (!vec) return go(w8a8_quantize_kernel<E, 512, false, kS>, 512);
    const int per_sm = (M + sm_count() - 1) / sm_count();
    if (per_sm <= 2 && K > 8192) return go(w8a8_quantize_kernel<E, 1024, true, kS>, 1024);
    if (per_sm <= 2) return go(w8a8_quantize_kernel<E, 512, true, kS>, 512);
    if (per_sm <= 8) return go(w8a8_quantize_kernel<E, 256, true, kS>, 256);
    return go(w8a8_quantize_kernel<E, 128, true, kS>, 128);
  };
  const std::true_type yes;
  const std::false_type no;
  const int rc = half ? (input_scale ? quantize(__half(), yes) : quantize(__half(), no))
                      : (input_scale ? quantize(__nv_bfloat16(), yes) : quantize(__nv_bfloat16(), no));
  if (rc != PARE_OK) return rc;

  p.step = q.step;
  p.sums = q.sums;
  if (f.splits) {
    FewParams cp = fp;
    cp.w = p;
    return half ? launch(w8a8_few_kernel<__half, true>, f.blocks, kFewThreads, kFewSmem, few_smem, f.splits, tw, tx, cp)
                : launch(w8a8_few_kernel<__nv_bfloat16, true>, f.blocks, kFewThreads, kFewSmem, few_smem, f.splits, tw, tx, cp);
  }
  p.mt = g.mt;
  p.mtiles = g.mtiles;
  p.stages = g.stages;
  const size_t smem = 1024 + (size_t)g.stages * (kWBytes + g.mt / 2 * kUnitK) + 512;
  const PairParams pp{p, g.tiles, g.splits};
  return half ? launch(w8a8_pair_kernel<__half>, g.blocks, kThreads, kMaxSmem, smem, 2 * g.splits, tw, tx, pp)
              : launch(w8a8_pair_kernel<__nv_bfloat16>, g.blocks, kThreads, kMaxSmem, smem, 2 * g.splits, tw, tx, pp);
}

}  // extern "C"
