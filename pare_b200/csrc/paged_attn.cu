// Attention of new tokens' queries over the paged 8-bit KV cache (paged_cache.cu), sm_100a.
//
//   out[t][hq] = softmax_j(q[t][hq] . K_j * scale) V_j over the positions j <= position of token t in its request,
// K_j, V_j = code * scale of the block for blocks that are full, the open rows (16-bit) for the rest.  Query head hq reads KV head
// hq / (Hq / H); up to eight query heads that share a KV head sit in the eight columns of the warp-level MMA, so the cache is
// read once for all of them.  The reference leaves attention to its caller (pare/kv_cache.py:183-186).
//
// Mathematics.  Codes are integers of at most 127: exact in fp16, so S = code . q and O' = code^T . P run on fp16 operands with fp32
// sums, and the block's scales multiply S and O' outside (one number per 16 tokens).  q is fp16 as it is, or bf16 times a power of
// two per head that puts its largest magnitude into [256, 512): every bf16 value within 2^-22 of that is exact, smaller ones are
// within 2^-34 of the largest.  Softmax runs online: a reference value per head which only moves when a score passes it by more than
// 2^kSlack (one vote per 16 tokens instead of a reduction); probabilities are kept times 2^kBias of that, so those down to 2^-18 of
// the reference are normal fp16 numbers and none passes 2^15.  Their sum is taken before their rounding to fp16.
//
// Work.  Units of 16 tokens of one (token, group of heads), counted by the step's tables; each thread block takes one contiguous run
// of units, all runs equally long, so ragged lengths balance by themselves and the host needs to know none of them.  Inside a run the
// warps take units in turn; each warp feeds itself through a ring of its own (cp.async, no barrier between warps), and their
// (maximum, sum, O) meet in shared memory at the end of a tile.  Tiles that span thread blocks leave their parts in the workspace for
// a second kernel.  Nothing in the workspace outlives the call, no counters: calls on any streams and replays of any graphs do not
// meet there.
#include <type_traits>

#include "paged.cuh"

namespace pare {
namespace {

using namespace paged;

constexpr int kHeads = 8;                  // query heads of a tile (MMA columns)
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBias = 4.f, kSlack = 11.f;

template <int D>
struct Shape {
  static constexpr int kStageBytes = 2 * kUnit * D;           // codes of 16 tokens: keys, then values
  static constexpr int kStages = D == 128 ? 6 : 8;
  static constexpr int kRing = kStages * kStageBytes;         // per warp
  static constexpr int kPitch = D + 4;                        // floats per head of a warp's O at the end of a tile
  static constexpr int kMergeFloats = kHeads * kPitch + 2 * kHeads;
  static_assert(kMergeFloats * 4 <= kRing, "the ring holds a warp's result");
  static constexpr size_t kSmem = (size_t)kWarps * (kRing + kStages * 8);
  static constexpr int kPartFloats = kHeads * D + 2 * kHeads; // a part in the workspace: O, maxima, sums
};

struct PagedAttnParams {
  const void* q;
  int64_t q_st, q_sh;
  void* out;
  int64_t o_st, o_sh;
  const int* token_request;
  const int* positions;
  const int* seq_lens;
  const int* unit_start;
  const int* table;
  int64_t ld_table;
  const int8_t* k_codes;
  const int8_t* v_codes;
  const float* k_scale;
  const float* v_scale;
  const void* tail_k;
  const void* tail_v;
  float* parts;
  float scale_log2;
  int T, R, H, group, sub, bs_log2, num_blocks, max_blocks;   // sub: tiles of eight heads per KV head
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Two bytes (selector 0x4140: bytes 0, 1; 0x4342: bytes 2, 3) of four codes + 128 -> the codes as two fp16 numbers: under the
// mantissa of 1024 a byte u reads 1024 + u, and 1024 + 128 is taken off again, exactly.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t w) {
  const uint32_t r = __byte_perm(w, 0x64646464u, SEL);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&r), __float2half2_rn(1152.f));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Largest over the eight lanes that hold the same heads (lane = 4 g + t: over g)
__device__ __forceinline__ float max_over_g(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float sum_over_g(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Units of a run per thread block: equal shares, but at least one unit per warp.
__device__ __forceinline__ int64_t run_units(int64_t total, int blocks) {
  const int64_t each = (total + blocks - 1) / blocks;
  return each < kWarps ? kWarps : each;
}

template <typename T, int D>
struct Tile {
  using S = Shape<D>;
  static constexpr int kJ = D / 64;              // 16-byte chunks of a key row per lane
  static constexpr int kW = D / 32;              // words of four value channels per lane and token: channels (D / 8) g ..
  uint32_t qh[kJ][4][2];                         // query operand, fp16: channels 16 (t + 4 j) + 4 w + {0, 1}, {2, 3} of head g
  float o[2 * kW][4];                            // O of channels (D / 8) g + 2 i, + 1 x heads 2 t, 2 t + 1
  float m0, m1, l0, l1;                          // reference (base 2) and partial sums of heads 2 t, 2 t + 1
  float f0, f1;                                  // score factors of those heads (softmax scale, log2 e, 1 / power of two)

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < 2 * kW; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    m0 = m1 = -INFINITY;
    l0 = l1 = 0.f;
  }

  // row: the query of head g of the tile (nullptr: a column without a head)
  __device__ __forceinline__ void load_q(const T* row, float scale_log2, int lane) {
    const int t = lane & 3;
    uint4 w[kJ][2];
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      w[j][0] = w[j][1] = make_uint4(0, 0, 0, 0);
      if (row) {
        const uint4* at = reinterpret_cast<const uint4*>(row + 16 * (t + 4 * j));
        w[j][0] = at[0];
        w[j][1] = at[1];
      }
    }
    float back = 1.f;
    if (std::is_same<T, __nv_bfloat16>::value) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(w[j][e].x & 0x7fff7fffu, w[j][e].y & 0x7fff7fffu),
                                       __vmaxu2(w[j][e].z & 0x7fff7fffu, w[j][e].w & 0x7fff7fffu)));
      uint32_t bits = max(top & 0xffffu, top >> 16);
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
      int e = (int)(bits >> 7) - 127;                        // exponent of the largest magnitude
      if (bits == 0 || e == 128) e = 8;                      // nothing to scale (zeros; infinities and NaN stay what they are)
      const int up = min(max(8 - e, -120), 120);
      const float f = __int_as_float((127 + up) << 23);
      back = __int_as_float((127 - up) << 23);
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2) {
          uint32_t* x = reinterpret_cast<uint32_t*>(&w[j][e2]);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = pack_half2(__uint_as_float(x[i] << 16) * f, __uint_as_float(x[i] & 0xffff0000u) * f);
        }
    }
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const uint32_t* x = reinterpret_cast<const uint32_t*>(w[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) qh[j][i][0] = x[2 * i], qh[j][i][1] = x[2 * i + 1];
    }
    f0 = __shfl_sync(0xffffffffu, back, 8 * t) * scale_log2;        // lane 4 g with g = 2 t
    f1 = __shfl_sync(0xffffffffu, back, 8 * t + 4) * scale_log2;
  }

  // Scores (already in base 2; hidden ones -inf) of tokens g, g + 8 x heads 2 t, 2 t + 1 -> probabilities in place
  __device__ __forceinline__ void softmax(float (&s)[4]) {
    const bool passed = s[0] > m0 + kSlack || s[2] > m0 + kSlack || s[1] > m1 + kSlack || s[3] > m1 + kSlack;
    if (__any_sync(0xffffffffu, passed)) {
      const float n0 = fmaxf(m0, max_over_g(fmaxf(s[0], s[2]))), n1 = fmaxf(m1, max_over_g(fmaxf(s[1], s[3])));
      const float a0 = n0 == m0 ? 1.f : ex2(m0 - n0), a1 = n1 == m1 ? 1.f : ex2(m1 - n1);
      m0 = n0;
      m1 = n1;
      l0 *= a0;
      l1 *= a1;
#pragma unroll
      for (int i = 0; i < 2 * kW; ++i) {
        o[i][0] *= a0;
        o[i][1] *= a1;
        o[i][2] *= a0;
        o[i][3] *= a1;
      }
    }
    const float b0 = m0 == -INFINITY ? 0.f : m0 - kBias, b1 = m1 == -INFINITY ? 0.f : m1 - kBias;
    s[0] = ex2(s[0] - b0);
    s[1] = ex2(s[1] - b1);
    s[2] = ex2(s[2] - b0);
    s[3] = ex2(s[3] - b1);
    l0 += s[0] + s[2];
    l1 += s[1] + s[3];
  }

  // 16 tokens in 8 bits from a stage of the ring; `seen`: how many of them are visible
  __device__ __forceinline__ void quantized_unit(uint32_t stage, float ks, float vs, int seen, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float acc[kJ][4];
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
      const int chunk = D == 128 ? (t + 4 * j) ^ ((g & 1) << 2) : t;
      const uint4 lo = lds128(stage + g * D + chunk * 16), hi = lds128(stage + (g + 8) * D + chunk * 16);
      const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, b[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t ua = a[w] ^ 0x80808080u, ub = b[w] ^ 0x80808080u;
        mma16816<__half>(acc[j], codes_to_half2<0x4140>(ua), codes_to_half2<0x4140>(ub), codes_to_half2<0x4342>(ua),
                         codes_to_half2<0x4342>(ub), qh[j][w][0], qh[j][w][1]);
      }
    }
    const float s0 = ks * f0, s1 = ks * f1;
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = acc[0][i];
      if (kJ == 2) x += acc[kJ - 1][i];
      s[i] = x * ((i & 1) ? s1 : s0);
    }
    if (seen < kUnit) {
      if (g >= seen) s[0] = s[1] = -INFINITY;
      if (g + 8 >= seen) s[2] = s[3] = -INFINITY;
    }
    softmax(s);
    const uint32_t p0 = transpose8x8(pack_half2(s[0], s[1])), p1 = transpose8x8(pack_half2(s[2], s[3]));
    const uint32_t vbase = stage + kUnit * D;
    uint32_t v[4][kW];   // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 x channels (D / 8) g ..
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 2 * t + (e & 1) + (e >> 1) * 8;
      if constexpr (D == 128) {
        const uint4 x = lds128(vbase + row * D + ((g ^ (2 * t)) << 4));
        v[e][0] = x.x, v[e][1] = x.y, v[e][2] = x.z, v[e][3] = x.w;
      } else {
        const uint2 x = lds64(vbase + row * D + (((g >> 1) ^ t) << 4) + ((g & 1) << 3));
        v[e][0] = x.x, v[e][1] = x.y;
      }
    }
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      // the four channels of two neighbouring tokens side by side, then to fp16 pairs (token, next token)
      const uint32_t ab0 = __byte_perm(v[0][w], v[1][w], 0x5140) ^ 0x80808080u, ab1 = __byte_perm(v[0][w], v[1][w], 0x7362) ^ 0x80808080u;
      const uint32_t cd0 = __byte_perm(v[2][w], v[3][w], 0x5140) ^ 0x80808080u, cd1 = __byte_perm(v[2][w], v[3][w], 0x7362) ^ 0x80808080u;
      float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
      mma16816<__half>(x, codes_to_half2<0x4140>(ab0), codes_to_half2<0x4342>(ab0), codes_to_half2<0x4140>(cd0),
                       codes_to_half2<0x4342>(cd0), p0, p1);
      mma16816<__half>(y, codes_to_half2<0x4140>(ab1), codes_to_half2<0x4342>(ab1), codes_to_half2<0x4140>(cd1),
                       codes_to_half2<0x4342>(cd1), p0, p1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[2 * w][i] = fmaf(vs, x[i], o[2 * w][i]);
        o[2 * w + 1][i] = fmaf(vs, y[i], o[2 * w + 1][i]);
      }
    }
  }

  // Up to 16 open tokens in 16 bits, from global memory (L2: a request's open rows are few).  Hidden rows are never loaded: what
  // lies there (later tokens, leftovers) may be infinite.  bf16 probabilities have too few digits: value + what its rounding left.
  __device__ __forceinline__ void open_unit(const T* k, const T* v, const T* q_row, float scale_log2, int seen, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      uint4 a[2], b[2], q[2];
      a[0] = a[1] = b[0] = b[1] = q[0] = q[1] = make_uint4(0, 0, 0, 0);
      const int c = 16 * (t + 4 * j);
      if (g < seen) a[0] = *reinterpret_cast<const uint4*>(k + g * D + c), a[1] = *reinterpret_cast<const uint4*>(k + g * D + c + 8);
      if (g + 8 < seen) b[0] = *reinterpret_cast<const uint4*>(k + (g + 8) * D + c), b[1] = *reinterpret_cast<const uint4*>(k + (g + 8) * D + c + 8);
      if (q_row) q[0] = *reinterpret_cast<const uint4*>(q_row + c), q[1] = *reinterpret_cast<const uint4*>(q_row + c + 8);
      const uint32_t* wa = reinterpret_cast<const uint32_t*>(a);
      const uint32_t* wb = reinterpret_cast<const uint32_t*>(b);
      const uint32_t* wq = reinterpret_cast<const uint32_t*>(q);
#pragma unroll
      for (int w = 0; w < 4; ++w) mma16816<T>(acc, wa[2 * w], wb[2 * w], wa[2 * w + 1], wb[2 * w + 1], wq[2 * w], wq[2 * w + 1]);
    }
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = acc[i] * scale_log2;
    if (g >= seen) s[0] = s[1] = -INFINITY;
    if (g + 8 >= seen) s[2] = s[3] = -INFINITY;
    softmax(s);
    uint32_t p0, p1, r0 = 0, r1 = 0;
    if constexpr (std::is_same<T, __half>::value) {
      p0 = transpose8x8(pack_half2(s[0], s[1]));
      p1 = transpose8x8(pack_half2(s[2], s[3]));
    } else {
      const uint32_t a = pack_bf2(s[0], s[1]), b = pack_bf2(s[2], s[3]);
      auto lo = [](uint32_t w) { return __uint_as_float(w << 16); };
      auto hi = [](uint32_t w) { return __uint_as_float(w & 0xffff0000u); };
      p0 = transpose8x8(a);
      p1 = transpose8x8(b);
      r0 = transpose8x8(pack_bf2(s[0] - lo(a), s[1] - hi(a)));
      r1 = transpose8x8(pack_bf2(s[2] - lo(b), s[3] - hi(b)));
    }
#pragma unroll
    for (int c = 0; c < kW / 2; ++c) {   // eight channels at a time
      uint4 x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 2 * t + (e & 1) + (e >> 1) * 8;
        x[e] = row < seen ? *reinterpret_cast<const uint4*>(v + row * D + (D / 8) * g + 8 * c) : make_uint4(0, 0, 0, 0);
      }
      const uint32_t* a = reinterpret_cast<const uint32_t*>(&x[0]);
      const uint32_t* b = reinterpret_cast<const uint32_t*>(&x[1]);
      const uint32_t* d = reinterpret_cast<const uint32_t*>(&x[2]);
      const uint32_t* e = reinterpret_cast<const uint32_t*>(&x[3]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t a0 = __byte_perm(a[w], b[w], 0x5410), a1 = __byte_perm(a[w], b[w], 0x7632);
        const uint32_t a2 = __byte_perm(d[w], e[w], 0x5410), a3 = __byte_perm(d[w], e[w], 0x7632);
        mma16816<T>(o[4 * c + w], a0, a1, a2, a3, p0, p1);
        if constexpr (!std::is_same<T, __half>::value) mma16816<T>(o[4 * c + w], a0, a1, a2, a3, r0, r1);
      }
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) paged_attn_kernel(const PagedAttnParams p) {
  using S = Shape<D>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int s_t;
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int tiles = p.H * p.sub;       // tiles of eight heads per token
  pdl_wait();
  const int64_t total = (int64_t)p.unit_start[p.T] * tiles, run = run_units(total, gridDim.x);
  const int64_t u0 = blockIdx.x * run, u1 = min(u0 + run, total);
  if (u0 >= u1) return;
  for (int i = threadIdx.x; i < p.T; i += kThreads) {
    const int64_t a = (int64_t)p.unit_start[i] * tiles, b = (int64_t)p.unit_start[i + 1] * tiles;
    if (a <= u0 && u0 < b) s_t = i;
  }
  __syncthreads();
  int t = s_t;

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem + warp * S::kRing);
  float* s_scale = reinterpret_cast<float*>(smem + kWarps * S::kRing) + warp * S::kStages * 2;
  float* mine = reinterpret_cast<float*>(smem + warp * S::kRing);
  Tile<T, D> tile;

  int units = p.unit_start[t + 1] - p.unit_start[t];
  const int64_t base = (int64_t)p.unit_start[t] * tiles;
  int h = (int)((u0 - base) / units), j0 = (int)(u0 - base - (int64_t)h * units);
  for (int64_t u = u0; u < u1;) {
    const int n = (int)min((int64_t)(units - j0), u1 - u);    // units j0 .. j0 + n - 1 of tile (t, h)
    const int r = p.token_request[t], pos = p.positions[t], end = p.seq_lens[r];
    const int held = end >> p.bs_log2 << p.bs_log2, nq = min(pos + 1, held), nq_units = (nq + kUnit - 1) / kUnit;
    const int hk = h / p.sub, head0 = hk * p.group + (h - hk * p.sub) * kHeads, heads = min(kHeads, (hk + 1) * p.group - head0);
    const T* q_row = g < heads ? reinterpret_cast<const T*>(p.q) + t * p.q_st + (head0 + g) * p.q_sh : nullptr;
    const int* row_table = p.table + r * p.ld_table;
    const int mine_n = n > warp ? (n - warp + kWarps - 1) / kWarps : 0;   // this warp's units: j0 + warp + i * kWarps

    // block ids and scales of 32 of this warp's units at a time, one per lane
    int ids = -1;
    float kss = 0.f, vss = 0.f;
    auto issue = [&](int i) {
      if (i < mine_n) {
        if ((i & 31) == 0) {
          const int j = j0 + warp + (i + lane) * kWarps;
          ids = -1;
          kss = vss = __int_as_float(0x7fffffff);               // a block that is not in the pool: NaN
          if (i + lane < mine_n && j < nq_units) {
            const int blk = j * kUnit >> p.bs_log2;
            ids = blk < p.max_blocks ? row_table[blk] : -1;
            if (ids >= 0 && ids < p.num_blocks) {
              kss = p.k_scale[(int64_t)ids * p.H + hk];
              vss = p.v_scale[(int64_t)ids * p.H + hk];
            } else {
              ids = -1;
            }
          }
        }
        const int j = j0 + warp + i * kWarps, id = __shfl_sync(0xffffffffu, ids, i & 31);
        const float ks = __shfl_sync(0xffffffffu, kss, i & 31), vs = __shfl_sync(0xffffffffu, vss, i & 31);
        if (j < nq_units) {
          const int slot = i % S::kStages;
          const uint32_t dst = ring + slot * S::kStageBytes;
          const int64_t src = id < 0 ? 0 : (((int64_t)id * p.H + hk) << p.bs_log2) * D + ((j * kUnit) & ((1 << p.bs_log2) - 1)) * D;
          const int bytes = id < 0 ? 0 : 16;
#pragma unroll
          for (int e = 0; e < kUnit * D / 512; ++e) {
            const int at = e * 32 + lane;          // 16-byte chunk of the piece
            const int row = at / (D / 16), c = at % (D / 16);
            const int ck = D == 128 ? c ^ ((row & 1) << 2) : c, cv = D == 128 ? c ^ (((row >> 1) & 3) << 1) : c ^ ((row >> 1) & 3);
            cp_async16(dst + row * D + ck * 16, p.k_codes + src + at * 16, bytes);
            cp_async16(dst + kUnit * D + row * D + cv * 16, p.v_codes + src + at * 16, bytes);
          }
          if (lane == 0) {
            s_scale[2 * slot] = ks;
            s_scale[2 * slot + 1] = vs;
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    tile.reset();
#pragma unroll 1
    for (int i = 0; i < S::kStages - 1; ++i) issue(i);
    tile.load_q(q_row, p.scale_log2, lane);
#pragma unroll 1
    for (int i = 0; i < mine_n; ++i) {
      const int j = j0 + warp + i * kWarps;
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
      __syncwarp();
      if (j < nq_units) {
        const int slot = i % S::kStages;
        const float ks = s_scale[2 * slot], vs = s_scale[2 * slot + 1];
        tile.quantized_unit(ring + slot * S::kStageBytes, ks, vs, nq - j * kUnit, lane);
      } else {
        const int from = (j - nq_units) * kUnit;
        const int64_t at = ((((int64_t)r * p.H + hk) << p.bs_log2) + from) * D;
        tile.open_unit(reinterpret_cast<const T*>(p.tail_k) + at, reinterpret_cast<const T*>(p.tail_v) + at, q_row, p.scale_log2,
                       pos + 1 - nq - from, lane);
      }
      __syncwarp();
      issue(i + S::kStages - 1);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();

    // ---- the warps' results meet: [8 heads][D + 4], maxima, sums per warp, over its ring ----
    const float l0 = sum_over_g(tile.l0), l1 = sum_over_g(tile.l1);
    if (g == 0) {
      mine[kHeads * S::kPitch + 2 * t4] = tile.m0;
      mine[kHeads * S::kPitch + 2 * t4 + 1] = tile.m1;
      mine[kHeads * S::kPitch + kHeads + 2 * t4] = l0;
      mine[kHeads * S::kPitch + kHeads + 2 * t4 + 1] = l1;
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int c = (D / 8) * g + 2 * i;
      *reinterpret_cast<float2*>(mine + (2 * t4) * S::kPitch + c) = make_float2(tile.o[i][0], tile.o[i][2]);
      *reinterpret_cast<float2*>(mine + (2 * t4 + 1) * S::kPitch + c) = make_float2(tile.o[i][1], tile.o[i][3]);
    }
    __syncthreads();
    {
      const int head = warp;   // eight warps, eight heads
      const float* all = reinterpret_cast<const float*>(smem);
      constexpr int kStep = S::kRing / 4;
      const int live = min(n, kWarps);
      float top = -INFINITY, sum = 0.f, x[D / 32];
#pragma unroll
      for (int c = 0; c < D / 32; ++c) x[c] = 0.f;
      for (int w = 0; w < live; ++w) top = fmaxf(top, all[w * kStep + kHeads * S::kPitch + head]);
      for (int w = 0; w < live; ++w) {
        const float m = all[w * kStep + kHeads * S::kPitch + head];
        const float f = m == top ? 1.f : ex2(m - top);
        sum = fmaf(f, all[w * kStep + kHeads * S::kPitch + kHeads + head], sum);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) x[c] = fmaf(f, all[w * kStep + head * S::kPitch + 32 * c + lane], x[c]);
      }
      if (n == units) {
        if (head < heads) {
          T* out = reinterpret_cast<T*>(p.out) + t * p.o_st + (head0 + head) * p.o_sh;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) out[32 * c + lane] = from_float<T>(x[c] / sum);
        }
      } else {   // slot 0: a tile that thread blocks before this one began; slot 1: one that this one begins
        float* part = p.parts + ((int64_t)blockIdx.x * 2 + (j0 == 0 ? 1 : 0)) * S::kPartFloats;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) part[head * D + 32 * c + lane] = x[c];
        if (lane == 0) {
          part[kHeads * D + head] = top;
          part[kHeads * D + kHeads + head] = sum;
        }
      }
    }
    __syncthreads();
    u += n;
    j0 = 0;
    if (++h == tiles && u < u1) {
      h = 0;
      do {
        ++t;
        units = p.unit_start[t + 1] - p.unit_start[t];
      } while (units == 0);
    }
  }
}

// Tiles that span thread blocks: their parts, in order.  One thread block per tile, one warp per head.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) paged_merge_kernel(const PagedAttnParams p, int blocks) {
  using S = Shape<D>;
  pdl_wait();
  const int tiles = p.H * p.sub, t = blockIdx.x / tiles, h = blockIdx.x - t * tiles;
  const int64_t total = (int64_t)p.unit_start[p.T] * tiles, run = run_units(total, blocks);
  const int units = p.unit_start[t + 1] - p.unit_start[t];
  const int64_t a = (int64_t)p.unit_start[t] * tiles + (int64_t)h * units;
  const int first = (int)(a / run), last = units ? (int)((a + units - 1) / run) : first;
  if (first == last) return;
  const int head = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = h / p.sub, head0 = hk * p.group + (h - hk * p.sub) * kHeads, heads = min(kHeads, (hk + 1) * p.group - head0);
  if (head >= heads) return;
  auto part_of = [&](int b) { return p.parts + ((int64_t)b * 2 + (b == first ? 1 : 0)) * S::kPartFloats; };
  float top = -INFINITY;
  for (int b = first + lane; b <= last; b += 32) top = fmaxf(top, part_of(b)[kHeads * D + head]);
  top = warp_max(top);
  float sum = 0.f, x[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) x[c] = 0.f;
#pragma unroll 4
  for (int b = first; b <= last; ++b) {
    const float* part = part_of(b);
    const float m = part[kHeads * D + head], f = m == top ? 1.f : ex2(m - top);
    sum = fmaf(f, part[kHeads * D + kHeads + head], sum);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) x[c] = fmaf(f, part[head * D + 32 * c + lane], x[c]);
  }
  T* out = reinterpret_cast<T*>(p.out) + t * p.o_st + (head0 + head) * p.o_sh;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) out[32 * c + lane] = from_float<T>(x[c] / sum);
}

int attn_blocks() { return sm_count(); }

}  // namespace
}  // namespace pare

extern "C" {

using namespace pare;
using namespace pare::paged;

size_t pare_paged_attn_workspace_bytes(int D) {
  if (D != 64 && D != 128) return 0;
  return (size_t)attn_blocks() * 2 * (kHeads * D + 2 * kHeads) * sizeof(float);
}

int pare_paged_attn(const void* q, int dtype, int64_t q_stride_t, int64_t q_stride_h, const void* step, int R, int T, int block_size,
                    const int32_t* block_table, int64_t ld_table, int max_blocks, const int8_t* k_codes, const int8_t* v_codes,
                    const float* k_scale, const float* v_scale, const void* tail_k, const void* tail_v, int num_blocks, int Hq, int H,
                    int D, void* out, int64_t out_stride_t, int64_t out_stride_h, float softmax_scale, void* workspace,
                    size_t workspace_bytes, void* stream) {
  PARE_REQUIRE(step && block_table && k_codes && v_codes && k_scale && v_scale && tail_k && tail_v, PARE_ERR_SHAPE);
  PARE_REQUIRE(R > 0 && R <= kMaxRequests && T >= 0 && num_blocks > 0 && H > 0 && Hq > 0 && Hq % H == 0 && max_blocks > 0 &&
                   ld_table >= max_blocks,
               PARE_ERR_SHAPE);
  PARE_REQUIRE(dtype == PARE_F16 || dtype == PARE_BF16, PARE_ERR_DTYPE);
  PARE_REQUIRE(block_size_ok(block_size) && (D == 64 || D == 128) && T <= kMaxQueryTokens, PARE_ERR_UNSUPPORTED);
  if (T == 0) return PARE_OK;
  PARE_REQUIRE(q && out, PARE_ERR_SHAPE);
  PARE_REQUIRE(aligned16(q) && (q_stride_t | q_stride_h) % 8 == 0 && aligned16(step) && aligned16(k_codes) && aligned16(v_codes) &&
                   aligned16(tail_k) && aligned16(tail_v) && aligned16(workspace),
               PARE_ERR_ALIGN);
  PARE_REQUIRE(workspace && workspace_bytes >= pare_paged_attn_workspace_bytes(D), PARE_ERR_WORKSPACE);
  const int group = Hq / H, sub = (group + kHeads - 1) / kHeads;
  PARE_REQUIRE((int64_t)T * H * sub < (int64_t)1 << 31, PARE_ERR_UNSUPPORTED);
  const StepLayout s(R, T, block_size);
  const int* w = reinterpret_cast<const int*>(step);
  PagedAttnParams p{q, q_stride_t, q_stride_h, out, out_stride_t, out_stride_h, w + s.token_request, w + s.positions, w + s.seq_lens,
                    w + s.unit_start, block_table, ld_table, k_codes, v_codes, k_scale, v_scale, tail_k, tail_v,
                    reinterpret_cast<float*>(workspace), softmax_scale * kLog2e, T, R, H, group, sub,
                    block_size == 16 ? 4 : block_size == 32 ? 5 : 6, num_blocks, max_blocks};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int blocks = attn_blocks();
  auto go = [&](auto kern, auto merge, size_t smem) {
    if (!ensure_smem_attr(reinterpret_cast<const void*>(kern), (int)smem)) return (int)PARE_ERR_CUDA;
    int rc = launch_pdl(kern, dim3(blocks), dim3(kThreads), smem, st, p);
    if (rc != PARE_OK) return rc;
    rc = launch_pdl(merge, dim3(T * H * sub), dim3(kThreads), 0, st, p, blocks);
    return rc != PARE_OK ? rc : launch_status();
  };
  if (dtype == PARE_F16)
    return D == 64 ? go(paged_attn_kernel<__half, 64>, paged_merge_kernel<__half, 64>, Shape<64>::kSmem)
                   : go(paged_attn_kernel<__half, 128>, paged_merge_kernel<__half, 128>, Shape<128>::kSmem);
  return D == 64 ? go(paged_attn_kernel<__nv_bfloat16, 64>, paged_merge_kernel<__nv_bfloat16, 64>, Shape<64>::kSmem)
                 : go(paged_attn_kernel<__nv_bfloat16, 128>, paged_merge_kernel<__nv_bfloat16, 128>, Shape<128>::kSmem);
}

}  // extern "C"
