// Attention of new tokens' queries over the paged 8-bit KV cache (paged_cache.cu), sm_100a.
//
//   out[t][hq] = softmax_j(q[t][hq] . K_j * scale) V_j over the positions j <= position of token t in its request,
// K_j, V_j = code * scale of the block for blocks that are full, the open rows (16-bit) for the rest.  Query head hq reads KV head
// hq / (Hq / H); up to eight query heads that share a KV head sit in the eight columns of the warp-level MMA, so the cache is
// read once for all of them.  The reference leaves attention to its caller (pare/kv_cache.py:183-186).
//
// Mathematics.  Codes are integers of at most 127: exact in fp16, so S = code . q and O' = code^T . P run on fp16 operands with fp32
// sums, and the block's scales multiply S and O' outside (one number per 16 tokens).  q is fp16 as it is, or bf16 times a power of
// two per head that puts its largest magnitude into [256, 512), where that is 2^-112 or more: every bf16 value within 2^-22 of that is
// exact, smaller ones are within 2^-33 of the largest.  Softmax runs online: a reference value per head which only moves when a score
// passes it by more than 2^kSlack (one vote per 16 tokens instead of a reduction); probabilities are kept times 2^kBias of that, so those
// down to 2^-18 of the reference are normal fp16 numbers and none passes 2^15.  Their sum is taken before they become two fp16 numbers
// each (those of open rows two of the rows' type).  Values above 2^112 / tokens may overflow the sums.
//
// Work.  Units of 16 tokens of one (token, group of heads), counted by the step's tables; each WARP takes one contiguous run of
// units, all runs equally long, so ragged lengths balance by themselves and the host needs to know none of them.  A warp feeds
// itself through a ring of its own (cp.async, no barrier between warps) and waits for nobody.  Tiles that span warps leave their
// parts in the workspace for a second kernel.  Nothing in the workspace outlives the call, no counters: calls on any streams and
// replays of any graphs do not meet there.
//
// A tile's eight columns are heads of one token, or, where a step has more rows than requests, heads of up to eight tokens of a request.
//
// Bound: the cache's bytes for long contexts, instructions (conversion of codes: 0.61 of the issue slots there, 0.50 for ragged requests) close
// behind; one sequence is a chain of dependent reads.  Both launches, of many in a graph, and how much of that the second one adds:
// 16 x 32768 tokens, 28 / 4 heads 100 us (540 MB: 0.82 of the copy rate), 8; 64 requests of up to 3600 tokens, 32 / 8 heads, bf16 62 us (0.65), 7;
// one of 4096 tokens 13.3 us, 4.7; three tokens of 12 requests over 1500 on average, D = 64 20.4 us, 6.4.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace pare {
namespace {

using namespace paged;

constexpr int kHeads = 8;                  // query heads of a tile (MMA columns)
constexpr int kWarpsPerSm = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBias = 4.f, kSlack = 11.f;
constexpr float kLowest = -3e38f;          // a reference below every score, and finite
constexpr int kMinRun = 3;                 // units of a warp's run at least

template <int D>
struct Shape {
  static constexpr int kStageBytes = 2 * kUnit * D;           // codes of 16 tokens: keys, then values
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kChunks = kUnit * D / 512;             // 16-byte chunks of a unit's keys (or values) per lane
  static constexpr int kRing = kStages * kStageBytes;         // per warp
  // An SM's warps in one thread block: of two, one runs ahead and leaves the other alone at the end (16 x 32768 tokens: 76 and 88 us, 86
  // with one).  Not for short heads, whose calls are short.
  static constexpr int kWarps = D == 128 ? kWarpsPerSm : kWarpsPerSm / 2, kThreads = kWarps * 32, kBlocksPerSm = kWarpsPerSm / kWarps;
  static constexpr size_t kSmem = (size_t)kWarps * kRing;
  static constexpr int kPartFloats = kHeads * D + 2 * kHeads; // a part in the workspace: O as the lanes hold it, maxima, sums
};

struct PagedAttnParams {
  const void* q;
  int64_t q_st, q_sh;
  void* out;
  int64_t o_st, o_sh;
  const int4* info;          // [T] request, position, length after the step, number in the request's rows
  const int* unit_start;     // [T + 1], of tiles of `pack` tokens
  const int* table;
  int64_t ld_table;
  const int8_t* k_codes;
  const int8_t* v_codes;
  const float* k_scale;
  const float* v_scale;
  const void* tail_k;
  const void* tail_v;
  float* parts;              // [warp][2]: of a tile that warps before it began, of one that it begins
  float scale_log2;
  int T, R, H, group, sub, bs_log2, num_blocks, max_blocks;   // sub: tiles of eight heads per KV head
  int pack, per_group;       // tokens of a tile at most, 256 / group rounded up
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
// A product that begins a sum (mma16816 adds to one)
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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

// Which of a tile's tokens a column belongs to: c / group for the groups that share tiles
template <bool PACKED>
__device__ __forceinline__ int token_of(const PagedAttnParams& p, int c) {
  return PACKED ? c * p.per_group >> 8 : 0;
}

// Where a column of a tile goes, nullptr if it is nobody's.  A tile's columns are the `heads` heads of its first token, of the next, ..;
// `earlier` tokens before the last one, which is token t.
template <typename T, bool PACKED>
__device__ __forceinline__ T* column_out(const PagedAttnParams& p, int t, int c, int earlier, int head0, int heads) {
  const int token = token_of<PACKED>(p, c), head = c - token * p.group;
  return token <= earlier && head < heads ? reinterpret_cast<T*>(p.out) + (int64_t)(t - earlier + token) * p.o_st + (int64_t)(head0 + head) * p.o_sh
                                          : nullptr;
}

// Units of a run: equal shares, but not so few that the parts outweigh the work.
__device__ __forceinline__ int64_t run_units(int64_t total, int warps) {
  const int64_t each = (total + warps - 1) / warps;
  return each < kMinRun ? kMinRun : each;
}

template <typename T, int D, bool PACKED>
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
    m0 = m1 = kLowest;
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

  // Sums of products of tokens g, g + 8 x heads 2 t, 2 t + 1, their factors to scores in base 2, and how many of the tokens are visible to
  // those heads (`least`: to any) -> probabilities in place
  __device__ __forceinline__ void softmax(float (&s)[4], float s0, float s1, int least, int seen0, int seen1, int g) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fmaf(s[i], (i & 1) ? s1 : s0, (i & 1) ? kBias - m1 : kBias - m0);
    if (least < kUnit) {
      if (g >= seen0) x[0] = -INFINITY;
      if (g >= seen1) x[1] = -INFINITY;
      if (g + 8 >= seen0) x[2] = -INFINITY;
      if (g + 8 >= seen1) x[3] = -INFINITY;
    }
    if (__any_sync(0xffffffffu, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) > kBias + kSlack)) {
      // the reference moves up to the largest score
      float t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = x[i] == -INFINITY ? -INFINITY : s[i] * ((i & 1) ? s1 : s0);
      const float n0 = fmaxf(m0, max_over_g(fmaxf(t[0], t[2]))), n1 = fmaxf(m1, max_over_g(fmaxf(t[1], t[3])));
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
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (x[i] != -INFINITY) x[i] = fmaf(s[i], (i & 1) ? s1 : s0, (i & 1) ? kBias - m1 : kBias - m0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = ex2(x[i]);
    l0 += s[0] + s[2];
    l1 += s[1] + s[3];
  }

  // 16 tokens in 8 bits from a stage of the ring; `least`, `seen0`, `seen1`: how many of them are visible
  __device__ __forceinline__ void quantized_unit(uint32_t stage, float ks, float vs, int least, int seen0, int seen1, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float acc[kJ][4];
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const int chunk = D == 128 ? (t + 4 * j) ^ ((g & 1) << 2) : t;
      const uint4 lo = lds128(stage + g * D + chunk * 16), hi = lds128(stage + (g + 8) * D + chunk * 16);
      const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, b[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t ua = a[w] ^ 0x80808080u, ub = b[w] ^ 0x80808080u;
        const uint32_t c0 = codes_to_half2<0x4140>(ua), c1 = codes_to_half2<0x4140>(ub), c2 = codes_to_half2<0x4342>(ua), c3 = codes_to_half2<0x4342>(ub);
        if (w == 0) mma16816_first(acc[j], c0, c1, c2, c3, qh[j][w][0], qh[j][w][1]);
        else mma16816<__half>(acc[j], c0, c1, c2, c3, qh[j][w][0], qh[j][w][1]);
      }
    }
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = kJ == 2 ? acc[0][i] + acc[kJ - 1][i] : acc[0][i];
    softmax(s, ks * f0, ks * f1, least, seen0, seen1, g);
    // a block that a head does not see at all may have a scale that is not finite
    const float vs0 = PACKED && seen0 <= 0 ? 0.f : vs, vs1 = PACKED && seen1 <= 0 ? 0.f : vs;
    // Rounding a probability to fp16 is off by up to 2^-11 of it, which changes a tenth of bf16 results by a step and is as much as the
    // rounding of an fp16 result.  So it is two numbers, the second what the first left: off by 2^-22.
    const uint32_t h0 = pack_half2(s[0], s[1]), h1 = pack_half2(s[2], s[3]), p0 = transpose8x8(h0), p1 = transpose8x8(h1);
    const float2 e0 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), e1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
    const uint32_t r0 = transpose8x8(pack_half2(s[0] - e0.x, s[1] - e0.y)), r1 = transpose8x8(pack_half2(s[2] - e1.x, s[3] - e1.y));
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
      const uint32_t a[4] = {codes_to_half2<0x4140>(ab0), codes_to_half2<0x4342>(ab0), codes_to_half2<0x4140>(cd0), codes_to_half2<0x4342>(cd0)};
      const uint32_t b[4] = {codes_to_half2<0x4140>(ab1), codes_to_half2<0x4342>(ab1), codes_to_half2<0x4140>(cd1), codes_to_half2<0x4342>(cd1)};
      float x[4], y[4];
      mma16816_first(x, a[0], a[1], a[2], a[3], p0, p1);
      mma16816_first(y, b[0], b[1], b[2], b[3], p0, p1);
      mma16816<__half>(x, a[0], a[1], a[2], a[3], r0, r1);
      mma16816<__half>(y, b[0], b[1], b[2], b[3], r0, r1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[2 * w][i] = fmaf((i & 1) ? vs1 : vs0, x[i], o[2 * w][i]);
        o[2 * w + 1][i] = fmaf((i & 1) ? vs1 : vs0, y[i], o[2 * w + 1][i]);
      }
    }
  }

  // Up to 16 open tokens in 16 bits: the keys in one stage of the ring, the values in another.  Rows that are hidden to a head (later
  // tokens, leftovers) were not loaded, they are zeros: what lies there may be infinite.  Values that some of the heads see (`most`
  // rows are visible to any, `least` to all; v_rows: where they are) are added one by one.  Probabilities in two terms, in the rows' type.
  __device__ __forceinline__ void open_unit(uint32_t stage_k, uint32_t stage_v, const T* q_row, const T* v_rows, float scale_log2, int least, int most,
                                            int seen0, int seen1, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      uint4 a[2], b[2], q[2];
      q[0] = q[1] = make_uint4(0, 0, 0, 0);
      const int c = 16 * (t + 4 * j);
      if (q_row) q[0] = *reinterpret_cast<const uint4*>(q_row + c), q[1] = *reinterpret_cast<const uint4*>(q_row + c + 8);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t at = stage_k + (((c / 8 + e) ^ (g & 1)) << 4);
        a[e] = lds128(at + g * 2 * D);
        b[e] = lds128(at + (g + 8) * 2 * D);
      }
      const uint32_t* wa = reinterpret_cast<const uint32_t*>(a);
      const uint32_t* wb = reinterpret_cast<const uint32_t*>(b);
      const uint32_t* wq = reinterpret_cast<const uint32_t*>(q);
#pragma unroll
      for (int w = 0; w < 4; ++w) mma16816<T>(acc, wa[2 * w], wb[2 * w], wa[2 * w + 1], wb[2 * w + 1], wq[2 * w], wq[2 * w + 1]);
    }
    float s[4] = {acc[0], acc[1], acc[2], acc[3]};
    softmax(s, scale_log2, scale_log2, least, seen0, seen1, g);
#pragma unroll 1
    for (int row = PACKED ? max(least, 0) : kUnit; row < min(most, kUnit); ++row) {
      const float y0 = __shfl_sync(0xffffffffu, row < 8 ? s[0] : s[2], 4 * (row & 7) + t), y1 = __shfl_sync(0xffffffffu, row < 8 ? s[1] : s[3], 4 * (row & 7) + t);
      const T* v = v_rows + row * D + (D / 8) * g;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint32_t two = *reinterpret_cast<const uint32_t*>(v + 2 * i);
        const T* e = reinterpret_cast<const T*>(&two);
        if (row < seen0) o[i][0] = fmaf(y0, to_float<T>(e[0]), o[i][0]), o[i][2] = fmaf(y0, to_float<T>(e[1]), o[i][2]);
        if (row < seen1) o[i][1] = fmaf(y1, to_float<T>(e[0]), o[i][1]), o[i][3] = fmaf(y1, to_float<T>(e[1]), o[i][3]);
      }
    }
    uint32_t p0, p1, r0, r1;
    if constexpr (std::is_same<T, __half>::value) {
      const uint32_t a = pack_half2(s[0], s[1]), b = pack_half2(s[2], s[3]);
      const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a)), fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
      p0 = transpose8x8(a);
      p1 = transpose8x8(b);
      r0 = transpose8x8(pack_half2(s[0] - fa.x, s[1] - fa.y));
      r1 = transpose8x8(pack_half2(s[2] - fb.x, s[3] - fb.y));
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
      for (int e = 0; e < 4; ++e) x[e] = lds128(stage_v + (2 * t + (e & 1) + (e >> 1) * 8) * 2 * D + ((((D / 64) * g + c) ^ open_value_swizzle(t)) << 4));
      const uint32_t* a = reinterpret_cast<const uint32_t*>(&x[0]);
      const uint32_t* b = reinterpret_cast<const uint32_t*>(&x[1]);
      const uint32_t* d = reinterpret_cast<const uint32_t*>(&x[2]);
      const uint32_t* e = reinterpret_cast<const uint32_t*>(&x[3]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t a0 = __byte_perm(a[w], b[w], 0x5410), a1 = __byte_perm(a[w], b[w], 0x7632);
        const uint32_t a2 = __byte_perm(d[w], e[w], 0x5410), a3 = __byte_perm(d[w], e[w], 0x7632);
        mma16816<T>(o[4 * c + w], a0, a1, a2, a3, p0, p1);
        mma16816<T>(o[4 * c + w], a0, a1, a2, a3, r0, r1);
      }
    }
  }

  // 16-byte chunks of a row of open values are moved by this (t: half the row's number modulo 4), so that the eight lanes of a
  // shared-memory phase (two g, four t) meet eight different banks
  __device__ static __forceinline__ int open_value_swizzle(int t) { return D == 128 ? (t & 1) | ((t >> 1) << 2) : 2 * t; }
};

template <typename T, int D, bool PACKED>
__global__ void __launch_bounds__(Shape<D>::kThreads, Shape<D>::kBlocksPerSm) paged_attn_kernel(const PagedAttnParams p) {
  using S = Shape<D>;
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int tiles = p.H * p.sub;       // tiles of eight heads per token
  const int me = warp * gridDim.x + blockIdx.x;      // a few runs spread over all SMs
  pdl_wait();
  pdl_launch_dependents();      // not before: the second launch reads the step before it waits for this one
  // The last token that begins at or before this run: 32 candidates a round, the first round together with the number of units
  const int all = p.unit_start[p.T], spread = (p.T + 31) / 32;
  const int mark = lane * spread < p.T ? p.unit_start[lane * spread] : 0x7fffffff;
  const int64_t total = (int64_t)all * tiles, run = run_units(total, gridDim.x * S::kWarps);
  const int64_t u0 = me * run, u1 = min(u0 + run, total);
  if (u0 >= u1) return;
  const int x = (int)(u0 / tiles), k0 = 31 - __clz(__ballot_sync(0xffffffffu, mark <= x));
  int t = k0 * spread;
  for (int n = min(spread, p.T - t); n > 1;) {
    const int step = (n + 31) / 32, at = lane * step;
    const int k = 31 - __clz(__ballot_sync(0xffffffffu, at < n && p.unit_start[t + min(at, n - 1)] <= x));
    t += k * step;
    n = min(step, n - k * step);
  }

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem + warp * S::kRing);
  Tile<T, D, PACKED> tile;

  // Where this lane's 16-byte chunks of a unit go in a stage: chunk e * 32 + lane of the keys at at_k + 512 e, of the values at
  // at_v[e & 1] + 512 e (the pattern that spreads rows over banks repeats after two rounds)
  uint32_t at_k, at_v[2];
  {
    const int row = lane / (D / 16), c = lane % (D / 16);
    at_k = row * D + (D == 128 ? c ^ ((row & 1) << 2) : c) * 16;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = row + e * (512 / D);
      at_v[e] = kUnit * D + row * D + (D == 128 ? c ^ (((r >> 1) & 3) << 1) : c ^ ((r >> 1) & 3)) * 16;
    }
  }

  int first_unit = p.unit_start[t], units = p.unit_start[t + 1] - first_unit;
  int4 info = p.info[t];
  const int64_t base = (int64_t)first_unit * tiles;
  int h = (int)((u0 - base) / units), j0 = (int)(u0 - base - (int64_t)h * units);
  for (int64_t u = u0; u < u1;) {
    const int n = (int)min((int64_t)(units - j0), u1 - u);    // units j0 .. j0 + n - 1 of tile (t, h)
    const int r = info.x, pos = info.y, end = info.z;
    const int held = end >> p.bs_log2 << p.bs_log2, nq = min(pos + 1, held), nq_units = (nq + kUnit - 1) / kUnit;
    const int hk = h / p.sub, head0 = hk * p.group + (h - hk * p.sub) * kHeads, heads = min(kHeads, (hk + 1) * p.group - head0);
    const int earlier = PACKED ? info.w & (p.pack - 1) : 0;                // tokens of the tile before its last one, t
    const int g_token = token_of<PACKED>(p, g), g_head = g - g_token * p.group;
    // how many tokens the columns 2 t4, 2 t4 + 1 see less than that one
    const int behind0 = PACKED ? earlier - token_of<PACKED>(p, 2 * t4) : 0, behind1 = PACKED ? earlier - token_of<PACKED>(p, 2 * t4 + 1) : 0;
    const T* q_row = g_token <= earlier && g_head < heads
                         ? reinterpret_cast<const T*>(p.q) + (t - earlier + g_token) * p.q_st + (head0 + g_head) * p.q_sh : nullptr;
    const int* row_table = p.table + r * p.ld_table;
    const int n8 = max(0, min(n, nq_units - j0));             // units in 8 bits, then units of open rows: two entries of the ring each
    const int entries = n8 + 2 * (n - n8);

    // Block ids and scales of 32 units at a time, one unit per lane.  Loads run ahead by the depth of the ring, so the scales of
    // the next 32 wait in registers of their own.
    int ids = -1, slot_in = 0;
    float ks_next = 0.f, vs_next = 0.f, kss = 0.f, vss = 0.f;
    auto issue = [&](int i) {
      if (i < n8) {
        if ((i & 31) == 0) {
          ids = -1;
          ks_next = vs_next = __int_as_float(0x7fffffff);       // a block that is not in the pool: NaN
          if (i + lane < n8) {
            const int blk = (j0 + i + lane) * kUnit >> p.bs_log2;
            ids = blk < p.max_blocks ? row_table[blk] : -1;
            if (ids < 0 || ids >= p.num_blocks) ids = -1;
          }
          if (ids >= 0) {
            ks_next = p.k_scale[(int64_t)ids * p.H + hk];
            vs_next = p.v_scale[(int64_t)ids * p.H + hk];
          }
        }
        const int id = __shfl_sync(0xffffffffu, ids, i & 31);
        const uint32_t dst = ring + slot_in * S::kStageBytes;
        const int64_t src = id < 0 ? 0 : ((((int64_t)id * p.H + hk) << p.bs_log2) + (((j0 + i) * kUnit) & ((1 << p.bs_log2) - 1))) * D;
        const int bytes = id < 0 ? 0 : 16;
        const int8_t* sk = p.k_codes + src + lane * 16;
        const int8_t* sv = p.v_codes + src + lane * 16;
#pragma unroll
        for (int e = 0; e < S::kChunks; ++e) cp_async16(dst + at_k + e * 512, sk + e * 512, bytes);
#pragma unroll
        for (int e = 0; e < S::kChunks; ++e) cp_async16(dst + at_v[e & 1] + e * 512, sv + e * 512, bytes);
      } else if (i < entries) {
        const int from = (j0 + n8 - nq_units + (i - n8) / 2) * kUnit;      // first row
        const bool values = (i - n8) & 1;
        const int seen = pos + 1 - nq - from - (values ? earlier : 0);     // rows visible to any head (keys), to all (values)
        const T* src = reinterpret_cast<const T*>(values ? p.tail_v : p.tail_k) + ((((int64_t)r * p.H + hk) << p.bs_log2) + from) * D;
        const uint32_t dst = ring + slot_in * S::kStageBytes;
#pragma unroll 1
        for (int e = 0; e < 2 * S::kChunks; ++e) {
          const int row = (e * 32 + lane) / (D / 8), c = (e * 32 + lane) % (D / 8);
          const int to = c ^ (values ? Tile<T, D, PACKED>::open_value_swizzle((row >> 1) & 3) : row & 1);
          const bool there = row < seen;
          cp_async16(dst + row * 2 * D + to * 16, there ? src + row * D + c * 8 : src, there ? 16 : 0);
        }
      }
      if (++slot_in == S::kStages) slot_in = 0;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    tile.reset();
#pragma unroll 1
    for (int i = 0; i < S::kStages - 1; ++i) issue(i);
    tile.load_q(q_row, p.scale_log2, lane);
    int slot = 0;
#pragma unroll 1
    for (int i = 0; i < n8; ++i) {
      if ((i & 31) == 0) kss = ks_next, vss = vs_next;
      const float ks = __shfl_sync(0xffffffffu, kss, i & 31), vs = __shfl_sync(0xffffffffu, vss, i & 31);
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
      __syncwarp();
      const int seen = pos + 1 - (j0 + i) * kUnit;
      tile.quantized_unit(ring + slot * S::kStageBytes, ks, vs, seen - earlier, seen - behind0, seen - behind1, lane);
      if (++slot == S::kStages) slot = 0;
      __syncwarp();
      issue(i + S::kStages - 1);
    }
#pragma unroll 1
    for (int i = n8; i < entries; i += 2) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 3) : "memory");
      __syncwarp();
      const int next = slot + 1 == S::kStages ? 0 : slot + 1;
      const int from = (j0 + n8 - nq_units + (i - n8) / 2) * kUnit, seen = pos + 1 - nq - from;
      tile.open_unit(ring + slot * S::kStageBytes, ring + next * S::kStageBytes, q_row,
                     reinterpret_cast<const T*>(p.tail_v) + ((((int64_t)r * p.H + hk) << p.bs_log2) + from) * D, p.scale_log2, seen - earlier, seen,
                     seen - behind0, seen - behind1, lane);
      slot = next + 1 == S::kStages ? 0 : next + 1;
      __syncwarp();
      issue(i + S::kStages - 1);
      issue(i + S::kStages);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();

    const float l0 = sum_over_g(tile.l0), l1 = sum_over_g(tile.l1);
    if (n == units) {
      const float y0 = 1.f / l0, y1 = 1.f / l1;
      T* out0 = column_out<T, PACKED>(p, t, 2 * t4, earlier, head0, heads);
      T* out1 = column_out<T, PACKED>(p, t, 2 * t4 + 1, earlier, head0, heads);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const int c = (D / 8) * g + 2 * i;
        if (out0) out0[c] = from_float<T>(tile.o[i][0] * y0), out0[c + 1] = from_float<T>(tile.o[i][2] * y0);
        if (out1) out1[c] = from_float<T>(tile.o[i][1] * y1), out1[c + 1] = from_float<T>(tile.o[i][3] * y1);
      }
    } else {
      float* part = p.parts + ((int64_t)me * 2 + (j0 == 0 ? 1 : 0)) * S::kPartFloats;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        reinterpret_cast<float4*>(part)[i * 32 + lane] = make_float4(tile.o[i][0], tile.o[i][1], tile.o[i][2], tile.o[i][3]);
      if (g == 0) {
        *reinterpret_cast<float2*>(part + kHeads * D + 2 * t4) = make_float2(tile.m0, tile.m1);
        *reinterpret_cast<float2*>(part + kHeads * D + kHeads + 2 * t4) = make_float2(l0, l1);
      }
    }
    u += n;
    j0 = 0;
    if (++h == tiles && u < u1) {
      h = 0;
      do {
        ++t;
        first_unit += units;
        units = p.unit_start[t + 1] - first_unit;
      } while (units == 0);
      info = p.info[t];
    }
  }
}

// Tiles that span warps.  A warp takes one piece of a tile's O (float4 per lane as the attention's lanes held it: channels
// (D / 8) g + 2 i, + 1 x heads 2 t, 2 t + 1).  Many tiles have few parts each, or most of them (one
// far longer than the others is added up by one warp a piece): a thread block per tile, a warp per piece.  Few tiles have
// many (one sequence: 86): GROUPS warps share a piece, each every GROUPS-th part, and are added up in order.  A warp alone gets
// through one instruction in about eight cycles, so what is serial counts: 8 tiles of 4096 tokens, both kernels, 22.7 / 15.8 / 13.1 / 12.7 us
// with 2 / 4 / 8 / 16 groups (six parts in flight and the step read before the wait have saved another 0.8 us since); 64 tiles of 32768
// tokens 101 / 99 / 99 / 106 us, 108 with one.
template <typename T, int D, int GROUPS, bool PACKED>
__global__ void __launch_bounds__(GROUPS > 1 ? GROUPS * 32 : D * 2) paged_merge_kernel(const PagedAttnParams p, int warps) {
  using S = Shape<D>;
  constexpr int kFlight = GROUPS == 16 ? 6 : 4;     // parts in flight per warp
  __shared__ float4 s_o[GROUPS][32], s_ml[GROUPS][32];
  const int tiles = p.H * p.sub, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int group = GROUPS > 1 ? warp : 0, piece = GROUPS > 1 ? blockIdx.y : warp;
  // The step was complete before the first launch let this one begin; its parts are there, and its readers of `out` gone, after the wait.
  bool waited = false;
  const int64_t total = (int64_t)p.unit_start[p.T] * tiles, run = run_units(total, warps);
  auto run_of = [&](int64_t u) { return total >> 32 ? (int)(u / run) : (int)((uint32_t)u / (uint32_t)run); };
  for (int job = blockIdx.x; job < p.T * tiles; job += gridDim.x) {
    const int t = job / tiles, h = job - t * tiles;
    const int first_unit = p.unit_start[t], units = p.unit_start[t + 1] - first_unit;
    const int64_t a = (int64_t)first_unit * tiles + (int64_t)h * units;
    const int first = run_of(a), last = units ? run_of(a + units - 1) : first;
    if (first == last) continue;
    if (!waited) {
      waited = true;
      pdl_wait();
    }
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float2 top = make_float2(-INFINITY, -INFINITY), l = make_float2(0.f, 0.f);
    auto add = [&](const float2& m, const float2& s, const float4& x) {
      const float n0 = fmaxf(top.x, m.x), n1 = fmaxf(top.y, m.y);
      const float a0 = n0 == top.x ? 1.f : ex2(top.x - n0), a1 = n1 == top.y ? 1.f : ex2(top.y - n1);
      const float f0 = n0 == m.x ? 1.f : ex2(m.x - n0), f1 = n1 == m.y ? 1.f : ex2(m.y - n1);
      top = make_float2(n0, n1);
      l = make_float2(fmaf(a0, l.x, f0 * s.x), fmaf(a1, l.y, f1 * s.y));
      o = make_float4(fmaf(a0, o.x, f0 * x.x), fmaf(a1, o.y, f1 * x.y), fmaf(a0, o.z, f0 * x.z), fmaf(a1, o.w, f1 * x.w));
    };
    for (int b = first + group; b <= last; b += GROUPS * kFlight) {
      float2 m[kFlight], s[kFlight];
      float4 x[kFlight];
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        const int at = b + i * GROUPS;
        const float* part = p.parts + ((int64_t)at * 2 + (at == first ? 1 : 0)) * S::kPartFloats;
        if (at <= last) {
          m[i] = *reinterpret_cast<const float2*>(part + kHeads * D + 2 * t4);
          s[i] = *reinterpret_cast<const float2*>(part + kHeads * D + kHeads + 2 * t4);
          x[i] = reinterpret_cast<const float4*>(part)[piece * 32 + lane];
        }
      }
#pragma unroll
      for (int i = 0; i < kFlight; ++i)
        if (b + i * GROUPS <= last) add(m[i], s[i], x[i]);
    }
    if (GROUPS > 1) {
      __syncthreads();     // the tile before has been read
      s_o[group][lane] = o;
      s_ml[group][lane] = make_float4(top.x, top.y, l.x, l.y);
      __syncthreads();
      if (group) continue;
#pragma unroll
      for (int w = 1; w < GROUPS; ++w) {
        const float4 ml = s_ml[w][lane];
        if (first + w <= last) add(make_float2(ml.x, ml.y), make_float2(ml.z, ml.w), s_o[w][lane]);
      }
    }
    const int hk = h / p.sub, head0 = hk * p.group + (h - hk * p.sub) * kHeads, heads = min(kHeads, (hk + 1) * p.group - head0);
    const int earlier = PACKED ? p.info[t].w & (p.pack - 1) : 0, c = (D / 8) * g + 2 * piece;
    T *out0, *out1;
    if constexpr (PACKED) {
      out0 = column_out<T, PACKED>(p, t, 2 * t4, earlier, head0, heads);
      out1 = column_out<T, PACKED>(p, t, 2 * t4 + 1, earlier, head0, heads);
    } else {
      out0 = reinterpret_cast<T*>(p.out) + t * p.o_st + (int64_t)(head0 + 2 * t4) * p.o_sh;
      out1 = 2 * t4 + 1 < heads ? out0 + p.o_sh : nullptr;
      if (2 * t4 >= heads) out0 = nullptr;
    }
    if (out0) out0[c] = from_float<T>(o.x / l.x), out0[c + 1] = from_float<T>(o.z / l.x);
    if (out1) out1[c] = from_float<T>(o.y / l.y), out1[c + 1] = from_float<T>(o.w / l.y);
  }
  if (!waited) pdl_wait();      // what comes after this launch comes after the first one too
}

size_t workspace_of(int D) { return (size_t)sm_count() * kWarpsPerSm * 2 * (kHeads * D + 2 * kHeads) * sizeof(float); }

}  // namespace
}  // namespace pare

extern "C" {

using namespace pare;
using namespace pare::paged;

size_t pare_paged_attn_workspace_bytes(int D) {
  if (D != 64 && D != 128) return 0;
  return workspace_of(D);
}

int pare_paged_attn(const void* q, int64_t q_stride_t, int64_t q_stride_h, const pare_paged_layer* l, const pare_paged_tables* tb, int Hq,
                    void* out, int64_t out_stride_t, int64_t out_stride_h, float softmax_scale, void* workspace, size_t workspace_bytes,
                    void* stream) {
  const int rc = check(l, tb);
  if (rc != PARE_OK) return rc;
  const int T = tb->T, H = l->H, D = l->D;
  PARE_REQUIRE(Hq > 0 && Hq % H == 0, PARE_ERR_SHAPE);
  PARE_REQUIRE(T <= kMaxQueryTokens, PARE_ERR_UNSUPPORTED);
  if (T == 0) return PARE_OK;
  PARE_REQUIRE(q && out, PARE_ERR_SHAPE);
  PARE_REQUIRE(aligned16(q) && (q_stride_t | q_stride_h) % 8 == 0 && aligned16(workspace), PARE_ERR_ALIGN);
  PARE_REQUIRE(workspace && workspace_bytes >= workspace_of(D), PARE_ERR_WORKSPACE);
  const int group = Hq / H, sub = (group + kHeads - 1) / kHeads, packs = !packs_tokens(tb->R, T) || group > 4 ? 0 : group == 1 ? 3 : group == 2 ? 2 : 1;
  PARE_REQUIRE((int64_t)T * H * sub < (int64_t)1 << 31, PARE_ERR_UNSUPPORTED);
  // the step counts its units in 32 bits
  PARE_REQUIRE(T * ((int64_t)tb->max_blocks * l->block_size / kUnit + 2) < (int64_t)1 << 31, PARE_ERR_UNSUPPORTED);
  const StepLayout s(tb->R, T, l->block_size);
  const int* w = reinterpret_cast<const int*>(tb->step);
  const PagedAttnParams p{q, q_stride_t, q_stride_h, out, out_stride_t, out_stride_h, reinterpret_cast<const int4*>(w + s.info),
                          w + s.unit_start + packs * s.unit_stride, tb->block_table, tb->ld_table, l->k_codes, l->v_codes, l->k_scale, l->v_scale, l->tail_k, l->tail_v,
                          reinterpret_cast<float*>(workspace), softmax_scale * kLog2e, T, tb->R, H, group, sub,
                          l->block_size == 16 ? 4 : l->block_size == 32 ? 5 : 6, l->num_blocks, tb->max_blocks,
                          1 << packs, (256 + group - 1) / group};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto tag, auto dim, auto packed) {
    using E = decltype(tag);
    constexpr int kD = decltype(dim)::value;
    constexpr bool kPacked = decltype(packed)::value;
    const auto kern = paged_attn_kernel<E, kD, kPacked>;
    const int sms = sm_count();
    if (!ensure_smem_attr(reinterpret_cast<const void*>(kern), (int)Shape<kD>::kSmem)) return (int)PARE_ERR_CUDA;
    int status = launch_pdl(kern, dim3(sms * Shape<kD>::kBlocksPerSm), dim3(Shape<kD>::kThreads), Shape<kD>::kSmem, st, p);
    if (status != PARE_OK) return status;
    const int jobs = T * H * sub, warps = sms * kWarpsPerSm;
    auto merge = [&](auto kernel, int groups) {
      return groups > 1 ? launch_pdl(kernel, dim3(jobs, kD / 16), dim3(groups * 32), 0, st, p, warps)
                        : launch_pdl(kernel, dim3(std::min(jobs, 32 * sms)), dim3(2 * kD), 0, st, p, warps);
    };
    if (8 * jobs <= sms) status = merge(paged_merge_kernel<E, kD, 16, kPacked>, 16);
    else if (jobs <= sms) status = merge(paged_merge_kernel<E, kD, 8, kPacked>, 8);
    else status = merge(paged_merge_kernel<E, kD, 1, kPacked>, 1);
    return status != PARE_OK ? status : launch_status();
  };
  auto by_dim = [&](auto tag, auto dim) { return packs ? go(tag, dim, std::true_type()) : go(tag, dim, std::false_type()); };
  auto by_type = [&](auto dim) { return l->dtype == PARE_F16 ? by_dim(__half(), dim) : by_dim(__nv_bfloat16(), dim); };
  return D == 64 ? by_type(std::integral_constant<int, 64>()) : by_type(std::integral_constant<int, 128>());
}

}  // extern "C"
