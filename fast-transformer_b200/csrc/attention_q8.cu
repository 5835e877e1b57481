// Attention of one token (decode) or a verify block of T tokens per row over an 8-bit KV cache
// (e4m3 codes, one fp32 scale per (row, KV head, block of slots)), sm_100a.
//
//   s[c] = (q . kcode[c]) * ks[c / block] * scale,  p[c] = 2^(s[c] log2 e - m),
//   out  = sum_c p[c] * vs[c / block] * vcode[c] / sum_c p[c]
// over the slots a token sees (decode: [0, position]; block: the reference's chain rule,
// engine/kernels/decode_attention.py:286-292); a token that sees none gives zeros.
//
// The codes are never expanded in memory: a warp converts its e4m3 fragments to f16 (exact) on
// the way into mma.sync m16n8k16, and the scales, uniform over a warp's 16 slots, fold into
// scalars. K's multiplies the scores. V's joins the exponent: the value product takes
// p'[c] = 2^(s[c] + log2 vs - M) with a pivot M of its own over s + log2 vs, so a block's scale
// can neither overflow nor wash out P's f16 range, while the denominator sums 2^(s - m) in
// fp32. Q is scaled by a power of two to f16's range (exact for any bf16 row).
//
// Bound by the bytes of codes; 148 persistent CTAs cut the 128-slot tiles of all (row, KV head,
// member group) units into equal contiguous slices, so ragged rows balance. A run of tiles that
// covers its unit writes the output; others leave (O, M, m, l) partials, merged in CTA order by
// a second launch (no counters, no atomics: two calls never share state).
//  * Warp 8 is the producer: one lane issues a TMA load per K and V tile (128 rows of D bytes,
//    swizzled by the row's length), 16 lanes copy the tile's per-slice scales with cp.async; both
//    complete on the stage's mbarrier.
//  * Warps 0-7 take 16 slots each: S^T[16 x 8 NG] = K Q^T, lazy pivot (it moves only when a score
//    passes it by more than 8, one vote), O^T += V^T P^T.
//  * Members = the T * G query heads that share a KV head, in groups of 8 NG columns.
#include "q8.cuh"

namespace fb {
namespace attn8 {

constexpr int kTile = 128;
constexpr int kWarps = 8;  // 16 slots each
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kMaxBatch = 1024;
constexpr int kScales = 2 * kWarps;  // per stage: K and V scale of each 16-slot slice
constexpr float kSlack = 8.f;        // log2 a score may pass the pivot by: p <= 2^8, exact enough in f16

struct Params {
  const __nv_bfloat16* q;  // [B, T, Hq, D]
  const float* key_scales;
  const float* value_scales;
  const int64_t* position;
  const int64_t* chain;  // [B]; nullptr: decode (T = 1)
  int per_row;
  __nv_bfloat16* out;  // [B, T, Hq, D]
  float* acc;          // [ctas + units, width, D]
  float4* stats;       // [ctas + units, width]: M, m, l
  int batch, tokens, q_heads, kv_heads, groups, capacity, block, blocks, ctas;
  int members;  // T * G
  int chunks;   // member groups per (row, KV head)
  int width;    // members of a chunk (the last may hold fewer)
  float scale_log2;
  unsigned* err;
};

// Slots row b's last token sees, clamped to the cache; 0: the row is empty.
__device__ __forceinline__ int row_length(const Params& p, int b) {
  const long long n = p.position[p.per_row ? b : 0];
  if (n < 0) return 0;
  return n > p.capacity - p.tokens ? p.capacity : static_cast<int>(n) + p.tokens;
}
__device__ __forceinline__ int tiles_of(int len) { return (len + kTile - 1) / kTile; }
__device__ __forceinline__ long long slice_start(long long total, int i, int ctas) { return total * i / ctas; }
__device__ __forceinline__ int slice_owner(long long total, long long tile, int ctas) {
  return static_cast<int>(((tile + 1) * ctas - 1) / total);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// x - y where y may be -inf (an empty running maximum): the pivot is then 0.
__device__ __forceinline__ float pivot(float m) { return m == -INFINITY ? 0.f : m; }

// sum p vs v / sum p from the two pivots' sums; zeros where nothing is seen, or only zero values.
__device__ __forceinline__ float finished(float O, float M, float m, float l) {
  if (l == 0.f || (M == -INFINITY && l > 0.f)) return 0.f;
  return O / l * exp2f(pivot(M) - pivot(m));
}

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile written by TMA with rows of D bytes:
// SWIZZLE_128B for D = 128, SWIZZLE_64B for D = 64.
template <int D>
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) {
  if constexpr (D == 128) return row * 128u + ((chunk ^ (row & 7u)) << 4);
  return row * 64u + ((chunk ^ ((row >> 1) & 3u)) << 4);
}

template <int D>
struct Smem {
  static constexpr int kTileBytes = kTile * D;
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kRing = kStages * 2 * kTileBytes;
  static constexpr int kScaleBytes = kStages * kScales * 4;
  static constexpr int kRedO = kWarps * D * 8 * 4;      // one 8-column group of every warp
  static constexpr int kRedStats = kWarps * 32 * 3 * 4;  // M, m, l of up to 32 columns
  static constexpr int kCum = ((kMaxBatch + 1) * 4 + 15) & ~15;
  static constexpr int kBars = 2 * kStages * 8;
  static constexpr int kTotal = 1024 + kRing + kScaleBytes + kRedO + kRedStats + kCum + kBars + 32;
};

// A consumer warp's state on one unit.
template <int D, int NG>
struct State {
  uint32_t q[NG][D / 16][2];  // B fragments: member column lane / 4 of each group
  float o[NG][D / 16][4];
  float m[NG][2], M[NG][2], l[NG][2];  // columns 2c, 2c + 1
  float qs[NG][2];                     // score multiplier of those columns: 2^e scale log2(e)
};

template <int D, int NG>
__device__ __forceinline__ void start_unit(State<D, NG>& a, const Params& p, int b, int h, int chunk, int lane) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int member = chunk * p.width + n * 8 + g;
    const bool live = n * 8 + g < p.width && member < p.members;
    const int t = live ? member / p.groups : 0;
    const int head = h * p.groups + (live ? member % p.groups : 0);
    const __nv_bfloat16* row = p.q + ((static_cast<size_t>(b) * p.tokens + t) * p.q_heads + head) * D;
    float x[D / 16][4];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const uint2 w = live ? *reinterpret_cast<const uint2*>(row + k * 16 + 4 * c) : make_uint2(0u, 0u);
      x[k][0] = bf16_lo(w.x), x[k][1] = bf16_hi(w.x), x[k][2] = bf16_lo(w.y), x[k][3] = bf16_hi(w.y);
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[k][e]));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // the row's largest magnitude to [2^14, 2^15): every value keeps its bits unless it is 2^-28 of it
    const int up = top > 0.f && top < INFINITY ? 14 - ilogbf(top) : 0;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      a.q[n][k][0] = pack_f16x2(ldexpf(x[k][0], up), ldexpf(x[k][1], up));
      a.q[n][k][1] = pack_f16x2(ldexpf(x[k][2], up), ldexpf(x[k][3], up));
    }
    const float mine = ldexpf(p.scale_log2, -up);  // of column g; this thread's scores are 2c and 2c + 1
    a.qs[n][0] = __shfl_sync(0xffffffffu, mine, 8 * c);
    a.qs[n][1] = __shfl_sync(0xffffffffu, mine, 8 * c + 4);
#pragma unroll
    for (int k = 0; k < D / 16; ++k) a.o[n][k][0] = a.o[n][k][1] = a.o[n][k][2] = a.o[n][k][3] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      a.m[n][e] = a.M[n][e] = -INFINITY;
      a.l[n][e] = 0.f;
    }
  }
}

// O^T += V^T P^T for this warp's 16 slots. Each register of a transposed load holds two dims of two
// slots; one byte permute and two conversions make the A fragments of dims 2g (rows 0-7 of the
// product) and 2g + 1 (rows 8-15). keep0 / keep1 mask the bytes of slots (2c, 2c+1) and 8 later.
template <int D, int NG>
__device__ __forceinline__ void value_product(float (&o)[NG][D / 16][4], uint32_t tile, int row, int half,
                                              uint32_t keep0, uint32_t keep1, const uint32_t (&pb)[NG][2]) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    uint32_t r[4];
    ldmatrix_x4_trans(tile + swizzled<D>(row, 2 * i + half), r[0], r[1], r[2], r[3]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t w0 = __byte_perm(r[2 * j] & keep0, 0, 0x3120), w1 = __byte_perm(r[2 * j + 1] & keep1, 0, 0x3120);
      const uint32_t a0 = q8::e4m3x2_to_f16x2(w0 & 0xffffu), a1 = q8::e4m3x2_to_f16x2(w0 >> 16);
      const uint32_t a2 = q8::e4m3x2_to_f16x2(w1 & 0xffffu), a3 = q8::e4m3x2_to_f16x2(w1 >> 16);
#pragma unroll
      for (int n = 0; n < NG; ++n) mma_f16(o[n][2 * i + j], a0, a1, a2, a3, pb[n][0], pb[n][1]);
    }
  }
}

// Whether token t of a row sees `slot`: the prefix [0, position] and, past it, the chain's tokens up
// to its own, or (t >= chain, an alternative to token 1) its own alone.
__device__ __forceinline__ bool sees(int slot, int len, int position, int t, int chain) {
  if (slot >= len) return false;
  return slot <= position || (t < chain ? slot <= position + t : slot == position + t);
}

// Whether this warp's 16 rows of a tile hold a NaN code.
template <int D>
__device__ __forceinline__ bool any_nan(uint32_t tile, int warp, int lane) {
  bool found = false;
  for (int i = lane; i < 16 * D / 4; i += 32) {
    uint32_t w;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(tile + warp * 16 * D + i * 4) : "memory");
    w &= 0x7f7f7f7fu;  // a byte of 0x7f: adding 1 reaches its top bit
    found = found || ((w + 0x01010101u) & 0x80808080u) != 0;
  }
  return __any_sync(0xffffffffu, found);
}

// One 128-slot tile starting at slot `first`: this warp's 16 slots of it. `len`: slots of the row;
// `position`: its first token's slot; ks, vs: the slice's scales.
template <int D, int NG>
__device__ __forceinline__ void attend_tile(State<D, NG>& a, const Params& p, uint32_t kt, uint32_t vt, int first,
                                            int len, int position, int chain, int chunk, float ks, float vs, int warp,
                                            int lane) {
  const int slice = first + warp * 16;
  if (slice >= len) return;
  const int g = lane >> 2, c = lane & 3;
  const int row = warp * 16 + (lane & 15), half = lane >> 4;
  float s[NG][4];
#pragma unroll
  for (int n = 0; n < NG; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    uint32_t r[4];
    ldmatrix_x4(kt + swizzled<D>(row, 2 * i + half), r[0], r[1], r[2], r[3]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t a0 = q8::e4m3x2_to_f16x2(r[2 * j] & 0xffffu), a2 = q8::e4m3x2_to_f16x2(r[2 * j] >> 16);
      const uint32_t a1 = q8::e4m3x2_to_f16x2(r[2 * j + 1] & 0xffffu), a3 = q8::e4m3x2_to_f16x2(r[2 * j + 1] >> 16);
#pragma unroll
      for (int n = 0; n < NG; ++n) mma_f16(s[n], a0, a1, a2, a3, a.q[n][2 * i + j][0], a.q[n][2 * i + j][1]);
    }
  }
  const float lv = log2f(vs);  // -inf for a block of zeros
  // every member sees slots [0, position]; past them the chain rule decides per token
  const bool tail = slice + 16 > (p.chain != nullptr ? position + 1 : len);
  uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
#pragma unroll
  for (int n = 0; n < NG; ++n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[n][e] *= a.qs[n][e & 1] * ks;
  }
  if (tail) {
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int slot = slice + g + (e >> 1) * 8;
        const int t = p.chain != nullptr ? (chunk * p.width + n * 8 + 2 * c + (e & 1)) / p.groups : 0;
        if (!sees(slot, len, position, t, chain)) s[n][e] = -INFINITY;
      }
    // slots past the row hold anything, NaN codes too: a zero weight must not meet them
    const int left = len - slice;
    keep0 = (2 * c < left ? 0xffffu : 0u) | (2 * c + 1 < left ? 0xffff0000u : 0u);
    keep1 = (2 * c + 8 < left ? 0xffffu : 0u) | (2 * c + 9 < left ? 0xffff0000u : 0u);
  }
  bool moves = false;
#pragma unroll
  for (int n = 0; n < NG; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      moves = moves || fmaxf(s[n][e], s[n][e + 2]) > fminf(a.m[n][e], a.M[n][e] - lv) + kSlack;
  if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float m = fmaxf(a.m[n][e], top), M = fmaxf(a.M[n][e], top + lv);
        const float fl = ex2(a.m[n][e] - pivot(m)), fo = ex2(a.M[n][e] - pivot(M));
        a.m[n][e] = m;
        a.M[n][e] = M;
        a.l[n][e] *= fl;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          a.o[n][k][e] *= fo;
          a.o[n][k][e + 2] *= fo;
        }
      }
  }
  uint32_t pb[NG][2];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a.l[n][e & 1] += ex2(s[n][e] - pivot(a.m[n][e & 1]));
      w[e] = ex2(s[n][e] + lv - pivot(a.M[n][e & 1]));
    }
    pb[n][0] = movmatrix_trans(pack_f16x2(w[0], w[1]));
    pb[n][1] = movmatrix_trans(pack_f16x2(w[2], w[3]));
  }
  if (tail && p.chain != nullptr && any_nan<D>(vt, warp, lane)) {
    // A NaN in a slot that only some members see: their zero weights must not meet it, so each
    // member's column is kept from a product of its own, over the slots it sees. Never taken on
    // sound values.
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll 1
      for (int col = 0; col < 8 && n * 8 + col < p.width; ++col) {
        const int t = (chunk * p.width + n * 8 + col) / p.groups;
        uint32_t k0 = 0u, k1 = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int slot = slice + 2 * c + (e & 1) + (e >> 1) * 8;
          if (!sees(slot, len, position, t, chain)) continue;
          (e < 2 ? k0 : k1) |= (e & 1) ? 0xffff0000u : 0xffffu;
        }
        const uint32_t one[1][2] = {{pb[n][0], pb[n][1]}};
        float o[1][D / 16][4] = {};
        value_product<D, 1>(o, vt, row, half, k0, k1, one);
        if (col >> 1 != c) continue;  // this thread's columns are 2c and 2c + 1
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          (col & 1 ? a.o[n][k][1] : a.o[n][k][0]) += col & 1 ? o[0][k][1] : o[0][k][0];
          (col & 1 ? a.o[n][k][3] : a.o[n][k][2]) += col & 1 ? o[0][k][3] : o[0][k][2];
        }
      }
    return;
  }
  value_product<D, NG>(a.o, vt, row, half, keep0, keep1, pb);
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"r"(kWarps * 32) : "memory"); }

// Sums the eight warps' states (in warp order) and either writes the unit's output or leaves
// its partials in `slot`.
template <int D, int NG>
__device__ void finish_run(State<D, NG>& a, const Params& p, int b, int h, int chunk, bool whole, size_t slot,
                           float* red_o, float* red_stats, int warp, int lane) {
  const int g = lane >> 2, c = lane & 3, tid = threadIdx.x;
#pragma unroll
  for (int n = 0; n < NG; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = a.l[n][e];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
      if (g == 0) {
        float* st = red_stats + (warp * 32 + n * 8 + 2 * c + e) * 3;
        st[0] = a.M[n][e], st[1] = a.m[n][e], st[2] = l;
      }
    }
  const int members = min(p.width, p.members - chunk * p.width);
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    if (n * 8 >= members) break;  // uniform
    consumers_sync();             // the last group's reads are done
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      float* dst = red_o + (warp * D + 16 * k + 2 * g) * 8 + 2 * c;
      *reinterpret_cast<float2*>(dst) = make_float2(a.o[n][k][0], a.o[n][k][1]);
      *reinterpret_cast<float2*>(dst + 8) = make_float2(a.o[n][k][2], a.o[n][k][3]);
    }
    consumers_sync();
    for (int e = tid; e < 8 * D; e += kWarps * 32) {
      const int col = e / D, d = e % D, in_chunk = n * 8 + col;
      if (in_chunk >= members) break;
      float M = -INFINITY, m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        M = fmaxf(M, red_stats[(w * 32 + in_chunk) * 3]);
        m = fmaxf(m, red_stats[(w * 32 + in_chunk) * 3 + 1]);
      }
      float O = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* st = red_stats + (w * 32 + in_chunk) * 3;
        O += red_o[(w * D + d) * 8 + col] * ex2(st[0] - pivot(M));
        l += st[2] * ex2(st[1] - pivot(m));
      }
      if (whole) {
        const int member = chunk * p.width + in_chunk;
        const int t = member / p.groups, head = h * p.groups + member % p.groups;
        p.out[((static_cast<size_t>(b) * p.tokens + t) * p.q_heads + head) * D + d] =
            __float2bfloat16_rn(finished(O, M, m, l));
      } else {
        p.acc[(slot * p.width + in_chunk) * D + d] = O;
        if (d == 0) p.stats[slot * p.width + in_chunk] = make_float4(M, m, l, 0.f);
      }
    }
  }
  consumers_sync();  // red_stats is free for the next run
}

template <int D, int NG>
__global__ void __launch_bounds__(kThreads, 1)
    attention_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ Params p) {
  using S = Smem<D>;
  constexpr int NS = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* stage_scales = reinterpret_cast<float*>(base + S::kRing);
  float* red_o = reinterpret_cast<float*>(base + S::kRing + S::kScaleBytes);
  float* red_stats = red_o + S::kRedO / 4;
  int* cum = reinterpret_cast<int*>(red_stats + S::kRedStats / 4);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(cum) + S::kCum);
  uint64_t* empty = full + NS;
  volatile int* misc = reinterpret_cast<volatile int*>(empty + NS);  // [0..2]: first row, unit, tile; [3]: abort

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int B = p.batch, per_row = p.kv_heads * p.chunks;  // units of a row
  if (warp == kWarps && lane == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1 + kScales);  // the tiles' bytes and 16 scale copies
      mbar_init(&empty[s], kWarps);
    }
    fence_barrier_init();
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    misc[3] = 0;
  }
  pdl_wait();
  pdl_trigger();
  // ---- plan: tiles before each row, this CTA's slice and where it begins ----
  if (warp == 0) {
    int running = 0;
    if (lane == 0) cum[0] = 0;
    for (int b0 = 0; b0 < B; b0 += 32) {
      const int b = b0 + lane;
      int x = b < B ? tiles_of(row_length(p, b)) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (b < B) cum[b + 1] = running + x;
      running += __shfl_sync(0xffffffffu, x, 31);
    }
  }
  __syncthreads();
  const long long total = static_cast<long long>(per_row) * cum[B];
  const long long t0 = slice_start(total, blockIdx.x, p.ctas), t1 = slice_start(total, blockIdx.x + 1, p.ctas);
  const int count = static_cast<int>(t1 - t0);
  if (count <= 0) return;
  if (warp == 0) {
    for (int b0 = 0; b0 < B; b0 += 32) {
      const int b = b0 + lane;
      const bool hit = b < B && static_cast<long long>(per_row) * cum[b] <= t0 &&
                       t0 < static_cast<long long>(per_row) * cum[b + 1];
      if (hit) {
        const int n = cum[b + 1] - cum[b];
        const long long off = t0 - static_cast<long long>(per_row) * cum[b];
        misc[0] = b;
        misc[1] = static_cast<int>(off / n);
        misc[2] = static_cast<int>(off % n);
      }
      if (__any_sync(0xffffffffu, hit)) break;
    }
  }
  __syncthreads();
  int b = misc[0], u = misc[1], j = misc[2];  // row, unit of the row (KV head, chunk), tile
  int n = cum[b + 1] - cum[b];

  if (warp == kWarps) {
    // ================================ producer ================================
    int issued = 0;
    for (int k = 0; k < count; ++k) {
      const int s = k % NS;
      bool ok = misc[3] == 0;
      if (ok && k >= NS && !mbar_wait_bounded(&empty[s], ((k / NS) - 1) & 1)) {
        if (lane == 0) raise_error(p.err, kErrTimeoutEmpty);
        misc[3] = 1;
        ok = false;
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      const size_t pair = static_cast<size_t>(b) * p.kv_heads + u / p.chunks;
      if (lane == 0) {
        uint8_t* kt = base + s * 2 * S::kTileBytes;
        const int row = static_cast<int>(pair * p.capacity) + j * kTile;
        mbar_arrive_expect_tx(&full[s], 2 * S::kTileBytes);
        tma_load_2d(kt, &kmap, &full[s], 0, row);
        tma_load_2d(kt + S::kTileBytes, &vmap, &full[s], 0, row);
      }
      if (lane < kScales) {
        const int i = min((j * kTile + (lane & 7) * 16) / p.block, p.blocks - 1);
        const float* src = (lane < 8 ? p.key_scales : p.value_scales) + pair * p.blocks + i;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(stage_scales + s * kScales + lane)),
                     "l"(src)
                     : "memory");
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[s])) : "memory");
      }
      issued = k + 1;
      if (++j == n) {
        j = 0;
        if (++u == per_row) {
          u = 0;
          do ++b;
          while (b < B && cum[b + 1] == cum[b]);
          if (b < B) n = cum[b + 1] - cum[b];
        }
      }
    }
    // after an abort: let the copies in flight land before the block's shared memory is released
    if (misc[3] != 0)
      for (int k = issued > NS ? issued - NS : 0; k < issued; ++k) mbar_wait_bounded(&full[k % NS], (k / NS) & 1);
    return;
  }

  // ================================ consumers ================================
  int len = row_length(p, b);
  int position = static_cast<int>(min(p.position[p.per_row ? b : 0], static_cast<int64_t>(p.capacity)));
  int chain = p.chain != nullptr ? static_cast<int>(p.chain[b]) : 1;
  int run_first = j;
  State<D, NG> a;
  start_unit<D, NG>(a, p, b, u / p.chunks, u % p.chunks, lane);
  for (int k = 0; k < count; ++k) {
    const int s = k % NS;
    bool ok = misc[3] == 0;
    if (ok && !mbar_wait_bounded(&full[s], (k / NS) & 1)) {
      raise_error(p.err, kErrTimeoutFull);
      misc[3] = 1;
    }
    const uint32_t kt = smem_u32(base + s * 2 * S::kTileBytes);
    // an aborted launch still takes every barrier below, on whatever the stage holds
    const float ks = stage_scales[s * kScales + warp], vs = stage_scales[s * kScales + 8 + warp];
    attend_tile<D, NG>(a, p, kt, kt + S::kTileBytes, j * kTile, len, position, chain, u % p.chunks, ks, vs, warp, lane);
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
    const int run_b = b, run_u = u, run_last = j, run_n = n;
    bool ends = k == count - 1;
    if (++j == n) {
      j = 0;
      ends = true;
      if (++u == per_row) {
        u = 0;
        do ++b;
        while (b < B && cum[b + 1] == cum[b]);
      }
    }
    if (!ends) continue;
    const size_t slot = blockIdx.x + static_cast<size_t>(run_b) * per_row + run_u;
    finish_run<D, NG>(a, p, run_b, run_u / p.chunks, run_u % p.chunks, run_first == 0 && run_last == run_n - 1, slot,
                      red_o, red_stats, warp, lane);
    if (k != count - 1) {
      n = cum[b + 1] - cum[b];
      len = row_length(p, b);
      position = static_cast<int>(min(p.position[p.per_row ? b : 0], static_cast<int64_t>(p.capacity)));
      chain = p.chain != nullptr ? static_cast<int>(p.chain[b]) : 1;
      run_first = j;
      start_unit<D, NG>(a, p, b, u / p.chunks, u % p.chunks, lane);
    }
  }
}

// One CTA per unit: merges the runs of the CTAs that shared it, in CTA order, and writes the
// zeros of empty rows.
constexpr int kMergeThreads = 128;

template <int D>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const __grid_constant__ Params p) {
  __shared__ int s_before, s_total;
  pdl_wait();
  pdl_trigger();
  const int per_row = p.kv_heads * p.chunks;
  const int b = blockIdx.x / per_row, u = blockIdx.x % per_row;
  const int h = u / p.chunks, chunk = u % p.chunks;
  if (threadIdx.x == 0) s_before = s_total = 0;
  __syncthreads();
  int before = 0, total = 0;
  for (int r = threadIdx.x; r < p.batch; r += kMergeThreads) {
    const int n = tiles_of(row_length(p, r));
    total += n;
    if (r < b) before += n;
  }
  if (before) atomicAdd(&s_before, before);
  if (total) atomicAdd(&s_total, total);
  __syncthreads();
  const int n = tiles_of(row_length(p, b));
  const int members = min(p.width, p.members - chunk * p.width);
  const long long T = static_cast<long long>(per_row) * s_total;
  const long long first = static_cast<long long>(per_row) * s_before + static_cast<long long>(u) * n;
  const int lo = n > 0 ? slice_owner(T, first, p.ctas) : 0, hi = n > 0 ? slice_owner(T, first + n - 1, p.ctas) : 0;
  if (n > 0 && lo == hi) return;  // one run covered the unit and wrote its output
  for (int e = threadIdx.x; e < members * D; e += kMergeThreads) {
    const int in_chunk = e / D, d = e % D, member = chunk * p.width + in_chunk;
    float M = -INFINITY, m = -INFINITY, O = 0.f, l = 0.f;
    if (n > 0) {
      for (int i = lo; i <= hi; ++i) {
        if (slice_start(T, i, p.ctas) >= slice_start(T, i + 1, p.ctas)) continue;  // an empty slice wrote nothing
        const float4 st = p.stats[(static_cast<size_t>(i) + blockIdx.x) * p.width + in_chunk];
        M = fmaxf(M, st.x);
        m = fmaxf(m, st.y);
      }
      for (int i = lo; i <= hi; ++i) {
        if (slice_start(T, i, p.ctas) >= slice_start(T, i + 1, p.ctas)) continue;
        const size_t at = (static_cast<size_t>(i) + blockIdx.x) * p.width + in_chunk;
        const float4 st = p.stats[at];
        O += p.acc[at * D + d] * ex2(st.x - pivot(M));
        l += st.z * ex2(st.y - pivot(m));
      }
    }
    const int t = member / p.groups, head = h * p.groups + member % p.groups;
    p.out[((static_cast<size_t>(b) * p.tokens + t) * p.q_heads + head) * D + d] =
        __float2bfloat16_rn(finished(O, M, m, l));
  }
}

// Columns of a unit: the least number of equal member groups of at most 24 (D = 128: the
// accumulators of 32 would not fit the registers) or 32 columns.
void chunk_members(Params* p, int head_dim) {
  const int most = head_dim == 128 ? 24 : 32;
  p->members = p->tokens * p->groups;
  p->chunks = (p->members + most - 1) / most;
  p->width = (p->members + p->chunks - 1) / p->chunks;
  p->chunks = (p->members + p->width - 1) / p->width;
}

size_t acc_bytes(const Params& p, int head_dim) {
  const size_t slots = static_cast<size_t>(p.ctas) + static_cast<size_t>(p.batch) * p.kv_heads * p.chunks;
  return (slots * p.width * head_dim * sizeof(float) + 255) & ~size_t(255);
}

size_t workspace_bytes(const Params& p, int head_dim) {
  const size_t slots = static_cast<size_t>(p.ctas) + static_cast<size_t>(p.batch) * p.kv_heads * p.chunks;
  return acc_bytes(p, head_dim) + slots * p.width * sizeof(float4);
}

int shape(Params* p, int batch, int tokens, int q_heads, int kv_heads, int head_dim, int capacity, int block) {
  if (batch <= 0 || tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || capacity <= 0) return FB_ERR_ARG;
  if ((head_dim != 64 && head_dim != 128) || !q8::valid_block(block)) return FB_ERR_SHAPE;
  if (q_heads % kv_heads != 0 || batch > kMaxBatch || tokens > capacity) return FB_ERR_SHAPE;
  if (static_cast<long long>(tokens) * (q_heads / kv_heads) > 65536) return FB_ERR_SHAPE;
  if (static_cast<long long>(batch) * kv_heads * capacity >= (1ll << 31)) return FB_ERR_SHAPE;  // tensor-map rows
  p->batch = batch;
  p->tokens = tokens;
  p->q_heads = q_heads;
  p->kv_heads = kv_heads;
  p->groups = q_heads / kv_heads;
  p->capacity = capacity;
  p->block = block;
  p->blocks = (capacity + block - 1) / block;
  p->ctas = sm_count();
  chunk_members(p, head_dim);
  return static_cast<long long>(batch) * kv_heads * p->chunks >= (1ll << 31) ? FB_ERR_SHAPE : FB_OK;
}

template <int D, int NG>
int launch(const CUtensorMap& km, const CUtensorMap& vm, const Params& p, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return FB_ERR_LAUNCH;
  if (dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(attention_kernel<D, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::kTotal) !=
        cudaSuccess)
      return FB_ERR_LAUNCH;
    if (dev < 64) configured[dev] = true;
  }
  const int st = launch_ex(attention_kernel<D, NG>, dim3(p.ctas), dim3(kThreads), Smem<D>::kTotal, stream, 1, km, vm, p);
  if (st != FB_OK) return st;
  return launch_ex(merge_kernel<D>, dim3(p.batch * p.kv_heads * p.chunks), dim3(kMergeThreads), 0, stream, 1, p);
}

template <int D>
int launch_groups(const CUtensorMap& km, const CUtensorMap& vm, const Params& p, cudaStream_t stream) {
  if (p.width <= 8) return launch<D, 1>(km, vm, p, stream);
  if (p.width <= 16) return launch<D, 2>(km, vm, p, stream);
  if (p.width <= 24) return launch<D, 3>(km, vm, p, stream);
  if constexpr (D == 64) return launch<D, 4>(km, vm, p, stream);
  return FB_ERR_SHAPE;
}

}  // namespace attn8
}  // namespace fb

using namespace fb;

extern "C" size_t fb_attention_q8_workspace(int batch, int tokens, int q_heads, int kv_heads, int head_dim,
                                            int capacity, int block) {
  attn8::Params p;
  if (attn8::shape(&p, batch, tokens, q_heads, kv_heads, head_dim, capacity, block) != FB_OK) return 0;
  return attn8::workspace_bytes(p, head_dim);
}

extern "C" int fb_attention_q8(const void* q, const void* keys, const void* values, const float* key_scales,
                               const float* value_scales, const int64_t* position, int per_row, const int64_t* chain,
                               void* out, void* workspace, size_t workspace_bytes, int batch, int tokens, int q_heads,
                               int kv_heads, int head_dim, int capacity, int block, float scale, void* stream) {
  if (!q || !keys || !values || !key_scales || !value_scales || !position || !out || !workspace) return FB_ERR_ARG;
  attn8::Params p;
  int st = attn8::shape(&p, batch, tokens, q_heads, kv_heads, head_dim, capacity, block);
  if (st != FB_OK) return st;
  if ((chain == nullptr && tokens != 1) || (chain != nullptr && !per_row)) return FB_ERR_ARG;
  if (workspace_bytes < attn8::workspace_bytes(p, head_dim)) return FB_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0 || (reinterpret_cast<uintptr_t>(q) & 7u) != 0)
    return FB_ERR_ARG;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.key_scales = key_scales;
  p.value_scales = value_scales;
  p.position = position;
  p.chain = chain;
  p.per_row = per_row ? 1 : 0;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.acc = static_cast<float*>(workspace);
  p.stats = reinterpret_cast<float4*>(static_cast<uint8_t*>(workspace) + attn8::acc_bytes(p, head_dim));
  p.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  p.err = error_word();
  const uint64_t rows = static_cast<uint64_t>(batch) * kv_heads * capacity;
  CUtensorMap km, vm;
  st = encode_u8_2d(&km, keys, rows, head_dim, attn8::kTile);
  if (st != FB_OK) return st;
  st = encode_u8_2d(&vm, values, rows, head_dim, attn8::kTile);
  if (st != FB_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return head_dim == 128 ? attn8::launch_groups<128>(km, vm, p, s) : attn8::launch_groups<64>(km, vm, p, s);
}
