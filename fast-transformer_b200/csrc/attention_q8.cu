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
// p'[c] = 2^(s[c] - m + log2 vs - r) with a pivot r of its own over s - m + log2 vs, so a block's scale
// can neither overflow nor wash out P's f16 range, while the denominator sums 2^(s - m) in
// fp32. r is kept relative to m: where scores are so large that their own rounding passes 1, the result is
// still a mean of values. r is set 7 below the largest exponent, so that P fills f16's range from the top and
// weights down to 2^-32 of the largest count. (With r at the largest, those below 2^-25 of it became zero in
// the numerator alone: all that stood behind one leading slot, however many, could be lost.) Q is scaled by a
// power of two to f16's range (exact for any bf16 row).
//
// Bound by the bytes of codes. Members = the T * G query heads that share a KV head, in groups of
// 8 NG columns; a unit = (row, KV head, member group); its tiles are 128 slots of K and V. A CTA is
// a producer warp (one lane issues a TMA load per K and V tile, 16 lanes copy the tile's scales
// with cp.async; both complete on the stage's mbarrier) and consumer warps; two CTAs share an SM: one
// streams while the other starts or ends. S^T[16 x 8 NG] = K Q^T, a lazy pivot (it moves only when a
// score passes it by kSlack, one vote), O^T += V^T P^T.
//  * One column group: four consumers of two 16-slot slices each, whole in registers; a warp needs no
//    other until the end.
//  * More: the conversions and products of a tile, not its bytes, fill its time, and O^T of every warp
//    would not fit the registers. Eight consumers: each scores its slice, P^T goes to shared memory, and
//    each multiplies all of it by its 16 dims of V. One barrier a tile (the vote), O held once.
// Work is cut in one of two ways:
//  * Few units, or short rows: a cluster of C CTAs per unit (interleaved tiles), merged by pushing each
//    partial to its output's owner through distributed shared memory: one launch, no workspace.
//  * Many units of long rows: a persistent grid cuts the tiles of all units into equal contiguous slices, so
//    ragged rows balance. A run of tiles that covers its unit writes the output; others leave
//    (O, M, m, l) partials that a second launch merges in CTA order. No counters, no atomics:
//    calls share nothing.
// Measured (D = 128, blocks of 64): 16 rows x 8320 slots, 32 + 8 heads 45.4 us, 6.0 TB/s (0.92 of a copy's rate);
// 64 rows of 1024 to 32768 slots 352 us, 6.3 TB/s; one row of 2048 slots 6.1 us (5.4 from L2), most of it launch, the
// chain position - tile - product, all of it behind the dependency wait, and the merge; 8 rows x 4101 slots x 5
// tokens 28 us, 2.4 TB/s: 0.36 of the issue slots, the warps waiting on each other's weights, on conversions and on
// shared memory.
#include <atomic>
#include <type_traits>

#include "q8.cuh"

namespace fb {
namespace attn8 {

constexpr int kSlices = 8;  // of 16 slots
constexpr int kTile = 16 * kSlices;
template <int NG>
constexpr int kConsumers = NG == 1 ? 4 : kSlices;  // warps
template <int NG>
constexpr int kThreads = (kConsumers<NG> + 1) * 32;
constexpr int kMaxBatch = 1024;
constexpr int kScales = 2 * kSlices;  // per stage: K and V scale of each 16-slot slice
constexpr int kMaxCluster = 16;      // above 8: the non-portable cluster size attribute
constexpr float kLift = 7.f;         // log2 of the largest p' when its pivot moves
constexpr float kSlack = 15.f;       // log2 of p' or p at which the pivots move: f16 ends at 65504 (p stays in fp32; a test
                                     // of its own against less cost 2 us of 27 with 20 members)

struct Params {
  const __nv_bfloat16* q;  // [B, T, Hq, D]
  const float* key_scales;
  const float* value_scales;
  const int64_t* position;
  const int64_t* chain;  // [B]; nullptr: decode (T = 1)
  int per_row;
  __nv_bfloat16* out;  // [B, T, Hq, D]
  float* acc;          // [ctas + units, width, D]
  float4* stats;       // [ctas + units, width]: r, m, l
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
__host__ __device__ __forceinline__ int tiles_of(int len) { return (len + kTile - 1) / kTile; }
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

// The pivot of nothing: finite, so that 2^(x - pivot) needs no test.
constexpr float kNone = -3.402823466e38f;
// A pivot relative to one m, relative to another that lies `by` below.
__device__ __forceinline__ float shifted(float r, float by) { return fmaxf(kNone, r + by); }

// sum p vs v / sum p from the two pivots' sums; zeros where nothing is seen, or only zero values.
__device__ __forceinline__ float finished(float O, float r, float l) {
  if (l == 0.f || (r == kNone && l > 0.f)) return 0.f;
  return O / l * exp2f(r);
}

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile written by TMA with rows of D bytes:
// SWIZZLE_128B for D = 128, SWIZZLE_64B for D = 64.
template <int D>
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) {
  if constexpr (D == 128) return row * 128u + ((chunk ^ (row & 7u)) << 4);
  return row * 64u + ((chunk ^ ((row >> 1) & 3u)) << 4);
}

template <int D, int NG>
struct Smem {
  static constexpr int kTileBytes = kTile * D;
  // two CTAs per SM (asserted below): what the buffers of more column groups leave
  static constexpr int kStages = D == 128 ? (NG == 1 ? 3 : 2) : (NG == 1 ? 5 : 4);
  static constexpr int kRing = kStages * 2 * kTileBytes;
  static constexpr int kScaleBytes = kStages * kScales * 4;
  // queries as B fragments, [group][32 dims][lane], then every column's score multiplier and token
  static constexpr int kFragments = NG * 8 * D * 2;
  static constexpr int kQuery = NG == 1 ? 0 : kFragments + NG * 8 * 8;
  // P^T as B fragments, [slice pair][group][lane][slice], of two tiles in turn
  static constexpr int kWeights = NG == 1 ? 0 : 2 * kSlices * NG * 32 * 8;
  // one group: half the dims of every warp; more: the O of warps that share dims with others
  static constexpr int kRedO = NG == 1 ? 4 * D / 2 * 8 * 4 : kSlices * NG * 32 * 16 / 2 * (D == 64);
  static constexpr int kRedStats = NG == 1 ? kConsumers<NG> * 8 * 3 * 4 : 0;  // r, m, l
  // persistent form: tile counts before each row; cluster form: O received as an owner
  // ([rank][chunk], C * 2 ceil(n / 2C) < n + 2C values) and every rank's r, m, l
  static constexpr int kCum = ((kMaxBatch + 1) * 4 + 15) & ~15;
  static constexpr int kRecvO = (NG * 8 * D + 2 * kMaxCluster) * 4;
  static constexpr int kRecvStats = kMaxCluster * NG * 8 * 3 * 4;
  static constexpr int kShared = kCum > kRecvO + kRecvStats ? kCum : kRecvO + kRecvStats;
  static constexpr int kBars = 2 * kStages * 8;
  static constexpr int kTotal =
      1024 + kRing + kScaleBytes + kQuery + kWeights + kRedO + kRedStats + kShared + kBars + 64;
  static_assert(kTotal + 1024 <= 228 * 1024 / 2, "two CTAs per SM");
  static_assert((kScaleBytes + kQuery + kWeights + kRedO + kRedStats + kShared) % 16 == 0, "mbarrier alignment");

  uint8_t* ring;
  float* scales;
  uint8_t* query;
  uint8_t* weights;
  float* red_o;
  float* red_stats;
  int* cum;
  float* recv_o;
  float* recv_stats;
  uint64_t* full;
  uint64_t* empty;
  volatile int* misc;  // [0..2]: first row, unit, tile; [3]: abort; [4 + warp]: 1 + the tile of its last move

  __device__ explicit Smem(uint8_t* raw) {
    ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    scales = reinterpret_cast<float*>(ring + kRing);
    query = ring + kRing + kScaleBytes;
    weights = query + kQuery;
    red_o = reinterpret_cast<float*>(weights + kWeights);
    red_stats = red_o + kRedO / 4;
    cum = reinterpret_cast<int*>(red_stats + kRedStats / 4);
    recv_o = reinterpret_cast<float*>(cum);
    recv_stats = recv_o + kRecvO / 4;
    full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(cum) + kShared);
    empty = full + kStages;
    misc = reinterpret_cast<volatile int*>(empty + kStages);
  }
};

// A consumer warp's state on one unit. One column group: its slices' share of O^T, and the query's B
// fragments. More: 16 dims of the unit's O^T and pivots that all warps hold alike; queries are read
// from shared memory for every tile.
template <int D, int NG>
struct State {
  static constexpr int kDims = NG == 1 ? D / 16 : 1;
  uint32_t q[NG == 1 ? D / 16 : 1][2];
  float o[NG][kDims][4];
  float m[NG][2], r[NG][2], l[NG][2];  // columns 2c, 2c + 1
  float qs[NG][2];                     // score multiplier of those columns: 2^e scale log2(e)
};

template <int NG>
__device__ __forceinline__ void consumers_sync() {
  asm volatile("bar.sync 1, %0;" ::"r"(kConsumers<NG> * 32) : "memory");
}
// The same barrier; whether any consumer thread says so.
template <int NG>
__device__ __forceinline__ bool consumers_any(bool x) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(any)
      : "r"(x ? 1u : 0u), "r"(kConsumers<NG> * 32)
      : "memory");
  return any != 0;
}

template <int D, int NG>
__device__ __forceinline__ void clear(State<D, NG>& a) {
#pragma unroll
  for (int n = 0; n < NG; ++n) {
#pragma unroll
    for (int k = 0; k < State<D, NG>::kDims; ++k) a.o[n][k][0] = a.o[n][k][1] = a.o[n][k][2] = a.o[n][k][3] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      a.m[n][e] = a.r[n][e] = kNone;
      a.l[n][e] = 0.f;
    }
  }
}

// The unit's queries as f16 B fragments: lane (g, c) holds dims 16 k + 4 c .. + 3 of member column
// g, the order in which K's fragments hold the dims. The row's largest magnitude is scaled to
// [2^14, 2^15): every value keeps its bits unless it is below 2^-28 of it.
template <int D, int NG>
__device__ __forceinline__ void start_unit(State<D, NG>& a, const Params& p, uint8_t* query, int b, int h, int chunk,
                                           int warp, int lane) {
  using S = Smem<D, NG>;
  const int g = lane >> 2, c = lane & 3;
  if (NG > 1) consumers_sync<NG>();  // the last unit's queries and totals have been read
  if (warp < NG || NG == 1) {         // shared queries: a warp converts a group
    const int col = NG == 1 ? g : warp * 8 + g, member = chunk * p.width + col;
    const bool live = col < p.width && member < p.members;
    const int t = live ? member / p.groups : 0;
    const int head = h * p.groups + (live ? member - t * p.groups : 0);
    const __nv_bfloat16* row = p.q + ((static_cast<size_t>(b) * p.tokens + t) * p.q_heads + head) * D;
    uint2 w[D / 16];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      w[k] = live ? *reinterpret_cast<const uint2*>(row + k * 16 + 4 * c) : make_uint2(0u, 0u);
      top = fmaxf(fmaxf(top, fmaxf(fabsf(bf16_lo(w[k].x)), fabsf(bf16_hi(w[k].x)))),
                  fmaxf(fabsf(bf16_lo(w[k].y)), fabsf(bf16_hi(w[k].y))));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^up in two factors: |up| reaches 147
    const int exponent = static_cast<int>(__float_as_uint(top) >> 23);  // 0: zero or subnormal; 255: not finite
    const int up = top > 0.f && exponent < 255 ? 14 + 127 - max(exponent, 1) : 0;
    const int first = up / 2;
    const float f0 = __uint_as_float(static_cast<uint32_t>(127 + first) << 23);
    const float f1 = __uint_as_float(static_cast<uint32_t>(127 + up - first) << 23);
    uint32_t f[D / 16][2];
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      f[k][0] = pack_f16x2(bf16_lo(w[k].x) * f0 * f1, bf16_hi(w[k].x) * f0 * f1);
      f[k][1] = pack_f16x2(bf16_lo(w[k].y) * f0 * f1, bf16_hi(w[k].y) * f0 * f1);
      if constexpr (NG == 1) {
        a.q[k][0] = f[k][0];
        a.q[k][1] = f[k][1];
      }
    }
    const float multiplier = p.scale_log2 / f0 / f1;  // of column g; this thread's scores are 2c and 2c + 1
    if constexpr (NG == 1) {
      a.qs[0][0] = __shfl_sync(0xffffffffu, multiplier, 8 * c);
      a.qs[0][1] = __shfl_sync(0xffffffffu, multiplier, 8 * c + 4);
    } else {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        reinterpret_cast<uint4*>(query)[(warp * (D / 32) + i) * 32 + lane] =
            make_uint4(f[2 * i][0], f[2 * i][1], f[2 * i + 1][0], f[2 * i + 1][1]);
      if (c == 0) {
        reinterpret_cast<float*>(query + S::kFragments)[col] = multiplier;
        reinterpret_cast<int*>(query + S::kFragments)[NG * 8 + col] = t;
      }
    }
  }
  if constexpr (NG > 1) {
    consumers_sync<NG>();
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) a.qs[n][e] = reinterpret_cast<const float*>(query + S::kFragments)[n * 8 + 2 * c + e];
  }
  clear<D, NG>(a);
}

// A register of a transposed load of V holds two dims of two slots; one byte permute and two conversions
// make the A fragments of dims 2g (rows 0-7 of the product) and 2g + 1 (rows 8-15). r0 holds slots
// (2c, 2c + 1) of 16, r1 those 8 later; pick0 / pick1 are their permutes: kPick, or with selectors of 4 (a
// zero byte) for slots left out.
constexpr uint32_t kPick = 0x3120u;

__device__ __forceinline__ void value_fragments(uint32_t (&f)[4], uint32_t r0, uint32_t r1, uint32_t pick0,
                                                uint32_t pick1) {
  q8::e4m3x4_to_f16x4(__byte_perm(r0, 0, pick0), f[0], f[1]);
  q8::e4m3x4_to_f16x4(__byte_perm(r1, 0, pick1), f[2], f[3]);
}

// O^T += V^T P^T for 16 slots and every dim (`row`: this lane's row of the tile, `half`: its 16-byte
// chunk's parity).
template <int D>
__device__ __forceinline__ void value_product(float (&o)[D / 16][4], uint32_t tile, int row, int half, uint32_t pick0,
                                              uint32_t pick1, const uint32_t (&pb)[2]) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    uint32_t r[4], f[4];
    ldmatrix_x4_trans(tile + swizzled<D>(row, 2 * i + half), r[0], r[1], r[2], r[3]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      value_fragments(f, r[2 * j], r[2 * j + 1], pick0, pick1);
      mma_f16(o[2 * i + j], f[0], f[1], f[2], f[3], pb[0], pb[1]);
    }
  }
}

// The permute that keeps slot 2c (result bytes 0 and 2) and slot 2c + 1 (bytes 1 and 3), or not.
__device__ __forceinline__ uint32_t pick_slots(bool even, bool odd) {
  return (even ? kPick & 0x0f0fu : 0x0404u) | (odd ? kPick & 0xf0f0u : 0x4040u);
}

// Whether token t of a row sees `slot`: the prefix [0, position] and, past it, the chain's tokens up
// to its own, or (t >= chain, an alternative to token 1) its own alone.
__device__ __forceinline__ bool sees(int slot, int len, int position, int t, int chain) {
  if (slot >= len) return false;
  return slot <= position || (t < chain ? slot <= position + t : slot == position + t);
}

// Whether a byte of w is a NaN code (0x7f or 0xff): adding 1 reaches its top bit.
__device__ __forceinline__ bool has_nan(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }

// Whether rows [row0, row0 + 16) of a tile hold a NaN code.
template <int D>
__device__ __forceinline__ bool any_nan(uint32_t tile, int row0, int lane) {
  bool found = false;
  for (int i = lane; i < 16 * D / 4; i += 32) {
    uint32_t w;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(tile + row0 * D + i * 4) : "memory");
    found = found || has_nan(w);
  }
  return __any_sync(0xffffffffu, found);
}

// log2 of a scale; exact for powers of two, -inf for 0.
__device__ __forceinline__ float log2_scale(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One column group: this warp's slices 2 w and 2 w + 1 of the 128-slot tile that starts at slot
// `first`, side by side (two independent chains hide each other's latency). `len`: slots of the row;
// `position`: its first token's slot; scales: the tile's, K then V.
template <int D>
__device__ __forceinline__ void attend_tile(State<D, 1>& a, const Params& p, const Smem<D, 1>&, const float* scales,
                                            uint32_t kt, uint32_t vt, int, bool, int first, int len, int position,
                                            int chain, int chunk, int warp, int lane) {
  constexpr int H = 2;
  const int g = lane >> 2, c = lane & 3, half = lane >> 4;
  const int slice = first + warp * 32;
  if (slice >= len) return;
  const int row = warp * 32 + (lane & 15);
  float s[H][4], s2[H][4];
#pragma unroll
  for (int x = 0; x < H; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[x][e] = s2[x][e] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int x = 0; x < H; ++x) {
      uint32_t r[4], k0[4], k1[4];
      ldmatrix_x4(kt + swizzled<D>(row + 16 * x, 2 * i + half), r[0], r[1], r[2], r[3]);
      q8::e4m3x4_to_f16x4(r[0], k0[0], k0[2]);
      q8::e4m3x4_to_f16x4(r[1], k0[1], k0[3]);
      q8::e4m3x4_to_f16x4(r[2], k1[0], k1[2]);
      q8::e4m3x4_to_f16x4(r[3], k1[1], k1[3]);
      // two chains of products: half the latency
      mma_f16(s[x], k0[0], k0[1], k0[2], k0[3], a.q[2 * i][0], a.q[2 * i][1]);
      mma_f16(s2[x], k1[0], k1[1], k1[2], k1[3], a.q[2 * i + 1][0], a.q[2 * i + 1][1]);
    }
  float lv[H];
#pragma unroll
  for (int x = 0; x < H; ++x) {
    const bool live = slice + 16 * x < len;  // past the row a scale can be anything
    const float ks = live ? scales[warp * 2 + x] : 1.f;
    lv[x] = live ? log2_scale(scales[kSlices + warp * 2 + x]) : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s[x][e] = __fmul_rn(s[x][e] + s2[x][e], a.qs[0][e & 1] * ks);
  }
  // every member sees slots [0, position]; past them the chain rule decides per token
  const bool tail = slice + 16 * H > (p.chain != nullptr ? position + 1 : len);
  if (tail) {
#pragma unroll
    for (int x = 0; x < H; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int slot = slice + 16 * x + g + (e >> 1) * 8;
        const int t = p.chain != nullptr ? (chunk * p.width + 2 * c + (e & 1)) / p.groups : 0;
        if (!sees(slot, len, position, t, chain)) s[x][e] = -INFINITY;
      }
  }
  bool moves = false;
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int x = 0; x < H; ++x) {
      const float over = fmaxf(s[x][e], s[x][e + 2]) - a.m[0][e];
      moves = moves || fmaxf(over, over + lv[x] - a.r[0][e]) > kSlack;
    }
  if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float top[H], m = a.m[0][e];
#pragma unroll
      for (int x = 0; x < H; ++x) {
        top[x] = fmaxf(s[x][e], s[x][e + 2]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], off));
        m = fmaxf(m, top[x]);
      }
      const float by = a.m[0][e] - m;
      float r = shifted(a.r[0][e], by);
#pragma unroll
      for (int x = 0; x < H; ++x) r = fmaxf(r, top[x] - m + lv[x] - kLift);
      const float fl = ex2(by), fo = ex2(a.r[0][e] + by - r);
      a.m[0][e] = m;
      a.r[0][e] = r;
      a.l[0][e] *= fl;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        a.o[0][k][e] *= fo;
        a.o[0][k][e + 2] *= fo;
      }
    }
  }
  uint32_t pb[H][2];
#pragma unroll
  for (int x = 0; x < H; ++x) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[x][e] -= a.m[0][e & 1];
      y[e] = s[x][e] + lv[x] - a.r[0][e & 1];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = ex2(y[e]);
    a.l[0][0] += ex2(s[x][0]) + ex2(s[x][2]);
    a.l[0][1] += ex2(s[x][1]) + ex2(s[x][3]);
    pb[x][0] = movmatrix_trans(pack_f16x2(y[0], y[1]));
    pb[x][1] = movmatrix_trans(pack_f16x2(y[2], y[3]));
  }
  if (!tail) {
#pragma unroll
    for (int x = 0; x < H; ++x) value_product<D>(a.o[0], vt, row + 16 * x, half, kPick, kPick, pb[x]);
    return;
  }
#pragma unroll
  for (int x = 0; x < H; ++x) {
    const int left = len - slice - 16 * x;
    // A NaN in a slot that only some members see: their zero weights must not meet it, so each
    // member's column is kept from a product of its own, over the slots it sees. Never taken on
    // sound values.
    if (p.chain != nullptr && left > 0 && any_nan<D>(vt, row - (lane & 15) + 16 * x, lane)) {
#pragma unroll 1
      for (int col = 0; col < p.width; ++col) {
        const int t = (chunk * p.width + col) / p.groups;
        bool seen[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          seen[e] = sees(slice + 16 * x + 2 * c + (e & 1) + (e >> 1) * 8, len, position, t, chain);
        float o[D / 16][4] = {};
        value_product<D>(o, vt, row + 16 * x, half, pick_slots(seen[0], seen[1]), pick_slots(seen[2], seen[3]), pb[x]);
        if (col >> 1 != c) continue;  // this thread's columns are 2c and 2c + 1
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          (col & 1 ? a.o[0][k][1] : a.o[0][k][0]) += col & 1 ? o[k][1] : o[k][0];
          (col & 1 ? a.o[0][k][3] : a.o[0][k][2]) += col & 1 ? o[k][3] : o[k][2];
        }
      }
      continue;
    }
    // slots past the row hold anything, NaN codes too: a zero weight must not meet them
    value_product<D>(a.o[0], vt, row + 16 * x, half, pick_slots(2 * c < left, 2 * c + 1 < left),
                     pick_slots(2 * c + 8 < left, 2 * c + 9 < left), pb[x]);
  }
}

// More column groups: warp w scores slice w, then multiplies every slice's weights by its 16 dims (with
// head_dim 64 half of the slices: warps w and w + 4 share dims).
template <int D, int NG>
__device__ __forceinline__ void attend_tile(State<D, NG>& a, const Params& p, const Smem<D, NG>& sm,
                                            const float* scales, uint32_t kt, uint32_t vt, int k, bool fresh, int first,
                                            int len, int position, int chain, int chunk, int warp, int lane) {
  using S = Smem<D, NG>;
  const int g = lane >> 2, c = lane & 3;
  const int slice = first + warp * 16;
  const int clear = p.chain != nullptr ? position + 1 : len;  // slots that every member sees
  auto token = [&](int col) { return reinterpret_cast<const int*>(sm.query + S::kFragments)[NG * 8 + col]; };
  float s[NG][4];
#pragma unroll
  for (int n = 0; n < NG; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
  float ks = 0.f, lv = 0.f;
  if (slice < len) {
    const int row = warp * 16 + (lane & 15), half = lane >> 4;
    const uint4* query = reinterpret_cast<const uint4*>(sm.query) + lane;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      uint32_t r[4], k0[4], k1[4];
      ldmatrix_x4(kt + swizzled<D>(row, 2 * i + half), r[0], r[1], r[2], r[3]);
      q8::e4m3x4_to_f16x4(r[0], k0[0], k0[2]);
      q8::e4m3x4_to_f16x4(r[1], k0[1], k0[3]);
      q8::e4m3x4_to_f16x4(r[2], k1[0], k1[2]);
      q8::e4m3x4_to_f16x4(r[3], k1[1], k1[3]);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const uint4 q = query[(n * (D / 32) + i) * 32];
        mma_f16(s[n], k0[0], k0[1], k0[2], k0[3], q.x, q.y);
        mma_f16(s[n], k1[0], k1[1], k1[2], k1[3], q.z, q.w);
      }
    }
    ks = scales[warp];
    lv = log2_scale(scales[kSlices + warp]);
  }
  uint32_t hidden = 0;  // a bit per score
  if (slice + 16 > clear) {
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!sees(slice + g + (e >> 1) * 8, len, position, token(n * 8 + 2 * c + (e & 1)), chain))
          hidden |= 1u << (n * 4 + e);
  }
  // The slice's weights, into this warp's half of its pair's fragments
  uint2* weights =
      reinterpret_cast<uint2*>(sm.weights + k % 2 * (S::kWeights / 2)) + warp / 2 * NG * 64 + lane * 2 + warp % 2;
  float l[NG][2];
  // Weights on the pivots so far: one barrier a tile, unless they have to move, as in a run's first tile. They
  // move once at most: they are worked out with the same roundings as x and y, which are monotone, so that no x is
  // above 0 then and no y above 8, kLift rounded to a step of at most 8 (where steps are 16 and more it rounds to
  // 0). A product fused into x would break that where scores round by more than kSlack.
  for (;; fresh = false) {
    if (!fresh) {
      float top = 0.f;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float x[4], y[4];  // s - m and s - m + log2 vs - r
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = __fmul_rn(s[n][e], a.qs[n][e & 1] * ks) - a.m[n][e & 1];
          y[e] = x[e] + lv - a.r[n][e & 1];
        }
        if (hidden != 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (hidden >> (n * 4 + e) & 1) x[e] = y[e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(x[e], y[e]));
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = ex2(y[e]);
        weights[n * 64] = make_uint2(movmatrix_trans(pack_f16x2(y[0], y[1])), movmatrix_trans(pack_f16x2(y[2], y[3])));
        l[n][0] = ex2(x[0]) + ex2(x[2]);
        l[n][1] = ex2(x[1]) + ex2(x[3]);
      }
      if (!consumers_any<NG>(top > kSlack && sm.misc[4 + warp] != k + 1)) break;
    }
    if (lane == 0) sm.misc[4 + warp] = k + 1;  // once a tile, whatever the scores
    __syncwarp();
    // [warp][column], where the last tile's weights were: everyone has multiplied by them (a run's first
    // tile: start_unit)
    float2* tops = reinterpret_cast<float2*>(sm.weights + (k + 1) % 2 * (S::kWeights / 2));
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float by = a.qs[n][e] * ks;
        float top = fmaxf(hidden >> (n * 4 + e) & 1 ? -INFINITY : __fmul_rn(s[n][e], by),
                          hidden >> (n * 4 + e + 2) & 1 ? -INFINITY : __fmul_rn(s[n][e + 2], by));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        if (g == 0) tops[warp * NG * 8 + n * 8 + 2 * c + e] = make_float2(top, lv);
      }
    consumers_sync<NG>();
    // of column `lane`: its m, which becomes the largest score if that is larger, and the largest score - m +
    // log2 vs, with the roundings of the loop above, less kLift
    float m_lane = kNone, r_lane = -INFINITY;
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float m = __shfl_sync(0xffffffffu, a.m[n][e], (lane & 7) >> 1);
        if (lane / 8 == n && lane % 2 == e) m_lane = m;
      }
    if (lane < NG * 8) {
#pragma unroll
      for (int w = 0; w < kConsumers<NG>; ++w) m_lane = fmaxf(m_lane, tops[w * NG * 8 + lane].x);
#pragma unroll
      for (int w = 0; w < kConsumers<NG>; ++w) {
        const float2 t = tops[w * NG * 8 + lane];
        r_lane = fmaxf(r_lane, t.x - m_lane + t.y);
      }
      r_lane -= kLift;
    }
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float m = __shfl_sync(0xffffffffu, m_lane, n * 8 + 2 * c + e), by = a.m[n][e] - m;
        const float r = fmaxf(shifted(a.r[n][e], by), __shfl_sync(0xffffffffu, r_lane, n * 8 + 2 * c + e));
        const float fl = ex2(by), fo = ex2(a.r[n][e] + by - r);
        a.m[n][e] = m;
        a.r[n][e] = r;
        a.l[n][e] *= fl;
        a.o[n][0][e] *= fo;
        a.o[n][0][e + 2] *= fo;
      }
  }
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    a.l[n][0] += l[n][0];
    a.l[n][1] += l[n][1];
  }
  constexpr int kChunks = D / 16, kShare = kSlices * kChunks / kConsumers<NG>;
  const int dims = warp % kChunks, from = warp / kChunks * kShare;
  const uint4* pairs = reinterpret_cast<const uint4*>(sm.weights + k % 2 * (S::kWeights / 2)) + lane;
  if (first + kTile <= clear) {
#pragma unroll
    for (int y0 = 0; y0 < kShare; y0 += 2) {
      uint32_t r[4];
      ldmatrix_x4_trans(vt + swizzled<D>(16 * (from + y0) + lane, dims), r[0], r[1], r[2], r[3]);
      uint32_t f0[4], f1[4];
      value_fragments(f0, r[0], r[1], kPick, kPick);
      value_fragments(f1, r[2], r[3], kPick, kPick);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const uint4 pb = pairs[((from + y0) / 2 * NG + n) * 32];
        mma_f16(a.o[n][0], f0[0], f0[1], f0[2], f0[3], pb.x, pb.y);
        mma_f16(a.o[n][0], f1[0], f1[1], f1[2], f1[3], pb.z, pb.w);
      }
    }
    return;
  }
  // the row's last tiles; kept small, since their code shares the instruction cache with the loop above
#pragma unroll 1
  for (int y = from; y < from + kShare; ++y) {
    const int at = first + 16 * y, left = len - at;
    if (left <= 0) break;
    uint32_t r[4], f[4];
    ldmatrix_x4_trans(vt + swizzled<D>(16 * y + (lane & 15), dims), r[0], r[1], r[2], r[3]);  // twice the slice
    bool nan = false;
    if (at + 16 > clear && p.chain != nullptr && lane < 16 && lane < left) {
      const uint32_t src = vt + swizzled<D>(16 * y + lane, dims);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(src + 4 * i) : "memory");
        nan = nan || has_nan(w);
      }
    }
    if (__any_sync(0xffffffffu, nan)) {
      // A NaN in a slot that only some members see: as above, a product for each of them.
#pragma unroll 1
      for (int col = 0; col < p.width; ++col) {
        const int t = token(col), group = col / 8;
        bool seen[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) seen[e] = sees(at + 2 * c + (e & 1) + (e >> 1) * 8, len, position, t, chain);
        value_fragments(f, r[0], r[1], pick_slots(seen[0], seen[1]), pick_slots(seen[2], seen[3]));
        const uint2 pb = reinterpret_cast<const uint2*>(pairs + (y / 2 * NG + group) * 32)[y % 2];
        float o[4] = {};
        mma_f16(o, f[0], f[1], f[2], f[3], pb.x, pb.y);
        if ((col & 7) >> 1 != c) continue;  // this thread's columns are 2c and 2c + 1
#pragma unroll
        for (int n = 0; n < NG; ++n)
          if (n == group) {
            a.o[n][0][0] += col & 1 ? 0.f : o[0];
            a.o[n][0][1] += col & 1 ? o[1] : 0.f;
            a.o[n][0][2] += col & 1 ? 0.f : o[2];
            a.o[n][0][3] += col & 1 ? o[3] : 0.f;
          }
      }
      continue;
    }
    // slots past the row hold anything, NaN codes too: a zero weight must not meet them
    value_fragments(f, r[0], r[1], pick_slots(2 * c < left, 2 * c + 1 < left),
                    pick_slots(2 * c + 8 < left, 2 * c + 9 < left));
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const uint2 pb = reinterpret_cast<const uint2*>(pairs + (y / 2 * NG + n) * 32)[y % 2];
      mma_f16(a.o[n][0], f[0], f[1], f[2], f[3], pb.x, pb.y);
    }
  }
}

// Sums the consumer warps' states in warp order: sink(in_chunk, d, O, r, m, l) for every live column and
// dim.
template <int D, typename Sink>
__device__ __forceinline__ void reduce_warps(State<D, 1>& a, const Smem<D, 1>& sm, int members, int warp, int lane,
                                             Sink sink) {
  constexpr int NG = 1, kWarps = kConsumers<1>;
  float *red_o = sm.red_o, *red_stats = sm.red_stats;
  const int g = lane >> 2, c = lane & 3, tid = threadIdx.x;
#pragma unroll
  for (int n = 0; n < NG; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = a.l[n][e];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
      if (g == 0) {
        float* st = red_stats + (warp * NG * 8 + n * 8 + 2 * c + e) * 3;
        st[0] = a.r[n][e], st[1] = a.m[n][e], st[2] = l;
      }
    }
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {  // half of the dims each
    constexpr int n = 0;
    const int k0 = pass * (D / 32);
    if (pass > 0) consumers_sync<NG>();  // the last pass's reads are done
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      float* dst = red_o + (warp * (D / 2) + 16 * k + 2 * g) * 8 + 2 * c;
      *reinterpret_cast<float2*>(dst) = make_float2(a.o[n][k0 + k][0], a.o[n][k0 + k][1]);
      *reinterpret_cast<float2*>(dst + 8) = make_float2(a.o[n][k0 + k][2], a.o[n][k0 + k][3]);
    }
    consumers_sync<NG>();
#pragma unroll
    for (int e0 = 0; e0 < 8 * (D / 2); e0 += kWarps * 32) {
      const int e = e0 + tid, col = e / (D / 2), d = e % (D / 2), in_chunk = n * 8 + col;
      if (in_chunk >= members) break;
      const float* st = red_stats + in_chunk * 3;
      float m = kNone, r = kNone, O = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, st[w * NG * 24 + 1]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) r = fmaxf(r, st[w * NG * 24] + (st[w * NG * 24 + 1] - m));
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float by = st[w * NG * 24 + 1] - m;
        O += red_o[(w * (D / 2) + d) * 8 + col] * ex2(st[w * NG * 24] + by - r);
        l += st[w * NG * 24 + 2] * ex2(by);
      }
      sink(in_chunk, k0 * 16 + d, O, r, m, l);
    }
  }
}

// More column groups: what the warps tell each other after `k` tiles, where the next tile's weights would go.
template <int D, int NG>
struct Totals {
  float* l;        // [warp][column]: denominators of the warp's slices
  float2* pivots;  // [column]: r, m
  float4* stats;   // [column]: r, m, l
  __device__ Totals(const Smem<D, NG>& sm, int k) {
    l = reinterpret_cast<float*>(sm.weights + k % 2 * (Smem<D, NG>::kWeights / 2));
    pivots = reinterpret_cast<float2*>(l + kConsumers<NG> * NG * 8);
    stats = reinterpret_cast<float4*>(pivots + NG * 8);
  }
  // A column's r, m and l, summed in warp order.
  __device__ float4 column(int col) const {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kConsumers<NG>; ++w) sum += l[w * NG * 8 + col];
    return make_float4(pivots[col].x, pivots[col].y, sum, 0.f);
  }
};

// Each warp ends with O of its dims; with head_dim 64 the first of the two that share dims.
template <int D, int NG>
__device__ __forceinline__ void join_warps(State<D, NG>& a, const Smem<D, NG>& sm, const Totals<D, NG>& totals,
                                           int warp, int lane) {
  constexpr int kChunks = D / 16;
  const int g = lane >> 2, c = lane & 3;
  float4* other = reinterpret_cast<float4*>(sm.red_o) + warp % kChunks * NG * 32 + lane;
#pragma unroll
  for (int n = 0; n < NG; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = n * 8 + 2 * c + e;
      float l = a.l[n][e];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
      if (g == 0) totals.l[warp * NG * 8 + col] = l;
      if (g == 0 && warp == 0) totals.pivots[col] = make_float2(a.r[n][e], a.m[n][e]);
    }
    if (warp >= kChunks) other[n * 32] = make_float4(a.o[n][0][0], a.o[n][0][1], a.o[n][0][2], a.o[n][0][3]);
  }
  consumers_sync<NG>();
  if (kChunks < kConsumers<NG> && warp < kChunks) {
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const float4 v = other[n * 32];
      a.o[n][0][0] += v.x, a.o[n][0][1] += v.y, a.o[n][0][2] += v.z, a.o[n][0][3] += v.w;
    }
  }
}

// sink(column, dim, value, value of the next dim) for the live columns of this thread.
template <int D, int NG, typename Sink>
__device__ __forceinline__ void each_pair(const State<D, NG>& a, int members, int warp, int lane, Sink sink) {
  if (warp >= D / 16) return;
#pragma unroll
  for (int n = 0; n < NG; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = n * 8 + 2 * (lane & 3) + e;
      if (col < members) sink(col, 16 * warp + 2 * (lane >> 2), a.o[n][0][e], a.o[n][0][e + 2]);
    }
}

template <int D>
__device__ __forceinline__ __nv_bfloat16* out_row(const Params& p, int b, int h, int member) {
  const int t = member / p.groups, head = h * p.groups + member - t * p.groups;
  return p.out + ((static_cast<size_t>(b) * p.tokens + t) * p.q_heads + head) * D;
}
template <int D>
__device__ __forceinline__ void write_out(const Params& p, int b, int h, int member, int d, float O, float r, float l) {
  out_row<D>(p, b, h, member)[d] = __float2bfloat16_rn(finished(O, r, l));
}

template <int D, int NG>
__device__ __forceinline__ void init_barriers(const Smem<D, NG>& sm, const CUtensorMap* kmap, const CUtensorMap* vmap) {
  for (int s = 0; s < Smem<D, NG>::kStages; ++s) {
    mbar_init(&sm.full[s], 1 + kScales);  // the tiles' bytes and the scale copies
    mbar_init(&sm.empty[s], kConsumers<NG>);
  }
  fence_barrier_init();
  prefetch_tensormap(kmap);
  prefetch_tensormap(vmap);
  for (int i = 3; i < 4 + kSlices; ++i) sm.misc[i] = 0;
}

// Producer warp: tile j of `pair` into stage k % stages. False after an abort.
template <int D, int NG>
__device__ __forceinline__ bool load_tile(const Smem<D, NG>& sm, const Params& p, const CUtensorMap* kmap,
                                          const CUtensorMap* vmap, int k, int pair, int j, int lane) {
  using S = Smem<D, NG>;
  const int s = k % S::kStages;
  bool ok = sm.misc[3] == 0;
  if (ok && k >= S::kStages && !mbar_wait_bounded(&sm.empty[s], ((k / S::kStages) - 1) & 1)) {
    raise_error(p.err, kErrTimeoutEmpty);
    sm.misc[3] = 1;
    ok = false;
  }
  if (!__all_sync(0xffffffffu, ok)) return false;
  if (lane == 0) {
    uint8_t* kt = sm.ring + s * 2 * S::kTileBytes;
    const int row = pair * p.capacity + j * kTile;
    mbar_arrive_expect_tx(&sm.full[s], 2 * S::kTileBytes);
    tma_load_2d(kt, kmap, &sm.full[s], 0, row);
    tma_load_2d(kt + S::kTileBytes, vmap, &sm.full[s], 0, row);
  }
  if (lane < kScales) {
    const int i = min((j * kTile + (lane % kSlices) * 16) / p.block, p.blocks - 1);
    const float* src = (lane < kSlices ? p.key_scales : p.value_scales) + static_cast<size_t>(pair) * p.blocks + i;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(sm.scales + s * kScales + lane)), "l"(src)
                 : "memory");
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&sm.full[s])) : "memory");
  }
  return true;
}

// After an abort: copies in flight land before the CTA's shared memory is released.
template <int D, int NG>
__device__ __forceinline__ void drain(const Smem<D, NG>& sm, int issued) {
  constexpr int NS = Smem<D, NG>::kStages;
  if (sm.misc[3] != 0)
    for (int k = issued > NS ? issued - NS : 0; k < issued; ++k) mbar_wait_bounded(&sm.full[k % NS], (k / NS) & 1);
}

// Consumer warp: tile j of a row with `len` slots from stage k % stages. After an abort the barriers
// that follow are still taken, on whatever the stage holds.
template <int D, int NG>
__device__ __forceinline__ void consume_tile(State<D, NG>& a, const Smem<D, NG>& sm, const Params& p, int k,
                                             bool fresh, int j, int len, int position, int chain, int chunk, int warp,
                                             int lane) {
  using S = Smem<D, NG>;
  const int s = k % S::kStages;
  if (sm.misc[3] == 0 && !mbar_wait_bounded(&sm.full[s], (k / S::kStages) & 1)) {
    raise_error(p.err, kErrTimeoutFull);
    sm.misc[3] = 1;
  }
  __syncwarp();
  const uint32_t kt = smem_u32(sm.ring + s * 2 * S::kTileBytes);
  attend_tile(a, p, sm, sm.scales + s * kScales, kt, kt + S::kTileBytes, k, fresh, j * kTile, len, position, chain,
              chunk, warp, lane);
  __syncwarp();
  if (lane == 0) mbar_arrive(&sm.empty[s]);
}

__device__ __forceinline__ int first_position(const Params& p, int b) {
  return static_cast<int>(min(p.position[p.per_row ? b : 0], static_cast<int64_t>(p.capacity)));
}

// Tokens of row b's chain: all of a longer one, none of a negative one.
__device__ __forceinline__ int chain_of(const Params& p, int b) {
  if (p.chain == nullptr) return 1;
  return static_cast<int>(max(static_cast<int64_t>(0), min(p.chain[b], static_cast<int64_t>(p.tokens))));
}

// ------------------------------------------------------------------------------ cluster form
template <int D, int NG>
__global__ void __launch_bounds__(kThreads<NG>, 2)
    cluster_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                   const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  const Smem<D, NG> sm(smem_raw);
  constexpr int kWarps = kConsumers<NG>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = gridDim.x, rank = blockIdx.x;  // cluster dims (C, 1, 1)
  const int pair = blockIdx.y / p.chunks, chunk = blockIdx.y % p.chunks;
  const int b = pair / p.kv_heads, h = pair % p.kv_heads;
  cluster_arrive_relaxed();  // this CTA runs: its shared memory may be written once all have said so
  if (warp == kWarps && lane == 0) init_barriers(sm, &kmap, &vmap);
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int len = row_length(p, b), n = tiles_of(len);
  const int count = n > rank ? (n - rank + C - 1) / C : 0;  // tiles rank, rank + C, ...
  if (warp == kWarps) {
    int k = 0;
    while (k < count && load_tile(sm, p, &kmap, &vmap, k, pair, rank + k * C, lane)) ++k;
    drain(sm, k);
    __syncwarp();
    cluster_wait();  // every thread of the cluster takes the same two barrier phases
    cluster_sync();
    return;
  }
  const int position = first_position(p, b);
  const int chain = chain_of(p, b);
  const int members = min(p.width, p.members - chunk * p.width);
  State<D, NG> a;
  start_unit<D, NG>(a, p, sm.query, b, h, chunk, warp, lane);
  for (int k = 0; k < count; ++k)
    consume_tile(a, sm, p, k, k == 0, rank + k * C, len, position, chain, chunk, warp, lane);
  // values of an owner: an even number, so that pairs stay together; e / share for e < 2^16
  const int total = members * D, share = (total + 2 * C - 1) / (2 * C) * 2;
  const uint32_t magic = (0xffffffffu / share) + 1;
  auto push_stats = [&](int col, int to, float r, float m, float l) {
    const uint32_t at = map_shared(smem_u32(sm.recv_stats + (rank * NG * 8 + col) * 3), to);
    st_cluster_f32(at, r);
    st_cluster_f32(at + 4, m);
    st_cluster_f32(at + 8, l);
  };
  auto push_to = [&](int e) {
    const int owner = __umulhi(e, magic);
    return map_shared(smem_u32(sm.recv_o + rank * share + e - owner * share), owner);
  };
  if constexpr (NG == 1) {
    cluster_wait();  // every CTA of the cluster runs
    reduce_warps(a, sm, members, warp, lane, [&](int col, int d, float O, float r, float m, float l) {
      st_cluster_f32(push_to(col * D + d), O);
      if (d < C) push_stats(col, d, r, m, l);  // one thread per rank passes this column's statistics on
    });
  } else {
    const Totals<D, NG> totals(sm, count);
    join_warps(a, sm, totals, warp, lane);
    cluster_wait();  // every CTA of the cluster runs
    each_pair(a, members, warp, lane, [&](int col, int d, float O0, float O1) {
      st_cluster_f32x2(push_to(col * D + d), O0, O1);
    });
    if (lane < members) {
      const float4 st = totals.column(lane);
      for (int to = warp; to < C; to += kWarps) push_stats(lane, to, st.x, st.y, st.z);
    }
  }
  cluster_sync();  // every partial has landed; nobody touches another CTA's memory after this
  // a rank's weight in a column's output, in place of its r; a column that sees nothing, or only zero
  // values, is marked by l = 0
  for (int c0 = 0; c0 < NG * 8; c0 += kWarps * 2) {
    const int col = c0 + static_cast<int>(threadIdx.x) / 16, q = threadIdx.x & 15;
    static_assert(kMaxCluster == 16, "a rank per lane of half a warp");
    const bool on = col < members && q < C;
    float* st = sm.recv_stats + (q * NG * 8 + col) * 3;
    const float r_q = on ? st[0] : kNone, m_q = on ? st[1] : kNone;
    float m = m_q;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float by = m_q - m;
    float r = shifted(r_q, by);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, off));
    float l = on ? st[2] * ex2(by) : 0.f;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    if (on) {
      st[0] = ex2(r_q + by - r) * finished(1.f, r, l);
      st[2] = r == kNone && l > 0.f ? 0.f : l;
    }
  }
  consumers_sync<NG>();
  const int low = rank * share, high = min(total, low + share);
  for (int e = low + 2 * static_cast<int>(threadIdx.x); e < high; e += 2 * kWarps * 32) {
    const int col = e / D;
    const float* st = sm.recv_stats + col * 3;
    float O0 = 0.f, O1 = 0.f;
    for (int q = 0; q < C; ++q) {
      const float2 v = *reinterpret_cast<const float2*>(sm.recv_o + q * share + e - low);
      const float w = st[q * NG * 8 * 3];
      O0 += v.x * w;
      O1 += v.y * w;
    }
    const bool none = st[2] == 0.f;
    *reinterpret_cast<__nv_bfloat162*>(out_row<D>(p, b, h, chunk * p.width + col) + e % D) =
        __floats2bfloat162_rn(none ? 0.f : O0, none ? 0.f : O1);
  }
}

// --------------------------------------------------------------------------- persistent form
template <int D, int NG>
__global__ void __launch_bounds__(kThreads<NG>, 2)
    persistent_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                      const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  const Smem<D, NG> sm(smem_raw);
  constexpr int kWarps = kConsumers<NG>;
  const int* cum = sm.cum;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int B = p.batch, per_row = p.kv_heads * p.chunks;  // units of a row
  if (warp == kWarps && lane == 0) init_barriers(sm, &kmap, &vmap);
  pdl_wait();
  pdl_trigger();
  // ---- plan: tiles before each row, this CTA's slice and where it begins ----
  if (warp == 0) {
    int running = 0;
    if (lane == 0) sm.cum[0] = 0;
    for (int b0 = 0; b0 < B; b0 += 32) {
      const int b = b0 + lane;
      int x = b < B ? tiles_of(row_length(p, b)) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (b < B) sm.cum[b + 1] = running + x;
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
        const int off = static_cast<int>(t0 - static_cast<long long>(per_row) * cum[b]);  // < 2^31: tiles of one row
        sm.misc[0] = b;
        sm.misc[1] = off / n;
        sm.misc[2] = off % n;
      }
      if (__any_sync(0xffffffffu, hit)) break;
    }
  }
  __syncthreads();
  int b = sm.misc[0], u = sm.misc[1], j = sm.misc[2];  // row, unit of the row (KV head, chunk), tile
  int n = cum[b + 1] - cum[b];

  if (warp == kWarps) {
    int k = 0;
    for (; k < count; ++k) {
      if (!load_tile(sm, p, &kmap, &vmap, k, b * p.kv_heads + u / p.chunks, j, lane)) break;
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
    drain(sm, k);
    return;
  }

  int run_first = 0, len = 0, position = 0, chain = 1;
  bool starts = true;
  State<D, NG> a;
  for (int k = 0; k < count; ++k) {
    if (starts) {
      n = cum[b + 1] - cum[b];
      len = row_length(p, b);
      position = first_position(p, b);
      chain = chain_of(p, b);
      run_first = j;
      start_unit<D, NG>(a, p, sm.query, b, u / p.chunks, u % p.chunks, warp, lane);
    }
    consume_tile(a, sm, p, k, starts, j, len, position, chain, u % p.chunks, warp, lane);
    const int run_b = b, run_u = u, run_last = j;
    starts = k == count - 1;
    if (++j == n) {
      j = 0;
      starts = true;
      if (++u == per_row) {
        u = 0;
        do ++b;
        while (b < B && cum[b + 1] == cum[b]);
      }
    }
    if (!starts) continue;
    // the run ends: its unit's output, or partials for the merge
    const int h = run_u / p.chunks, chunk = run_u % p.chunks;
    const size_t slot = blockIdx.x + static_cast<size_t>(run_b) * per_row + run_u;
    const bool whole = run_first == 0 && run_last == n - 1;
    const int members = min(p.width, p.members - chunk * p.width);
    if constexpr (NG == 1) {
      consumers_sync<NG>();  // the last run's reductions are read
      reduce_warps(a, sm, members, warp, lane, [&](int col, int d, float O, float r, float m, float l) {
        if (whole) {
          write_out<D>(p, run_b, h, chunk * p.width + col, d, O, r, l);
        } else {
          p.acc[(slot * p.width + col) * D + d] = O;
          if (d == 0) p.stats[slot * p.width + col] = make_float4(r, m, l, 0.f);
        }
      });
    } else {
      const Totals<D, NG> totals(sm, k + 1);
      join_warps(a, sm, totals, warp, lane);
      if (warp == 0 && lane < members) {
        const float4 st = totals.column(lane);
        if (whole)
          totals.stats[lane] = st;
        else
          p.stats[slot * p.width + lane] = st;
      }
      if (whole) consumers_sync<NG>();
      each_pair(a, members, warp, lane, [&](int col, int d, float O0, float O1) {
        if (whole) {
          const float4 st = totals.stats[col];
          __nv_bfloat16* out = out_row<D>(p, run_b, h, chunk * p.width + col) + d;
          *reinterpret_cast<__nv_bfloat162*>(out) =
              __floats2bfloat162_rn(finished(O0, st.x, st.z), finished(O1, st.x, st.z));
        } else {
          *reinterpret_cast<float2*>(p.acc + (slot * p.width + col) * D + d) = make_float2(O0, O1);
        }
      });
    }
  }
}

// One CTA per (unit, 8 columns): merges the runs of the CTAs that shared the unit, in CTA order, and
// writes the zeros of empty rows. The plan is worked out before the wait (the positions were
// there before the first launch passed its own); after it a unit of at most four runs takes one
// round trip to L2: statistics and accumulators are loaded together.
constexpr int kMergeThreads = 256;
constexpr int kMergeRuns = 4;

template <int D>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const __grid_constant__ Params p) {
  __shared__ int s_before, s_total;
  const int per_row = p.kv_heads * p.chunks;
  const int b = blockIdx.x / per_row, u = blockIdx.x % per_row;
  const int h = u / p.chunks, chunk = u % p.chunks, col0 = blockIdx.y * 8;
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
  const int members = min(8, min(p.width, p.members - chunk * p.width) - col0);
  const long long T = static_cast<long long>(per_row) * s_total;
  const long long first = static_cast<long long>(per_row) * s_before + static_cast<long long>(u) * n;
  const int lo = n > 0 ? slice_owner(T, first, p.ctas) : 0, hi = n > 0 ? slice_owner(T, first + n - 1, p.ctas) : 0;
  const bool sparse = T < p.ctas;  // some slices are empty: their CTAs wrote nothing
  pdl_wait();
  pdl_trigger();
  if (n > 0 && lo == hi) return;  // one run covered the unit and wrote its output
  for (int e = threadIdx.x; e < members * D; e += kMergeThreads) {
    const int col = col0 + e / D, d = e % D;
    float r = kNone, m = kNone, O = 0.f, l = 0.f;
    if (n > 0) {
      const float4* st = p.stats + (static_cast<size_t>(lo) + blockIdx.x) * p.width + col;
      const float* acc = p.acc + ((static_cast<size_t>(lo) + blockIdx.x) * p.width + col) * D + d;
      for (int i0 = 0; i0 <= hi - lo; i0 += kMergeRuns) {
        float4 s[kMergeRuns];
        float v[kMergeRuns];
        float to_m = m;
#pragma unroll
        for (int i = 0; i < kMergeRuns; ++i) {
          const int run = i0 + i;
          const bool on = run <= hi - lo &&
                          !(sparse && slice_start(T, lo + run, p.ctas) == slice_start(T, lo + run + 1, p.ctas));
          s[i] = on ? __ldcg(st + static_cast<size_t>(run) * p.width) : make_float4(kNone, kNone, 0.f, 0.f);
          v[i] = on ? __ldcg(acc + static_cast<size_t>(run) * p.width * D) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < kMergeRuns; ++i) to_m = fmaxf(to_m, s[i].y);
        float to_r = shifted(r, m - to_m);
#pragma unroll
        for (int i = 0; i < kMergeRuns; ++i) to_r = fmaxf(to_r, s[i].x + (s[i].y - to_m));
        O *= ex2(r + (m - to_m) - to_r);
        l *= ex2(m - to_m);
        r = to_r;
        m = to_m;
#pragma unroll
        for (int i = 0; i < kMergeRuns; ++i) {
          O += v[i] * ex2(s[i].x + (s[i].y - m) - r);
          l += s[i].z * ex2(s[i].y - m);
        }
      }
    }
    write_out<D>(p, b, h, chunk * p.width + col, d, O, r, l);
  }
}

// Columns of a unit: the least number of equal member groups of at most 32 columns.
void chunk_members(Params* p) {
  constexpr int kMost = 32;
  p->members = p->tokens * p->groups;
  p->chunks = (p->members + kMost - 1) / kMost;
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

int shape(Params* p, const fb_q8_cache& cache, int tokens, int q_heads) {
  const int batch = cache.batch, kv_heads = cache.kv_heads, capacity = cache.capacity;
  const int head_dim = cache.head_dim, block = cache.block;
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
  p->ctas = 2 * sm_count();
  chunk_members(p);
  const long long row_units = static_cast<long long>(kv_heads) * p->chunks;
  return batch * row_units >= (1ll << 31) || row_units * tiles_of(capacity) >= (1ll << 31) ? FB_ERR_SHAPE : FB_OK;
}

constexpr int kMaxDevices = 64;

template <int D, int NG>
bool configure() {
  static std::atomic<bool> configured[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev < kMaxDevices && configured[dev]) return true;
  const int bytes = Smem<D, NG>::kTotal;
  if (cudaFuncSetAttribute(cluster_kernel<D, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
      cudaFuncSetAttribute(persistent_kernel<D, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return false;
  if (cudaFuncSetAttribute(cluster_kernel<D, NG>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    cudaGetLastError();  // no clusters above 8: the occupancy query then reports none
  if (dev < kMaxDevices) configured[dev] = true;
  return true;
}

// Clusters of c CTAs that the device holds at once (0 if unknown), kept per device.
template <int D, int NG>
int resident_clusters(int c) {
  static std::atomic<int> cache[kMaxDevices][kMaxCluster + 1];  // count + 1; 0: not asked
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < kMaxDevices && cache[dev][c] != 0) return cache[dev][c] - 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c, 1);
  cfg.blockDim = dim3(kThreads<NG>);
  cfg.dynamicSmemBytes = Smem<D, NG>::kTotal;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, cluster_kernel<D, NG>, &cfg) != cudaSuccess || n < 0) {
    cudaGetLastError();
    n = 0;
  }
  if (dev < kMaxDevices) cache[dev][c] = n + 1;
  return n;
}

// Tiles of the cache up to which units past one an SM get a CTA each; beyond, the persistent form's slices, whose
// merge and partials cost more than uneven rows do at few tiles. us, CTA per unit against slices, rows of 8 KV heads:
// decode of 64 x 4101 slots 86 against 92 (lengths from an eighth on 63 against 70), 64 x 4608 93 against 102, 24 x 4101
// 38 against 43 (34 against 33), and past the border 64 x 8197 159 against 172 (115 against 108), 24 x 8197 69 against 72
// (63 against 50): even rows of any length would stay with a CTA each, ragged ones would not. Verify blocks of 5
// tokens, 20 members: 20 x 2053 44 against 46, 32 x 4101 77 against 99, 64 x 4101 150 against 176, 20 x 8197 144 against
// 110; the rule is wrong for 20 x 4101, whose 160 units leave most SMs with one of two CTAs: 77 against 68 (66 against 53).
constexpr int kUnitTiles = 36;

// The cluster size of a launch, 0 for the persistent form. Up to a unit per SM: the largest whose clusters are
// all resident at once, no larger than the cache has tiles. us by size (0: persistent): 64 units of 33 tiles, 20
// members 0 43, 1 56, 2 33, 4 28 (taken), 8 36; 128 units of 65 tiles 0 54, 1 53, 2 45 (taken), 4 49; 8 units of 16 tiles 4
// 7.0, 8 5.8, 16 6.1 (taken); 10 units of 8 tiles, D = 64, 4 5.1, 8 4.6 (taken); 16 units of 7 tiles, 32 members, D = 64
// 4 9.7, 7 10.1 (taken). Near the top a size is within 0.4 of the next: the merge grows as the tiles shrink.
template <int D, int NG>
int cluster_size(const Params& p) {
  const int units = p.batch * p.kv_heads * p.chunks, tiles = tiles_of(p.capacity);
  if (units > 65535) return 0;
  if (units > sm_count()) return tiles <= kUnitTiles ? 1 : 0;
  for (int c = tiles < kMaxCluster ? tiles : kMaxCluster; c >= 1; --c)
    if (resident_clusters<D, NG>(c) >= units) return c;
  return 0;
}

template <int D, int NG>
int launch(const CUtensorMap& km, const CUtensorMap& vm, const Params& p, int cluster, cudaStream_t stream) {
  const int units = p.batch * p.kv_heads * p.chunks;
  constexpr int bytes = Smem<D, NG>::kTotal;
  if (cluster > 0)
    return launch_ex(cluster_kernel<D, NG>, dim3(cluster, units), dim3(kThreads<NG>), bytes, stream, cluster, km, vm,
                     p);
  const int st = launch_ex(persistent_kernel<D, NG>, dim3(p.ctas), dim3(kThreads<NG>), bytes, stream, 1, km, vm, p);
  if (st != FB_OK) return st;
  return launch_ex(merge_kernel<D>, dim3(units, (p.width + 7) / 8), dim3(kMergeThreads), 0, stream, 1, p);
}

// Calls f(head dim, column groups) as compile-time constants.
template <int D, typename F>
auto with_groups(const Params& p, F f) {
  using std::integral_constant;
  if (p.width <= 8) return f(integral_constant<int, D>(), integral_constant<int, 1>());
  if (p.width <= 16) return f(integral_constant<int, D>(), integral_constant<int, 2>());
  if (p.width <= 24) return f(integral_constant<int, D>(), integral_constant<int, 3>());
  return f(integral_constant<int, D>(), integral_constant<int, 4>());
}
template <typename F>
auto with_shape(const Params& p, int head_dim, F f) {
  return head_dim == 128 ? with_groups<128>(p, f) : with_groups<64>(p, f);
}

// The cluster size a shape runs with (0: persistent), or an error.
int plan(const Params& p, int head_dim) {
  return with_shape(p, head_dim, [&](auto d, auto ng) {
    constexpr int D = decltype(d)::value, NG = decltype(ng)::value;
    return configure<D, NG>() ? cluster_size<D, NG>(p) : static_cast<int>(FB_ERR_LAUNCH);
  });
}

}  // namespace attn8
}  // namespace fb

using namespace fb;

extern "C" size_t fb_attention_q8_workspace(const fb_q8_cache* cache, int tokens, int q_heads) {
  attn8::Params p;
  if (cache == nullptr || attn8::shape(&p, *cache, tokens, q_heads) != FB_OK) return ~size_t(0);
  int devices = 0;
  if (cudaGetDeviceCount(&devices) != cudaSuccess || devices == 0) {
    cudaGetLastError();  // a host that sizes memory without a device: the most any form takes
    return attn8::workspace_bytes(p, cache->head_dim);
  }
  const int cluster = attn8::plan(p, cache->head_dim);
  if (cluster < 0) return ~size_t(0);  // the launch would fail too: no size to keep
  return cluster > 0 ? 0 : attn8::workspace_bytes(p, cache->head_dim);
}

extern "C" int fb_attention_q8(const void* q, const fb_q8_cache* cache, const int64_t* position, int per_row,
                               const int64_t* chain, void* out, void* workspace, size_t workspace_bytes, int tokens,
                               int q_heads, float scale, void* stream) {
  if (!q || !cache || !position || !out) return FB_ERR_ARG;
  if (!cache->keys || !cache->values || !cache->key_scales || !cache->value_scales) return FB_ERR_ARG;
  attn8::Params p;
  int st = attn8::shape(&p, *cache, tokens, q_heads);
  if (st != FB_OK) return st;
  if ((chain == nullptr && tokens != 1) || (chain != nullptr && !per_row)) return FB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) & 7u) != 0 || (reinterpret_cast<uintptr_t>(out) & 3u) != 0) return FB_ERR_ARG;
  const int head_dim = cache->head_dim;
  const int cluster = attn8::plan(p, head_dim);
  if (cluster < 0) return cluster;
  if (cluster == 0) {
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return FB_ERR_ARG;
    if (workspace_bytes < attn8::workspace_bytes(p, head_dim)) return FB_ERR_WORKSPACE;
    p.acc = static_cast<float*>(workspace);
    p.stats = reinterpret_cast<float4*>(static_cast<uint8_t*>(workspace) + attn8::acc_bytes(p, head_dim));
  } else {
    p.acc = nullptr;
    p.stats = nullptr;
  }
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.key_scales = cache->key_scales;
  p.value_scales = cache->value_scales;
  p.position = position;
  p.chain = chain;
  p.per_row = per_row ? 1 : 0;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  p.err = error_word();
  const uint64_t rows = static_cast<uint64_t>(p.batch) * p.kv_heads * p.capacity;
  CUtensorMap km, vm;
  st = encode_u8_2d(&km, cache->keys, rows, head_dim, attn8::kTile);
  if (st != FB_OK) return st;
  st = encode_u8_2d(&vm, cache->values, rows, head_dim, attn8::kTile);
  if (st != FB_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return attn8::with_shape(p, head_dim, [&](auto d, auto ng) {
    return attn8::launch<decltype(d)::value, decltype(ng)::value>(km, vm, p, cluster, s);
  });
}
