// Fused per-head Q/K RMSNorm + rotate-half RoPE + append to an 8-bit KV cache, and the move of
// one slot inside it (sm_100a).
//
//   inv = rsqrt(mean(x^2) + eps);  w = x * inv * gain;  out = w * cos + rot(w) * sin
// in fp32 from the bf16 projection output to the one rounding: Q to bf16, K and V to e4m3. (The
// bf16 cache's append rounds to bf16 four times on the way, because the engine it replaces does;
// an 8-bit cache has no such counterpart, so nothing is rounded twice here.)
//
// Scales: a block's scale is the least power of two that brings the largest finite magnitude of
// its slots to at most 448. A token that starts a block sets it anew (whatever the slots held);
// one that joins a block with earlier slots can only raise it, and then the earlier codes are
// rounded once to the new scale, which changes only codes that fall into e4m3's subnormals.
//
// A block has one owner CTA: it holds every new value of the block in registers, reduces the
// largest magnitude through shared memory, and is the only reader and writer of the block's
// codes and scale. No atomics. Q heads run in CTAs of their own, a warp per token and run of heads.
//
// A prompt is bound by instruction issue (0.75 per cycle) and close behind by bytes (the packed projection
// in, Q and the codes out): a head's D values lie on D / 8 lanes, four dims of each half, so that RoPE's
// partners meet in a lane (no shuffles but the norm's); gains are folded into cos and sin once per token; the
// arithmetic runs in fp32 pairs; and a warp issues all the loads of its rows before it uses one. 8192 tokens of
// 32 + 8 heads of 128: 36.9 us, 5.1 TB/s, 0.78 of the floor. (Of the steps: loads that waited for one another
// 55 us; a launch each for Q heads and blocks 50; all cos and sin loaded at once, three CTAs per SM, 49;
// gains, cos and sin applied one by one, and single fp32 operations, 43; eight heads a warp instead of sixteen 39.)
// A decode step is bound by latency: 16 rows 2.9 us.
#include <initializer_list>

#include "q8.cuh"

namespace fb {
namespace q8 {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBlock = 64;
constexpr int kE = 8;  // values of a lane

struct AppendParams {
  const void* packed;
  int splits;
  const __nv_bfloat16* q_weight;
  const __nv_bfloat16* k_weight;
  float q_eps, k_eps;
  const __nv_bfloat16* cos;
  const __nv_bfloat16* sin;
  const int64_t* position;
  const int64_t* phases;
  __nv_bfloat16* query;
  uint8_t* keys;
  uint8_t* values;
  float* key_scales;
  float* value_scales;
  int batch, tokens, q_heads, kv_heads, capacity, block, block_shift, blocks, mode, table;
  int query_ctas;   // CTAs [0, query_ctas) do Q heads
  int query_heads;  // of a warp's token
  int runs;         // warps of a token: ceil(q_heads / query_heads)
  int touched;      // cache blocks a row's tokens can touch
  unsigned* err;
};

// Slot of a row's first token; negative: the row holds no sequence (nothing is appended). Held where a token's
// offset cannot carry it past 64 bits; anything from the capacity on is past the cache alike.
constexpr long long kFar = 1ll << 61;
__device__ __forceinline__ long long first_slot(const AppendParams& p, int b) {
  if (p.mode == 1) return 0;
  return min(static_cast<long long>(p.position[p.mode == 2 ? b : 0]), kFar);
}

// The cos/sin row of token t of row b. Whole tables have at least `capacity` rows: a phase
// outside them is reported (unless the row is empty) and read at the nearest end.
__device__ __forceinline__ long long phase_row(const AppendParams& p, int b, int t, long long start) {
  const int row = b * p.tokens + t;
  if (!p.table) return p.mode == 2 ? row : t;
  long long offset = p.phases != nullptr ? p.phases[row] : t;
  offset = max(-kFar, min(offset, kFar));
  long long phase = max(-kFar, start) + offset;
  if (phase < 0 || phase >= p.capacity) {
    if (start >= 0) raise_error(p.err, kErrBadShape);
    phase = phase < 0 ? 0 : p.capacity - 1;
  }
  return phase;
}

// How a row of D values lies on a warp: D / 8 lanes, 32 / that many rows side by side; a lane holds dims
// d0 .. d0 + 3 and D / 2 + d0 .. D / 2 + d0 + 3, d0 = 4 (lane % kLanes).
template <int D>
struct Lanes {
  static constexpr int kLanes = D / kE, kRows = 32 / kLanes;
};

__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[kE]) {
  x[0] = bf16_lo(w.x), x[1] = bf16_hi(w.x), x[2] = bf16_lo(w.y), x[3] = bf16_hi(w.y);
  x[4] = bf16_lo(w.z), x[5] = bf16_hi(w.z), x[6] = bf16_lo(w.w), x[7] = bf16_hi(w.w);
}

// A lane's eight bf16 values of a row, src at its d0.
template <int D>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* src) {
  const uint2 a = *reinterpret_cast<const uint2*>(src), b = *reinterpret_cast<const uint2*>(src + D / 2);
  return make_uint4(a.x, a.y, b.x, b.y);
}

// A lane's values of a row of the packed projection, `off` its first element: bf16, or fp32 split partials
// summed in split order and rounded to bf16 (the projection's own rounding).
template <int D, bool kSplit>
__device__ __forceinline__ void load_packed8(const AppendParams& p, size_t off, size_t split_stride, float (&x)[kE]) {
  if constexpr (!kSplit) {
    unpack8(load8<D>(static_cast<const __nv_bfloat16*>(p.packed) + off), x);
    return;
  }
  const float* src = static_cast<const float*>(p.packed) + off;
  constexpr int kBatch = 4;  // slabs in flight before their in-order adds
  for (int s0 = 0; s0 < p.splits; s0 += kBatch) {
    float4 y[kBatch][2];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (s0 + j < p.splits) {
        y[j][0] = __ldcg(reinterpret_cast<const float4*>(src + (s0 + j) * split_stride));
        y[j][1] = __ldcg(reinterpret_cast<const float4*>(src + (s0 + j) * split_stride + D / 2));
      }
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (s0 + j < p.splits) {
        const float v[kE] = {y[j][0].x, y[j][0].y, y[j][0].z, y[j][0].w, y[j][1].x, y[j][1].y, y[j][1].z, y[j][1].w};
#pragma unroll
        for (int e = 0; e < kE; ++e) x[e] = s0 + j == 0 ? v[e] : x[e] + v[e];
      }
  }
#pragma unroll
  for (int e = 0; e < kE; ++e) x[e] = bf16_round(x[e]);
}

// gain * cos and the partner's -+ gain * sin of a lane's dims, in pairs: RoPE of x * inv * gain is then
// inv * (x c + partner s).
struct Rotation {
  float2 c[kE / 2], s[kE / 2];
  __device__ __forceinline__ Rotation(const uint4& gain, const uint4& cos, const uint4& sin) {
    float g[kE], cs[kE], sn[kE];
    unpack8(gain, g);
    unpack8(cos, cs);
    unpack8(sin, sn);
#pragma unroll
    for (int i = 0; i < kE / 2; ++i) {
      const int e = 2 * i;
      const float sign = i < kE / 4 ? -1.f : 1.f;
      c[i] = make_float2(g[e] * cs[e], g[e + 1] * cs[e + 1]);
      s[i] = make_float2(sign * g[e ^ 4] * sn[e], sign * g[(e + 1) ^ 4] * sn[e + 1]);
    }
  }
};

// RMSNorm + RoPE of the rows on a warp, in place, in fp32.
template <int D>
__device__ __forceinline__ void norm_rope_fp32(float (&x)[kE], float eps, const Rotation& r) {
  constexpr int kLanes = Lanes<D>::kLanes;
  float2 v[kE / 2], sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kE / 2; ++i) {
    v[i] = make_float2(x[2 * i], x[2 * i + 1]);
    sum = fma2(v[i], v[i], sum);
  }
  float ss = sum.x + sum.y;
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float inv = rsqrtf(ss / static_cast<float>(D) + eps);
#pragma unroll
  for (int i = 0; i < kE / 2; ++i) v[i] = mul2(v[i], make_float2(inv, inv));
#pragma unroll
  for (int i = 0; i < kE / 2; ++i) {
    const float2 out = fma2(v[i ^ 2], r.s[i], mul2(v[i], r.c[i]));
    x[2 * i] = out.x;
    x[2 * i + 1] = out.y;
  }
}

// Four values times `factor` to packed codes; kChecked: anything that is not finite to the NaN code.
template <bool kChecked>
__device__ __forceinline__ uint32_t codes4(const float* x, float factor) {
  if constexpr (kChecked)
    return to_e4m3x2(x[0] * factor, x[1] * factor) | (to_e4m3x2(x[2] * factor, x[3] * factor) << 16);
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * factor, x[1] * factor), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * factor, x[3] * factor), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

template <int D, bool kChecked>
__device__ __forceinline__ void store_codes8(uint8_t* dst, const float (&x)[kE], float factor) {
  *reinterpret_cast<uint32_t*>(dst) = codes4<kChecked>(x, factor);
  *reinterpret_cast<uint32_t*>(dst + D / 2) = codes4<kChecked>(x + 4, factor);
}

template <int D>
__device__ __forceinline__ void load_codes8(const uint8_t* src, float (&x)[kE]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(src + i * (D / 2));
    const float2 a = e4m3x2_to_float2(w & 0xffffu), b = e4m3x2_to_float2(w >> 16);
    x[4 * i] = a.x, x[4 * i + 1] = a.y, x[4 * i + 2] = b.x, x[4 * i + 3] = b.y;
  }
}

constexpr uint32_t kInfinity = 0x7f800000u;  // bits: anything from here on is not finite

// The largest magnitude, or NaN (its bits order as magnitudes do; NaN above infinity above all).
__device__ __forceinline__ float largest_magnitude(const float (&x)[kE], float so_far) {
#pragma unroll
  for (int e = 0; e < kE; e += 2)
    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(so_far) : "f"(fabsf(x[e])), "f"(fabsf(x[e + 1])));
  return so_far;
}

// Largest finite magnitude (NaN and infinities do not set a scale).
__device__ __forceinline__ float finite_max(const float (&x)[kE], float so_far) {
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    const float a = fabsf(x[e]);
    so_far = a < INFINITY ? fmaxf(so_far, a) : so_far;
  }
  return so_far;
}

// One launch does both. A decode step's CTAs of Q heads come first; a prompt's CTAs of either kind are spread
// evenly, so that the blocks' chains of loads, norm, barrier and stores hide behind the Q heads' bytes.
template <int D, bool kSplit, bool kPrompt>
__global__ void __launch_bounds__(kThreads, kSplit || !kPrompt ? 2 : 4) append_kernel(const AppendParams p) {
  constexpr int kLanes = Lanes<D>::kLanes, kRows = Lanes<D>::kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / kLanes, d0 = lane % kLanes * 4;
  const int width = (p.q_heads + 2 * p.kv_heads) * D;
  const size_t split_stride = static_cast<size_t>(p.batch) * p.tokens * width;
  pdl_wait();
  pdl_trigger();

  const int cta = static_cast<int>(blockIdx.x);
  int block_cta = cta - p.query_ctas;  // the CTA's number among those with blocks
  bool takes_block = block_cta >= 0;
  if (kPrompt) {
    const long long block_ctas = gridDim.x - p.query_ctas;
    block_cta = static_cast<int>(cta * block_ctas / gridDim.x);  // CTAs with blocks before this one
    takes_block = (cta + 1) * block_ctas / gridDim.x > block_cta;
  }
  if (!takes_block) {
    // ---- query_heads heads of one token, kRows side by side ----
    const unsigned item = static_cast<unsigned>(kPrompt ? cta - block_cta : cta) * kWarps + warp;  // < 2^31 + kWarps
    const unsigned nth_row = item / p.runs;
    const int head0 = static_cast<int>(item - nth_row * p.runs) * p.query_heads;
    if (nth_row >= static_cast<unsigned>(p.batch * p.tokens)) return;
    const int row = static_cast<int>(nth_row), b = row / p.tokens, t = row - b * p.tokens;
    const int heads = min(p.query_heads, p.q_heads - head0);
    constexpr int kMost = 4;  // loads in flight
    const size_t in = static_cast<size_t>(row) * width + head0 * D + d0;
    __nv_bfloat16* out = p.query + (static_cast<size_t>(row) * p.q_heads + head0) * D + d0;
    // rows of lanes past the last head repeat it and store nothing
    uint4 raw[kMost];  // the first heads', on their way before the position and its phase are known
    auto load = [&](int h0) {
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.packed) + in;
#pragma unroll
      for (int i = 0; i < kMost; ++i)
        raw[i] = load8<D>(src + static_cast<size_t>(min(h0 + i * kRows + sub, heads - 1)) * D);
    };
    if (!kSplit) load(0);
    const size_t phase = static_cast<size_t>(phase_row(p, b, t, first_slot(p, b))) * D + d0;
    const Rotation rotation(load8<D>(p.q_weight + d0), load8<D>(p.cos + phase), load8<D>(p.sin + phase));
    auto finish = [&](float (&x)[kE], int h) {
      norm_rope_fp32<D>(x, p.q_eps, rotation);
      if (h >= heads) return;
      __nv_bfloat16* dst = out + static_cast<size_t>(h) * D;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
      *reinterpret_cast<uint2*>(dst + D / 2) = make_uint2(pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    };
    if constexpr (kSplit) {
      for (int h = sub; h - sub < heads; h += kRows) {
        float x[kE];
        load_packed8<D, true>(p, in + static_cast<size_t>(min(h, heads - 1)) * D, split_stride, x);
        finish(x, h);
      }
    } else {
      for (int h0 = 0;;) {
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          if (h0 + i * kRows >= heads) break;  // warp-uniform
          float x[kE];
          unpack8(raw[i], x);
          finish(x, h0 + i * kRows + sub);
        }
        h0 += kMost * kRows;
        if (h0 >= heads) break;
        load(h0);
      }
    }
    return;
  }

  // ---- one cache block of one (row, KV head, K or V) ----
  __shared__ uint32_t s_largest[kWarps];
  __shared__ float s_finite[kWarps];
  int item = block_cta;
  const int nth = item % p.touched;
  item /= p.touched;
  const bool is_value = item & 1;
  const int pair = item >> 1;
  const int b = pair / p.kv_heads, h = pair - b * p.kv_heads;
  const long long start = first_slot(p, b);
  if (start < 0 || start >= p.capacity) {  // whole CTA: an empty row, or every token past the cache
    if (start >= 0 && threadIdx.x == 0) raise_error(p.err, kErrBadShape);
    return;
  }
  const long long at = (start >> p.block_shift) + nth;  // block index
  const long long low = at << p.block_shift;
  if (low >= start + p.tokens) return;
  if (low >= p.capacity) {
    if (threadIdx.x == 0) raise_error(p.err, kErrBadShape);  // tokens past the cache
    return;
  }
  uint8_t* codes = (is_value ? p.values : p.keys) + (static_cast<size_t>(pair) * p.capacity + low) * D + d0;
  float* scale_at = (is_value ? p.value_scales : p.key_scales) + static_cast<size_t>(pair) * p.blocks + at;
  const bool joins = start > low;  // the block holds earlier slots
  const float before = joins ? *scale_at : 0.f;

  // this lane's slots of the block: warp * kRows + sub, and every kStride from there
  const int head = p.q_heads + (is_value ? p.kv_heads : 0) + h;
  constexpr int kStride = kWarps * kRows, kSlots = kMaxBlock / kStride;
  const int slot0 = warp * kRows + sub;
  // slots that get a token
  const int from = static_cast<int>(start > low ? start - low : 0);
  long long last = start + p.tokens - low;
  if (last > p.capacity - low) {
    if (threadIdx.x == 0) raise_error(p.err, kErrBadShape);  // tokens past the cache
    last = p.capacity - low;
  }
  const int to = static_cast<int>(last < p.block ? last : p.block);
  // Every load of the lane's slots is issued before one is used. Slots that get no token count as zeros: a
  // warp skips those of a pass where it has none that does, else they read the nearest such slot's token.
  auto passes = [&](int i) {
    const int first = warp * kRows + i * kStride;
    return first < to && first + kRows > from;
  };
  float x[kSlots][kE];
  uint4 raw[kSlots], cos[2], sin[2], gain;  // cos and sin of two slots at a time: registers
  auto token = [&](int i) { return static_cast<int>(low - start) + min(max(slot0 + i * kStride, from), to - 1); };
  auto load_phase = [&](int i) {
    if (is_value || !passes(i)) return;
    const size_t phase = static_cast<size_t>(phase_row(p, b, token(i), start)) * D + d0;
    cos[i & 1] = load8<D>(p.cos + phase);
    sin[i & 1] = load8<D>(p.sin + phase);
  };
  if (!is_value) gain = load8<D>(p.k_weight + d0);
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    raw[i] = make_uint4(0u, 0u, 0u, 0u);
    if (!passes(i)) continue;
    const size_t off = (static_cast<size_t>(b) * p.tokens + token(i)) * width + head * D + d0;
    if constexpr (kSplit)
      load_packed8<D, true>(p, off, split_stride, x[i]);
    else
      raw[i] = load8<D>(static_cast<const __nv_bfloat16*>(p.packed) + off);
  }
#pragma unroll
  for (int i = 0; i < 2 && i < kSlots; ++i) load_phase(i);
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int slot = slot0 + i * kStride;
    if (!kSplit) unpack8(raw[i], x[i]);
    if (slot < from || slot >= to)
#pragma unroll
      for (int e = 0; e < kE; ++e) x[i][e] = 0.f;
    if (!is_value && passes(i)) norm_rope_fp32<D>(x[i], p.k_eps, Rotation(gain, cos[i & 1], sin[i & 1]));  // zeros stay
    if (i + 2 < kSlots) load_phase(i + 2);
    top = largest_magnitude(x[i], top);
  }
  uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if (lane == 0) s_largest[warp] = bits;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) bits = max(bits, s_largest[w]);
  float largest = __uint_as_float(bits);
  const bool sound = bits < kInfinity;
  if (!sound) {  // some value is not finite (the whole CTA agrees): the largest of the others
    largest = 0.f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) largest = finite_max(x[i], largest);
    largest = warp_max(largest);
    if (lane == 0) s_finite[warp] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) largest = fmaxf(largest, s_finite[w]);
  }
  const float after = fmaxf(least_scale(largest), before);
  const float inverse = 1.f / after;
  if (joins && after > before) {
    const float ratio = before * inverse;
    for (int slot = slot0; slot < from; slot += kStride) {
      float old[kE];
      load_codes8<D>(codes + static_cast<size_t>(slot) * D, old);
      store_codes8<D, true>(codes + static_cast<size_t>(slot) * D, old, ratio);
    }
  }
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int slot = slot0 + i * kStride;
    if (slot < from || slot >= to) continue;
    if (sound)
      store_codes8<D, false>(codes + static_cast<size_t>(slot) * D, x[i], inverse);
    else
      store_codes8<D, true>(codes + static_cast<size_t>(slot) * D, x[i], inverse);
  }
  if (threadIdx.x == 0) *scale_at = after;
}

// One slot per row moved inside an 8-bit store [planes, B, Hkv, C, D] (scales [planes, B, Hkv,
// blocks]): a warp per (plane, row, head) reads slot move_from's value and writes it at move_to
// as an append there would: move_to becomes its block's newest slot, a first slot sets the
// block's scale, a later one can only raise it (the block's earlier codes are then rounded once).
// 36 layers x 16 rows x 8 heads of 128, K and V: 3.2 us within a block, 4.8 across blocks (a chain of two loads, a
// reduction and a store), 32 where every move raises the scale of a block with 63 slots before it (149 MB
// read and written, 22.6 us of a copy; a warp rescales two slots at a time).
template <int D>
__global__ void __launch_bounds__(128) relocate_kernel(uint8_t* store, float* scales, int planes, int batch,
                                                       int kv_heads, int capacity, int block, int blocks,
                                                       const int64_t* move_from, const int64_t* move_to,
                                                       unsigned* err) {
  constexpr int kLanes = Lanes<D>::kLanes;
  pdl_wait();
  pdl_trigger();
  const long long item = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, sub = lane / kLanes, rows = 32 / kLanes;
  if (item >= static_cast<long long>(planes) * batch * kv_heads) return;
  const int row = static_cast<int>(item / kv_heads % batch);
  const long long source = move_from[row], target = move_to[row];
  if (source < 0) return;
  if (source >= capacity || target < 0 || target >= capacity) {
    if (lane == 0) raise_error(err, kErrBadShape);
    return;
  }
  uint8_t* codes = store + static_cast<size_t>(item) * capacity * D + lane % kLanes * 4;
  float* s = scales + static_cast<size_t>(item) * blocks;
  const long long to_block = target / block, low = to_block * block;
  if (source / block == to_block) {  // one scale: the codes move as they are
    if (sub < 2)
      *reinterpret_cast<uint32_t*>(codes + target * D + sub * (D / 2)) =
          *reinterpret_cast<const uint32_t*>(codes + source * D + sub * (D / 2));
    return;
  }
  float x[kE];
  load_codes8<D>(codes + source * D, x);
  const float from_scale = s[source / block], before = s[to_block];
#pragma unroll
  for (int e = 0; e < kE; ++e) x[e] *= from_scale;
  const float wanted = least_scale(warp_max(finite_max(x, 0.f)));
  const bool joins = target > low;
  const float after = joins ? fmaxf(wanted, before) : wanted;
  const float inverse = 1.f / after;
  if (joins && after > before)
    for (long long slot = low + sub; slot < target; slot += rows) {
      float old[kE];
      load_codes8<D>(codes + slot * D, old);
      store_codes8<D, true>(codes + slot * D, old, before * inverse);
    }
  if (sub == 0) store_codes8<D, true>(codes + target * D, x, inverse);
  __syncwarp();
  if (lane == 0) s[to_block] = after;
}

constexpr long long kPromptRows = 1024;

template <int D, bool kSplit>
int launch_append(const AppendParams& p, long long rows, long long ctas, cudaStream_t s) {
  auto* kernel = rows < kPromptRows ? append_kernel<D, kSplit, false> : append_kernel<D, kSplit, true>;
  return launch_ex(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0, s, 1, p);
}

}  // namespace q8
}  // namespace fb

using namespace fb;

extern "C" int fb_qk_norm_rope_append_q8(const void* packed, int packed_splits, const void* q_weight,
                                         const void* k_weight, float q_eps, float k_eps, const void* cos,
                                         const void* sin, const int64_t* position, const int64_t* phases,
                                         void* query, const fb_q8_cache* cache, int tokens, int q_heads, int mode,
                                         int table, void* stream) {
  if (!packed || !q_weight || !k_weight || !cos || !sin || !position || !query || !cache) return FB_ERR_ARG;
  if (!cache->keys || !cache->values || !cache->key_scales || !cache->value_scales) return FB_ERR_ARG;
  const int batch = cache->batch, kv_heads = cache->kv_heads, capacity = cache->capacity, head_dim = cache->head_dim;
  const int block = cache->block;
  if (batch <= 0 || tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || capacity <= 0 || packed_splits < 0)
    return FB_ERR_ARG;
  if (mode < 0 || mode > 2 || (table && mode == 1) || (phases && !table)) return FB_ERR_ARG;
  if ((head_dim != 64 && head_dim != 128) || !q8::valid_block(block) || tokens > capacity) return FB_ERR_SHAPE;
  // vector loads of the inputs and stores of the queries
  for (const void* q : {packed, q_weight, k_weight, cos, sin, static_cast<const void*>(query),
                        static_cast<const void*>(cache->keys), static_cast<const void*>(cache->values)})
    if (reinterpret_cast<uintptr_t>(q) & 15u) return FB_ERR_ARG;
  q8::AppendParams p;
  p.packed = packed;
  p.splits = packed_splits;
  p.q_weight = static_cast<const __nv_bfloat16*>(q_weight);
  p.k_weight = static_cast<const __nv_bfloat16*>(k_weight);
  p.q_eps = q_eps;
  p.k_eps = k_eps;
  p.cos = static_cast<const __nv_bfloat16*>(cos);
  p.sin = static_cast<const __nv_bfloat16*>(sin);
  p.position = position;
  p.phases = phases;
  p.query = static_cast<__nv_bfloat16*>(query);
  p.keys = static_cast<uint8_t*>(cache->keys);
  p.values = static_cast<uint8_t*>(cache->values);
  p.key_scales = cache->key_scales;
  p.value_scales = cache->value_scales;
  p.batch = batch;
  p.tokens = tokens;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.capacity = capacity;
  p.block = block;
  p.block_shift = block == 16 ? 4 : block == 32 ? 5 : 6;
  p.blocks = (capacity + block - 1) / block;
  p.mode = mode;
  p.table = table ? 1 : 0;
  p.err = error_word();
  // a prompt starts on a block; elsewhere the first token can be a block's last slot
  p.touched = mode == 1 ? (tokens + block - 1) / block : (tokens + block - 2) / block + 1;
  // a prompt's warps take sixteen heads of a token (its rotation is worked out once for them), a few rows' the
  // least that fills a load, so that more warps share them
  const long long rows = static_cast<long long>(batch) * tokens;
  p.query_heads = rows >= q8::kPromptRows ? 16 : 32 * q8::kE / head_dim;
  p.runs = (q_heads + p.query_heads - 1) / p.query_heads;
  const long long query_ctas = (rows * p.runs + q8::kWarps - 1) / q8::kWarps;
  const long long ctas = query_ctas + 2ll * batch * kv_heads * p.touched;
  if (ctas >= (1ll << 31) || rows * p.runs >= (1ll << 31)) return FB_ERR_SHAPE;
  p.query_ctas = static_cast<int>(query_ctas);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    return packed_splits ? q8::launch_append<128, true>(p, rows, ctas, s)
                         : q8::launch_append<128, false>(p, rows, ctas, s);
  return packed_splits ? q8::launch_append<64, true>(p, rows, ctas, s) : q8::launch_append<64, false>(p, rows, ctas, s);
}

extern "C" int fb_spec_relocate_q8(void* store, float* scales, int planes, int batch, int kv_heads, int capacity,
                                   int head_dim, int block, const int64_t* move_from, const int64_t* move_to,
                                   void* stream) {
  if (!store || !scales || !move_from || !move_to || planes <= 0 || batch <= 0 || kv_heads <= 0 || capacity <= 0)
    return FB_ERR_ARG;
  if ((head_dim != 64 && head_dim != 128) || !q8::valid_block(block)) return FB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(store) & 3u) return FB_ERR_ARG;  // codes move four at a time
  const long long warps = static_cast<long long>(planes) * batch * kv_heads;
  if ((warps + 3) / 4 >= (1ll << 31)) return FB_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>((warps + 3) / 4)), threads(128);
  const int blocks = (capacity + block - 1) / block;
  uint8_t* codes = static_cast<uint8_t*>(store);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    return launch_ex(q8::relocate_kernel<128>, grid, threads, 0, s, 1, codes, scales, planes, batch, kv_heads,
                     capacity, block, blocks, move_from, move_to, error_word());
  return launch_ex(q8::relocate_kernel<64>, grid, threads, 0, s, 1, codes, scales, planes, batch, kv_heads, capacity,
                   block, blocks, move_from, move_to, error_word());
}
