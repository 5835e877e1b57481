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
// codes and scale. No atomics. Q heads run in CTAs of their own, a warp per (token, head).
#include "q8.cuh"
#include "rope_math.cuh"

namespace fb {
namespace q8 {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBlock = 64;
constexpr int kPerWarp = kMaxBlock / kWarps;  // slots of a block a warp holds

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
  int batch, tokens, q_heads, kv_heads, capacity, block, blocks, mode, table;
  int query_ctas;      // CTAs [0, query_ctas) do Q heads
  int touched;         // cache blocks a row's tokens can touch
  unsigned* err;
};

// Slot of a row's first token; negative: the row holds no sequence (nothing is appended).
__device__ __forceinline__ long long first_slot(const AppendParams& p, int b) {
  if (p.mode == 1) return 0;
  return p.position[p.mode == 2 ? b : 0];
}

// The cos/sin row of token t of row b. Whole tables have at least `capacity` rows: a phase
// outside them is reported (unless the row is empty) and read at the nearest end.
__device__ __forceinline__ long long phase_row(const AppendParams& p, int b, int t, long long start) {
  const int row = b * p.tokens + t;
  if (!p.table) return p.mode == 2 ? row : t;
  long long phase = start + (p.phases != nullptr ? p.phases[row] : t);
  if (phase < 0 || phase >= p.capacity) {
    if (start >= 0) raise_error(p.err, kErrBadShape);
    phase = phase < 0 ? 0 : p.capacity - 1;
  }
  return phase;
}

// RMSNorm + RoPE of one head on a warp, lane l holding dims [l*E, l*E + E): in place, in fp32.
template <int D>
__device__ __forceinline__ void norm_rope_fp32(float (&x)[D / 32], const float (&gain)[D / 32], float eps,
                                               const float (&cs)[D / 32], const float (&sn)[D / 32], int lane) {
  constexpr int E = D / 32;
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) ss += x[e] * x[e];
  const float inv = __frsqrt_rn(warp_sum(ss) / static_cast<float>(D) + eps);
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = x[e] * inv * gain[e];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float partner = __shfl_xor_sync(0xffffffffu, x[e], 16);
    x[e] = x[e] * cs[e] + (lane < 16 ? -partner : partner) * sn[e];
  }
}

template <int E>
__device__ __forceinline__ void store_codes(uint8_t* dst, const float (&x)[E], float inverse) {
  const uint32_t lo = to_e4m3x2(x[0] * inverse, x[1] * inverse);
  if constexpr (E == 4)
    *reinterpret_cast<uint32_t*>(dst) = lo | (to_e4m3x2(x[2] * inverse, x[3] * inverse) << 16);
  else
    *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(lo);
}

template <int E>
__device__ __forceinline__ void load_codes(const uint8_t* src, float (&x)[E]) {
  if constexpr (E == 4) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(src);
    const float2 a = e4m3x2_to_float2(w & 0xffffu), b = e4m3x2_to_float2(w >> 16);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  } else {
    const float2 a = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(src));
    x[0] = a.x, x[1] = a.y;
  }
}

// Largest finite magnitude of E values (NaN and infinities do not set a scale).
template <int E>
__device__ __forceinline__ float finite_max(const float (&x)[E], float so_far) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float a = fabsf(x[e]);
    so_far = a < INFINITY ? fmaxf(so_far, a) : so_far;
  }
  return so_far;
}

template <int D>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendParams p) {
  constexpr int E = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int d0 = lane * E;
  const int width = (p.q_heads + 2 * p.kv_heads) * D;
  const size_t split_stride = static_cast<size_t>(p.batch) * p.tokens * width;
  pdl_wait();
  pdl_trigger();

  if (static_cast<int>(blockIdx.x) < p.query_ctas) {
    const long long item = static_cast<long long>(blockIdx.x) * kWarps + warp;
    const long long rows = static_cast<long long>(p.batch) * p.tokens;
    if (item >= rows * p.q_heads) return;
    const int row = static_cast<int>(item / p.q_heads), head = static_cast<int>(item % p.q_heads);
    const int b = row / p.tokens, t = row % p.tokens;
    float x[E], gain[E], cs[E], sn[E];
    rope::load_packed_values<E, 8>(p.packed, p.splits, static_cast<size_t>(row) * width + head * D + d0, split_stride, x);
    rope::load_bf16<E>(p.q_weight + d0, gain);
    const size_t phase = static_cast<size_t>(phase_row(p, b, t, first_slot(p, b))) * D + d0;
    rope::load_bf16<E>(p.cos + phase, cs);
    rope::load_bf16<E>(p.sin + phase, sn);
    norm_rope_fp32<D>(x, gain, p.q_eps, cs, sn, lane);
    __nv_bfloat16* dst = p.query + (static_cast<size_t>(row) * p.q_heads + head) * D + d0;
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(x[0], x[1]);
    return;
  }

  // ---- one cache block of one (row, KV head, K or V) ----
  __shared__ float s_largest[kWarps];
  int item = blockIdx.x - p.query_ctas;
  const int nth = item % p.touched;
  item /= p.touched;
  const bool is_value = item & 1;
  const int pair = item >> 1;
  const int b = pair / p.kv_heads, h = pair % p.kv_heads;
  const long long start = first_slot(p, b);
  if (start < 0) return;  // whole CTA
  const long long at = start / p.block + nth;  // block index
  const long long low = at * p.block;
  if (low >= p.capacity || low >= start + p.tokens) {
    if (low < start + p.tokens && threadIdx.x == 0) raise_error(p.err, kErrBadShape);  // tokens past the cache
    return;
  }
  uint8_t* codes = (is_value ? p.values : p.keys) + (static_cast<size_t>(pair) * p.capacity + low) * D + d0;
  float* scale_at = (is_value ? p.value_scales : p.key_scales) + static_cast<size_t>(pair) * p.blocks + at;
  const bool joins = start > low;  // the block holds earlier slots
  const float before = joins ? *scale_at : 0.f;

  const int head = p.q_heads + (is_value ? p.kv_heads : 0) + h;
  float gain[E];
  if (!is_value) rope::load_bf16<E>(p.k_weight + d0, gain);
  float x[kPerWarp][E];
  float largest = 0.f;
#pragma unroll
  for (int i = 0; i < kPerWarp; ++i) {
    const int offset = warp + i * kWarps;
    const long long t = low + offset - start;
    if (offset >= p.block || t < 0 || t >= p.tokens) continue;  // warp-uniform
    if (low + offset >= p.capacity) {
      if (lane == 0) raise_error(p.err, kErrBadShape);
      continue;
    }
    const size_t row = static_cast<size_t>(b) * p.tokens + t;
    rope::load_packed_values<E, 2>(p.packed, p.splits, row * width + head * D + d0, split_stride, x[i]);
    if (!is_value) {
      float cs[E], sn[E];
      const size_t phase = static_cast<size_t>(phase_row(p, b, static_cast<int>(t), start)) * D + d0;
      rope::load_bf16<E>(p.cos + phase, cs);
      rope::load_bf16<E>(p.sin + phase, sn);
      norm_rope_fp32<D>(x[i], gain, p.k_eps, cs, sn, lane);
    }
    largest = finite_max<E>(x[i], largest);
  }
  largest = warp_max(largest);
  if (lane == 0) s_largest[warp] = largest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) largest = fmaxf(largest, s_largest[w]);
  const float after = fmaxf(least_scale(largest), before);
  const float inverse = 1.f / after;
  if (joins && after > before) {
    const float ratio = before * inverse;
    for (int offset = warp; offset < p.block && low + offset < start; offset += kWarps) {
      float old[E];
      load_codes<E>(codes + static_cast<size_t>(offset) * D, old);
      store_codes<E>(codes + static_cast<size_t>(offset) * D, old, ratio);
    }
  }
#pragma unroll
  for (int i = 0; i < kPerWarp; ++i) {
    const int offset = warp + i * kWarps;
    const long long t = low + offset - start;
    if (offset >= p.block || t < 0 || t >= p.tokens || low + offset >= p.capacity) continue;
    store_codes<E>(codes + static_cast<size_t>(offset) * D, x[i], inverse);
  }
  if (threadIdx.x == 0) *scale_at = after;
}

// One slot per row moved inside an 8-bit store [planes, B, Hkv, C, D] (scales [planes, B, Hkv,
// blocks]): a warp per (plane, row, head) reads slot move_from's value and writes it at move_to
// as an append there would: move_to becomes its block's newest slot, a first slot sets the
// block's scale, a later one can only raise it (the block's earlier codes are then rounded once).
template <int D>
__global__ void __launch_bounds__(128) relocate_kernel(uint8_t* store, float* scales, int planes, int batch,
                                                       int kv_heads, int capacity, int block, int blocks,
                                                       const int64_t* move_from, const int64_t* move_to,
                                                       unsigned* err) {
  constexpr int E = D / 32;
  pdl_wait();
  pdl_trigger();
  const long long item = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= static_cast<long long>(planes) * batch * kv_heads) return;
  const int row = static_cast<int>(item / kv_heads % batch);
  const long long source = move_from[row], target = move_to[row];
  if (source < 0) return;
  if (source >= capacity || target < 0 || target >= capacity) {
    if (lane == 0) raise_error(err, kErrBadShape);
    return;
  }
  uint8_t* codes = store + static_cast<size_t>(item) * capacity * D + lane * E;
  float* s = scales + static_cast<size_t>(item) * blocks;
  const long long to_block = target / block, low = to_block * block;
  float x[E];
  load_codes<E>(codes + source * D, x);
  const float from_scale = s[source / block], before = s[to_block];
  if (source / block == to_block) {  // one scale: the codes move as they are
    store_codes<E>(codes + target * D, x, 1.f);
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] *= from_scale;
  const float wanted = least_scale(warp_max(finite_max<E>(x, 0.f)));
  const bool joins = target > low;
  const float after = joins ? fmaxf(wanted, before) : wanted;
  const float inverse = 1.f / after;
  if (joins && after > before)
    for (long long slot = low; slot < target; ++slot) {
      float old[E];
      load_codes<E>(codes + slot * D, old);
      store_codes<E>(codes + slot * D, old, before * inverse);
    }
  store_codes<E>(codes + target * D, x, inverse);
  __syncwarp();
  if (lane == 0) s[to_block] = after;
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
  p.blocks = (capacity + block - 1) / block;
  p.mode = mode;
  p.table = table ? 1 : 0;
  p.err = error_word();
  // a prompt starts on a block; elsewhere the first token can be a block's last slot
  p.touched = mode == 1 ? (tokens + block - 1) / block : (tokens + block - 2) / block + 1;
  const long long heads = static_cast<long long>(batch) * tokens * q_heads;
  const long long query_ctas = (heads + q8::kWarps - 1) / q8::kWarps;
  const long long ctas = query_ctas + 2ll * batch * kv_heads * p.touched;
  if (ctas >= (1ll << 31) || static_cast<long long>(batch) * tokens >= (1ll << 31)) return FB_ERR_SHAPE;
  p.query_ctas = static_cast<int>(query_ctas);
  const dim3 grid(static_cast<unsigned>(ctas)), threads(q8::kThreads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch_ex(q8::append_kernel<128>, grid, threads, 0, s, 1, p);
  return launch_ex(q8::append_kernel<64>, grid, threads, 0, s, 1, p);
}

extern "C" int fb_spec_relocate_q8(void* store, float* scales, int planes, int batch, int kv_heads, int capacity,
                                   int head_dim, int block, const int64_t* move_from, const int64_t* move_to,
                                   void* stream) {
  if (!store || !scales || !move_from || !move_to || planes <= 0 || batch <= 0 || kv_heads <= 0 || capacity <= 0)
    return FB_ERR_ARG;
  if ((head_dim != 64 && head_dim != 128) || !q8::valid_block(block)) return FB_ERR_SHAPE;
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
