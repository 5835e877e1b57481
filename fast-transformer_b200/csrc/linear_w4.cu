// Projections with 4-bit weights and group scales, y[M, N] = x[M, K] @ W[N, K]^T for M <= 64 rows,
// W[n, k] = code[n, k] * scale[n, k / group], codes -8..7 (sm_100a).
//
// Bound by the packed codes (N K / 2 bytes) at few rows. They are laid out once
// (fb_w4_pack) in the order the product reads them: tiles of 16 rows x 64 columns, 512 bytes, in
// which lane l's 16 bytes are its A fragments of four mma.sync m16n8k16 (the weights are the
// 16-row operand, x the 8-column one, so a single row of x wastes 7/8 of nothing but tensor
// time). A warp streams its tiles with one 16-byte load per lane and tile, straight into
// registers: no shared memory, no barrier on the stream.
//
// Unpacking is exact: a nibble q = code + 8 in the low mantissa bits of 128.0 is the bf16 number
// 128 + q; subtracting 136 leaves the code. x stays bf16, products accumulate in fp32 over at
// most 64 columns, then multiply by the group's scale in fp32 into the row's total: W itself is
// never rounded.
//
// A cluster of `splits` CTAs owns a contiguous range of row tiles, each CTA a contiguous K range,
// its warps the 64-column chunks of that range in turn. Warps are summed through shared memory and
// CTAs through distributed shared memory, both in order: one launch, no workspace, the same bits
// every time, and the result leaves finished (bf16, fp32 or SwiGLU).
#include <cuda_bf16.h>

#include "common.cuh"

namespace fb {
namespace w4 {

constexpr int kRows = 16;    // rows of a tile
constexpr int kChunk = 64;   // columns of a tile
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxRows = 64;

enum Epilogue : int { kBf16 = 0, kFp32 = 1, kSwiGLU = 2 };

struct Params {
  const __nv_bfloat16* x;
  const uint4* packed;       // [tiles, chunks, 32]
  const uint32_t* scales;    // [tiles, groups, 8]: bf16 scales of rows g (low half) and g + 8
  void* out;
  int m, n, k, tiles, chunks, groups, epilogue;
};

__device__ __forceinline__ uint4 load_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Two nibbles (bits 0-3 and 16-19 of w >> shift) to the bf16 pair of their codes.
__device__ __forceinline__ uint32_t codes_bf16x2(uint32_t w) {
  uint32_t biased;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(biased) : "r"(w));  // (w & mask) | 128.0
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&biased), __floats2bfloat162_rn(136.f, 136.f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Row tile of position v in the order a CTA walks: SwiGLU weights hold 64 gate rows, then their 64 up
// rows; the walk pairs each gate tile with its up tile.
__device__ __forceinline__ int tile_of(int v, int epilogue) {
  return epilogue == kSwiGLU ? (v & ~7) | ((v & 1) << 2) | ((v >> 1) & 3) : v;
}

template <int MT, int R>
struct Shape {
  static constexpr int kCols = MT * 8;
  static constexpr int kVals = R * kRows * kCols;  // outputs of a pass
  static constexpr int kSmem = kWarps * kVals * 4;
};

// SEG: scale segments of a chunk (2: groups of 32).
template <int MT, int R, int SEG>
__global__ void __launch_bounds__(kThreads, 1) linear_w4_kernel(const Params p) {
  using S = Shape<MT, R>;
  extern __shared__ __align__(16) float vals[];  // [warp][column m][row n of the pass]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int splits = gridDim.x, rank = blockIdx.x;
  pdl_trigger();
  const int unit = p.epilogue == kSwiGLU ? 2 : 1;  // tiles that stay together
  const int units = p.tiles / unit;
  const int t0 = static_cast<int>(static_cast<long long>(units) * blockIdx.y / gridDim.y) * unit;
  const int t1 = static_cast<int>(static_cast<long long>(units) * (blockIdx.y + 1) / gridDim.y) * unit;
  const int c0 = static_cast<int>(static_cast<long long>(p.chunks) * rank / splits);
  const int c1 = static_cast<int>(static_cast<long long>(p.chunks) * (rank + 1) / splits);
  const int first = c0 + warp;
  const int count = c1 > first ? (c1 - first + kWarps - 1) / kWarps : 0;
  pdl_wait();

  for (int t = t0; t < t1; t += R) {
    float total[R][MT][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) total[r][mt][0] = total[r][mt][1] = total[r][mt][2] = total[r][mt][3] = 0.f;
    const uint4* src[R];
    const uint32_t* scale_src[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int tile = tile_of(min(t + r, t1 - 1), p.epilogue);
      src[r] = p.packed + (static_cast<size_t>(tile) * p.chunks + first) * 32 + lane;
      scale_src[r] = p.scales + static_cast<size_t>(tile) * p.groups * 8 + g;
    }
    for (int i = 0; i < count; ++i) {
      const int chunk = first + i * kWarps;
      uint4 w[R];
      uint32_t sc[R][SEG];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        w[r] = load_stream(src[r] + static_cast<size_t>(i) * kWarps * 32);
#pragma unroll
        for (int e = 0; e < SEG; ++e) {
          const int group = SEG == 2 ? 2 * chunk + e : static_cast<int>(static_cast<long long>(chunk) * p.groups / p.chunks);
          sc[r][e] = __ldg(scale_src[r] + group * 8);
        }
      }
      uint4 xb[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int row = mt * 8 + g, col = chunk * kChunk + hh * 32 + c * 8;
          xb[mt][hh] = row < p.m && col < p.k
                           ? *reinterpret_cast<const uint4*>(p.x + static_cast<size_t>(row) * p.k + col)
                           : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t words[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
        float acc[MT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j == 0 || (SEG == 2 && j == 2)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.f;
          }
          const uint32_t a0 = codes_bf16x2(words[j]), a1 = codes_bf16x2(words[j] >> 4);
          const uint32_t a2 = codes_bf16x2(words[j] >> 8), a3 = codes_bf16x2(words[j] >> 12);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const uint4 v = xb[mt][j >> 1];
            mma_bf16_16816(acc[mt], a0, a1, a2, a3, (j & 1) ? v.z : v.x, (j & 1) ? v.w : v.y);
          }
          if (j == 3 || (SEG == 2 && j == 1)) {
            const uint32_t s = sc[r][SEG == 2 ? j >> 1 : 0];
            const float s0 = bf16_lo(s), s1 = bf16_hi(s);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              total[r][mt][0] += acc[mt][0] * s0;
              total[r][mt][1] += acc[mt][1] * s0;
              total[r][mt][2] += acc[mt][2] * s1;
              total[r][mt][3] += acc[mt][3] * s1;
            }
          }
        }
      }
    }
    // ---- sum the warps, then the cluster's CTAs, each in order ----
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          vals[warp * S::kVals + (mt * 8 + 2 * c + (e & 1)) * (R * kRows) + r * kRows + g + (e >> 1) * 8] = total[r][mt][e];
    __syncthreads();
    const int live = min(R, t1 - t) * kRows;  // rows of this pass
    for (int e = threadIdx.x; e < S::kVals; e += kThreads) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < kWarps; ++q) v += vals[q * S::kVals + e];
      vals[e] = v;  // slot e of warp 0's area: read by this thread alone
    }
    if (splits > 1) {
      cluster_sync();
    } else {
      __syncthreads();
    }
    const uint32_t local = smem_u32(vals);
    auto value = [&](int at) {
      if (splits == 1) return vals[at];
      float v = 0.f;
      for (int q = 0; q < splits; ++q) v += ld_cluster_f32(map_shared(local + at * 4, q));
      return v;
    };
    if (p.epilogue == kSwiGLU) {
      // the pass holds gate tile, up tile, gate tile, up tile ...
      const int width = p.n / 2, half = live / 2;
      for (int e = rank * kThreads + threadIdx.x; e < p.m * half; e += splits * kThreads) {
        const int m = e / half, f = e % half, pairn = f / kRows, row = f % kRows;
        const int at = m * (R * kRows) + pairn * 2 * kRows + row;
        const float gate = bf16_round(value(at)), up = bf16_round(value(at + kRows));
        const int tile = tile_of(t + 2 * pairn, kSwiGLU);
        const int feature = (tile >> 3) * 64 + (tile & 3) * kRows + row;
        if (feature < width)
          static_cast<__nv_bfloat16*>(p.out)[static_cast<size_t>(m) * width + feature] =
              __float2bfloat16_rn(bf16_round(gate / (1.0f + expf(-gate))) * up);
      }
    } else {
      for (int e = rank * kThreads + threadIdx.x; e < p.m * live; e += splits * kThreads) {
        const int m = e / live, row = e % live, n = t * kRows + row;
        if (n >= p.n) continue;
        const float v = value(m * (R * kRows) + row);
        if (p.epilogue == kFp32)
          static_cast<float*>(p.out)[static_cast<size_t>(m) * p.n + n] = v;
        else
          static_cast<__nv_bfloat16*>(p.out)[static_cast<size_t>(m) * p.n + n] = __float2bfloat16_rn(v);
      }
    }
    if (splits > 1) {
      cluster_sync();  // nobody overwrites a tile another CTA still reads
    } else {
      __syncthreads();
    }
  }
}

// codes int8 [N, K], scales bf16 [N, K / group] -> the packed tiles and scales. One thread a word.
__global__ void pack_kernel(const int8_t* codes, const __nv_bfloat16* scales, uint32_t* packed, uint32_t* packed_scales,
                            int n, int k, int group, int tiles, int chunks, int groups) {
  pdl_wait();
  const long long words = static_cast<long long>(tiles) * chunks * 128;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < words;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int j = i & 3, lane = (i >> 2) & 31;
    const long long tc = i >> 7;
    const int chunk = static_cast<int>(tc % chunks), tile = static_cast<int>(tc / chunks);
    const int g = lane >> 2, c = lane & 3;
    const int col = chunk * kChunk + (j >> 1) * 32 + c * 8 + (j & 1) * 4;
    uint32_t word = 0;
    for (int nib = 0; nib < 8; ++nib) {
      const int row = tile * kRows + g + (nib & 1) * 8;
      const int at = col + ((nib >> 1) & 1) * 2 + (nib >> 2);
      const int code = row < n && at < k ? codes[static_cast<size_t>(row) * k + at] : 0;
      word |= static_cast<uint32_t>((code + 8) & 15) << (4 * nib);
    }
    packed[i] = word;
  }
  const long long scale_words = static_cast<long long>(tiles) * groups * 8;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < scale_words;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int g = i & 7;
    const int at = static_cast<int>((i >> 3) % groups), tile = static_cast<int>((i >> 3) / groups);
    uint32_t word = 0;
    for (int hi = 0; hi < 2; ++hi) {
      const int row = tile * kRows + g + hi * 8;
      if (row < n && at < k / group)
        word |= static_cast<uint32_t>(__bfloat16_as_ushort(scales[static_cast<size_t>(row) * (k / group) + at])) << (16 * hi);
    }
    packed_scales[i] = word;
  }
}

// The weights' values, each rounded once to bf16: what the library product of a prompt reads.
__global__ void __launch_bounds__(256) dequantize_kernel(const uint32_t* packed, const uint32_t* scales, __nv_bfloat16* out,
                                                         int n, int k, int group, int tiles, int chunks, int groups) {
  pdl_wait();
  const long long words = static_cast<long long>(tiles) * chunks * 128;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < words;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int j = i & 3, lane = (i >> 2) & 31;
    const long long tc = i >> 7;
    const int chunk = static_cast<int>(tc % chunks), tile = static_cast<int>(tc / chunks);
    const int g = lane >> 2, c = lane & 3;
    const int col = chunk * kChunk + (j >> 1) * 32 + c * 8 + (j & 1) * 4;
    if (col >= k) continue;
    const uint32_t word = packed[i], s = scales[(static_cast<size_t>(tile) * groups + col / group) * 8 + g];
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const int row = tile * kRows + g + hi * 8;
      if (row >= n) continue;
      const float f = hi ? bf16_hi(s) : bf16_lo(s);
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = static_cast<float>(static_cast<int>((word >> (4 * (hi + (e >> 1) * 2 + (e & 1) * 4))) & 15u) - 8) * f;
      *reinterpret_cast<uint2*>(out + static_cast<size_t>(row) * k + col) =
          make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
  }
}

int tiles_of(int n) { return (n + kRows - 1) / kRows; }
int chunks_of(int k) { return (k + kChunk - 1) / kChunk; }
int groups_of(int k, int group) { return group == 32 ? 2 * chunks_of(k) : k / group; }

bool valid(int n, int k, int group) {
  return n > 0 && k > 0 && n % 8 == 0 && (group == 32 || group == 64 || group == 128) && k % group == 0 &&
         n < (1 << 27) && k < (1 << 27);
}

template <int MT, int R, int SEG>
int launch(const Params& p, int splits, int clusters, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return FB_ERR_LAUNCH;
  constexpr int kSmem = Shape<MT, R>::kSmem;
  if (kSmem > 48 * 1024 && (dev >= 64 || !configured[dev])) {
    if (cudaFuncSetAttribute(linear_w4_kernel<MT, R, SEG>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) !=
        cudaSuccess)
      return FB_ERR_LAUNCH;
    if (dev < 64) configured[dev] = true;
  }
  return launch_ex(linear_w4_kernel<MT, R, SEG>, dim3(splits, clusters), dim3(kThreads), kSmem, stream, splits, p);
}

template <int MT, int R>
int launch_segments(const Params& p, int group, int splits, int clusters, cudaStream_t s) {
  return group == 32 ? launch<MT, R, 2>(p, splits, clusters, s) : launch<MT, R, 1>(p, splits, clusters, s);
}

}  // namespace w4
}  // namespace fb

using namespace fb;

extern "C" size_t fb_w4_packed_bytes(int n, int k, int group) {
  if (!w4::valid(n, k, group)) return 0;
  return static_cast<size_t>(w4::tiles_of(n)) * w4::chunks_of(k) * 512;
}

extern "C" size_t fb_w4_scale_bytes(int n, int k, int group) {
  if (!w4::valid(n, k, group)) return 0;
  return static_cast<size_t>(w4::tiles_of(n)) * w4::groups_of(k, group) * 32;
}

extern "C" int fb_w4_pack(const int8_t* codes, const void* scales, void* packed, void* packed_scales, int n, int k,
                          int group, void* stream) {
  if (!codes || !scales || !packed || !packed_scales) return FB_ERR_ARG;
  if (!w4::valid(n, k, group)) return FB_ERR_SHAPE;
  return launch_ex(w4::pack_kernel, dim3(sm_count() * 8), dim3(256), 0, static_cast<cudaStream_t>(stream), 1, codes,
                   static_cast<const __nv_bfloat16*>(scales), static_cast<uint32_t*>(packed),
                   static_cast<uint32_t*>(packed_scales), n, k, group, w4::tiles_of(n), w4::chunks_of(k),
                   w4::groups_of(k, group));
}

extern "C" int fb_w4_dequantize(const void* packed, const void* packed_scales, void* out, int n, int k, int group,
                                void* stream) {
  if (!packed || !packed_scales || !out) return FB_ERR_ARG;
  if (!w4::valid(n, k, group)) return FB_ERR_SHAPE;
  return launch_ex(w4::dequantize_kernel, dim3(sm_count() * 8), dim3(256), 0, static_cast<cudaStream_t>(stream), 1,
                   static_cast<const uint32_t*>(packed), static_cast<const uint32_t*>(packed_scales),
                   static_cast<__nv_bfloat16*>(out), n, k, group, w4::tiles_of(n), w4::chunks_of(k),
                   w4::groups_of(k, group));
}

extern "C" int fb_linear_w4(const void* x, const void* packed, const void* packed_scales, void* out, int m, int n,
                            int k, int group, int epilogue, void* stream) {
  if (!x || !packed || !packed_scales || !out || m <= 0) return FB_ERR_ARG;
  if (epilogue < w4::kBf16 || epilogue > w4::kSwiGLU) return FB_ERR_ARG;
  if (!w4::valid(n, k, group) || m > w4::kMaxRows) return FB_ERR_SHAPE;
  if (epilogue == w4::kSwiGLU && n % 128 != 0) return FB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(packed)) & 15u) return FB_ERR_ARG;
  w4::Params p;
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.packed = static_cast<const uint4*>(packed);
  p.scales = static_cast<const uint32_t*>(packed_scales);
  p.out = out;
  p.m = m;
  p.n = n;
  p.k = k;
  p.tiles = w4::tiles_of(n);
  p.chunks = w4::chunks_of(k);
  p.groups = w4::groups_of(k, group);
  p.epilogue = epilogue;
  // Two CTAs over K halve what each reads of x; clusters fill the machine once.
  const int units = epilogue == w4::kSwiGLU ? p.tiles / 2 : p.tiles;
  const int splits = p.chunks >= 2 * w4::kWarps ? 2 : 1;
  int clusters = sm_count() / splits;
  if (clusters > units) clusters = units;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (m <= 8) return w4::launch_segments<1, 4>(p, group, splits, clusters, s);
  if (m <= 16) return w4::launch_segments<2, 4>(p, group, splits, clusters, s);
  if (m <= 32) return w4::launch_segments<4, 2>(p, group, splits, clusters, s);
  return w4::launch_segments<8, 2>(p, group, splits, clusters, s);
}
