// Projections with 4-bit weights and group scales, y[M, N] = x[M, K] @ W[N, K]^T for M <= 64 rows,
// W[n, k] = code[n, k] * scale[n, k / group], codes -8..7 (sm_100a, tcgen05).
//
// Bound by the packed codes (N K / 2 bytes) and, as built, by their unpacking (0.13 us of the ALU pipe for a
// block of 128 x 128 codes, which arrives in 0.19 us of an SM's share of the bandwidth), which is why the
// products leave the warps altogether: a thread owns one of a tile's 128 weight rows, unpacks its
// codes to bf16 and stores them to tensor memory, where they are the A operand of
// tcgen05.mma (D[128 x M'] += A[128 x 16] B[16 x M'], B = x in shared memory, M' = M padded to 16,
// 32 or 64). Each scale group accumulates in its own D columns; the thread that owns the row reads
// them back, multiplies by its scale in fp32 and adds them to its row's totals in registers. (A
// first form with mma.sync spent twice the instructions on fragments, addends and scaling.)
//
// Measured (us, weights from HBM, rates of codes and scales): 24576 x 4096, group 128, M = 16 20.0, 2.6 TB/s
// (without the conversion about 15, the rest is the 192 tiles' uneven share of 148 SMs and 5 us of launch, fill and
// merge); 4096 x 12288, group 32, M = 5 12.0, 2.4 TB/s; 6144 x 4096, M = 64 12.7; 4096 x 1024, group 64, M = 1 4.8.
//
// Unpacking is exact: a nibble q = code + 8 in the low mantissa bits of 128.0 is the bf16 number
// 128 + q; subtracting 136 leaves the code. W itself is never rounded, x stays bf16.
//
// Work: a cluster of `splits` CTAs owns a 128-row tile and cuts its 128-column blocks into equal
// contiguous ranges, one per CTA. (Clusters of several tiles, for evener waves, gained 9% at 24576 x 4096
// and lost 15% at small sizes.) The packed layout keeps a block's codes and scales together, so a block is
// one bulk copy (8 KB and 256 bytes a group) and two boxes of x. Warp roles: two sets of four unpacking warps
// that take parts in turn, each with its A and D, a producer and an MMA warp, whose issue sits behind
// elect.sync (behind `lane == 0` it took four times as long). Up to 32 rows two CTAs share an SM (but for 17 to 32
// rows in groups of 32, whose A and D take 384 of the 512 tensor memory columns). The CTAs' totals are pushed to the
// owner of each output through distributed shared memory and added in rank order: one launch, no workspace, the same
// bits every time, and the result leaves finished (bf16, fp32 or SwiGLU).
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "tcgen05.cuh"

namespace fb {
namespace w4 {

constexpr int kRows = 128;   // rows of a tile: the TMEM lanes
constexpr int kBlock = 128;  // columns of a block
constexpr int kRun = 32;     // columns of 16 bytes of codes
constexpr int kRunBytes = kRows * 16;
constexpr int kMaxRows = 64;
constexpr int kMaxSplits = 8;  // portable cluster size
constexpr int kSets = 2, kUnpackWarps = 4 * kSets, kProducerWarp = kUnpackWarps, kMmaWarp = kUnpackWarps + 1;
constexpr int kThreads = (kUnpackWarps + 2) * 32;

enum Epilogue : int { kBf16 = 0, kFp32 = 1, kSwiGLU = 2 };

// The packed layout: tile by tile, in each its blocks of 128 columns (the last may hold fewer runs):
// per run of 32 columns 16 bytes of codes a row, then per scale group 2 bytes a row.
struct Layout {
  int tiles, k, group_shift;  // a group is 1 << group_shift columns
  int block_bytes;            // of a whole block
  size_t tile_bytes;
  __host__ __device__ int blocks() const { return (k + kBlock - 1) / kBlock; }
  __host__ __device__ int columns(int block) const {
    const int left = k - block * kBlock;
    return left < kBlock ? left : kBlock;
  }
  __host__ __device__ int bytes(int block) const {
    const int c = columns(block);
    return c / kRun * kRunBytes + (c >> group_shift) * kRows * 2;
  }
  __host__ __device__ size_t at(int tile, int block) const {
    return tile * tile_bytes + static_cast<size_t>(block) * block_bytes;
  }
};

struct Params {
  const uint8_t* packed;
  void* out;
  int m, n, epilogue;
  Layout layout;
  unsigned* err;
};

// Copies `bytes` (a multiple of 16) of static weights, evicted first from L2.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// D (tensor memory) += A (tensor memory, one row per lane, two bf16 per column) * B (shared memory).
__device__ __forceinline__ void mma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u));
}

// One lane of a converged warp. The compiler sees that what the warp computed before is uniform and
// keeps the products' operands in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
  return r != 0;
}

// 16 consecutive 32-bit columns of this warp's lanes; complete after tcgen05.wait::st.
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The constants of the unpacking, kept in registers (a LOP3 takes one immediate).
struct Magic {
  uint32_t mask, base, bias;
  __device__ Magic() {
    asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(mask));
    asm volatile("mov.b32 %0, 0x43004300;" : "=r"(base));  // 128.0 twice
    asm volatile("mov.b32 %0, 0xc308c308;" : "=r"(bias));  // -136.0 twice
  }
};

// Two nibbles (bits 0-3 and 16-19 of w) to the bf16 pair of their codes.
__device__ __forceinline__ uint32_t codes_bf16x2(uint32_t w, const Magic& k) {
  uint32_t biased, v;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(biased) : "r"(w), "r"(k.mask), "r"(k.base));  // (w & mask) | 128.0
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(biased), "r"(k.bias));
  return v;
}

// M: padded rows of x (the products' N); SEGS: scale groups of a block.
template <int M_, int SEGS_>
struct Config {
  static constexpr int M = M_, SEGS = SEGS_;
  // A block is unpacked and multiplied in one part, or in two where its groups' D would not fit.
  static constexpr int PARTS = SEGS * M > 192 ? 2 : 1, kPart = kBlock / PARTS, GROUPS = SEGS / PARTS;
  // tensor memory: per set an A buffer of kPart / 2 columns and a D of M columns a group. Two CTAs share
  // the SM's 512 columns where that and the registers of M totals a thread allow it.
  static constexpr int kA = kPart / 2, kD = kA * kSets;  // columns of A, first column of D
  static constexpr int kTmem = M <= 32 && kD + kSets * GROUPS * M <= 256 ? 256 : 512;
  static_assert(kD + kSets * GROUPS * M <= kTmem, "tensor memory");
  static constexpr int kCtas = 512 / kTmem;
  static constexpr int kBoxBytes = M * 128;  // 64 columns of x
  static constexpr int kX = 2 * kBoxBytes;
  static constexpr int kW = 9 * 1024;  // codes and at most four groups' scales
  static constexpr int kStage = kX + kW;
  // totals received as an owner: [rank][set][column][local row], at most 2 ceil(64 / S) S <= 142 rows
  static constexpr int kRecv = kSets * 142 * M * 4;
  static constexpr int kFree = (228 * 1024) / kCtas - 1024 - 1024 - kRecv - 256;
  static constexpr int NS = kFree / kStage > 8 ? 8 : kFree / kStage;
  static constexpr int kTotal = 1024 + NS * kStage + kRecv + 256;
  static_assert(kTotal <= 227 * 1024, "shared memory");
  // An odd number of stages gives a stage to the two sets in turn, so a set sees every other phase of its
  // barrier and must not come back before the other's use has landed. The MMA warp takes parts in order:
  // while part u is missing a set waits for at most part u + 3.
  static_assert(NS >= 4 && kSets == 2, "a stage's next use lies beyond a set's lead");
};

template <typename C>
__global__ void __launch_bounds__(kThreads, C::kCtas)
    linear_w4_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ Params p) {
  constexpr int M = C::M, GROUPS = C::GROUPS, PARTS = C::PARTS, NS = C::NS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* recv = reinterpret_cast<float*>(ring + NS * C::kStage);
  uint64_t* full = reinterpret_cast<uint64_t*>(recv + C::kRecv / 4);  // copies -> everyone, per stage
  uint64_t* empty = full + NS;         // unpackers (codes read) and MMA lane (x read) -> producer
  uint64_t* a_full = empty + NS;       // set's unpackers -> MMA lane: A written, the last D read
  uint64_t* d_full = a_full + kSets;   // MMA lane -> set's unpackers: products done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_full + kSets);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * NS + 2 * kSets) * 8 + 8 <= 256, "barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = gridDim.x, rank = blockIdx.x;
  const int tile = blockIdx.y, blocks = p.layout.blocks();  // of a tile; this CTA: [b0, b0 + count)
  const int b0 = blocks * rank / splits, count = blocks * (rank + 1) / splits - b0;
  const int parts = count * PARTS;  // part i: stage i / PARTS % NS
  // the row's last block may be short: its parts have tail_columns(which) columns, others kPart
  const int short_block = p.layout.k % kBlock != 0 && b0 + count == blocks ? count - 1 : -1;
  auto tail_columns = [&](int which) { return max(0, min(C::kPart, p.layout.k % kBlock - which * C::kPart)); };
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], (4 + 1) * PARTS);
    }
    for (int i = 0; i < kSets; ++i) {
      mbar_init(&a_full[i], 4);
      mbar_init(&d_full[i], 1);
    }
    fence_barrier_init();
    prefetch_tensormap(&xmap);
    *abort_flag = 0;
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(static_cast<uint32_t>(C::kTmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (splits > 1) cluster_arrive_relaxed();  // this CTA runs: its memory may be written once all have said so
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;

  // A bounded wait; false (and the abort flag) when it or another wait gave up.
  auto wait = [&](uint64_t* bar, uint32_t parity, unsigned what) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag == 0 && mbar_wait_bounded(bar, parity)) return true;
    if (*abort_flag == 0) raise_error(p.err, what);
    *abort_flag = 1;
    return false;
  };

  if (warp == kProducerWarp) {
    const uint64_t policy = l2_evict_first_policy();
    auto weights = [&](int i, int s) {
      const int bytes = p.layout.bytes(b0 + i);
      const uint8_t* src = p.packed + p.layout.at(tile, b0 + i);
      if (elect_one()) {
        mbar_arrive_expect_tx(&full[s], bytes + C::kX);
        bulk_load(ring + s * C::kStage + C::kX, src, bytes, &full[s], policy);
      }
      __syncwarp();
    };
    auto inputs = [&](int i, int s) {
      const int column = (b0 + i) * kBlock;
      uint8_t* at = ring + s * C::kStage;
      if (elect_one()) {
        tma_load_2d(at, &xmap, &full[s], column, 0);
        tma_load_2d(at + C::kBoxBytes, &xmap, &full[s], column + 64, 0);
      }
      __syncwarp();
    };
    // weights are static: the ring fills before the wait on the previous kernel
    const int pre = count < NS ? count : NS;
    for (int i = 0; i < pre; ++i) weights(i, i);
    pdl_wait();
    for (int i = 0; i < pre; ++i) inputs(i, i);
    int i = pre;
    for (int s = 0, phase = 0; i < count; ++i) {  // stage i % NS, i / NS - 1 uses of it done
      if (!__all_sync(0xffffffffu, wait(&empty[s], phase, kErrTimeoutEmpty))) break;
      weights(i, s);
      inputs(i, s);
      if (++s == NS) s = 0, phase ^= 1;
    }
    if (*abort_flag != 0)  // copies in flight land before the CTA's shared memory is released
      for (int k = i > NS ? i - NS : 0; k < i; ++k) mbar_wait_bounded(&full[k % NS], (k / NS) & 1);
    __syncwarp();
    if (splits > 1) cluster_wait();
  } else if (warp == kMmaWarp) {
    constexpr uint32_t kIdesc = tc::idesc_bf16(kRows, M, false, false);
    constexpr int kPer = C::kPart / 16 / GROUPS;  // products of a group
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t ring_desc = tc::desc_sw128(smem_u32(ring), 16, 1024);
    for (int i = 0, s = 0, turn = 0; i < parts; ++i) {
      const int set = i % kSets;
      const int steps = (i / PARTS == short_block ? tail_columns(i % PARTS) : C::kPart) / 16;
      // the set has seen this stage land, and read D of its last part, before it wrote A
      if (!__all_sync(0xffffffffu, wait(&a_full[set], turn, kErrTimeoutMma))) break;
      tc::fence_after();
      const uint64_t xdesc = ring_desc + (s * C::kStage + i % PARTS * C::kBoxBytes) / 16;
      const uint32_t d = tmem_u + C::kD + set * GROUPS * M, a = tmem_u + set * C::kA;
      if (elect_one()) {
        if (steps == C::kPart / 16) {
#pragma unroll
          for (int kk = 0; kk < C::kPart / 16; ++kk)
            mma_bf16_ts(d + kk / kPer * M, a + kk * 8, xdesc + (kk / 4 * C::kBoxBytes + kk % 4 * 32) / 16, kIdesc,
                        kk % kPer != 0);
        } else {
          for (int kk = 0; kk < steps; ++kk)
            mma_bf16_ts(d + kk / kPer * M, a + kk * 8, xdesc + (kk / 4 * C::kBoxBytes + kk % 4 * 32) / 16, kIdesc,
                        kk % kPer != 0);
        }
        tc::commit(&empty[s]);
        tc::commit(&d_full[set]);
      }
      __syncwarp();
      if (set == kSets - 1) turn ^= 1;
      if (i % PARTS == PARTS - 1 && ++s == NS) s = 0;
    }
    if (splits > 1) cluster_wait();
  } else {
    // ============================ unpacking warps: a thread per row ============================
    const Magic magic;
    const int set = warp / 4, row = threadIdx.x % kRows;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp % 4 * 32) << 16);
    const uint32_t a_lanes = lanes + set * C::kA, d_lanes = lanes + C::kD + set * GROUPS * M;
    constexpr int kRuns = C::kPart / kRun;
    uint4 codes[kRuns];
    float scale[GROUPS];
    // The set's parts set, set + kSets, ... lie kSets / PARTS stages apart; with two parts a block a set takes
    // the same one of every block.
    constexpr int kStageStep = kSets / PARTS;
    const int which = PARTS == 1 ? 0 : set;
    const int tail_groups = tail_columns(which) >> p.layout.group_shift;
    const int tail_scales = p.layout.k % kBlock / kRun * kRunBytes;
    int s = set / PARTS, phase = 0;  // of the next fetch
    // Part i's codes and scales to registers; this warp is then done with the stage.
    auto fetch = [&](int i) {
      if (!__all_sync(0xffffffffu, wait(&full[s], phase, kErrTimeoutFull))) return false;
      const uint8_t* at = ring + s * C::kStage + C::kX;
#pragma unroll
      for (int r = 0; r < kRuns; ++r)  // runs and groups past the last block's columns read what is not used
        codes[r] = *reinterpret_cast<const uint4*>(at + (which * kRuns + r) * kRunBytes + row * 16);
      const uint8_t* scales =
          at + (i / PARTS == short_block ? tail_scales : kBlock / kRun * kRunBytes) + row * 2;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        scale[g] = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(scales + (which * GROUPS + g) * kRows * 2));
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      s += kStageStep;
      if (s >= NS) s -= NS, phase ^= 1;
      return true;
    };
    const int share = (64 + splits - 1) / splits;  // features (rows f and f + 64) of an owner
    const int f64 = row & 63, owner = f64 / share, local = (row >> 6) * share + f64 - owner * share;
    float total[M];
#pragma unroll
    for (int m = 0; m < M; ++m) total[m] = 0.f;
    bool ok = set >= parts || fetch(set);
    if (splits > 1) cluster_wait();  // every CTA of the cluster runs
    int turn = 0;
    for (int i = set; ok && i < parts; i += kSets) {  // this set's parts
      const int groups = i / PARTS == short_block ? tail_groups : GROUPS;
      // A is free: the products of this set's last block were waited for below
#pragma unroll
      for (int r = 0; r < kRuns; ++r) {
        const uint32_t words[4] = {codes[r].x, codes[r].y, codes[r].z, codes[r].w};
        uint32_t a[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[4 * j] = codes_bf16x2(words[j], magic);
          a[4 * j + 1] = codes_bf16x2(words[j] >> 4, magic);
          a[4 * j + 2] = codes_bf16x2(words[j] >> 8, magic);
          a[4 * j + 3] = codes_bf16x2(words[j] >> 12, magic);
        }
        st16(a_lanes + r * 16, a);
      }
      wait_st();
      tc::fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_full[set]);
      float f[GROUPS];
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) f[g] = scale[g];
      ok = i + kSets >= parts || fetch(i + kSets);  // while the part multiplies
      ok = ok && __all_sync(0xffffffffu, wait(&d_full[set], turn, kErrTimeoutMma));
      if (!ok) break;
      turn ^= 1;
      tc::fence_after();
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        if (g >= groups) break;
#pragma unroll
        for (int c = 0; c < M; c += 16) {
          float v[16];
          tc::ld16(d_lanes + g * M + c, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) total[c + e] += v[e] * f[g];
        }
      }
      tc::fence_before();  // the next a_full says that D was read
    }
    if (ok) {
      const uint32_t dst =
          map_shared(smem_u32(recv + (rank * kSets + set) * M * 2 * share + local), owner);
#pragma unroll
      for (int m = 0; m < M; ++m)
        if (m < p.m) st_cluster_f32(dst + m * 2 * share * 4, total[m]);
    }
    pdl_wait();  // the output may still be read by an earlier kernel
  }

  __syncwarp();
  // ---- each output at its owner: the totals of the CTAs and sets that had blocks of its tile, in order ----
  if (splits > 1)
    cluster_sync();  // every total has landed; nobody touches another CTA's memory after this
  else
    __syncthreads();
  const int share = (64 + splits - 1) / splits;
  const int mine = min(share, 64 - rank * share), wide = p.epilogue == kSwiGLU ? mine : 2 * mine;
  if (warp < kUnpackWarps && wide > 0) {
    const int per = kUnpackWarps * 32 / wide;  // columns that the threads cover at once
    const int at = threadIdx.x % wide, m0 = threadIdx.x / wide;
    const int hi = at >= mine ? 1 : 0, f = at - hi * mine;
    const int n = tile * kRows + hi * 64 + rank * share + f;
    auto sum = [&](int m, int half) {
      const float* src = recv + m * 2 * share + half * share + f;
      float v = src[0];
      for (int q = 1; q < splits * kSets; ++q) v += src[q * M * 2 * share];
      return v;
    };
    for (int m = m0; m0 < per && n < p.n && m < p.m; m += per) {
      if (p.epilogue == kSwiGLU) {
        const float gate = bf16_round(sum(m, 0)), up = bf16_round(sum(m, 1));
        static_cast<__nv_bfloat16*>(p.out)[static_cast<size_t>(m) * (p.n / 2) + tile * 64 + rank * share + f] =
            __float2bfloat16_rn(bf16_round(gate / (1.0f + expf(-gate))) * up);
      } else if (p.epilogue == kFp32) {
        static_cast<float*>(p.out)[static_cast<size_t>(m) * p.n + n] = sum(m, hi);
      } else {
        static_cast<__nv_bfloat16*>(p.out)[static_cast<size_t>(m) * p.n + n] = __float2bfloat16_rn(sum(m, hi));
      }
    }
  }
  // every product was waited for (or the launch aborted): the tensor memory can go
  tc::fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(static_cast<uint32_t>(C::kTmem)));
  }
}

// Word i of all codes, tile by tile, run by run: columns col .. col + 7 of a row, at byte `at`. Nibbles b and
// b + 4 hold columns col + 2 b and col + 2 b + 1: one register of the unpacking.
struct Word {
  int row, col;
  size_t at;
  __device__ Word(long long i, const Layout& l) {
    const int runs = l.k / kRun, lane_row = static_cast<int>(i >> 2) % kRows;
    const long long tr = i / (4 * kRows);
    const int tile = static_cast<int>(tr / runs), run = static_cast<int>(tr % runs);
    row = tile * kRows + lane_row;
    col = run * kRun + (i & 3) * 8;
    at = l.at(tile, run / (kBlock / kRun)) + (run % (kBlock / kRun)) * kRunBytes + lane_row * 16 + (i & 3) * 4;
  }
};

// Byte of the scale of a row's group.
__device__ __forceinline__ size_t scale_at(const Layout& l, int row, int group) {
  const int per = kBlock >> l.group_shift, block = group / per, tile = row / kRows;
  return l.at(tile, block) + l.columns(block) / kRun * kRunBytes + (group % per) * kRows * 2 + row % kRows * 2;
}

// codes int8 [N, K], scales bf16 [N, K / group] -> the packed layout; rows past N get code 0, scale 0.
__global__ void pack_kernel(const int8_t* codes, const __nv_bfloat16* scales, uint8_t* packed, int n, const Layout l) {
  pdl_wait();
  const long long first = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  const long long words = static_cast<long long>(l.tiles) * kRows * (l.k / 8);
  for (long long i = first; i < words; i += step) {
    const Word w(i, l);
    uint32_t word = 0;
    for (int e = 0; e < 8; ++e) {
      const int code = w.row < n ? codes[static_cast<size_t>(w.row) * l.k + w.col + e] : 0;
      word |= static_cast<uint32_t>((code + 8) & 15) << (4 * (e / 2) + 16 * (e & 1));
    }
    *reinterpret_cast<uint32_t*>(packed + w.at) = word;
  }
  const int groups = l.k >> l.group_shift;
  for (long long i = first; i < static_cast<long long>(l.tiles) * kRows * groups; i += step) {
    const int row = static_cast<int>(i / groups), group = static_cast<int>(i % groups);
    *reinterpret_cast<__nv_bfloat16*>(packed + scale_at(l, row, group)) =
        row < n ? scales[static_cast<size_t>(row) * groups + group] : __float2bfloat16_rn(0.f);
  }
}

// The weights' values, each rounded once to bf16: what the library product of a prompt reads.
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* packed, __nv_bfloat16* out, int n,
                                                         const Layout l) {
  pdl_wait();
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  const long long words = static_cast<long long>(l.tiles) * kRows * (l.k / 8);
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < words; i += step) {
    const Word w(i, l);
    if (w.row >= n) continue;
    const uint32_t word = *reinterpret_cast<const uint32_t*>(packed + w.at);
    const float f = __bfloat162float(
        *reinterpret_cast<const __nv_bfloat16*>(packed + scale_at(l, w.row, w.col >> l.group_shift)));
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = static_cast<float>(static_cast<int>((word >> (4 * (e / 2) + 16 * (e & 1))) & 15u) - 8) * f;
    *reinterpret_cast<uint4*>(out + static_cast<size_t>(w.row) * l.k + w.col) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
}

bool valid(int n, int k, int group) {
  return n > 0 && k > 0 && n % 8 == 0 && (group == 32 || group == 64 || group == 128) && k % group == 0 &&
         n < (1 << 23) && k < (1 << 27) && static_cast<long long>(n) * k <= 1ll << 34;  // Word's 32-bit row count
}

Layout layout_of(int n, int k, int group) {
  Layout l;
  l.tiles = (n + kRows - 1) / kRows;
  l.k = k;
  l.group_shift = group == 32 ? 5 : group == 64 ? 6 : 7;
  l.block_bytes = kBlock / kRun * kRunBytes + kBlock / group * kRows * 2;
  l.tile_bytes = static_cast<size_t>(k) / kRun * kRunBytes + static_cast<size_t>(k) / group * kRows * 2;
  return l;
}

constexpr int kMaxDevices = 64;

// Clusters of `splits` CTAs of a kernel that the device holds at once, kept per device.
template <typename C>
int resident_clusters(int splits) {
  static std::atomic<int> cache[kMaxDevices][kMaxSplits + 1];  // count + 1; 0: not asked
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < kMaxDevices && cache[dev][splits] != 0) return cache[dev][splits] - 1;
  if (cudaFuncSetAttribute(linear_w4_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kTotal) != cudaSuccess)
    return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, 1);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kTotal;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, linear_w4_kernel<C>, &cfg) != cudaSuccess || n < 0) {
    cudaGetLastError();
    n = 0;
  }
  if (dev < kMaxDevices) cache[dev][splits] = n + 1;
  return n;
}

// What a CTA costs beside its stream, in blocks: 3 us at 0.35 us a block.
constexpr int kFixed = 8;

// K splits: the least waves x (blocks of a CTA + what it costs beside them). Clusters that the device holds:
// the occupancy query counts one CTA per SM for kernels with tensor memory. Two share an SM where kCtas is 2,
// so a cluster of S also fits wherever one of S / 2 does with a CTA to an SM. At M = 16 it takes 8 for
// 4096 x 12288 (11.5 us; 6: 12.7, 4: 14.9, 1: 42.1) and 1 for 24576 x 4096 (20.0; 2: 20.5, 4: 24.8, 8: 41.4); at
// M = 64 2 for 6144 x 4096 (12.7; 1: 19.3, 4: 17.8). It does not count the merge, which grows with the cluster: 4
// would be better than its 5 for 6144 x 4096 at M = 16 (7.9 against 8.8) and than its 8 for 4096 x 1024 at M = 1
// (4.1 against 4.8).
template <typename C>
int launch(const CUtensorMap& xm, const Params& p, cudaStream_t stream) {
  const int blocks = p.layout.blocks(), tiles = p.layout.tiles;
  if (tiles > 65535) return FB_ERR_SHAPE;
  int best = 0;
  long long best_cost = 0;
  for (int splits = 1; splits <= kMaxSplits && splits <= blocks; ++splits) {
    int slots = resident_clusters<C>(splits) * C::kCtas;
    if (C::kCtas > 1) slots = std::max(slots, resident_clusters<C>((splits + 1) / 2));
    if (slots <= 0) continue;
    const long long waves = (tiles + slots - 1) / slots;
    const long long cost = waves * ((blocks + splits - 1) / splits + kFixed);
    if (best == 0 || cost < best_cost) {
      best = splits;
      best_cost = cost;
    }
  }
  if (best == 0) return FB_ERR_LAUNCH;
  return launch_ex(linear_w4_kernel<C>, dim3(best, tiles), dim3(kThreads), C::kTotal, stream, best, xm, p);
}

template <int M>
int launch_groups(const CUtensorMap& xm, const Params& p, cudaStream_t s) {
  if (p.layout.group_shift == 5) return launch<Config<M, 4>>(xm, p, s);
  if (p.layout.group_shift == 6) return launch<Config<M, 2>>(xm, p, s);
  return launch<Config<M, 1>>(xm, p, s);
}

}  // namespace w4
}  // namespace fb

using namespace fb;

extern "C" size_t fb_w4_packed_bytes(int n, int k, int group) {
  if (!w4::valid(n, k, group)) return 0;
  const w4::Layout l = w4::layout_of(n, k, group);
  return l.tiles * l.tile_bytes;
}

extern "C" int fb_w4_pack(const int8_t* codes, const void* scales, void* packed, int n, int k, int group,
                          void* stream) {
  if (!codes || !scales || !packed) return FB_ERR_ARG;
  if (!w4::valid(n, k, group)) return FB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(packed) & 15u) return FB_ERR_ARG;
  return launch_ex(w4::pack_kernel, dim3(sm_count() * 8), dim3(256), 0, static_cast<cudaStream_t>(stream), 1, codes,
                   static_cast<const __nv_bfloat16*>(scales), static_cast<uint8_t*>(packed), n,
                   w4::layout_of(n, k, group));
}

extern "C" int fb_w4_dequantize(const void* packed, void* out, int n, int k, int group, void* stream) {
  if (!packed || !out) return FB_ERR_ARG;
  if (!w4::valid(n, k, group)) return FB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(packed) | reinterpret_cast<uintptr_t>(out)) & 15u) return FB_ERR_ARG;
  return launch_ex(w4::dequantize_kernel, dim3(sm_count() * 8), dim3(256), 0, static_cast<cudaStream_t>(stream), 1,
                   static_cast<const uint8_t*>(packed), static_cast<__nv_bfloat16*>(out), n, w4::layout_of(n, k, group));
}

extern "C" int fb_linear_w4(const void* x, const void* packed, void* out, int m, int n, int k, int group, int epilogue,
                            void* stream) {
  if (!x || !packed || !out || m <= 0) return FB_ERR_ARG;
  if (epilogue < w4::kBf16 || epilogue > w4::kSwiGLU) return FB_ERR_ARG;
  if (!w4::valid(n, k, group) || m > w4::kMaxRows) return FB_ERR_SHAPE;
  if (epilogue == w4::kSwiGLU && n % 128 != 0) return FB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(packed)) & 15u) return FB_ERR_ARG;
  w4::Params p;
  p.packed = static_cast<const uint8_t*>(packed);
  p.out = out;
  p.m = m;
  p.n = n;
  p.epilogue = epilogue;
  p.layout = w4::layout_of(n, k, group);
  p.err = error_word();
  const int rows = m <= 16 ? 16 : m <= 32 ? 32 : 64;
  CUtensorMap xm;
  const int st = encode_bf16_2d(&xm, x, m, k, k, 64, rows, true);
  if (st != FB_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 16) return w4::launch_groups<16>(xm, p, s);
  if (rows == 32) return w4::launch_groups<32>(xm, p, s);
  return w4::launch_groups<64>(xm, p, s);
}
