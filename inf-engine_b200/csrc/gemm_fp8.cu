// y[M, N] = x[M, K] w[N, K]^T with both operands in 8-bit floating point (e4m3): x with a scale for each row and 128 columns,
// w with a scale for each block of 128 x 128,
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b]  sum_{k in block b} x[m, k] w[n, k]
//
// inner and outer sums in float32, one rounding to the output's type.
//
// Four kernels, by the rows of x and the length of the weight (gemm_fp8 at the end holds the rules, with both sides measured):
//   few rows          registers and the matrix instructions for halves; bfloat16 rows may be quantised inside
//   a long weight     under up to 32 rows: the tensor cores, w as the larger operand, bound by the weight's bytes (5.6 TB/s)
//   tiles             128 x 128, K dealt out over a cluster where tiles are few
//   pairs             256 x 256 over two SMs: 4096 x 8192 x 8192 in 237 us (2.32 PFLOP/s; 276 us and 1.99 under the card's power
//                     cap).  The library's product of the same codes with one scale for all takes 190 and 220: the rest is the
//                     scaling of every block of 128, 2.1 thousand million multiply-adds out of tensor memory.
#include "fp8_codes.cuh"
#include <cooperative_groups.h>
#include <cuda.h>

namespace cg = cooperative_groups;

namespace {

enum { IE_E4M3 = 2 };      // dtype code of an operand that is quantised already
#define IE_NEEDS_SCRATCH -5  /* the rows are to be quantised, and there is no room for their codes */

struct Fp8Params {
  const uint8_t* x;
  const float* sx;
  const uint8_t* w;
  const float* sw;
  void* y;
  int M, N, K;
  long long ldx, sx_row, sx_col, ldw, ldy;
  int y_bf16;
  int y_vec;       // rows of y start on 16 bytes
  int split;       // blocks of a cluster that share a tile
  // the kernel ahead is the quantiser of x, whose blocks are past their own wait when one of this kernel starts: whatever wrote the
  // weights has finished then, so they may be asked for before this kernel's wait
  int early;
  // x in bfloat16 where the product quantises it itself; whether its rows can be read 16 bytes at a time
  const void* raw;
  int raw_vec;
};

// ------------------------------------------------------------------- tiles on the tensor cores
// One stage of the ring is one block of 128 codes of K (a 128-byte swizzle row), so one scale of x a row and one of w for 128
// columns hold for all of it: four MMAs of 32 codes make the block's sum in tensor memory from nothing, and eight warps add it,
// scaled, to the sums that they keep in registers, while the MMAs of the next block fill the other half of tensor memory.
constexpr int X_BYTES = 128 * GROUP, STAGE = 2 * X_BYTES, STAGES = 5;     // a block of K of 128 rows of x and 128 rows of w
// Twelve warps: TMA, MMA, two that do nothing, eight that sum.  A thread is launched with 168 registers (three warps a quarter of
// the SM); the first four warps hand some of theirs on: 4 * 56 + 8 * 224 = 12 * 168.
// (Only the wide tile, whose sums alone take 128 registers, needs it.)
constexpr int TILE_THREADS = 384;
constexpr int REGS_LAUNCH = 168, REGS_FEW = 56, REGS_MANY = 224;
static_assert(REGS_FEW + 2 * REGS_MANY <= 3 * REGS_LAUNCH, "a share beyond what the block was launched with is never given out");
constexpr unsigned SPIN_LIMIT = 1u << 20;
constexpr int AHEAD = 8;               // blocks of K that the scales are asked for ahead
constexpr int OUT_STAGE = 32 * 128;    // bytes of a summing warp's output tile: 32 rows x 128 bytes

__device__ int g_fp8_error = 0;

__device__ __forceinline__ uint32_t saddr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// an arrival at a barrier of any block of the cluster (an address of map_shared)
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t map_shared(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// one lane of a converged warp.  The warps that issue copies and MMAs run their loops whole and elect a lane for the issue alone:
// what all lanes compute alike stays in the uniform registers that those instructions take (with a loop run by lane 0, moving it
// there cost the MMA warp 900 cycles a block of K, of which its four MMAs are 512).
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(is));
  return is != 0;
}
// waits for a phase; false when the limit is reached or another thread of the block has given up
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const volatile int* failed) {
  for (unsigned i = 0; i < SPIN_LIMIT; ++i) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
    if (*failed) return false;
  }
  return false;
}
// PAIR: the bytes are counted at a barrier that may be the other block's
template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if (PAIR)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
// shared-memory descriptor: K-major rows of 128 bytes, 128-byte swizzle, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t smem_desc(uint32_t byte_addr) {
  return (uint64_t)((byte_addr & 0x3FFFF) >> 4) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// D float32, A and B e4m3, both K-major, m x n
__device__ __forceinline__ constexpr uint32_t instr_desc(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void mma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (PAIR)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// an arrival at the barrier (PAIR: at that of both blocks) when the MMAs so far have finished
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
}
// the registers are named, so that nothing that reads them moves ahead of the wait
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :: "memory");
}

// two float32 multiply-adds in one instruction: acc += c * f, each of the two rounded as a single one is
__device__ __forceinline__ void fma2(unsigned long long& acc, uint32_t c0, uint32_t c1, unsigned long long f) {
  asm("{\n.reg .b64 c;\nmov.b64 c, {%1, %2};\nfma.rn.f32x2 %0, c, %3, %0;\n}" : "+l"(acc) : "r"(c0), "r"(c1), "l"(f));
}
__device__ __forceinline__ unsigned long long pair(float a, float b) {
  return (unsigned long long)__float_as_uint(a) | ((unsigned long long)__float_as_uint(b) << 32);
}
__device__ __forceinline__ float low(unsigned long long v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high(unsigned long long v) { return __uint_as_float((uint32_t)(v >> 32)); }

// 128 bytes of a row of y that starts anywhere, from column n, by a warp whose lanes hold four bytes each. Halves that start
// between two words move up by one, so that all but the first and the last still leave as whole words.
// 2,805 x 1,075 x 256 from codes: 10.7 us, 2,039 x 3,701 x 4,759: 50.9; number by number 13.6 and 57.2, and 5.7 and 41.8 where rows of
// y start on 16 bytes (1,072 and 3,704 columns).
__device__ __forceinline__ void store_row(const Fp8Params& p, int m, int n, int lane, uint32_t v) {
  const uint32_t next = __shfl_down_sync(0xffffffffu, v, 1);
  if (m >= p.M) return;
  if (!p.y_bf16) {
    if (n + lane < p.N) ((uint32_t*)p.y)[m * p.ldy + n + lane] = v;
    return;
  }
  unsigned short* y = (unsigned short*)p.y + m * p.ldy + n;
  const int odd = (int)(((uintptr_t)y >> 1) & 1), e = 2 * lane + odd, end = min(64, p.N - n);
  if (odd) {
    if (lane == 0 && end > 0) y[0] = (unsigned short)v;
    v = __byte_perm(v, next, 0x5432);
  }
  if (e + 1 < end) *reinterpret_cast<uint32_t*>(y + e) = v;
  else if (e < end) y[e] = (unsigned short)v;
}
// 16 bytes of a row of y that starts on 16, from column n: number by number at the matrix's edge
__device__ __forceinline__ void store16(const Fp8Params& p, int m, int n, uint4 v) {
  const int per = p.y_bf16 ? 8 : 4;
  unsigned char* dst = (unsigned char*)p.y + ((long long)m * p.ldy + n) * (p.y_bf16 ? 2 : 4);
  if (n + per <= p.N) {
    *reinterpret_cast<uint4*>(dst) = v;
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (p.y_bf16) {
      if (n + 2 * j < p.N) reinterpret_cast<unsigned short*>(dst)[2 * j] = (unsigned short)w[j];
      if (n + 2 * j + 1 < p.N) reinterpret_cast<unsigned short*>(dst)[2 * j + 1] = (unsigned short)(w[j] >> 16);
    } else if (n + j < p.N) {
      reinterpret_cast<uint32_t*>(dst)[j] = w[j];
    }
  }
}
__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// four results of a row
__device__ __forceinline__ void store4(const Fp8Params& p, int m, int n, float4 v) {
  if (!p.y_vec || n + 4 > p.N) {
    const float s[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) {
        if (p.y_bf16) ((bf16*)p.y)[m * p.ldy + n + j] = __float2bfloat16_rn(s[j]);
        else ((float*)p.y)[m * p.ldy + n + j] = s[j];
      }
  } else if (p.y_bf16) {
    *reinterpret_cast<uint2*>((bf16*)p.y + m * p.ldy + n) = make_uint2(two_bf16(v.x, v.y), two_bf16(v.z, v.w));
  } else {
    *reinterpret_cast<float4*>((float*)p.y + m * p.ldy + n) = v;
  }
}

// PAIR: two blocks of a cluster make 256 x 256 of the result with MMAs over both SMs: each brings its 128 rows of x and HALF of the
// 256 rows of w, so a block of K is 32 KB an SM where a tile of 128 x 256 alone takes 48 KB (and at 512 cycles of MMAs asks more
// of the L2 than an SM gets from it).  The first block issues the MMAs; each block sums its own 128 rows.
// SPLIT: 128 x 128; a tile's blocks of K are dealt out to the blocks of a cluster, whose sums come together through each other's
// shared memory, in the order of K.  Neither: 128 x 128, a block walks over tiles.
template <bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(TILE_THREADS, 1) gemm_fp8_tile_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                        const __grid_constant__ CUtensorMap map_w, Fp8Params p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long bars[2 * STAGES + 4];     // full, empty, acc_full[2], acc_empty[2]
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  constexpr int TM = PAIR ? 256 : 128, TN = PAIR ? 256 : 128;          // the tile
  constexpr int COLS = TN / 2;                                         // columns of a summing warp: of one block of w's scales

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t ring = (saddr(smem_raw) + 1023u) & ~1023u;
  unsigned char* ring_ptr = smem_raw + (ring - saddr(smem_raw));
  const uint32_t full0 = saddr(&bars[0]), empty0 = saddr(&bars[STAGES]), acc_full0 = saddr(&bars[2 * STAGES]), acc_empty0 = acc_full0 + 16;
  const int k_blocks = (p.K + GROUP - 1) / GROUP, m_tiles = (p.M + TM - 1) / TM, tiles = m_tiles * ((p.N + TN - 1) / TN);
  const int per_tile = PAIR ? 2 : SPLIT ? p.split : 1;                 // blocks of a tile (a cluster), and which of them this is
  const int rank = (int)(blockIdx.x % per_tile);
  const int t0 = (int)(blockIdx.x / per_tile), t_step = SPLIT ? tiles : (int)(gridDim.x / per_tile);
  const int kb0 = SPLIT ? k_blocks * rank / p.split : 0, kb1 = SPLIT ? k_blocks * (rank + 1) / p.split : k_blocks;
  const int part = PAIR ? rank * 128 : 0;                              // this block's rows of x and of w in the tile

  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
    failed = 0;
    for (int s = 0; s < STAGES; ++s) {
      bar_init(full0 + 8 * s, 1);
      bar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      bar_init(acc_full0 + 8 * b, 1);
      bar_init(acc_empty0 + 8 * b, PAIR ? 16 : 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&tmem_slot)), "n"(2 * TN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&tmem_slot)), "n"(2 * TN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  if (PAIR) cg::this_cluster().sync();                                 // the other block's barriers and tensor memory are there
  else __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  pdl_trigger();                                       // a kernel that starts beside this one finds tensor memory taken, not this one
  if (warp < 4) {
    if (PAIR) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEW));
    if (warp == 0) {
      const uint32_t first_full = PAIR ? map_shared(full0, 0) : full0;
      int s = 0;
      uint32_t phase = 0;
      bool ok = true;
      // the ring's first round of the weight goes out before the codes of x are there
      const int ahead = p.early ? min(STAGES, kb1 - kb0) : 0;
      if (elect_one()) {
        for (int i = 0; i < ahead; ++i) {
          if (rank == 0 || !PAIR) bar_expect(full0 + 8 * i, (PAIR ? 2 : 1) * STAGE);
          tma_load<PAIR>(ring + i * STAGE + X_BYTES, &map_w, (kb0 + i) * GROUP, (t0 / m_tiles) * TN + part, first_full + 8 * i);
        }
      }
      __syncwarp();
      pdl_wait();
      for (int t = t0; t < tiles && ok; t += t_step) {
        const int m0 = (t % m_tiles) * TM + part, n0 = (t / m_tiles) * TN + part;        // tiles side by side share the weight
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = __all_sync(0xffffffffu, bar_wait(empty0 + 8 * s, phase ^ 1, &failed));
          if (!ok) { atomicExch(&g_fp8_error, 1); failed = 1; break; }
          const bool asked = t == t0 && kb - kb0 < ahead;
          if (elect_one()) {
            if (!asked && (rank == 0 || !PAIR)) bar_expect(full0 + 8 * s, (PAIR ? 2 : 1) * STAGE);
            tma_load<PAIR>(ring + s * STAGE, &map_x, kb * GROUP, m0, first_full + 8 * s);
            if (!asked) tma_load<PAIR>(ring + s * STAGE + X_BYTES, &map_w, kb * GROUP, n0, first_full + 8 * s);
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; phase ^= 1; }
        }
      }
      if (failed) for (int i = 0; i < 2048; ++i) __nanosleep(64);        // copies under way still land in this block's memory
    } else if (warp == 1 && (rank == 0 || !PAIR)) {
      pdl_wait();                                      // its waits have a limit: they begin when the kernel ahead is done
      int s = 0, buf = 0;
      uint32_t phase = 0, acc_phase = 1;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += t_step) {
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = __all_sync(0xffffffffu, bar_wait(acc_empty0 + 8 * buf, acc_phase, &failed));
          if (!ok) { atomicExch(&g_fp8_error, 2); failed = 1; break; }
          ok = __all_sync(0xffffffffu, bar_wait(full0 + 8 * s, phase, &failed));
          if (!ok) { atomicExch(&g_fp8_error, 3); failed = 1; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t a = smem_desc(ring + s * STAGE), b = smem_desc(ring + s * STAGE + X_BYTES);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < GROUP / 32; ++k)               // 32 codes on: 2 units of 16 bytes in the descriptor's address
              mma_fp8<PAIR>(tmem + (uint32_t)(buf * TN), a + 2 * k, b + 2 * k, instr_desc(TM, TN), k > 0 ? 1u : 0u);
            mma_commit<PAIR>(empty0 + 8 * s);                  // the stage has been read
            mma_commit<PAIR>(acc_full0 + 8 * buf);             // the block's sum is there
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; phase ^= 1; }
          buf ^= 1;
          acc_phase ^= buf == 0 ? 1u : 0u;
        }
      }
    }
  } else {
    if (PAIR) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_MANY));
    const int quarter = warp & 3, half = (warp - 4) >> 2;          // tensor memory lanes 32 quarter .., columns COLS half ..
    const uint32_t my_tmem = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * COLS);
    const uint32_t first_empty = PAIR ? map_shared(acc_empty0, 0) : acc_empty0;
    // The scales of a block come AHEAD blocks early into slots of the warp's own (a load of theirs takes as long as several blocks' MMAs),
    // on into the next tile: 32 of x side by side, then the one of w, copied once.  (Shared memory feeds the MMAs too: with a
    // copy of w's scale for every lane, 8 bytes apart, the copies took 300 of its cycles a block.)
    constexpr uint32_t SLOT = 36 * 4;
    const uint32_t slots = ring + STAGES * STAGE + 8 * OUT_STAGE + (warp - 4) * AHEAD * SLOT;
    int ahead_t = t0, ahead_kb = kb0, ahead_slot = 0;
    const float *ahead_sx = nullptr, *ahead_sw = nullptr;
    const auto ask = [&]() {
      if (ahead_t < tiles) {
        if (ahead_kb == kb0) {
          const int m = (ahead_t % m_tiles) * TM + part + quarter * 32 + lane, n = (ahead_t / m_tiles) * TN + half * COLS;
          ahead_sx = p.sx + min(m, p.M - 1) * p.sx_row + kb0 * p.sx_col;
          ahead_sw = p.sw + (long long)(min(n, p.N - 1) / GROUP) * k_blocks + kb0;
        }
        const uint32_t dst = slots + ahead_slot * SLOT;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4 * lane), "l"(ahead_sx) : "memory");
        if (lane == 0) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 128), "l"(ahead_sw) : "memory");
        ahead_sx += p.sx_col;
        ++ahead_sw;
        if (++ahead_kb == kb1) { ahead_kb = kb0; ahead_t += t_step; }
      }
      ahead_slot = (ahead_slot + 1) % AHEAD;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    pdl_wait();                                        // the scales of x come from the kernel ahead
    for (int i = 0; i < AHEAD - 1; ++i) ask();
    int it = 0;
    bool ok = true;
    for (int t = t0; t < tiles && ok; t += t_step) {
      const int m0 = (t % m_tiles) * TM + part + quarter * 32, n0 = (t / m_tiles) * TN + half * COLS;
      unsigned long long acc[COLS / 2];
#pragma unroll
      for (int j = 0; j < COLS / 2; ++j) acc[j] = 0ull;
#pragma unroll 1
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int buf = it & 1;
        ask();                                         // into the slot of the block before, which every lane has read
        asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
        __syncwarp();                                  // lane 0's copy of w's scale is there for all
        float fx, fw;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(fx) : "r"(slots + (it % AHEAD) * SLOT + 4 * lane) : "memory");
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(fw) : "r"(slots + (it % AHEAD) * SLOT + 128) : "memory");
        const unsigned long long f = pair(fx * fw, fx * fw);
        ok = bar_wait(acc_full0 + 8 * buf, (uint32_t)(it >> 1) & 1u, &failed);
        if (!ok) { atomicExch(&g_fp8_error, 4); failed = 1; }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // 16 columns are under way while the 16 before them are added
        uint32_t r[2][16];
        tmem_ld16(my_tmem + (uint32_t)(buf * TN), r[0]);
#pragma unroll
        for (int c = 0; c < COLS / 16; ++c) {
          tmem_ld_wait(r[c & 1]);
          if (c + 1 < COLS / 16) {
            tmem_ld16(my_tmem + (uint32_t)(buf * TN + 16 * (c + 1)), r[(c + 1) & 1]);
          } else {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");      // all of it is in registers
            __syncwarp();
            if (lane == 0) { if (PAIR) bar_arrive_cluster(first_empty + 8 * buf); else bar_arrive(acc_empty0 + 8 * buf); }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) fma2(acc[8 * c + j], r[c & 1][2 * j], r[c & 1][2 * j + 1], f);
        }
      }
      if (!ok) break;
      if (SPLIT) {
        // the ring is free: every copy has landed and every MMA that read it has finished
        float* row = reinterpret_cast<float*>(ring_ptr) + (quarter * 32 + lane) * (TN + 4) + half * COLS;
#pragma unroll
        for (int j = 0; j < COLS / 4; ++j)
          *reinterpret_cast<float4*>(row + 4 * j) = make_float4(low(acc[2 * j]), high(acc[2 * j]), low(acc[2 * j + 1]), high(acc[2 * j + 1]));
      } else {
        // a lane holds a row: 128 bytes of each of the warp's 32 rows go through shared memory and out as whole lines (16-byte units
        // swizzled by row, so that neither side has bank conflicts)
        unsigned char* stage = ring_ptr + STAGES * STAGE + (warp - 4) * OUT_STAGE;
        const int per = p.y_bf16 ? 64 : 32, sw8 = lane & 7;
#pragma unroll
        for (int c = 0; c < COLS / 32; ++c) {
          if (p.y_bf16) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint4 v;
              v.x = two_bf16(low(acc[16 * c + 4 * u]), high(acc[16 * c + 4 * u]));
              v.y = two_bf16(low(acc[16 * c + 4 * u + 1]), high(acc[16 * c + 4 * u + 1]));
              v.z = two_bf16(low(acc[16 * c + 4 * u + 2]), high(acc[16 * c + 4 * u + 2]));
              v.w = two_bf16(low(acc[16 * c + 4 * u + 3]), high(acc[16 * c + 4 * u + 3]));
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * (c & 1) + u) ^ sw8) << 4)) = v;
            }
            if ((c & 1) == 0) continue;
          } else {
#pragma unroll
            for (int u = 0; u < 8; ++u)
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((u ^ sw8) << 4)) =
                  make_uint4((uint32_t)acc[16 * c + 2 * u], (uint32_t)(acc[16 * c + 2 * u] >> 32), (uint32_t)acc[16 * c + 2 * u + 1],
                             (uint32_t)(acc[16 * c + 2 * u + 1] >> 32));
          }
          __syncwarp();
          const int first = n0 + 32 * c + 32 - per, u = lane & 7;
          if (p.y_vec) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = 4 * i + (lane >> 3), m = m0 + r, n = first + u * (per >> 3);
              const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((u ^ (r & 7)) << 4));
              if (m < p.M && n < p.N) store16(p, m, n, v);
            }
          } else {
            // rows of y start anywhere: a row at a time, four bytes a lane side by side
#pragma unroll 8
            for (int r = 0; r < 32; ++r) {
              const uint32_t v = *reinterpret_cast<const uint32_t*>(stage + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + ((lane & 3) << 2));
              store_row(p, m0 + r, first, lane, v);
            }
          }
          __syncwarp();
        }
      }
    }
  }

  asm volatile("cp.async.wait_all;" ::: "memory");
  if (SPLIT) {
    // every block of the cluster comes here, one whose waits ran out too
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    // each block adds up its share of the tile's rows that lie in the matrix, 4 columns a thread
    const int m0 = (t0 % m_tiles) * TM, n0 = (t0 / m_tiles) * TN, items = min(p.M - m0, 128) * (TN / 4);
    const int first = items * rank / p.split, end = items * (rank + 1) / p.split;
    for (int i = first + tid; i < end; i += TILE_THREADS) {
      const int r = i / (TN / 4), c = i % (TN / 4) * 4;
      float4 v[8];                                     // all under way at once: one after the other they are 8 trips to another SM
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < p.split) v[q] = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(cluster.map_shared_rank(ring_ptr, q)) + r * (TN + 4) + c);
      float4 s = v[0];
#pragma unroll
      for (int q = 1; q < 8; ++q)
        if (q < p.split) { s.x += v[q].x; s.y += v[q].y; s.z += v[q].z; s.w += v[q].w; }
      store4(p, m0 + r, n0 + c, s);
    }
    cluster.sync();                                    // a block's memory is read until here
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  if (PAIR) cg::this_cluster().sync();                 // the other block's MMAs read this one's memory, and its warps arrive here
  else __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(2 * TN) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(2 * TN) : "memory");
  }
}

// ------------------------------------------------------------------- a long weight under few rows
// Up to 32 rows of x: the weight's bytes are the bound, and it is the MMA's larger operand: 128 rows of w by TX rows of x a tile, a block
// of K a stage.  Nothing converts a code (on the matrix instructions for halves, the conversions of both operands take 96 cycles of an
// SM for 2 KB of the weight, which memory brings in 85), the ring holds 9 or 10 stages of 16 KB, and with TX columns a sum the tensor
// memory holds four blocks' sums, so the trip from MMA to summing warps and back is not waited for.  One scale of w holds for a
// whole tile, those of x go by columns.  SPLIT as above: the blocks of a cluster share a tile.
constexpr int THIN_THREADS = 256, THIN_SUMS = 4, THIN_LEAST = 4;       // TMA, MMA, two that do nothing, four that sum
template <int TX> constexpr int THIN_STAGE = (128 + TX) * GROUP;
template <int TX> constexpr int THIN_STAGES = TX == 16 ? 10 : 9;
template <int TX> constexpr int THIN_SMEM = 1024 + THIN_STAGES<TX> * THIN_STAGE<TX>;

template <int TX, bool SPLIT>
__global__ void __launch_bounds__(THIN_THREADS, 1) gemm_fp8_thin_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                        const __grid_constant__ CUtensorMap map_w, Fp8Params p) {
  constexpr int NS = THIN_STAGES<TX>, BYTES = THIN_STAGE<TX>, W_BYTES = 128 * GROUP, PITCH = 132;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long bars[2 * NS + 2 * THIN_SUMS];     // full, empty, acc_full, acc_empty
  __shared__ __align__(16) float scales[4][AHEAD][TX + 4];                     // of each summing warp: of x, then that of w
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  static_assert(TX * PITCH * 4 <= NS * BYTES, "the sums of a split tile fit the ring");

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t ring = (saddr(smem_raw) + 1023u) & ~1023u;
  unsigned char* ring_ptr = smem_raw + (ring - saddr(smem_raw));
  const uint32_t full0 = saddr(&bars[0]), empty0 = saddr(&bars[NS]), acc_full0 = saddr(&bars[2 * NS]), acc_empty0 = acc_full0 + 8 * THIN_SUMS;
  const int k_blocks = (p.K + GROUP - 1) / GROUP, tiles = (p.N + 127) / 128;
  const int rank = SPLIT ? (int)(blockIdx.x % p.split) : 0;
  const int t0 = SPLIT ? (int)(blockIdx.x / p.split) : (int)blockIdx.x, t_step = SPLIT ? tiles : (int)gridDim.x;
  const int kb0 = SPLIT ? k_blocks * rank / p.split : 0, kb1 = SPLIT ? k_blocks * (rank + 1) / p.split : k_blocks;

  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
    failed = 0;
    for (int s = 0; s < NS; ++s) {
      bar_init(full0 + 8 * s, 1);
      bar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < THIN_SUMS; ++b) {
      bar_init(acc_full0 + 8 * b, 1);
      bar_init(acc_empty0 + 8 * b, 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&tmem_slot)), "n"(THIN_SUMS * TX) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  pdl_trigger();                                       // a kernel that starts beside this one finds tensor memory taken, not this one

  if (warp == 0) {
    int s = 0;
    uint32_t phase = 0;
    bool ok = true;
    const int ahead = p.early ? min(NS, kb1 - kb0) : 0;              // the ring's first round of the weight, before x is there
    if (elect_one()) {
      for (int i = 0; i < ahead; ++i) {
        bar_expect(full0 + 8 * i, BYTES);
        tma_load<false>(ring + i * BYTES, &map_w, (kb0 + i) * GROUP, t0 * 128, full0 + 8 * i);
      }
    }
    __syncwarp();
    pdl_wait();
    for (int t = t0; t < tiles && ok; t += t_step) {
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = __all_sync(0xffffffffu, bar_wait(empty0 + 8 * s, phase ^ 1, &failed));
        if (!ok) { atomicExch(&g_fp8_error, 5); failed = 1; break; }
        const bool asked = t == t0 && kb - kb0 < ahead;
        if (elect_one()) {
          if (!asked) {
            bar_expect(full0 + 8 * s, BYTES);
            tma_load<false>(ring + s * BYTES, &map_w, kb * GROUP, t * 128, full0 + 8 * s);
          }
          tma_load<false>(ring + s * BYTES + W_BYTES, &map_x, kb * GROUP, 0, full0 + 8 * s);
        }
        __syncwarp();
        if (++s == NS) { s = 0; phase ^= 1; }
      }
    }
    if (failed) for (int i = 0; i < 2048; ++i) __nanosleep(64);      // copies under way still land in this block's memory
  } else if (warp == 1) {
    pdl_wait();                                        // its waits have a limit: they begin when the kernel ahead is done
    int s = 0, buf = 0;
    uint32_t phase = 0, acc_phase = 1;
    bool ok = true;
    for (int t = t0; t < tiles && ok; t += t_step) {
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = __all_sync(0xffffffffu, bar_wait(acc_empty0 + 8 * buf, acc_phase, &failed));
        if (!ok) { atomicExch(&g_fp8_error, 6); failed = 1; break; }
        ok = __all_sync(0xffffffffu, bar_wait(full0 + 8 * s, phase, &failed));
        if (!ok) { atomicExch(&g_fp8_error, 7); failed = 1; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t a = smem_desc(ring + s * BYTES), b = smem_desc(ring + s * BYTES + W_BYTES);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < GROUP / 32; ++k)
            mma_fp8<false>(tmem + (uint32_t)(buf * TX), a + 2 * k, b + 2 * k, instr_desc(128, TX), k > 0 ? 1u : 0u);
          mma_commit<false>(empty0 + 8 * s);
          mma_commit<false>(acc_full0 + 8 * buf);
        }
        __syncwarp();
        if (++s == NS) { s = 0; phase ^= 1; }
        if (++buf == THIN_SUMS) { buf = 0; acc_phase ^= 1; }
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3;                                    // tensor memory lanes, rows of w
    const uint32_t my_tmem = tmem + ((uint32_t)(quarter * 32) << 16);
    float (*mine)[TX + 4] = scales[quarter];
    const uint32_t slots = saddr(&scales[quarter][0][0]);
    // The scales of a block come AHEAD blocks early, a column of x a lane, on into the next tile
    int ahead_t = t0, ahead_kb = kb0, ahead_slot = 0;
    const auto ask = [&]() {
      if (ahead_t < tiles) {
        const uint32_t dst = slots + ahead_slot * (TX + 4) * 4;
        for (int j = lane; j < TX; j += 32)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4 * j), "l"(p.sx + min(j, p.M - 1) * p.sx_row + ahead_kb * p.sx_col) : "memory");
        if (lane == 0)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4 * TX), "l"(p.sw + (long long)ahead_t * k_blocks + ahead_kb) : "memory");
        if (++ahead_kb == kb1) { ahead_kb = kb0; ahead_t += t_step; }
      }
      ahead_slot = (ahead_slot + 1) % AHEAD;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    pdl_wait();                                                      // the scales of x come from the kernel ahead
    for (int i = 0; i < AHEAD - 1; ++i) ask();
    int it = 0, buf = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = t0; t < tiles && ok; t += t_step) {
      float acc[TX];
#pragma unroll
      for (int j = 0; j < TX; ++j) acc[j] = 0.f;
#pragma unroll 1
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        __syncwarp();                                                // every lane has read the slot that is filled next
        ask();
        asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
        __syncwarp();                                                // every lane's copies into this block's slot are there
        const float* sx = mine[it % AHEAD];
        const float sw = sx[TX];
        ok = bar_wait(acc_full0 + 8 * buf, acc_phase, &failed);
        if (!ok) { atomicExch(&g_fp8_error, 8); failed = 1; }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t r[TX / 16][16];
#pragma unroll
        for (int c = 0; c < TX / 16; ++c) tmem_ld16(my_tmem + (uint32_t)(buf * TX + 16 * c), r[c]);
#pragma unroll
        for (int c = 0; c < TX / 16; ++c) tmem_ld_wait(r[c]);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(acc_empty0 + 8 * buf);
#pragma unroll
        for (int j = 0; j < TX; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(sx + j);
          acc[j] = fmaf(__uint_as_float(r[j / 16][j % 16]), f.x * sw, acc[j]);
          acc[j + 1] = fmaf(__uint_as_float(r[j / 16][j % 16 + 1]), f.y * sw, acc[j + 1]);
          acc[j + 2] = fmaf(__uint_as_float(r[j / 16][j % 16 + 2]), f.z * sw, acc[j + 2]);
          acc[j + 3] = fmaf(__uint_as_float(r[j / 16][j % 16 + 3]), f.w * sw, acc[j + 3]);
        }
        if (++buf == THIN_SUMS) { buf = 0; acc_phase ^= 1; }
      }
      if (!ok) break;
      const int row = quarter * 32 + lane;
      if (SPLIT) {
        float* part = reinterpret_cast<float*>(ring_ptr);            // the ring is free: every MMA that read it has finished
#pragma unroll
        for (int j = 0; j < TX; ++j) part[j * PITCH + row] = acc[j];
      } else {
        const int n = t * 128 + row;
#pragma unroll
        for (int j = 0; j < TX; ++j)
          if (j < p.M && n < p.N) {
            if (p.y_bf16) ((bf16*)p.y)[j * p.ldy + n] = __float2bfloat16_rn(acc[j]);
            else ((float*)p.y)[j * p.ldy + n] = acc[j];
          }
      }
    }
  }

  asm volatile("cp.async.wait_all;" ::: "memory");
  if (SPLIT) {
    // every block of the cluster comes here, one whose waits ran out too
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int items = p.M * 32, first = items * rank / p.split, end = items * (rank + 1) / p.split;
    for (int i = first + tid; i < end; i += THIN_THREADS) {
      const int m = i / 32, c = i % 32 * 4;
      float4 v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < p.split) v[q] = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(cluster.map_shared_rank(ring_ptr, q)) + m * PITCH + c);
      float4 s = v[0];
#pragma unroll
      for (int q = 1; q < 8; ++q)
        if (q < p.split) { s.x += v[q].x; s.y += v[q].y; s.z += v[q].z; s.w += v[q].w; }
      if (t0 * 128 + c < p.N) store4(p, m, t0 * 128 + c, s);
    }
    cluster.sync();                                                  // a block's memory is read until here
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(THIN_SUMS * TX) : "memory");
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static std::atomic<EncodeTiledFn> known{nullptr};
  EncodeTiledFn fn = known.load(std::memory_order_acquire);
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      known.store(fn = (EncodeTiledFn)ptr, std::memory_order_release);
  }
  return fn;
}

// codes [rows, cols], row pitch ld bytes: boxes of `high` rows x 128 columns, zeros beyond the last column and row
int make_map(CUtensorMap* map, const void* base, int rows, int cols, long long ld, int high = 128) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return IE_BAD_SIZE;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)GROUP, (cuuint32_t)high};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? IE_OK : IE_BAD_ALIGN;
}

constexpr size_t TILE_SMEM = 1024 + STAGES * STAGE + 8 * OUT_STAGE + 8 * AHEAD * 36 * 4;

// clusters of `size` blocks of a kernel that the current device runs at once; `known`: what was asked before, by device and size
typedef std::atomic<int> FitTable[64][9];
int clusters_that_fit(int dev, const void* kernel, int threads, int smem, int size, FitTable& known) {
  int n = 0;
  if (dev < 64 && (n = known[dev][size].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = size * 1024;
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute a;
  a.id = cudaLaunchAttributeClusterDimension;
  a.val.clusterDim.x = size;
  a.val.clusterDim.y = a.val.clusterDim.z = 1;
  cfg.attrs = &a;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();                                // this size does not fit: nothing that a later launch should report
    return 0;
  }
  if (dev < 64) known[dev][size].store(n, std::memory_order_relaxed);
  return n;
}
// As many blocks as can share a tile with all tiles under way at once and `least` blocks of K each
template <typename Kernel>
int blocks_a_tile(Kernel kernel, int threads, int smem, long long tiles, int k_blocks, int least, FitTable& known) {
  int split = 1, dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return split;
  for (int s = 2; s <= 8 && least * s <= k_blocks; ++s)
    if (clusters_that_fit(dev, (const void*)kernel, threads, smem, s, known) >= tiles) split = s;
  return split;
}

template <bool PAIR, bool SPLIT>
int launch_tiles(Fp8Params p, int sms, cudaStream_t stream) {
  CUtensorMap mx, mw;
  int rc = make_map(&mx, p.x, p.M, p.K, p.ldx);
  if (rc) return rc;
  rc = make_map(&mw, p.w, p.N, p.K, p.ldw);
  if (rc) return rc;
  constexpr size_t SMEM = TILE_SMEM;
  static_assert(SMEM <= 232448 - 1024, "shared memory of a block");
  static_assert(128 * (128 + 4) * 4 <= STAGES * STAGE, "the sums of a split tile fit the ring");
  static OncePerDevice once;
  rc = once([] {
    cudaFuncAttributes a;
    const cudaError_t e = cudaFuncGetAttributes(&a, gemm_fp8_tile_kernel<PAIR, SPLIT>);
    if (e != cudaSuccess) return (int)e;
    if (PAIR && a.numRegs != REGS_LAUNCH) return IE_BAD_SIZE;           // built so that the shares do not add up
    return (int)cudaFuncSetAttribute(gemm_fp8_tile_kernel<PAIR, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM);
  });
  if (rc) return rc;
  const long long side = PAIR ? 256 : 128, tiles = ((p.M + side - 1) / side) * ((p.N + side - 1) / side);
  const long long cluster = PAIR ? 2 : SPLIT ? p.split : 1, room = sms / cluster;
  const long long blocks = cluster * (SPLIT || tiles < room ? tiles : room);
  if (tiles * cluster > 0x7fffffffLL || room < 1) return IE_BAD_SIZE;
  if (PAIR || SPLIT)
    return launch_k_cluster(gemm_fp8_tile_kernel<PAIR, SPLIT>, (int)cluster, (unsigned)blocks, TILE_THREADS, SMEM, stream, mx, mw, p);
  return launch_k(gemm_fp8_tile_kernel<PAIR, SPLIT>, (unsigned)blocks, TILE_THREADS, SMEM, stream, mx, mw, p);
}

template <int TX>
int launch_thin(Fp8Params p, int sms, cudaStream_t stream) {
  CUtensorMap mx, mw;
  int rc = make_map(&mx, p.x, p.M, p.K, p.ldx, TX);
  if (rc) return rc;
  rc = make_map(&mw, p.w, p.N, p.K, p.ldw);
  if (rc) return rc;
  static_assert(THIN_SMEM<TX> <= 232448 - 16 * 1024, "shared memory of a block");
  static OncePerDevice once;
  rc = once([] {
    const cudaError_t e = cudaFuncSetAttribute(gemm_fp8_thin_kernel<TX, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, THIN_SMEM<TX>);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(gemm_fp8_thin_kernel<TX, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, THIN_SMEM<TX>);
  });
  if (rc) return rc;
  static FitTable fits;
  const int tiles = (p.N + 127) / 128;
  p.split = blocks_a_tile(gemm_fp8_thin_kernel<TX, true>, THIN_THREADS, THIN_SMEM<TX>, tiles, (p.K + GROUP - 1) / GROUP, THIN_LEAST, fits);
  if (p.split > 1)
    return launch_k_cluster(gemm_fp8_thin_kernel<TX, true>, p.split, (unsigned)(tiles * p.split), THIN_THREADS, THIN_SMEM<TX>, stream, mx, mw, p);
  return launch_k(gemm_fp8_thin_kernel<TX, false>, (unsigned)(tiles < sms ? tiles : sms), THIN_THREADS, THIN_SMEM<TX>, stream, mx, mw, p);
}

// ------------------------------------------------------------------- few rows
// Up to 16 rows of x under a weight that is not long: the weight goes from memory straight into the registers that the matrix
// instruction reads, 16 bytes a lane, a block of K ahead of the one at work.  A warp holds 16 rows of w, the instruction's larger
// side, and 8 NT rows of x.  The codes become halves, which hold them exactly (an instruction for e4m3 exists, but is made of the
// same conversions, of both operands every time).  Long weights are bound by the conversions, so slots in shared memory with more blocks
// of K ahead do not help (4 x 8192 x 8192 took 22 us with four, 15.9 so); short ones by start and trips: 1 row under 2,048 columns takes 1.6 us
// and the weight's bytes at 4.5 TB/s, 8 rows under 8,192 columns 5.0 us at 512 rows of w and 5.9 at 2,048, four trips of a warp one after
// the other and the sum over 16.  The instruction wants of lane (g, t) two numbers from 2 t and two
// from 8 + 2 t of its 16; any other dealing of K serves as well if both operands share it, so lane t takes 16 neighbouring codes of 64,
// for four instructions.  ks warps share rows of w and deal out K where there are few rows of it; their sums come together in shared
// memory, in the order of K.

// 16 codes from column k on, zeros behind the last column (what lies there may be anything, NaN too)
__device__ __forceinline__ uint4 codes_to_the_end(const uint8_t* row, int k, int K) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k < K) {
    v = *reinterpret_cast<const uint4*>(row + k);
    const int n = K - k;
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n < 4 * j + 4) w[j] = n <= 4 * j ? 0u : w[j] & (0xffffffffu >> (8 * (4 * j + 4 - n)));
  }
  return v;
}
__device__ __forceinline__ uint4 stream_codes(const uint8_t* at) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
  return v;
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }
// four codes -> the first two and the last two as halves
__device__ __forceinline__ void halves(uint32_t codes, uint32_t& first, uint32_t& last) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(first), "=r"(last) : "r"(codes));
}
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same 16 x 2 numbers of a row of x in bfloat16, and their codes.  A group's 128 columns lie with the four lanes of a row, so its
// largest number is two exchanges away, and quantising here (as fp8_quantize.cu does) saves a kernel where the weight has few rows.
struct RawRow { uint4 u[2][2]; };
__device__ __forceinline__ RawRow raw_row(const bf16* row, int k, int K, bool whole) {
  RawRow r;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = k + 64 * c + 8 * h;
      if (whole) {
        r.u[c][h] = *reinterpret_cast<const uint4*>(row + at);
      } else {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = at + j < K ? __bfloat16_as_ushort(row[at + j]) : 0;
        r.u[c][h] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
      }
    }
  return r;
}
__device__ __forceinline__ void quantize_row(const RawRow& r, uint4 (&codes)[2], float& scale) {
  float m = 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int h = 0; h < 2; ++h) m = largest8(Raw8<bf16>{r.u[c][h]}, m);
#pragma unroll
  for (int o = 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const bool infinite = !finite(m);
  if (__any_sync(0xffffffffu, infinite)) {
    float f = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) f = largest_finite8(Raw8<bf16>{r.u[c][h]}, f);
#pragma unroll
    for (int o = 2; o > 0; o >>= 1) f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, o));
    m = f;
  }
  const int e = scale_exponent(m);
  scale = exp2i(e);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const uint2 a = codes8(Raw8<bf16>{r.u[c][0]}, exp2i(-e), infinite), b = codes8(Raw8<bf16>{r.u[c][1]}, exp2i(-e), infinite);
    codes[c] = make_uint4(a.x, a.y, b.x, b.y);
  }
}

// RAW: x comes in bfloat16 and is quantised here (one tile of 8 rows)
template <int NT, bool RAW, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS) gemm_fp8_few_kernel(Fp8Params p, int ks) {
  static_assert(!RAW || NT == 1, "registers for one tile of raw rows");
  __shared__ float sums[WARPS][16][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int groups = WARPS / ks, slice = warp % ks, k_blocks = (p.K + GROUP - 1) / GROUP;
  const int n0 = (blockIdx.x * groups + warp / ks) * 16;
  const int kb0 = k_blocks * slice / ks, kb1 = n0 < p.N ? k_blocks * (slice + 1) / ks : kb0;
  const uint8_t* rows[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) rows[i] = p.w + (long long)min(n0 + g + 8 * i, p.N - 1) * p.ldw + 16 * t;
  uint4 w[2][2][2];
  const auto ask = [&](uint4 (&to)[2][2], int kb) {
    const int k = kb * GROUP;
    if (k + GROUP <= p.K) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        to[i][0] = stream_codes(rows[i] + k);
        to[i][1] = stream_codes(rows[i] + k + 64);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        to[i][0] = codes_to_the_end(rows[i] - 16 * t, k + 16 * t, p.K);
        to[i][1] = codes_to_the_end(rows[i] - 16 * t, k + 16 * t + 64, p.K);
      }
    }
  };
  // x and the scales of a block: behind the kernel ahead's, so apart from the weight
  const float* sw = p.sw + (long long)(min(n0, p.N - 1) / GROUP) * k_blocks;      // 16 rows lie in one block of scales
  const uint8_t* x_row = p.x + min(g, p.M - 1) * p.ldx + 16 * t;
  const uint8_t* x_row8 = NT == 1 ? nullptr : p.x + min(8 + g, p.M - 1) * p.ldx + 16 * t;
  const float* sx = p.sx + min(2 * t, p.M - 1) * p.sx_row;                        // rows of x beyond the last make results that nobody reads
  uint4 xs[2][RAW ? 1 : NT][2];
  float fs[2][2 * NT + 1];
  RawRow raw[2];
  const bf16* raw_at = (const bf16*)p.raw + min(g, p.M - 1) * p.ldx;
  const auto ask_raw = [&](RawRow& to, float& f, int kb) {
    f = sw[kb];
    to = raw_row(raw_at, kb * GROUP + 16 * t, p.K, p.raw_vec && (kb + 1) * GROUP <= p.K);
  };
  const auto ask_x = [&](uint4 (&to)[NT][2], float (&f)[2 * NT + 1], int kb) {
    const int k = kb * GROUP;
    f[2 * NT] = sw[kb];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const uint8_t* row = i == 0 ? x_row : x_row8;
      if (k + GROUP <= p.K) {
        to[i][0] = *reinterpret_cast<const uint4*>(row + k);
        to[i][1] = *reinterpret_cast<const uint4*>(row + k + 64);
      } else {
        to[i][0] = codes_to_the_end(row - 16 * t, k + 16 * t, p.K);
        to[i][1] = codes_to_the_end(row - 16 * t, k + 16 * t + 64, p.K);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f[2 * i + j] = sx[(min(8 * i + 2 * t + j, p.M - 1) - min(2 * t, p.M - 1)) * p.sx_row + kb * p.sx_col];
    }
  };
  pdl_trigger();
  if (p.early && kb0 < kb1) ask(w[0], kb0);
  pdl_wait();
  if (!p.early && kb0 < kb1) ask(w[0], kb0);
  if (kb0 < kb1) {
    if constexpr (RAW) ask_raw(raw[0], fs[0][2 * NT], kb0);
    else ask_x(xs[0], fs[0], kb0);
  }
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;

  const auto add = [&](const uint4 (&from)[2][2], const uint4 (&x)[NT][2], const float (&f)[2 * NT + 1]) {
    float in[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) in[i][j] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t a0, a1, a2, a3, b0, b1;
        halves(word_of(from[0][c], j), a0, a2);
        halves(word_of(from[1][c], j), a1, a3);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          halves(word_of(x[i][c], j), b0, b1);
          mma_16x8x16(in[i], a0, a1, a2, a3, b0, b1);
        }
      }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(in[i][j], f[2 * i + (j & 1)] * f[2 * NT], acc[i][j]);
  };
  if constexpr (RAW) {
    const auto add_raw = [&](const uint4 (&from)[2][2], const RawRow& r, float fw) {
      uint4 x[1][2];
      float f[3], scale;
      quantize_row(r, x[0], scale);
      f[0] = __shfl_sync(0xffffffffu, scale, 8 * t);            // rows 2 t and 2 t + 1 of x are lanes 8 t .. and 8 t + 4 ..
      f[1] = __shfl_sync(0xffffffffu, scale, 8 * t + 4);
      f[2] = fw;
      add(from, x, f);
    };
    for (int kb = kb0; kb < kb1; kb += 2) {
      if (kb + 1 < kb1) { ask(w[1], kb + 1); ask_raw(raw[1], fs[1][2 * NT], kb + 1); }
      add_raw(w[0], raw[0], fs[0][2 * NT]);
      if (kb + 1 < kb1) {
        if (kb + 2 < kb1) { ask(w[0], kb + 2); ask_raw(raw[0], fs[0][2 * NT], kb + 2); }
        add_raw(w[1], raw[1], fs[1][2 * NT]);
      }
    }
  } else {
    for (int kb = kb0; kb < kb1; kb += 2) {
      if (kb + 1 < kb1) { ask(w[1], kb + 1); ask_x(xs[1], fs[1], kb + 1); }
      add(w[0], xs[0], fs[0]);
      if (kb + 1 < kb1) {
        if (kb + 2 < kb1) { ask(w[0], kb + 2); ask_x(xs[0], fs[0], kb + 2); }
        add(w[1], xs[1], fs[1]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[warp][g + 8 * (j >> 1)][8 * i + 2 * t + (j & 1)] = acc[i][j];
  __syncthreads();
  const int high = groups * 16;
  for (int i = threadIdx.x; i < high * p.M; i += 32 * WARPS) {
    const int r = i % high, m = i / high, n = blockIdx.x * high + r;
    if (n >= p.N) continue;
    float s = 0.f;
    for (int q = 0; q < ks; ++q) s += sums[(r >> 4) * ks + q][r & 15][m];
    if (p.y_bf16) ((bf16*)p.y)[m * p.ldy + n] = __float2bfloat16_rn(s);
    else ((float*)p.y)[m * p.ldy + n] = s;
  }
}

template <int NT, bool RAW>
int launch_few_rows(const Fp8Params& p, int sms, cudaStream_t stream) {
  const int groups = (p.N + 15) / 16, k_blocks = (p.K + GROUP - 1) / GROUP;
  // No more row tiles than SMs, and 16 blocks of K: one tile a block of 16 warps, each with a sixteenth of K (against 8 warps 1 x 2048 x 2048
  // 2.9 us and 4.0, 8 x 2048 x 8192 6.8 and 7.9)
  if (groups <= sms && k_blocks >= 16) return launch_k(gemm_fp8_few_kernel<NT, RAW, 16>, groups, 512, 0, stream, p, 16);
  int ks = 1;
  while (ks < 8 && (long long)groups * ks < 8LL * sms && 2 * ks <= k_blocks) ks *= 2;
  const int per = 8 / ks, grid = (groups + per - 1) / per;
  return launch_k(gemm_fp8_few_kernel<NT, RAW, 8>, grid, 256, 0, stream, p, ks);
}
int launch_few(const Fp8Params& p, int sms, cudaStream_t stream) {
  if (p.raw) return launch_few_rows<1, true>(p, sms, stream);
  return p.M <= 8 ? launch_few_rows<1, false>(p, sms, stream) : launch_few_rows<2, false>(p, sms, stream);
}

}  // namespace

// fp8_quantize.cu
int fp8_quantize_rows(const void* x, int dtype, void* codes, float* scales, int rows, int cols, long long ldx, long long ldc,
                      long long s_row, long long s_col, cudaStream_t stream);

// bytes of scratch that the product of unquantised rows takes, unless it quantises them itself: their codes, then their scales [K / 128][M]
static long long scratch_of(int M, int K) {
  if (M <= 0 || K <= 0) return 0;
  return (long long)M * ((K + 15) / 16 * 16) + 4LL * M * ((K + GROUP - 1) / GROUP);
}

// x: codes (x_dtype IE_E4M3, with sx) or float32 / bfloat16 rows, which are quantised into scratch first
static int gemm_fp8(const void* x, int x_dtype, const float* sx, const void* w, const float* sw, void* y, int y_dtype, int M, int N, int K,
                    long long ldx, long long sx_row, long long sx_col, long long ldw, long long ldy, void* scratch,
                    long long scratch_bytes, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return IE_OK;
  if (K <= 0) return IE_BAD_SIZE;
  if (y_dtype != IE_F32 && y_dtype != IE_BF16) return IE_BAD_DTYPE;
  if (((uintptr_t)w & 15) || ldw % 16) return IE_BAD_ALIGN;
  const int sms = device_sms();
  if (sms <= 0) return IE_BAD_SIZE;
  Fp8Params p;
  p.w = (const uint8_t*)w; p.sw = sw; p.y = y; p.M = M; p.N = N; p.K = K; p.ldw = ldw; p.ldy = ldy; p.y_bf16 = y_dtype == IE_BF16;
  p.y_vec = ((uintptr_t)y & 15) == 0 && ldy * (p.y_bf16 ? 2 : 4) % 16 == 0;
  p.split = 1;
  p.early = 0;
  p.raw = nullptr;
  // Up to 8 rows of a small weight: the kernel saved counts for more than quantising them in every block does, as long as a warp has two
  // blocks of K at most (8 x 4096 x 2048: 4.4 us either way, 8 x 2048 x 4096 4.4 against 4.5, and half of the host's time; 8 x 2048 x 8192
  // 7.7 against 6.8, 8 x 8192 x 2048 7.4 against 6.4)
  if (x_dtype == IE_BF16 && M <= 8 && N < 32 * sms && K <= (N <= 16 * sms ? 4096 : 2048)) {
    p.raw = x; p.raw_vec = ((uintptr_t)x & 15) == 0 && ldx % 8 == 0;
    p.x = nullptr; p.sx = nullptr; p.ldx = ldx; p.sx_row = p.sx_col = 0;
    return launch_few(p, sms, stream);
  }
  if (x_dtype != IE_E4M3) {
    if (scratch == nullptr || scratch_bytes < scratch_of(M, K)) return IE_NEEDS_SCRATCH;
    if ((uintptr_t)scratch & 15) return IE_BAD_ALIGN;
    const long long pitch = (K + 15) / 16 * 16;
    float* scales = reinterpret_cast<float*>((char*)scratch + M * pitch);
    const int rc = fp8_quantize_rows(x, x_dtype, scratch, scales, M, K, ldx, pitch, 1, M, stream);
    if (rc) return rc;
    x = scratch; ldx = pitch; sx = scales; sx_row = 1; sx_col = M;
    p.early = 1;
  }
  if (((uintptr_t)x & 15) || ldx % 16) return IE_BAD_ALIGN;
  p.x = (const uint8_t*)x; p.sx = sx; p.ldx = ldx; p.sx_row = sx_row; p.sx_col = sx_col;
  // A weight of 24 million codes and more pays for the start of the tensor cores' kernel (6 x 128256 x 2048: 47.7 us against 52.4, 16 x
  // 16384 x 2048: 9.4 against 12.6, but 8 x 8192 x 2048: 7.3 against 6.6, 1 x 2048 x 2048: 5.1 against 3.8)
  if (M <= 16) return (long long)N * K >= (24LL << 20) ? launch_thin<16>(p, sms, stream) : launch_few(p, sms, stream);
  // 32 rows: 32 x 2048 x 8192 9.4 us against 10.7 of the tiles below, 32 x 16384 x 2048 11.3 against 12.6 (at 64 rows 14.1 against 11.7)
  if (M <= 32) return launch_thin<32>(p, sms, stream);
  const long long tiles = (long long)((M + 127) / 128) * ((N + 127) / 128);
  // More tiles of 128 x 128 than SMs: pairs take less per result (512 x 8192 x 2048, 256 tiles: 15.8 us against 20.8; at 200 x 2048 x
  // 2048, 32 tiles, 13.4 against 9.3).
  if (M > 128 && tiles > sms) return launch_tiles<true, false>(p, sms, stream);
  // 77 x 2048 x 8192 takes 26.6 us unsplit, 10.9 by four, 10.0 by six (22 clusters fit, 16 tiles), 16.7 by eight (15 fit: two rounds)
  static FitTable fits;
  p.split = blocks_a_tile(gemm_fp8_tile_kernel<false, true>, TILE_THREADS, (int)TILE_SMEM, tiles, (K + GROUP - 1) / GROUP, 4, fits);
  return p.split > 1 ? launch_tiles<false, true>(p, sms, stream) : launch_tiles<false, false>(p, sms, stream);
}

// the entry: arguments as 64-bit words in the order above, which a caller converts in one go; sizes above SIZE_MOST are refused
extern "C" int ie_gemm_fp8(const long long* a) {
  if (beyond(a[7], a[8], a[9])) return IE_BAD_SIZE;
  // out and scratch over the scales (the caller has compared them with x, w and each other)
  const long long M = a[7], N = a[8], k_blocks = (a[9] + GROUP - 1) / GROUP, size = a[6] == IE_F32 ? 4 : 2;
  const Span out = {(uintptr_t)a[5], M, size * N, size * a[14]}, scratch = {(uintptr_t)a[15], 1, a[16], a[16]};
  const Span sw = scales_span((const void*)a[4], (N + GROUP - 1) / GROUP, k_blocks, k_blocks, 1);
  const Span sx = scales_span((const void*)a[2], M, k_blocks, a[11], a[12]);
  if (overlap(out, sw) || overlap(out, sx) || overlap(scratch, sw) || overlap(scratch, sx)) return IE_OVERLAP;
  return gemm_fp8((const void*)a[0], (int)a[1], (const float*)a[2], (const void*)a[3], (const float*)a[4], (void*)a[5], (int)a[6], (int)a[7],
                  (int)a[8], (int)a[9], a[10], a[11], a[12], a[13], a[14], (void*)a[15], a[16], (cudaStream_t)a[17]);
}

// reads and clears the word that a wait which ran out leaves (0: none)
extern "C" int ie_gemm_fp8_error() {
  int v = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_fp8_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_fp8_error, &zero, sizeof(int));
  return v;
}
