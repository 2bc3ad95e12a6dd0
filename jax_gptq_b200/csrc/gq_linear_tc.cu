// Products with packed weights for many tokens, on the tcgen05 tensor cores.
//
// A CTA computes 128 rows of W (the M of the MMA) times TILE columns of x (its
// N), walking along K in blocks of 128 positions:
//   D[row, col] += scale[row, granule] * sum_k (code - offset)[row, k] * x[col, k].
// code - offset is a whole number of at most 8 bits, exact in bf16 and fp16, so
// each granule is summed in tensor memory from exact products and multiplied by
// its scale in fp32 registers: nothing about the weights is rounded, as in the
// few-token form.  A granule's scale is one number per row, which is one number
// per thread of an epilogue warp (a thread owns a row of tensor memory).
//
// Roles (640 threads):
//   warp 0      TMA producer: x tiles of 128 positions (K-major, 128-byte
//               swizzle), several in flight;
//   warp 1      MMA issuer: A = decoded weights from TENSOR MEMORY, B = x from
//               shared memory.  The whole warp walks the loop, so that addresses
//               and descriptors stay in uniform registers, and one lane is
//               elected to issue;
//   warp 2      copies a block's codes and scales to shared memory;
//   warps 4-11  decode: a thread turns its row's codes of a block into 128 16-bit
//               numbers and stores them to one of 2 or 3 tensor-memory buffers.
//               The two groups of four warps take alternate blocks: one group
//               alone needed 2200 cycles a block, twice what the MMAs need;
//   warps 12-19 accumulate: granule sums from tensor memory into registers, two
//               columns a multiply-add (fma.rn.f32x2).
// Three accumulators (two in one form) are used in turn, one for each granule's MMAs over the
// tile's columns, or over half of them where the tile is wider than 128: filling
// one (512 cycles for 128 positions of 128 columns) and then reading it out takes
// about 1600 cycles with the signals in between, so with two the tensor pipe idled
// half the time.  In wide tiles each group of four accumulating warps has a half
// of the columns, else half of every granule's.
//
// Where there are fewer tiles than SMs, a cluster of up to 8 CTAs splits K: each
// leaves its sums in its own shared memory and adds up its share of the columns
// over the cluster in rank order.  No load uses multicast.
//
// Bound: 2048 tokens through 11008 x 4096 take 191 us in a short run with columns in
// order, 965 TFLOP/s, and 206 to 225 with the gather in long ones, 820 to 900: cuBLAS
// on weights already decoded takes 133 to 142 (8-bit codes: 225 us in order).  The
// roles take turns at tensor memory, which three accumulators and two decoded blocks
// fill.  Few tokens (37 float32 ones through 4096 x 4096: 17 us with the gather) are a
// chain of about 1600 cycles a block of K.
//
// Every wait is bounded (gq_set_wait_limit_ns): one that expires makes all roles
// leave their loops and records GQ_DEVERR_TIMEOUT, read by gq_device_status().
#include <cuda.h>

#include "gq_linear.cuh"

#include <algorithm>
#include <atomic>

namespace gq {
namespace lintc {

using namespace lin;

static __device__ int g_device_status = 0;
static __device__ uint64_t g_wait_limit_ns = kWaitLimitNs;

int read_status(int reset, int* out) {
  int v = 0;
  GQ_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_device_status, sizeof(int)));
  if (reset) {
    const int z = 0;
    GQ_CHECK_CUDA(cudaMemcpyToSymbol(g_device_status, &z, sizeof(int)));
  }
  *out = v;
  return GQ_OK;
}
int set_wait_limit(uint64_t ns) {
  GQ_CHECK_CUDA(cudaMemcpyToSymbol(g_wait_limit_ns, &ns, sizeof(ns)));
  return GQ_OK;
}

constexpr int THREADS = 640;
constexpr int BM = 128;
constexpr int A_COLS = KC / 2;  // tensor-memory columns of one decoded block
constexpr int TMEM_COLS = 512;
constexpr int MAX_SMEM = 227 * 1024;

// N: columns of an MMA, PARTS: MMAs side by side (1 or 2).
template <int WIDTH, int N, int PARTS, int G>
struct Cfg {
  static constexpr int TILE = N * PARTS;           // columns of x per CTA
  static constexpr int BOX = TILE * 128;           // bytes of 64 positions of the tile
  static constexpr int XSTAGE = 2 * BOX;           // a block of 128 positions
  static constexpr int STAGES = TILE > 128 ? 3 : 4;   // blocks of x
  // accumulators and decoded blocks: tensor memory has room for 3 of both only
  // with narrower MMAs; a tile of one part needs the decoded blocks more (128
  // tokens through 11008 x 4096: 26 us against 30), one of two the accumulators
  static constexpr int ACCS = N > 96 && PARTS == 1 ? 2 : 3;
  static constexpr int ASTAGES = N > 96 && PARTS == 2 ? 2 : 3;
  static constexpr int CODES = BM * KC * WIDTH / 8;        // a block's codes of 128 rows
  static constexpr int SCALES = BM * (KC / G) * 8;         // and its scales and offsets
  static constexpr int WSTAGE = CODES + SCALES;
  static constexpr int WSTAGES = TILE > 192 ? (G < 128 ? 2 : 3) : 4;
  // Where two groups of warps take a ring's slots in turn, a group meets a slot of an
  // odd ring only every second time round.  A wait for a phase returns at once while the
  // phase before it is still open, so a group that never waited for that one could take
  // a slot too early.  Odd rings therefore have two barriers a slot, used in turn: a
  // barrier's last use is then the same group's, which has waited for it.
  static constexpr int barriers(int slots) { return slots % 2 ? 2 * slots : slots; }
  static constexpr int W_FULL = barriers(WSTAGES);    // decoders: copied codes
  static constexpr int A_EMPTY = barriers(ASTAGES);   // decoders: room for a decoded block
  static constexpr int T_FULL = PARTS == 2 ? barriers(ACCS) : ACCS;  // accumulating groups
  static constexpr int PER = PARTS == 2 ? N : N / 2;  // columns per accumulating thread
  static constexpr int LD = PER % 16 == 0 ? 16 : 8;
  static constexpr int A0 = ACCS * N;                 // first tensor-memory column of the weights
  static constexpr int SUMS = TILE * BM * 4;       // a tile's sums in shared memory
  static constexpr int W0 = STAGES * XSTAGE;       // where the weights' stages begin
  static constexpr int USED = W0 + WSTAGES * WSTAGE;
  static constexpr int SMEM = (USED > SUMS ? USED : SUMS) + 1024;
  static_assert(ACCS * N + ASTAGES * A_COLS <= TMEM_COLS, "tensor memory");
  static_assert(SUMS <= W0, "sums only over x");
  static_assert(SMEM + 1024 <= MAX_SMEM, "shared memory");
};

struct Params {
  const uint4* qw;
  const float2* params;
  int64_t m;
  int nkc;       // blocks along K
  int row_blocks;  // blocks of 16 rows
  int tokens;
  int mt, nt;    // row tiles, column tiles
  int split;     // CTAs along K (the cluster size)
  void* y;
  int64_t ldy;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// The same without waiting at all (try_wait may hold the thread for a while).
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait; false when the deadline passed or another role gave up.  The
// clock is read on every 16th try only.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  uint64_t t0 = 0;
  for (uint32_t i = 0;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 15) != 15) continue;
    if (*abort_flag) return false;
    const uint64_t now = globaltimer_ns();
    if (t0 == 0) {
      t0 = now;
    } else if (now - t0 > g_wait_limit_ns) {
      *abort_flag = 1;
      atomicExch(&g_device_status, GQ_DEVERR_TIMEOUT);
      return false;
    }
  }
}
// The same for a whole warp, which stays converged: one lane polls.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity,
                                               volatile int* abort_flag) {
  int ok = 0;
  if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, abort_flag);
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
// Waits, within the limit, for what this thread itself has in flight, whether
// or not the roles have given up.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
  uint64_t t0 = 0;
  for (uint32_t i = 0; !mbar_try_wait(bar, parity); ++i) {
    if ((i & 15) != 15) continue;
    const uint64_t now = globaltimer_ns();
    if (t0 == 0) t0 = now;
    else if (now - t0 > g_wait_limit_ns) return;
  }
}
__device__ __forceinline__ void tma_load_2d(const CUtensorMap* map, uint64_t* bar, void* dst, int x,
                                            int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint64_t* bar, void* dst, int x,
                                            int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// K-major SW128 descriptor: 8-row groups of 1024 bytes.
__device__ __forceinline__ uint64_t make_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | 1ull << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 |
         2ull << 61;
}
// Executed by the whole warp; the thread with `leader` set issues.
__device__ __forceinline__ void umma(uint32_t leader, uint32_t d, uint32_t a, uint64_t b,
                                     uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accum), "r"(leader));
}
__device__ __forceinline__ void umma_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(
          smem_u32(bar)), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(addr));
}
// Waits for this thread's tensor-memory loads; the registers pass through, so
// that nothing that uses them moves above.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7])
               :
               : "memory");
}
// {a0, a1} = scale * {r0, r1} + {a0, a1}
__device__ __forceinline__ void fma2(float& a0, float& a1, uint32_t r0, uint32_t r1, float scale) {
  asm("{\n .reg .b64 a, r, s;\n mov.b64 a, {%0, %1};\n mov.b64 r, {%2, %3};\n mov.b64 s, {%4, %4};\n"
      " fma.rn.f32x2 a, r, s, a;\n mov.b64 {%0, %1}, a;\n}"
      : "+f"(a0), "+f"(a1)
      : "f"(__uint_as_float(r0)), "f"(__uint_as_float(r1)), "f"(scale));
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}

// Failure-path check of this file's bounded waits: a warp waits on an mbarrier that
// nothing arrives on, so the wait must give up after g_wait_limit_ns, record
// GQ_DEVERR_TIMEOUT, and return false; a second wait then sees the flag, and the
// drain, which goes on after it, ends by its own limit.  *observed gets 1 when all
// did so.  The kernel then simply returns.
__global__ void expire_wait_kernel(int* observed) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int abort_flag;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    mbar_init(&bar, 1);
  }
  __syncthreads();
  const bool first = mbar_wait_warp(&bar, 0, &abort_flag);
  const bool second = mbar_wait_warp(&bar, 0, &abort_flag);
  mbar_drain(&bar, 0);
  if (threadIdx.x == 0) *observed = !first && !second && abort_flag == 1 ? 1 : 0;
}

int launch_expire_test(int* observed, cudaStream_t st) {
  expire_wait_kernel<<<1, 32, 0, st>>>(observed);
  return check_launch("packed product expire_wait");
}

template <int WIDTH, typename T, int N, int PARTS, int G>
__global__ void __launch_bounds__(THREADS, 1)
many_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
            const __grid_constant__ CUtensorMap map_s, Params p) {
  using C = Cfg<WIDTH, N, PARTS, G>;
  constexpr bool BF16 = !std::is_same<T, __half>::value;
  constexpr int SPLIT = std::is_same<T, float>::value ? 3 : 1;
  constexpr int GPC = KC / G;            // granules per block
  constexpr int TOK = C::TILE / SPLIT;   // tokens per tile
  constexpr uint32_t IDESC = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) |
                             ((uint32_t)(N >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  __shared__ uint64_t x_full[C::STAGES], x_empty[C::STAGES], a_full[C::ASTAGES], a_empty[C::A_EMPTY];
  __shared__ uint64_t w_full[C::W_FULL], w_empty[C::WSTAGES];
  __shared__ uint64_t t_full[C::T_FULL], t_empty[C::ACCS], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&x_full[s], 1);
      mbar_init(&x_empty[s], 1);
    }
    for (int s = 0; s < C::ASTAGES; ++s) mbar_init(&a_full[s], 4);  // the decoding warps of a block
    for (int s = 0; s < C::A_EMPTY; ++s) mbar_init(&a_empty[s], 1);
    for (int s = 0; s < C::W_FULL; ++s) mbar_init(&w_full[s], 1);
    for (int s = 0; s < C::WSTAGES; ++s) mbar_init(&w_empty[s], 4);  // the decoding warps of a block
    for (int h = 0; h < C::T_FULL; ++h) mbar_init(&t_full[h], 1);
    for (int h = 0; h < C::ACCS; ++h) mbar_init(&t_empty[h], PARTS == 2 ? 4 : 8);  // the warps that read it
    mbar_init(&done, 1);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_slot)),
                 "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;

  // this CTA's tiles (one, where a cluster splits K) and its blocks of K
  const int rank = p.split > 1 ? (int)(blockIdx.x % p.split) : 0;
  const int first_tile = p.split > 1 ? (int)(blockIdx.x / p.split) : (int)blockIdx.x;
  const int step = p.split > 1 ? p.mt * p.nt : (int)gridDim.x;
  const int num_tiles = p.mt * p.nt;
  const int c0 = (int)((int64_t)p.nkc * rank / p.split), c1 = (int)((int64_t)p.nkc * (rank + 1) / p.split);

  // Registers: 640 threads start with 96 each; warps 0-3 keep 40, the decoders
  // 56, the accumulating warps take 160: 128 * 40 + 256 * 56 + 256 * 160 = 60416.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 1) {
      // Every barrier is looked at once before the MMAs ahead of it are issued, so
      // that the answer is there when it is needed.
      int s = 0, as = 0, acc = 0;
      uint32_t phase = 0, aphase = 0, tphase = 0;
      const uint32_t leader = elect_one();
      const int blocks = (c1 - c0) * ((num_tiles - first_tile + step - 1) / step);
      bool ok = true, x_ready = false, a_ready = false, t_ready = false;
      for (int n = 0; n < blocks; ++n) {
        ok = (x_ready || mbar_wait(&x_full[s], phase, abort_flag)) &&
             (a_ready || mbar_wait(&a_full[as], aphase, abort_flag));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t b_base = smem_u32(smem) + s * C::XSTAGE;
        const uint32_t a_base = tmem + C::A0 + as * A_COLS;
        uint64_t* const x_done = &x_empty[s];
        // (every second time round a ring, an odd one's second barriers)
        uint64_t* const a_done = &a_empty[as + (C::A_EMPTY > C::ASTAGES && aphase ? C::ASTAGES : 0)];
        if (++s == C::STAGES) {
          s = 0;
          phase ^= 1;
        }
        if (++as == C::ASTAGES) {
          as = 0;
          aphase ^= 1;
        }
#pragma unroll
        for (int gr = 0; gr < GPC; ++gr) {
#pragma unroll
          for (int h = 0; h < PARTS; ++h) {
            ok = ok && (t_ready || mbar_wait(&t_empty[acc], tphase ^ 1, abort_flag));
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int cur = acc;
            uint64_t* const t_done = &t_full[cur + (C::T_FULL > C::ACCS && tphase ? C::ACCS : 0)];
            if (++acc == C::ACCS) {
              acc = 0;
              tphase ^= 1;
            }
            t_ready = mbar_test(&t_empty[acc], tphase ^ 1);
            if (gr == GPC - 1 && h == PARTS - 1) {
              x_ready = mbar_test(&x_full[s], phase);
              a_ready = mbar_test(&a_full[as], aphase);
            }
            fence_after();
#pragma unroll
            for (int i = 0; i < G / 16; ++i) {
              const int kk = gr * (G / 16) + i;
              umma(leader, tmem + cur * N, a_base + kk * 8,
                   make_desc(b_base + (kk / 4) * C::BOX + h * N * 128 + (kk % 4) * 32), IDESC, i > 0);
            }
            umma_commit(leader, t_done);
          }
        }
        if (!ok) break;
        umma_commit(leader, a_done);
        umma_commit(leader, x_done);
      }
      umma_commit(leader, &done);  // whatever was issued is over before the block ends
      mbar_drain(&done, 0);
    } else if (warp == 0 || warp == 2) {
      // copies by tensor map: x; codes and scales of 8 blocks of 16 rows (rows
      // past the last block read as zeros)
      const int stages = warp == 0 ? C::STAGES : C::WSTAGES;
      const int fulls = warp == 0 ? C::STAGES : C::W_FULL;
      uint64_t* fb = warp == 0 ? x_full : w_full;
      uint64_t* eb = warp == 0 ? x_empty : w_empty;
      int s = 0, loads = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first_tile; ok && t < num_tiles; t += step) {
        const int col = (t / p.mt) * (TOK * SPLIT), rb0 = (t % p.mt) * (BM / ROWS);
        for (int c = c0; c < c1; ++c) {
          if (!(ok = mbar_wait_warp(&eb[s], phase ^ 1, abort_flag))) break;
          if (lane == 0) {
            uint64_t* const full = &fb[s + (fulls > stages && phase ? stages : 0)];
            if (warp == 0) {
              uint8_t* dst = smem + s * C::XSTAGE;
              mbar_expect_tx(full, C::XSTAGE);
              tma_load_2d(&map_x, full, dst, c * KC, col);
              tma_load_2d(&map_x, full, dst + C::BOX, c * KC + 64, col);
            } else {
              uint8_t* dst = smem + C::W0 + s * C::WSTAGE;
              mbar_expect_tx(full, C::WSTAGE);
              tma_load_3d(&map_w, full, dst, 0, c, rb0);
              tma_load_3d(&map_s, full, dst + C::CODES, 0, c, rb0);
            }
          }
          ++loads;
          if (++s == stages) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // Every stage was let go of: no arrival is still on its way.  Where the
      // roles gave up, the copies issued so far still land before the block ends.
      for (int i = 0; ok && i < stages; ++i) {
        ok = mbar_wait_warp(&eb[s], phase ^ 1, abort_flag);
        if (++s == stages) {
          s = 0;
          phase ^= 1;
        }
      }
      if (!ok && lane == 0)
        for (int i = 0; i < fulls; ++i) {
          const int issued = loads / fulls + (i < loads % fulls);
          if (issued > 0) mbar_drain(&fb[i], (issued - 1) & 1);
        }
    }
    __syncwarp();
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    constexpr int LPR = WIDTH;  // 16-byte loads per row and block: 4 or 8
    const int q4 = warp & 3;
    const int rt = q4 * 32 + lane;  // row of the tile
    const uint32_t lanes = (uint32_t)(q4 * 32) << 16;
    // n: blocks so far; this group takes every second one
    const int mine = (warp >> 2) & 1;
    uint32_t n = 0;
    bool ok = true;
    for (int t = first_tile; ok && t < num_tiles; t += step) {
      for (int c = c0; c < c1; ++c, ++n) {
        if ((n & 1) != mine) continue;
        const int ws = n % C::WSTAGES, as = n % C::ASTAGES;
        if (!(ok = mbar_wait_warp(&w_full[n % C::W_FULL], (n / C::W_FULL) & 1, abort_flag))) break;
        const uint8_t* stage = smem + C::W0 + ws * C::WSTAGE;
        const uint4* codes = reinterpret_cast<const uint4*>(stage) + rt * LPR;
        const float2* sc = reinterpret_cast<const float2*>(stage + C::CODES) +
                           (rt >> 4) * (GPC * ROWS) + (rt & 15);
        uint4 cur[LPR];
        float coff[GPC];
#pragma unroll
        for (int i = 0; i < LPR; ++i) cur[i] = codes[piece_at<WIDTH>(i, rt)];
#pragma unroll
        for (int i = 0; i < GPC; ++i) coff[i] = sc[i * ROWS].y;
        __syncwarp();
        if (lane == 0) mbar_arrive(&w_empty[ws]);
        // the MMAs of block n - ASTAGES are over (the first blocks have room at once)
        const uint32_t room = n + (C::A_EMPTY - C::ASTAGES);
        if (!(ok = mbar_wait_warp(&a_empty[room % C::A_EMPTY], ((room / C::A_EMPTY) & 1) ^ 1, abort_flag)))
          break;
        fence_after();
        const uint32_t dst = tmem + lanes + C::A0 + as * A_COLS;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t r[16];
          const uint32_t o = offset_operand<WIDTH, BF16>(coff[j * 32 / G]);
#pragma unroll
          for (int tq = 0; tq < 4; ++tq) {
            uint32_t w[2], v[4];
            if constexpr (WIDTH == 4) {
              w[0] = j == 0 ? cur[tq].x : j == 1 ? cur[tq].y : j == 2 ? cur[tq].z : cur[tq].w;
            } else {
              const uint4& q = cur[(j >> 1) * 4 + tq];
              w[0] = (j & 1) == 0 ? q.x : q.z;
              w[1] = (j & 1) == 0 ? q.y : q.w;
            }
            decode8<WIDTH, BF16>(w, o, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) r[4 * tq + e] = v[e];
          }
          tmem_st16(dst + 16 * j, r);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&a_full[as]);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
    const int q4 = warp & 3, part = (warp - 12) >> 2;  // part: which columns of each half
    const int rt = q4 * 32 + lane;
    const uint32_t lanes = (uint32_t)(q4 * 32) << 16;
    uint32_t u = 0;
    bool ok = true;
    for (int t = first_tile; ok && t < num_tiles; t += step) {
      const int row = (t % p.mt) * BM + rt;
      // the scales of a row, AHEAD granules before they are needed
      constexpr int AHEAD = GPC == 1 ? 2 : 4;
      const float2* pp = p.params + ((int64_t)min(row >> 4, p.row_blocks - 1) * p.nkc + c0) * (GPC * ROWS) + (row & 15);
      float acc[C::PER];
#pragma unroll
      for (int i = 0; i < C::PER; ++i) acc[i] = 0.f;
      const int granules = (c1 - c0) * GPC;
      float ahead[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        ahead[i] = i < granules ? __ldg(&pp->x) : 0.f;
        pp += ROWS;
      }
      for (int gr = 0; gr < granules; ++gr) {
        const float scale = ahead[0];
#pragma unroll
        for (int i = 0; i + 1 < AHEAD; ++i) ahead[i] = ahead[i + 1];
        if (gr + AHEAD < granules) ahead[AHEAD - 1] = __ldg(&pp->x);
        pp += ROWS;
        // wide tiles: this group's half of every granule; else every granule's
        // half of the columns
        const uint32_t st = PARTS == 2 ? 2 * u + part : u;  // number of the step
        const uint32_t buf = st % C::ACCS;
        ok = mbar_wait_warp(&t_full[st % C::T_FULL], (st / C::T_FULL) & 1, abort_flag);
        ++u;
        if (!ok) break;
        fence_after();
        const uint32_t src = tmem + lanes + buf * N + (PARTS == 2 ? 0 : part * C::PER);
        uint32_t r[2][C::LD];
        tmem_ld(src, r[0]);
#pragma unroll
        for (int i = 0; i < C::PER; i += C::LD) {
          uint32_t(&v)[C::LD] = r[(i / C::LD) & 1];
          tmem_wait(v);
          if (i + C::LD < C::PER) {
            tmem_ld(src + i + C::LD, r[(i / C::LD + 1) & 1]);
          } else {  // all is read: the MMAs may refill the accumulator
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&t_empty[buf]);
          }
#pragma unroll
          for (int e = 0; e < C::LD; e += 2) fma2(acc[i + e], acc[i + e + 1], v[e], v[e + 1], scale);
        }
      }
      if (!ok) break;
      const int tok0 = (t / p.mt) * TOK;
      const int col0 = part * C::PER;
      if (p.split == 1) {
        T* y = static_cast<T*>(p.y) + row;
        if (row < p.m) {
#pragma unroll
          for (int i = 0; i < C::PER; i += SPLIT) {
            const int tok = tok0 + (col0 + i) / SPLIT;
            float v = acc[i];
            if constexpr (SPLIT == 3) v = acc[i + 2] + acc[i + 1] + v;  // small terms first
            if (tok < p.tokens) store_out(y + (int64_t)tok * p.ldy, v);
          }
        }
      } else {
        // once every MMA of this CTA is over (the other group's half as well), the
        // stages of x have no reader left and take the sums
        if (!(ok = mbar_wait_warp(&done, 0, abort_flag))) break;
        float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int i = 0; i < C::PER; ++i) sums[(col0 + i) * BM + rt] = acc[i];
      }
    }
  }

  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(TMEM_COLS));
  }
  if (p.split > 1) {
    cluster_sync();  // every CTA's sums are in its shared memory
    const int row0 = (first_tile % p.mt) * BM, tok0 = (first_tile / p.mt) * TOK;
    const int ntok = min(TOK, p.tokens - tok0);
    const uint32_t base = smem_u32(smem);
    const int r = threadIdx.x % BM;
    if (row0 + r < p.m) {
      for (int tk = rank * (THREADS / BM) + (int)threadIdx.x / BM; tk < ntok;
           tk += p.split * (THREADS / BM)) {
        float v = 0.f;
#pragma unroll
        for (int sp = SPLIT - 1; sp >= 0; --sp) {
          float part = 0.f;
          for (int c = 0; c < p.split; ++c)
            part += ld_cluster(peer_addr(base + ((tk * SPLIT + sp) * BM + r) * 4, c));
          v += part;
        }
        store_out(static_cast<T*>(p.y) + (int64_t)(tok0 + tk) * p.ldy + row0 + r, v);
      }
    }
    cluster_sync();  // no CTA leaves while another reads its sums
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeTiledFn>(ptr);
  }();
  return fn;
}

// [blocks][along][inner] of `size`-byte elements, read 8 blocks at a time.
static int make_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int inner,
                    int64_t along, int64_t blocks, int size) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(GQ_ECUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)along, (cuuint64_t)blocks};
  cuuint64_t strides[2] = {(cuuint64_t)inner * size, (cuuint64_t)inner * size * along};
  cuuint32_t box[3] = {(cuuint32_t)inner, 1, BM / ROWS};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, type, 3, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(GQ_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return GQ_OK;
}

template <int WIDTH, typename T, int N, int PARTS, int G>
int launch(const CUtensorMap& map, const CUtensorMap& map_w, const Params& p, cudaStream_t st) {
  using C = Cfg<WIDTH, N, PARTS, G>;
  auto kernel = many_kernel<WIDTH, T, N, PARTS, G>;
  CUtensorMap map_s;  // [row blocks][blocks of K][16 rows x granules of a scale and an offset]
  GQ_TRY(make_map(&map_s, CU_TENSOR_MAP_DATA_TYPE_INT64, p.params, ROWS * (KC / G), p.nkc,
                  p.row_blocks, 8));
  static std::atomic<uint64_t> ready{0};  // devices on which the attribute is set
  int dev = 0;
  GQ_CHECK_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (dev > 63 || !(ready.load(std::memory_order_acquire) & bit)) {
    GQ_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    ready.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  const int tiles = p.mt * p.nt;
  cfg.gridDim = dim3((unsigned)(p.split > 1 ? tiles * p.split : std::min(tiles, sm_count())));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)p.split, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = p.split > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, map, map_w, map_s, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(GQ_ECUDA, "gq_linear: %s", cudaGetErrorString(e));
  }
  return check_launch("gq_linear many-token product");
}

// CTAs that K can be split over: each keeps 4 blocks.
inline int most_parts(int nkc) {
  int parts = 1;
  while (parts < 8 && nkc >= parts * 2 * 4) parts *= 2;
  return parts;
}

// Split K over a cluster while that fills idle SMs and leaves 4 blocks each.  Of
// clusters of 8, one CTA an SM, 14 run at once on a B200's 148 SMs (they do not cross
// its groups of SMs), and on other numbers of SMs in proportion: 128 tokens through
// 2048 x 8192 (16 tiles) take 28.4 us by 8 and 20.7 by 4, through 1792 x 8192 17.0 by 8.
inline int choose_split(int64_t tiles, int nkc, int sms) {
  const int most = most_parts(nkc);
  int split = 1;
  while (split < most && tiles * split * 2 <= (split == 4 ? sms * 14 / 148 * 8 : sms)) split *= 2;
  return split;
}

struct Tile {
  int n, parts;
  int tokens(int dtype) const { return n * parts / (dtype == 0 ? 3 : 1); }
};

// The columns of x per tile: what a CTA can hold, or less where narrower tiles, split
// along K as far as it goes, still take no more than half the SMs (more of them meet
// the limit on clusters above: 128 tokens through 1024 x 8192 16.6 us, by 64 columns
// 24.1).  255 tokens through 276 x 512 at granule 32: 19.3 us by 256 columns, 11.7 by
// 64; 61 float32 tokens through 96 x 4608: 20.2 by 192, 16.3 by 96.
inline Tile choose_tile(int width, int dtype, int64_t m, int64_t tokens, int nkc, int sms) {
  auto fits = [&](int each) {  // all in one tile, or tiles of so many tokens leave SMs idle
    return tokens <= each || ceil_div(m, BM) * ceil_div(tokens, each) * most_parts(nkc) <= sms / 2;
  };
  if (dtype == 0) return {96, fits(32) ? 1 : 2};  // three columns a token
  if (fits(64)) return {64, 1};
  if (fits(128)) return {128, 1};
  // 256 columns and the 8-bit codes' stages together exceed shared memory
  return {width == 4 ? 128 : 96, 2};
}

template <int WIDTH, typename T, int N, int PARTS>
int run_tile(const uint16_t* x, int64_t ldx, int64_t k, int granule, Params p, cudaStream_t st) {
  constexpr int SPLIT = std::is_same<T, float>::value ? 3 : 1;
  constexpr int TOK = (N * PARTS) / SPLIT;
  const int64_t cols = (int64_t)p.tokens * SPLIT;
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(GQ_ECUDA, "cuTensorMapEncodeTiled is unavailable");
  CUtensorMap map;
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)cols};
  cuuint64_t strides[1] = {(cuuint64_t)(ldx * 2)};
  cuuint32_t box[2] = {64, (cuuint32_t)(N * PARTS)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r =
      fn(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<uint16_t*>(x), dims, strides, box,
         estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(GQ_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  CUtensorMap map_w;  // a block's 16 rows of codes: 256 elements of 4 or 8 bytes
  GQ_TRY(make_map(&map_w, WIDTH == 4 ? CU_TENSOR_MAP_DATA_TYPE_INT32 : CU_TENSOR_MAP_DATA_TYPE_INT64,
                  p.qw, 256, p.nkc, p.row_blocks, WIDTH));
  p.mt = (int)ceil_div(p.m, BM);
  p.nt = (int)ceil_div(p.tokens, TOK);
  const int64_t tiles = (int64_t)p.mt * p.nt;
  GQ_REQUIRE(tiles < (1ll << 31), "gq_linear: too many tiles");
  p.split = choose_split(tiles, p.nkc, sm_count());
  if (granule == 128) return launch<WIDTH, T, N, PARTS, 128>(map, map_w, p, st);
  if (granule == 64) return launch<WIDTH, T, N, PARTS, 64>(map, map_w, p, st);
  return launch<WIDTH, T, N, PARTS, 32>(map, map_w, p, st);
}

template <int WIDTH, typename T>
int run_typed(const uint16_t* x, int64_t ldx, int64_t k, int granule, const Params& p,
              cudaStream_t st) {
  constexpr int DTYPE = std::is_same<T, float>::value ? 0 : std::is_same<T, __half>::value ? 2 : 1;
  const Tile t = choose_tile(WIDTH, DTYPE, p.m, p.tokens, p.nkc, sm_count());
  if constexpr (DTYPE == 0) {
    if (t.parts == 1) return run_tile<WIDTH, T, 96, 1>(x, ldx, k, granule, p, st);
    return run_tile<WIDTH, T, 96, 2>(x, ldx, k, granule, p, st);
  } else {
    if (t.parts == 2) return run_tile<WIDTH, T, WIDTH == 4 ? 128 : 96, 2>(x, ldx, k, granule, p, st);
    if (t.n == 64) return run_tile<WIDTH, T, 64, 1>(x, ldx, k, granule, p, st);
    return run_tile<WIDTH, T, 128, 1>(x, ldx, k, granule, p, st);
  }
}

// What gq_test_linear_form tells of a configuration.
template <int WIDTH, int N, int PARTS>
void describe(int granule, int64_t* form) {
  auto put = [&](auto c) {
    using C = decltype(c);
    const int rings[] = {C::WSTAGES, C::W_FULL, C::ASTAGES, C::A_EMPTY, C::ACCS, C::T_FULL};
    for (int v : rings) *form++ = v;
  };
  if (granule == 128) put(Cfg<WIDTH, N, PARTS, 128>{});
  else if (granule == 64) put(Cfg<WIDTH, N, PARTS, 64>{});
  else put(Cfg<WIDTH, N, PARTS, 32>{});
}

}  // namespace lintc

namespace lin {

void many_form(int64_t m, int64_t k, int bits, int granule, int dtype, int64_t tokens, int sms,
               int64_t* form) {
  using namespace lintc;
  const int width = bits <= 4 ? 4 : 8, nkc = (int)(k / KC);
  const Tile t = choose_tile(width, dtype, m, tokens, nkc, sms);
  const int64_t tiles = ceil_div(m, BM) * ceil_div(tokens, t.tokens(dtype));
  form[0] = t.n;
  form[1] = t.parts;
  form[2] = choose_split(tiles, nkc, sms);
  form[3] = tiles;
  form += 4;
  if (t.parts == 1) {
    if (t.n == 64) width == 4 ? describe<4, 64, 1>(granule, form) : describe<8, 64, 1>(granule, form);
    else if (t.n == 96) width == 4 ? describe<4, 96, 1>(granule, form) : describe<8, 96, 1>(granule, form);
    else width == 4 ? describe<4, 128, 1>(granule, form) : describe<8, 128, 1>(granule, form);
  } else if (t.n == 96) {
    width == 4 ? describe<4, 96, 2>(granule, form) : describe<8, 96, 2>(granule, form);
  } else {
    describe<4, 128, 2>(granule, form);
  }
}

int run_many(const uint32_t* qw, const float* params, int64_t m, int64_t k, int bits, int granule,
             const uint16_t* x, int64_t ldx, int dtype, int64_t tokens, void* y, int64_t ldy,
             cudaStream_t st) {
  lintc::Params p = {};
  p.qw = reinterpret_cast<const uint4*>(qw);
  p.params = reinterpret_cast<const float2*>(params);
  p.m = m;
  p.nkc = (int)(k / KC);
  p.row_blocks = (int)ceil_div(m, ROWS);
  p.tokens = (int)tokens;
  p.y = y;
  p.ldy = ldy;
  if (bits <= 4) {
    if (dtype == 0) return lintc::run_typed<4, float>(x, ldx, k, granule, p, st);
    if (dtype == 1) return lintc::run_typed<4, __nv_bfloat16>(x, ldx, k, granule, p, st);
    return lintc::run_typed<4, __half>(x, ldx, k, granule, p, st);
  }
  if (dtype == 0) return lintc::run_typed<8, float>(x, ldx, k, granule, p, st);
  if (dtype == 1) return lintc::run_typed<8, __nv_bfloat16>(x, ldx, k, granule, p, st);
  return lintc::run_typed<8, __half>(x, ldx, k, granule, p, st);
}

}  // namespace lin
}  // namespace gq
