// Products with packed weights, y = x W^T:
//   y[t, r] = sum_c x[t, c] * (code[r, c] + qmin - zero[r, g(c)]) * scale[r, g(c)]
// for the codes of gq_pack_codes (bits 1..8, any groups, act-order).  The
// reference only ever dequantizes (quant.py:37); this runs the packed form.
//
// Layout (gq_linear_layout, made once per weight).  Columns are put in group
// order and every group is padded to a multiple of the granule G (32, 64 or
// 128 columns), the whole to K, a multiple of 128; kmap[k] is the original
// column of position k or -1.  Codes are stored as 4-bit (bits <= 4) or 8-bit
// fields, in blocks of 16 rows x 128 positions: block (rb, kc) is 16 rows of
// 64 (128) bytes, contiguous, blocks of one rb following each other, so a
// warp that walks along K reads one contiguous stream.  Inside a block's row
// the bytes are ordered for the m16n8k16 fragments: position 32 j + 8 t + i is
// field i of word j of lane t of its quad, so one 16-byte load per lane and
// row holds the lane's share of 128 positions, and the other operand's
// matching 8 values (positions 32 j + 8 t ..) are 16 contiguous bytes of x.
// The 16-byte pieces of a row are permuted with the row (piece_at), so that
// eight threads that read one piece of eight rows from shared memory meet eight
// different bank groups.
// params[(rb * K / G + granule) * 16 + r] = {scale, offset}: offset = zero -
// qmin is a whole number (the quantizers round it), so the weight is
// (code - offset) * scale.
//
// Arithmetic.  code - offset is exact in bf16 and fp16 (at most 8 bits), so
// the tensor cores multiply x by whole numbers and add in fp32, and each
// granule's sum is multiplied by its scale once, in fp32: the weights are not
// rounded.  float32 x is split into three bf16 terms by truncation (8 + 8 + 8
// bits: the split is exact), which run as three columns of the same product
// and are added at the end.
#include "gq_linear.cuh"

#include <algorithm>

namespace gq {
namespace lin {

constexpr int WARPS = 8;     // warps of a product CTA, which split K
constexpr int MAX_PARTS = 8; // CTAs of a cluster, which split K again

// ---------------------------------------------------------------- layout

__device__ __forceinline__ uint32_t stream_code(const uint32_t* row, int64_t c, int bits) {
  const int64_t bit = c * bits;
  const int64_t w = bit >> 5;
  const int off = (int)(bit & 31);
  uint64_t v = row[w];
  if (off + bits > 32) v |= (uint64_t)row[w + 1] << 32;
  return (uint32_t)(v >> off) & ((1u << bits) - 1u);
}

// One thread per 32-bit word of the laid-out codes.
template <int WIDTH>
__global__ void layout_codes_kernel(const uint32_t* __restrict__ packed, int64_t m, int64_t ldp,
                                    int bits, const int32_t* __restrict__ kmap, int64_t nkc,
                                    uint32_t* __restrict__ qw, int64_t total_words) {
  constexpr int WPR = KC * WIDTH / 32;  // words per block row: 16 or 32
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total_words;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t rest = i / WPR;
    const int r = (int)(rest % ROWS);
    const int wi = ((int)(i % WPR) & 3) | piece_at<WIDTH>((int)(i % WPR) >> 2, r) << 2;
    const int64_t blk = rest / ROWS;
    const int64_t kc = blk % nkc, row = (blk / nkc) * ROWS + r;
    uint32_t out = 0;
    if (row < m) {
      const uint32_t* src = packed + row * ldp;
      if constexpr (WIDTH == 4) {
        const int t = wi >> 2, j = wi & 3;
        const int32_t* km = kmap + kc * KC + 32 * j + 8 * t;
#pragma unroll
        for (int f = 0; f < 8; ++f) {
          const int32_t c = km[f];
          if (c >= 0) {
            const uint32_t v = stream_code(src, c, bits);
            out |= __funnelshift_l(v, v, 3 + 4 * (f >> 1) + 16 * (f & 1));  // field at bit 3, 7, .. 31, wrapping
          }
        }
      } else {
        const int jh = wi >> 4, t = (wi >> 2) & 3, jl = (wi >> 1) & 1, h = wi & 1;
        const int32_t* km = kmap + kc * KC + 32 * (2 * jh + jl) + 8 * t + 4 * h;
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const int32_t c = km[f];
          if (c >= 0) out |= stream_code(src, c, bits) << (8 * f);
        }
      }
    }
    qw[i] = out;
  }
}

// bad: bit 0 = an offset that is not a whole number of 0 .. 2^bits - 1, bit 1 =
// a scale that is not finite.
__global__ void layout_params_kernel(const float* __restrict__ scales,
                                     const float* __restrict__ zeros, int64_t m, int64_t n_groups,
                                     float qmin, float omax, const int32_t* __restrict__ granule_group,
                                     int64_t ngran, float2* __restrict__ params, int64_t total,
                                     int* __restrict__ bad) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int r = (int)(i % ROWS);
    const int64_t rest = i / ROWS;
    const int64_t gr = rest % ngran, row = (rest / ngran) * ROWS + r;
    const int32_t g = granule_group[gr];
    float2 p = make_float2(0.f, 0.f);
    if (row < m && g >= 0) {
      p.x = scales[row * n_groups + g];
      p.y = __fsub_rn(zeros[row * n_groups + g], qmin);
      int b = 0;
      if (!(p.y >= 0.f && p.y <= omax) || rintf(p.y) != p.y) b |= 1;
      if (!(fabsf(p.x) <= 3.402823466e38f)) b |= 2;
      if (b) atomicOr(bad, b);
    }
    params[i] = p;
  }
}

// ------------------------------------------------- x in position order

// xp[(t * split + s) * K + k] = term s of x[t, kmap[k]] (0 where kmap is -1).
// One thread per 8 positions.
template <typename T, int SPLIT>
__global__ void __launch_bounds__(128) gather_kernel(const T* __restrict__ x, int64_t ldx,
                                                     const int32_t* __restrict__ kmap, int64_t K,
                                                     uint16_t* __restrict__ xp) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t t = blockIdx.y;
  const int64_t k = 8 * (blockIdx.x * (int64_t)blockDim.x + threadIdx.x);
  if (k >= K) return;
  const T* row = x + t * ldx;
  const int4 m0 = *reinterpret_cast<const int4*>(kmap + k);
  const int4 m1 = *reinterpret_cast<const int4*>(kmap + k + 4);
  const int32_t c[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
  uint32_t v[SPLIT][4];
#pragma unroll
  for (int s = 0; s < SPLIT; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[s][i] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int sh = 16 * (i & 1);
    if constexpr (SPLIT == 1) {
      const uint16_t b = c[i] >= 0 ? *reinterpret_cast<const uint16_t*>(row + c[i]) : (uint16_t)0;
      v[0][i >> 1] |= (uint32_t)b << sh;
    } else {
      // truncation keeps every term's sign and never overflows; an infinity or
      // NaN stays in the first term alone
      const float f = c[i] >= 0 ? *reinterpret_cast<const float*>(row + c[i]) : 0.f;
      const uint32_t u = __float_as_uint(f);
      uint32_t h = u & 0xffff0000u;
      uint32_t mid = 0, lo = 0;
      if ((u & 0x7f800000u) != 0x7f800000u) {
        const float r = __fsub_rn(f, __uint_as_float(h));
        mid = __float_as_uint(r) & 0xffff0000u;
        lo = __float_as_uint(__fsub_rn(r, __uint_as_float(mid)));
      } else if (u & 0x007fffffu) {
        h |= 0x00400000u;  // a NaN whose mantissa lies in the low half stays one
      }
      v[0][i >> 1] |= (h >> 16) << sh;
      v[1][i >> 1] |= (mid >> 16) << sh;
      v[2][i >> 1] |= (lo >> 16) << sh;
    }
  }
#pragma unroll
  for (int s = 0; s < SPLIT; ++s)
    *reinterpret_cast<uint4*>(xp + (t * SPLIT + s) * K + k) =
        make_uint4(v[s][0], v[s][1], v[s][2], v[s][3]);
}

// ------------------------------------------------------ few-token product

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weights are read once: they pass L1 by, where x stays.
__device__ __forceinline__ uint4 load_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

struct Args {
  const uint4* qw;
  const float2* params;
  const uint16_t* x;  // [cols, ldx] 16-bit values in position order
  int64_t ldx;
  int cols;           // columns of the product: tokens * split
  int64_t m;
  int nkc;            // K / 128
  void* y;
  int64_t ldy;
  int tokens;
};

// One cluster: 16 rows, up to 8 NT columns; the warps of its CTAs take
// contiguous shares of K and their sums are added in order.
// Bound: reading the weights, in the end; now the loads' latency that 24 warps an SM
// leave bare, most of all where a CTA begins (issue slots 48 % busy, the integer pipe
// 45 %), and whole rounds of CTAs.  1 token bf16 of 28672 x 8192: 33.3 us, 4.0 TB/s (4.04
// rounds); of 11008 x 4096 8.0 us, of 4096 x 4096 3.8 us, of 1024 x 1024 1.9 us.  Four
// warps a CTA and twice the CTAs take 9 to 15 us where 256 row blocks take 9; four
// blocks in flight spill.
template <int WIDTH, typename T, int NT, int G>
__global__ void __launch_bounds__(32 * WARPS, NT == 1 ? 3 : 2)
    few_kernel(Args a, int split, bool dependent) {
  constexpr bool BF16 = !std::is_same<T, __half>::value;
  constexpr int SPLIT = std::is_same<T, float>::value ? 3 : 1;
  constexpr int TOK = 8 * NT / SPLIT;  // whole tokens per CTA
  constexpr int JG = G / 32;           // 32-position steps per granule
  constexpr int GPC = KC / G;          // granules per block
  constexpr int LPR = WIDTH / 4;       // 16-byte loads per lane, row and block
  constexpr int DEPTH = 2;             // blocks in flight per warp; 3 and 4 spill or take a CTA
  __shared__ float red[WARPS][8 * NT][ROWS + 1];
  __shared__ float sums[MAX_PARTS][8 * NT * ROWS];  // of the cluster's CTAs, in its first one
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int parts = 1 << split;                 // CTAs of the cluster
  const int part = blockIdx.x & (parts - 1);    // this one's rank
  const int64_t rb = blockIdx.x >> split;
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int tok0 = blockIdx.y * TOK;
  const int col0 = tok0 * SPLIT;
  const int share = part * WARPS + warp;
  const int c0 = (a.nkc * share / WARPS) >> split, c1 = (a.nkc * (share + 1) / WARPS) >> split;
  const uint4* qrow = a.qw + (rb * a.nkc) * (ROWS * 4 * LPR);
  const float2* prow = a.params + (rb * a.nkc) * (int64_t)(GPC * ROWS);

  uint4 q[DEPTH][2][LPR];
  auto fetch = [&](int c, uint4 (&d)[2][LPR]) {
    const uint4* b = qrow + (int64_t)c * (ROWS * 4 * LPR);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int l = 0; l < LPR; ++l)
        d[h][l] = load_stream(b + (g + 8 * h) * (4 * LPR) + piece_at<WIDTH>(l * 4 + t, g));
  };
#pragma unroll
  for (int s = 0; s < DEPTH; ++s)
    if (c0 + s < c1) fetch(c0 + s, q[s]);
  if (dependent) asm volatile("griddepcontrol.wait;" ::: "memory");

  // a lane without a column reads the first one: columns do not mix
  const uint16_t* xr[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int col = col0 + 8 * i + g;
    xr[i] = a.x + (int64_t)(8 * i + g < TOK * SPLIT && col < a.cols ? col : col0) * a.ldx +
            (int64_t)c0 * KC + 8 * t;
  }
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;

  const float2* pc = prow + (int64_t)c0 * (GPC * ROWS) + g;
  float2 pv[DEPTH][GPC][2];
  auto fetch_p = [&](float2 (&d)[GPC][2]) {
#pragma unroll
    for (int gr = 0; gr < GPC; ++gr) {
      d[gr][0] = __ldg(pc + gr * ROWS);
      d[gr][1] = __ldg(pc + gr * ROWS + 8);
    }
    pc += GPC * ROWS;
  };
  if (c0 < c1) fetch_p(pv[0]);
  for (int cb = c0; cb < c1; cb += DEPTH) {
#pragma unroll
    for (int s = 0; s < DEPTH; ++s) {
      const int c = cb + s;
      if (c >= c1) break;
      uint4 xv[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) xv[i][j] = *reinterpret_cast<const uint4*>(xr[i] + 32 * j);
        xr[i] += KC;
      }
      if (c + 1 < c1) fetch_p(pv[(s + 1) % DEPTH]);
#pragma unroll
      for (int gr = 0; gr < GPC; ++gr) {
        const float2 p0 = pv[s][gr][0], p1 = pv[s][gr][1];
        const uint32_t o0 = offset_operand<WIDTH, BF16>(p0.y);
        const uint32_t o1 = offset_operand<WIDTH, BF16>(p1.y);
        float sum[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[i][e] = 0.f;
#pragma unroll
        for (int jj = 0; jj < JG; ++jj) {
          const int j = gr * JG + jj;
          uint32_t v0[4], v1[4];
          const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&q[s][0][0]) + j * LPR;
          const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&q[s][1][0]) + j * LPR;
          decode8<WIDTH, BF16>(w0, o0, v0);
          decode8<WIDTH, BF16>(w1, o1, v1);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            mma16816<BF16>(sum[i], v0[0], v1[0], v0[1], v1[1], xv[i][j].x, xv[i][j].y);
            mma16816<BF16>(sum[i], v0[2], v1[2], v0[3], v1[3], xv[i][j].z, xv[i][j].w);
          }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          acc[i][0] = fmaf(p0.x, sum[i][0], acc[i][0]);
          acc[i][1] = fmaf(p0.x, sum[i][1], acc[i][1]);
          acc[i][2] = fmaf(p1.x, sum[i][2], acc[i][2]);
          acc[i][3] = fmaf(p1.x, sum[i][3], acc[i][3]);
        }
      }
      if (c + DEPTH < c1) fetch(c + DEPTH, q[s]);
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      red[warp][8 * i + 2 * t + (e & 1)][g + 8 * (e >> 1)] = acc[i][e];
  __syncthreads();
  // every CTA is running: the first one's memory can be written to
  if (parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  for (int i = threadIdx.x; i < TOK * ROWS; i += 32 * WARPS) {
    const int r = i % ROWS, tk = i / ROWS;
    float v = 0.f;
#pragma unroll
    for (int s = SPLIT - 1; s >= 0; --s) {  // the small terms first
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) sum += red[w][tk * SPLIT + s][r];
      v += sum;
    }
    if (parts == 1) {
      const int64_t row = rb * ROWS + r;
      if (row < a.m && tok0 + tk < a.tokens)
        store_out(static_cast<T*>(a.y) + (int64_t)(tok0 + tk) * a.ldy + row, v);
    } else {
      asm volatile(
          "{\n.reg .b32 d;\nmapa.shared::cluster.u32 d, %0, 0;\n"
          "st.shared::cluster.f32 [d], %1;\n}" ::"r"((uint32_t)__cvta_generic_to_shared(&sums[part][i])),
          "f"(v)
          : "memory");
    }
  }
  if (parts == 1) return;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  if (part) return;  // nothing reads the memory of the others
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int i = threadIdx.x; i < TOK * ROWS; i += 32 * WARPS) {
    const int r = i % ROWS, tk = i / ROWS;
    const int64_t row = rb * ROWS + r;
    if (row >= a.m || tok0 + tk >= a.tokens) continue;
    float v = 0.f;
    for (int s = 0; s < parts; ++s) v += sums[s][i];
    store_out(static_cast<T*>(a.y) + (int64_t)(tok0 + tk) * a.ldy + row, v);
  }
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                   int cluster, bool dependent, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (dependent) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int WIDTH, typename T, int NT>
int run_few(const Args& a, int granule, bool dependent, cudaStream_t st) {
  constexpr int SPLIT = std::is_same<T, float>::value ? 3 : 1;
  constexpr int TOK = 8 * NT / SPLIT;
  const int64_t rbs = ceil_div(a.m, ROWS), groups = ceil_div(a.tokens, TOK);
  // K is split over a cluster while there are fewer CTAs than SMs and every warp
  // keeps a block: 1 token of 1024 x 8192 3.5 us by clusters of 4, 5.5 by single
  // CTAs; of 4096 x 4096 (256 row blocks) 6.8 by pairs, 4.3 without.
  int split = 0;
  while ((1 << split) < MAX_PARTS && (rbs * groups << split) < sm_count() && a.nkc >= 2 * WARPS << split) ++split;
  const dim3 grid((unsigned)(rbs << split), (unsigned)groups);
  cudaError_t e;
  if (granule == 128)
    e = launch(few_kernel<WIDTH, T, NT, 128>, grid, dim3(32 * WARPS), 0, st, 1 << split, dependent, a, split, dependent);
  else if (granule == 64)
    e = launch(few_kernel<WIDTH, T, NT, 64>, grid, dim3(32 * WARPS), 0, st, 1 << split, dependent, a, split, dependent);
  else
    e = launch(few_kernel<WIDTH, T, NT, 32>, grid, dim3(32 * WARPS), 0, st, 1 << split, dependent, a, split, dependent);
  if (e != cudaSuccess) return fail(GQ_ECUDA, "gq_linear: %s", cudaGetErrorString(e));
  return check_launch("gq_linear few-token product");
}

template <int WIDTH, typename T>
int run_typed(const Args& a, int granule, bool dependent, cudaStream_t st) {
  const int64_t tiles = ceil_div(a.cols, 8);
  if (tiles <= 1) return run_few<WIDTH, T, 1>(a, granule, dependent, st);
  if (tiles == 2) return run_few<WIDTH, T, 2>(a, granule, dependent, st);
  if constexpr (!std::is_same<T, float>::value) {  // 24 columns are 8 whole float32 tokens
    if (tiles > 3) return run_few<WIDTH, T, 4>(a, granule, dependent, st);
  }
  return run_few<WIDTH, T, 3>(a, granule, dependent, st);
}

// The columns of x that the few-token form takes: one CTA's, and 24 where the tcgen05
// form's row tiles alone fill the SMs.  32 against 33 tokens: 4096 x 4096 9.4 and 12.4
// us, 11008 x 4096 23.4 and 22.6, 28672 x 8192 94 and 71.
inline int few_columns(int dtype, int64_t m, int sms) {
  return dtype == 0 || m >= (int64_t)sms * 128 ? 24 : 32;
}

inline int64_t align256(int64_t b) { return (b + 255) & ~int64_t(255); }

}  // namespace lin
}  // namespace gq

extern "C" {

int gq_linear_layout(const uint32_t* packed, int64_t m, int64_t n, int64_t ldp, int bits, int sym,
                     const float* scales, const float* zeros, int64_t n_groups,
                     const int32_t* kmap, int64_t k, const int32_t* granule_group, int granule,
                     uint32_t* qw, float* params, int* bad, void* stream) {
  using namespace gq;
  GQ_REQUIRE(bits >= 1 && bits <= 8 && (!sym || bits >= 2), "gq_linear_layout: bad bits");
  GQ_REQUIRE(granule == 32 || granule == 64 || granule == 128,
             "gq_linear_layout: granule must be 32, 64 or 128");
  GQ_REQUIRE(m >= 0 && n >= 0 && n_groups >= 0 && ldp >= gq_packed_words(n, bits),
             "gq_linear_layout: bad shape");
  GQ_REQUIRE(k >= n && k % lin::KC == 0 && k < (1ll << 31),
             "gq_linear_layout: k must be a multiple of 128 that holds the %lld columns",
             (long long)n);
  GQ_REQUIRE(m < (1ll << 31), "gq_linear_layout: too many rows");
  GQ_REQUIRE(bad != nullptr, "gq_linear_layout: NULL bad");
  cudaStream_t st = as_stream(stream);
  GQ_CHECK_CUDA(cudaMemsetAsync(bad, 0, sizeof(int), st));
  if (m == 0 || k == 0) return GQ_OK;
  GQ_REQUIRE(packed && scales && zeros && kmap && granule_group && qw && params,
             "gq_linear_layout: NULL buffer");
  const int width = bits <= 4 ? 4 : 8;
  const int64_t rbs = ceil_div(m, lin::ROWS);
  const int64_t words = rbs * lin::ROWS * k * width / 32;
  const unsigned g1 = (unsigned)std::min<int64_t>(ceil_div(words, 256), sm_count() * 32);
  if (width == 4)
    lin::layout_codes_kernel<4><<<g1, 256, 0, st>>>(packed, m, ldp, bits, kmap, k / lin::KC, qw, words);
  else
    lin::layout_codes_kernel<8><<<g1, 256, 0, st>>>(packed, m, ldp, bits, kmap, k / lin::KC, qw, words);
  GQ_TRY(check_launch("gq_linear_layout codes"));
  const int64_t ngran = k / granule, total = rbs * lin::ROWS * ngran;
  const float qmin = sym ? (float)(1 - (1 << (bits - 1))) : 0.f;
  lin::layout_params_kernel<<<(unsigned)std::min<int64_t>(ceil_div(total, 256), sm_count() * 16), 256, 0, st>>>(
      scales, zeros, m, n_groups, qmin, (float)((1 << bits) - 1), granule_group, ngran,
      reinterpret_cast<float2*>(params), total, bad);
  return check_launch("gq_linear_layout params");
}

int gq_test_linear_form(int64_t m, int64_t k, int bits, int granule, int dtype, int64_t tokens,
                        int sms, int64_t* form) {
  using namespace gq;
  GQ_REQUIRE(form != nullptr && m >= 1 && m < (1ll << 31) && tokens >= 1 && tokens < (1ll << 29) &&
                 k >= 1 && k < (1ll << 31) && k % lin::KC == 0 && bits >= 1 && bits <= 8 &&
                 (granule == 32 || granule == 64 || granule == 128) && dtype >= 0 && dtype <= 2 &&
                 sms >= 1,
             "gq_test_linear_form: bad argument");
  for (int i = 0; i < 10; ++i) form[i] = 0;
  if (tokens * (dtype == 0 ? 3 : 1) > lin::few_columns(dtype, m, sms))
    lin::many_form(m, k, bits, granule, dtype, tokens, sms, form);
  return GQ_OK;
}

int64_t gq_linear_workspace_size(int64_t tokens, int64_t k, int dtype) {
  if (tokens <= 0 || k <= 0) return 256;
  return gq::lin::align256(tokens * (dtype == 0 ? 3 : 1) * k * 2);
}

int gq_linear(const uint32_t* qw, const float* params, const int32_t* kmap, int64_t m, int64_t n,
              int64_t k, int bits, int granule, int direct, const void* x, int dtype,
              int64_t tokens, int64_t ldx, void* y, int64_t ldy, void* workspace,
              int64_t workspace_bytes, void* stream) {
  using namespace gq;
  GQ_REQUIRE(dtype >= 0 && dtype <= 2, "gq_linear: dtype must be 0 (float32), 1 (bf16) or 2 (fp16)");
  GQ_REQUIRE(bits >= 1 && bits <= 8, "gq_linear: bad bits");
  GQ_REQUIRE(granule == 32 || granule == 64 || granule == 128,
             "gq_linear: granule must be 32, 64 or 128");
  GQ_REQUIRE(m >= 0 && n >= 1 && tokens >= 0 && m < (1ll << 31) && tokens < (1ll << 29),
             "gq_linear: bad shape");
  GQ_REQUIRE(k >= n && k % lin::KC == 0 && k < (1ll << 31), "gq_linear: bad k");
  GQ_REQUIRE(ldx >= n && ldy >= m, "gq_linear: leading dimension too small");
  if (m == 0 || tokens == 0) return GQ_OK;
  GQ_REQUIRE(qw && params && x && y && (direct || kmap), "gq_linear: NULL buffer");
  GQ_REQUIRE((reinterpret_cast<uintptr_t>(qw) & 15) == 0 && (reinterpret_cast<uintptr_t>(params) & 15) == 0,
             "gq_linear: the laid-out weights must be 16-byte aligned");
  // x is read in place when its columns already are the positions and its
  // rows can be read 16 bytes at a time
  const bool in_place = direct && k == n && dtype != 0 && ldx % 8 == 0 &&
                        (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  cudaStream_t st = as_stream(stream);
  lin::Args a;
  a.qw = reinterpret_cast<const uint4*>(qw);
  a.params = reinterpret_cast<const float2*>(params);
  a.m = m;
  a.nkc = (int)(k / lin::KC);
  a.y = y;
  a.ldy = ldy;
  a.tokens = (int)tokens;
  a.cols = (int)tokens * (dtype == 0 ? 3 : 1);
  if (in_place) {
    a.x = static_cast<const uint16_t*>(x);
    a.ldx = ldx;
  } else {
    GQ_REQUIRE(kmap != nullptr && (reinterpret_cast<uintptr_t>(kmap) & 15) == 0,
               "gq_linear: kmap must be 16-byte aligned");
    GQ_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0 &&
                   workspace_bytes >= gq_linear_workspace_size(tokens, k, dtype),
               "gq_linear: workspace too small or not 256-byte aligned");
    uint16_t* xp = static_cast<uint16_t*>(workspace);
    for (int64_t t0 = 0; t0 < tokens; t0 += 65535) {
      const dim3 grid((unsigned)ceil_div(k, 8 * 128), (unsigned)std::min<int64_t>(65535, tokens - t0));
      if (dtype == 0)
        lin::gather_kernel<float, 3><<<grid, 128, 0, st>>>(
            static_cast<const float*>(x) + t0 * ldx, ldx, kmap, k, xp + t0 * 3 * k);
      else
        lin::gather_kernel<uint16_t, 1><<<grid, 128, 0, st>>>(
            static_cast<const uint16_t*>(x) + t0 * ldx, ldx, kmap, k, xp + t0 * k);
      GQ_TRY(check_launch("gq_linear gather"));
    }
    a.x = xp;
    a.ldx = k;
  }
  if (a.cols > lin::few_columns(dtype, m, sm_count()))
    return lin::run_many(qw, params, m, k, bits, granule, a.x, a.ldx, dtype, tokens, y, ldy, st);
  const bool dep = !in_place;
  if (bits <= 4) {
    if (dtype == 0) return lin::run_typed<4, float>(a, granule, dep, st);
    if (dtype == 1) return lin::run_typed<4, __nv_bfloat16>(a, granule, dep, st);
    return lin::run_typed<4, __half>(a, granule, dep, st);
  }
  if (dtype == 0) return lin::run_typed<8, float>(a, granule, dep, st);
  if (dtype == 1) return lin::run_typed<8, __nv_bfloat16>(a, granule, dep, st);
  return lin::run_typed<8, __half>(a, granule, dep, st);
}

}  // extern "C"
