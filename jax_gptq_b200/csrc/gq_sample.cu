// Choice of the next token: temperature, top-k, top-p and min-p, then the
// inverse of what remains of the distribution at a given uniform number.
//
// Per row, with l the logits (NaN and -inf are excluded), M their maximum and
// e_i = exp((l_i - M) / temperature):
//   order the tokens by logit, largest first, equal ones by index;
//   top-k keeps the first k of them; top-p, of those, the ones before which
//   less than p of their mass lies; min-p, of those, the ones with e_i >= min_p;
//   the first always stays.  W = sum of e over the kept tokens;
//   token = the smallest index i with  sum of kept e_j, j <= i  >  u W.
// Temperature 0 (or below, or NaN) is the first largest logit; others count as at least
// 1e-37 and at most 1e36.  A row without any token gives -1 and -inf.
//
// Sums.  The choice turns on sums that lie next to a border, so e is computed
// in float64 and held as a whole number of 2^-S (S = 45 for up to 2^17 tokens):
// sums of whole numbers do not depend on the order of additions, so the shared
// memory atomics and the split over threads and blocks never change a result,
// and a term's rounding (2^-46 of the largest) is far below what a float32
// uniform resolves.  Terms below 2^-(S+1) are rounded to zero: they can not be drawn.
//
// Split.  A cluster of up to 8 blocks takes a row, each a contiguous part, each
// warp a contiguous part of that; parts of up to 64 KB are kept in shared memory,
// larger ones are read again from L2.  Passes over the row:
//   1. the maximum;
//   2. with top-k or top-p the number of tokens in 512 bins of log2 e (found in
//      float32: any function that keeps the order will do); without top-k each
//      warp's sum of e;
//   3. the bins tell down to which one a border can lie: the k-th token's, or the
//      first by which the sum is at least p (a bin's sum is at least its count
//      times its smallest e).  Tokens down to there, where they are at most 2048,
//      are collected and sorted by every block, and the borders read off their
//      running sum; up to 256 kept ones are drawn from right there.
//      Otherwise (flat distributions) top-k's border bin alone is sorted; for top-p
//      the bins' sums are estimated, and one pass adds up what lies before the place
//      where the border should be and collects the tokens around it.  Where that
//      misses, the counts also tell from which bin on the border can lie (a bin's sum
//      is at most its count times its largest e), one pass adds up what lies before
//      and 512 cells between the two, and the border's cell is sorted.  More than
//      2048 tokens in one (runs of equal logits) are resolved by radix passes over
//      the ordered bits;
//   4. with filters each warp's sum of the kept e and its number of tokens equal
//      to the border;
//   5. the block that holds u W finds the token in the part of one warp.
// Reading other blocks' shared memory is slow (a 16 KB histogram of all 8 blocks
// took 24000 cycles), so little is exchanged, by as many lanes at once as can be.
#include "gq_common.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>

namespace cg = cooperative_groups;

namespace gq {
namespace samp {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int BINS = 512;   // of log2 e, 11 to a power of two; one a thread
constexpr int MAX_CL = 8;
constexpr int LIST = 2048;  // tokens that are collected and sorted
constexpr int RANKED = 512; // up to so many by counting, more by a sorting network
constexpr int DIRECT = 256; // up to so many kept ones are drawn from without another pass
constexpr int MAX_STAGE = 64 * 1024;  // bytes of a row that a block keeps in shared memory

struct RowParam {  // a setting: one value, or one per row
  const void* rows;
  int kind;  // 0 value, 1 float32, 2 float64, 3 int32, 4 int64
  double value;
};
__device__ __forceinline__ double row_value(const RowParam& p, int64_t r) {
  switch (p.kind) {
    case 1: return (double)static_cast<const float*>(p.rows)[r];
    case 2: return static_cast<const double*>(p.rows)[r];
    case 3: return (double)static_cast<const int32_t*>(p.rows)[r];
    case 4: return (double)static_cast<const int64_t*>(p.rows)[r];
    default: return p.value;
  }
}

struct Args {
  const void* logits;
  int64_t ld;
  int64_t rows;
  int vocab;
  RowParam u, temperature, top_k, top_p, min_p;
  int64_t* tokens;
  float* logprobs;
  double scale;  // 2^S
  int limb;      // bits: 3 limbs hold a term, and 32 bits the sum of a block's
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }

// Bits of a float (not NaN) in its order; -0 and +0 are one value.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

// 2^(-j/32), the nearest doubles
constexpr int ROOTS = 32;
__device__ const uint64_t root_bits[ROOTS] = {
    0x3ff0000000000000ull, 0x3fef50765b6e4540ull, 0x3feea4afa2a490daull, 0x3fedfc97337b9b5full,
    0x3fed5818dcfba487ull, 0x3fecb720dcef9069ull, 0x3fec199bdd85529cull, 0x3feb7f76f2fb5e47ull,
    0x3feae89f995ad3adull, 0x3fea5503b23e255dull, 0x3fe9c49182a3f090ull, 0x3fe93737b0cdc5e5ull,
    0x3fe8ace5422aa0dbull, 0x3fe82589994cce13ull, 0x3fe7a11473eb0187ull, 0x3fe71f75e8ec5f74ull,
    0x3fe6a09e667f3bcdull, 0x3fe6247eb03a5585ull, 0x3fe5ab07dd485429ull, 0x3fe5342b569d4f82ull,
    0x3fe4bfdad5362a27ull, 0x3fe44e086061892dull, 0x3fe3dea64c123422ull, 0x3fe371a7373aa9cbull,
    0x3fe306fe0a31b715ull, 0x3fe29e9df51fdee1ull, 0x3fe2387a6e756238ull, 0x3fe1d4873168b9aaull,
    0x3fe172b83c7d517bull, 0x3fe11301d0125b51ull, 0x3fe0b5586cf9890full, 0x3fe059b0d3158574ull};
struct Roots {  // in shared memory, high and low words: one a bank each
  uint32_t hi[ROOTS], lo[ROOTS];
};

// 2^-y for 0 <= y < 1000, within 2^-47 of it: y is split at the nearest k/32,
// 2^-(k/32) is a table's entry with an exponent, and 2^-f, |f| <= 1/64, is the Taylor
// series to the 5th power (remainder below 2^-48).  N at a time, step by step: one
// alone is a chain of dependent float64 operations, and four warps a scheduler do not
// hide that.
template <int N>
__device__ __forceinline__ void exp2_neg(const Roots& roots, const double (&y)[N], double (&out)[N]) {
  constexpr double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the whole part
  constexpr double c[6] = {1.0, -0.6931471805599453, 0.24022650695910072, -0.05550410866482158,
                           0.009618129107628477, -0.0013333558146428443};  // (-ln 2)^n / n!
  double x[N];
  int k[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double s = fma(y[i], (double)ROOTS, magic);
    k[i] = __double2loint(s);
    x[i] = fma(s - magic, -1.0 / ROOTS, y[i]);
    out[i] = c[5];
  }
#pragma unroll
  for (int n = 4; n >= 0; --n)
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = fma(out[i], x[i], c[n]);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = k[i] & (ROOTS - 1);
    out[i] *= __hiloint2double((int)roots.hi[j] - ((k[i] << 15) & (int)0xfff00000), (int)roots.lo[j]);
  }
}

struct Row {
  double mx, c;  // the maximum, log2(e) / temperature
  double limit;  // terms with log2 e below -limit are zero: S + 2, where rounding makes them so too
  double scale;
  float top, low;  // the maximum; a logit whose term is zero
  bool plain;      // `low` is so, and (mx - l) c below 1000 for all l from there on
  const Roots* roots;
  // distance below the maximum in powers of two; false where the term is zero
  // (y is then any number)
  __device__ __forceinline__ bool distance(float l, double& y) const {
    y = l == top ? 0.0 : (mx - (double)l) * c;
    return y < limit;  // false for NaN
  }
  // the terms as whole numbers, 0 where !have
  template <int N>
  __device__ __forceinline__ void fixed(const double (&y)[N], const bool (&have)[N],
                                        uint64_t (&f)[N]) const {
    double e[N];
    exp2_neg(*roots, y, e);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const double t = fma(e[i], scale, 4503599627370496.0);  // + 2^52: whole number in the low bits
      f[i] = have[i] ? (uint64_t)__double_as_longlong(t) & 0xfffffffffffffull : 0;
    }
  }
  // the sum of four logits' terms (plain rows): those below `low` and NaN are raised to
  // it, and only the sum is freed of the four exponents of 2^52
  __device__ __forceinline__ uint64_t sum4(const float* l) const {
    double y[4], e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (mx - (double)fmaxf(l[i], low)) * c;
    exp2_neg(*roots, y, e);
    uint64_t sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sum += (uint64_t)__double_as_longlong(fma(e[i], scale, 4503599627370496.0));
    return sum - 4 * 0x4330000000000000ull;
  }
  __device__ __forceinline__ uint64_t fixed(float l) const {
    double y[1];
    const bool have[1] = {distance(l, y[0])};
    uint64_t f[1];
    if (!have[0]) y[0] = 0.0;
    fixed(y, have, f);
    return f[0];
  }
};

// The row's elements in units of VEC, aligned to 16 bytes: unit q holds
// elements VEC q - shift .. + VEC - 1.
template <typename T>
struct Units {
  static constexpr int VEC = 16 / sizeof(T);
  const T* row;
  int vocab, shift, count;
  __device__ __forceinline__ Units(const T* r, int v) : row(r), vocab(v) {
    shift = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    count = (v + shift + VEC - 1) / VEC;
  }
  // a unit's 16 bytes, NaN where there is no element
  __device__ __forceinline__ uint4 load(int q) const {
    const int i0 = q * VEC - shift;
    if (i0 >= 0 && i0 + VEC <= vocab) return __ldg(reinterpret_cast<const uint4*>(row + i0));
    using Bits = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
    struct alignas(16) Pack { Bits e[VEC]; } p;
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      p.e[e] = (i0 + e >= 0 && i0 + e < vocab)
                   ? reinterpret_cast<const Bits*>(row)[i0 + e]
                   : (Bits)(sizeof(T) == 4 ? 0x7fc00000u : std::is_same<T, __half>::value ? 0x7e00u : 0x7fc0u);
    uint4 raw;
    memcpy(&raw, &p, 16);
    return raw;
  }
  static __device__ __forceinline__ void values(const uint4& raw, float (&x)[VEC]) {
    struct alignas(16) Pack { T e[VEC]; } p;
    memcpy(&p, &raw, 16);
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = to_f<T>(p.e[e]);
  }
};

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Border {
  uint32_t key;   // tokens with a larger key are kept, of those with this key the first `ties`
  uint32_t ties;
};

struct Shared {
  Roots roots;
  uint32_t count[BINS];                // histogram over log2 e: tokens
  uint32_t mass[3][BINS];              // and sums, by limbs of a.limb bits
  union {
    alignas(16) unsigned long long keys[LIST];  // collected from the whole row, sorted
    struct {
      unsigned long long rmass[2][256];  // a radix pass, two buffers in turn
      uint32_t rcount[2][256];
    } radix;
  };
  unsigned long long list[LIST];       // collected in this block
  uint32_t list_n, kmin, kmax;
  unsigned long long term[DIRECT];     // a draw from the sorted list
  uint32_t index[DIRECT];
  uint64_t wmass[WARPS];               // per warp: what the draw walks through
  uint32_t wties[WARPS];
  float mx[WARPS];
  uint32_t amax[WARPS];
  unsigned long long smass[WARPS];     // scratch of the scans
  uint32_t scount[WARPS];
  float block_max;
  uint32_t block_arg;
  unsigned long long all_mass[MAX_CL * WARPS];  // every warp of the cluster
  uint32_t all_ties[MAX_CL * WARPS];
  int pick_warp;
  uint32_t pick_ties, pick_all_ties;
  unsigned long long pick_before, pick_total;
  int found;
  uint32_t found_count, found_own;
  unsigned long long found_mass, found_own_mass;
  int hit, last;
  double hit_y, last_y;
};

// Sorts E keys a thread, the largest first, by a bitonic network: keys E t .. E t + E - 1
// in thread t's registers, partners in other lanes by shuffles, in other warps through
// shared memory (10 of 66 steps of 2048 keys; 812 keys took 19000 cycles with all
// steps there, 9300 so).
template <int E>
__device__ __forceinline__ void sort_keys(unsigned long long* keys) {
  const int tid = threadIdx.x;
  struct alignas(16) Pack { unsigned long long k[E]; } v;
  __syncthreads();
  v = reinterpret_cast<const Pack*>(keys)[tid];
  auto exchange = [](unsigned long long mine, unsigned long long other, bool larger) {
    return (mine > other) == larger ? mine : other;
  };
  for (int k = 2; k <= E * THREADS; k *= 2) {
    for (int j = k / 2; j >= E; j /= 2) {
      const bool larger = ((E * tid & j) == 0) == ((E * tid & k) == 0);
      const int apart = j / E;  // threads
      Pack o;
      if (apart < 32) {
#pragma unroll
        for (int i = 0; i < E; ++i) o.k[i] = __shfl_xor_sync(0xffffffffu, v.k[i], apart);
      } else {
        __syncthreads();
        reinterpret_cast<Pack*>(keys)[tid] = v;
        __syncthreads();
        o = reinterpret_cast<const Pack*>(keys)[tid ^ apart];
      }
#pragma unroll
      for (int i = 0; i < E; ++i) v.k[i] = exchange(v.k[i], o.k[i], larger);
    }
#pragma unroll
    for (int j = E / 2; j > 0; j /= 2) {  // inside the thread
      if (j >= k) continue;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if ((i & j) == 0) {
          const bool larger = ((E * tid + i) & k) == 0;
          const unsigned long long x = v.k[i], y = v.k[i + j];
          const bool keep = (x > y) == larger;
          v.k[i] = keep ? x : y;
          v.k[i + j] = keep ? y : x;
        }
    }
  }
  __syncthreads();
  reinterpret_cast<Pack*>(keys)[tid] = v;
  __syncthreads();
}

// STAGED: the block's part of the row is kept in shared memory
template <typename T, bool STAGED>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(Args a) {
  constexpr int VEC = Units<T>::VEC;
  __shared__ Shared sh;
  extern __shared__ uint4 stage[];
  cg::cluster_group cl = cg::this_cluster();
  const int CL = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t r = blockIdx.x / CL;
  const T* row = static_cast<const T*>(a.logits) + r * a.ld;
  const Units<T> un(row, a.vocab);
  // this warp's units
  const int b0 = (int)((int64_t)un.count * rank / CL), b1 = (int)((int64_t)un.count * (rank + 1) / CL);
  auto warp_begin = [&](int w) { return b0 + (int)((int64_t)(b1 - b0) * w / WARPS); };
  const int w0 = warp_begin(warp), w1 = warp_begin(warp + 1);
  auto unit = [&](int q) { return STAGED ? stage[q - b0] : un.load(q); };
  // f(values, index of the first) for this lane's tokens, a unit at a time, NaN
  // where there is none
  auto each_unit = [&](auto&& f) {
    if (w0 + lane >= w1) return;
    uint4 next = unit(w0 + lane);  // one ahead: a row that is not staged comes from L2
    for (int q = w0 + lane; q < w1; q += 32) {
      float x[VEC];
      un.values(next, x);
      next = unit(min(q + 32, w1 - 1));
      f(x, q * VEC - un.shift);
    }
  };
  auto each_token = [&](auto&& f) {
    each_unit([&](const float (&x)[VEC], int i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f(x[e], i + e);
    });
  };
  // the same field of block c, read by lane c of every warp
  auto peer = [&](int c) { return cl.map_shared_rank(&sh, c); };

  const double temp = row_value(a.temperature, r);
  const double kd = row_value(a.top_k, r);
  const double p = row_value(a.top_p, r);
  const double mp = row_value(a.min_p, r);
  const double u = row_value(a.u, r);

  const uint64_t root = tid < ROOTS ? root_bits[tid] : 0;

  // ---- 1. the maximum (and for temperature 0 its first index)
  float mx = -INFINITY;
  uint32_t arg = 0xffffffffu;
  for (int q = w0 + lane; q < w1; q += 128) {  // four units in flight
    uint4 raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (q + 32 * i < w1) raw[i] = un.load(q + 32 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (q + 32 * i >= w1) break;
      if (STAGED) stage[q + 32 * i - b0] = raw[i];
      float x[VEC];
      un.values(raw[i], x);
      if (temp > 0.0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) mx = fmaxf(mx, x[e]);  // (not NaN)
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (x[e] > mx) {  // indices grow along a lane's walk: the first one stays
            mx = x[e];
            arg = (uint32_t)((q + 32 * i) * VEC - un.shift + e);
          }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, mx, o);
    const uint32_t oa = __shfl_xor_sync(0xffffffffu, arg, o);
    if (om > mx || (om == mx && oa < arg)) {
      mx = om;
      arg = oa;
    }
  }
  if (lane == 0) {
    sh.mx[warp] = mx;
    sh.amax[warp] = arg;
  }
  sh.count[tid] = sh.mass[0][tid] = sh.mass[1][tid] = sh.mass[2][tid] = 0;
  if (tid < ROOTS) {
    sh.roots.hi[tid] = (uint32_t)(root >> 32);
    sh.roots.lo[tid] = (uint32_t)root;
  }
  if (tid == 0) {
    sh.list_n = 0;
    sh.hit = sh.last = -1;
  }
  __syncthreads();
  if (warp == 0) {
    mx = lane < WARPS ? sh.mx[lane] : -INFINITY;
    arg = lane < WARPS ? sh.amax[lane] : 0xffffffffu;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, mx, o);
      const uint32_t oa = __shfl_xor_sync(0xffffffffu, arg, o);
      if (om > mx || (om == mx && oa < arg)) {
        mx = om;
        arg = oa;
      }
    }
    if (lane == 0) {
      sh.block_max = mx;
      sh.block_arg = arg;
    }
  }
  cl.sync();
  mx = lane < CL ? peer(lane)->block_max : -INFINITY;
  arg = lane < CL ? peer(lane)->block_arg : 0xffffffffu;
#pragma unroll
  for (int o = MAX_CL / 2; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, mx, o);
    const uint32_t oa = __shfl_xor_sync(0xffffffffu, arg, o);
    if (om > mx || (om == mx && oa < arg)) {
      mx = om;
      arg = oa;
    }
  }
  mx = __shfl_sync(0xffffffffu, mx, 0);
  arg = __shfl_sync(0xffffffffu, arg, 0);
  const bool none = !(mx > -INFINITY);
  if (none || !(temp > 0.0)) {
    if (rank == 0 && tid == 0) {
      a.tokens[r] = none ? -1 : (int64_t)arg;
      if (a.logprobs) a.logprobs[r] = none ? -INFINITY : 0.f;
    }
    cl.sync();  // no block leaves while another may read its shared memory
    return;
  }
  Row rw;
  rw.mx = (double)mx;
  rw.top = mx;
  rw.roots = &sh.roots;
  // bins are found in float32: 11 c has to be one, and where mx - l is infinite, between
  // numbers of opposite sign, the term has to be zero
  rw.c = 1.4426950408889634 / fmin(fmax(temp, 1e-37), 1e36);
  rw.scale = a.scale;
  rw.limit = (double)(((__double2hiint(a.scale) >> 20) & 0x7ff) - 1023) + 2.0;  // S + 2
  rw.low = __double2float_rd(rw.mx - 60.0 / rw.c);
  const double low_y = (rw.mx - (double)rw.low) * rw.c;  // 0 where the largest is huge, NaN where infinite
  rw.plain = rw.low > -INFINITY && low_y > 59.0 && low_y < 1000.0;
  const float cf = (float)rw.c;
  // bin of a token; the last bin holds only terms that are zero (46.45 powers of
  // two below the largest and further), and whatever is no token at all
  auto depth = [&](float l) {  // in bins
    const float y = l == mx ? 0.f : (mx - l) * cf;
    return fminf(y, 50.f) * 11.f;
  };
  auto bin_of = [&](float l) { return min(BINS - 1, (int)depth(l)); };
  const bool by_k = kd >= 1.0 && kd < (double)a.vocab;
  const uint32_t k = by_k ? (uint32_t)kd : 0;
  const bool by_p = p < 1.0;
  const bool by_min = mp > 0.0;
  // e >= min_p in powers of two below the largest; the largest itself stays
  const double floor_y = by_min ? fmax(-log2(mp), 0.0) : 0.0;

  // ---- 2. sums, tokens per bin
  if (by_k || by_p)
    each_token([&](float x, int) {
      const int b = bin_of(x);
      if (b < BINS - 1) atomicAdd(&sh.count[b], 1u);
    });
  auto sum_terms = [&] {  // each warp's sum of e
    uint64_t sum = 0;
    each_unit([&](const float (&x)[VEC], int) {
#pragma unroll
      for (int h = 0; h < VEC; h += 4) {
        if (rw.plain) {
          sum += rw.sum4(x + h);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) sum += rw.fixed(x[h + e]);
        }
      }
    });
    sum = warp_sum64(sum);
    if (lane == 0) sh.wmass[warp] = sum;
  };
  if (!by_k) sum_terms();
  if (lane == 0) sh.wties[warp] = 0;
  cl.sync();

  // ---- 3. borders
  Border border{0, 0xffffffffu};  // everything
  // exclusive prefixes over the threads, and the totals
  auto scan = [&](unsigned long long m, uint32_t n, unsigned long long& pm, uint32_t& pn,
                  unsigned long long& tm, uint32_t& tn) {
    unsigned long long im = m;
    uint32_t in = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long vm = __shfl_up_sync(0xffffffffu, im, o);
      const uint32_t vn = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) {
        im += vm;
        in += vn;
      }
    }
    __syncthreads();
    if (lane == 31) {
      sh.smass[warp] = im;
      sh.scount[warp] = in;
    }
    __syncthreads();
    unsigned long long wm = lane < WARPS ? sh.smass[lane] : 0;
    uint32_t wn = lane < WARPS ? sh.scount[lane] : 0;
#pragma unroll
    for (int o = 1; o < WARPS; o <<= 1) {
      const unsigned long long vm = __shfl_up_sync(0xffffffffu, wm, o);
      const uint32_t vn = __shfl_up_sync(0xffffffffu, wn, o);
      if (lane >= o) {
        wm += vm;
        wn += vn;
      }
    }
    tm = __shfl_sync(0xffffffffu, wm, WARPS - 1);
    tn = __shfl_sync(0xffffffffu, wn, WARPS - 1);
    const unsigned long long bm = __shfl_sync(0xffffffffu, wm, max(warp - 1, 0));
    const uint32_t bn = __shfl_sync(0xffffffffu, wn, max(warp - 1, 0));
    pm = im - m + (warp > 0 ? bm : 0);
    pn = in - n + (warp > 0 ? bn : 0);
  };
  // what the one thread that found something (what >= 0) says to all
  auto tell = [&](int what, uint32_t n, unsigned long long m, uint32_t own, unsigned long long own_m) {
    __syncthreads();
    if (tid == 0) sh.found = -1;
    __syncthreads();
    if (what >= 0) {
      sh.found = what;
      sh.found_count = n;
      sh.found_mass = m;
      sh.found_own = own;
      sh.found_own_mass = own_m;
    }
    __syncthreads();
    return sh.found;
  };
  // of `own` equal tokens, before which `msum` lies, those that begin before the target
  auto staying = [&](uint32_t own, unsigned long long each, unsigned long long msum, double target) {
    if (each == 0) return own;
    const double room = (target - (double)msum) / (double)each;
    uint32_t j = room >= (double)own ? own : room > 0.0 ? (uint32_t)room : 0u;
    while (j > 0 && !((double)(msum + (unsigned long long)(j - 1) * each) < target)) --j;
    while (j < own && (double)(msum + (unsigned long long)j * each) < target) ++j;
    return j;
  };
  // Collects this row's tokens that `pred` picks, as (bits in order, ~index): larger
  // is earlier.  The number of them over the whole row; if that is at most LIST they
  // are in the blocks' `list`s, block c's ending at `upto` of lane c.
  uint32_t upto = 0;
  auto listed = [&] {  // once every block's list is complete
    upto = lane < CL ? peer(lane)->list_n : 0;
#pragma unroll
    for (int o = 1; o < MAX_CL; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t n = __shfl_sync(0xffffffffu, upto, MAX_CL - 1);
    if (n > LIST) cl.sync();  // the lists are not read further and may be begun anew
    return n;
  };
  auto list_token = [&](float x, int i) {
    const uint32_t at = atomicAdd(&sh.list_n, 1u);
    if (at < LIST) sh.list[at] = (unsigned long long)ordered(x) << 32 | ~(uint32_t)i;
  };
  auto begin_list = [&] {
    __syncthreads();
    if (tid == 0) sh.list_n = 0;
    __syncthreads();
  };
  auto collect = [&](auto&& pred) {
    begin_list();
    each_token([&](float x, int i) {
      if (pred(x)) list_token(x, i);
    });
    cl.sync();
    return listed();
  };
  // The n <= LIST collected tokens of all blocks in `keys`, the earliest first.
  auto sorted = [&](uint32_t n) {
    // (only ranked ones need no full array)
    const uint32_t size = n <= RANKED ? (n + 31) & ~31u : n <= 2 * THREADS ? 2 * THREADS : LIST;
    for (uint32_t i = tid; i < size; i += THREADS) {
      unsigned long long key = 0;  // below every token
      uint32_t c = 0, from = 0;
#pragma unroll
      for (int o = 0; o < MAX_CL; ++o) {
        const uint32_t end = __shfl_sync(0xffffffffu, upto, o);
        if (o < CL && i >= end) {
          c = o + 1;
          from = end;
        }
      }
      if (i < n) key = peer(c)->list[i - from];
      sh.keys[i] = key;
    }
    if (n <= RANKED) {
      __syncthreads();
      unsigned long long key = 0;
      uint32_t at = 0;
      if (tid < n) {
        key = sh.keys[tid];
        for (uint32_t j = 0; j < n; j += 2) {  // (an odd last one meets a 0)
          const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&sh.keys[j]);
          at += (o.x > key) + (o.y > key);
        }
      }
      __syncthreads();
      if (tid < n) sh.keys[at] = key;
      __syncthreads();
      return;
    }
    if (n <= 2 * THREADS) sort_keys<2>(sh.keys);
    else sort_keys<4>(sh.keys);
  };
  auto sorted_value = [&](uint32_t i) { return from_ordered((uint32_t)(sh.keys[i] >> 32)); };
  // The terms of the first n sorted tokens, EACH a thread, with their running sum;
  // and the number of the last one that begins before `target` (at least the first).
  constexpr int EACH = LIST / THREADS;
  auto running = [&](uint32_t n, uint64_t (&f)[EACH], unsigned long long& pm,
                     unsigned long long& total) {
    double y[EACH];
    bool have[EACH];
#pragma unroll
    for (int h = 0; h < EACH; ++h) {
      have[h] = EACH * tid + h < n && rw.distance(sorted_value(EACH * tid + h), y[h]);
      y[h] = have[h] ? y[h] : 0.0;
    }
    rw.fixed(y, have, f);
    uint32_t pn, tn;
    scan(f[0] + f[1] + f[2] + f[3], 0, pm, pn, total, tn);
  };
  auto last_before = [&](uint32_t n, const uint64_t (&f)[EACH], unsigned long long pm, double target) {
    int mine = -1;
#pragma unroll
    for (int h = 0; h < EACH; ++h) {
      const bool stays = EACH * tid + h < n && (double)pm < target;
      pm += f[h];
      if (stays && !(EACH * tid + h + 1 < n && (double)pm < target)) mine = EACH * tid + h;
    }
    return (uint32_t)max(tell(mine, 0, 0, 0, 0), 0);
  };
  auto border_at = [&](uint32_t place, Border& out) {  // after sorted token number `place`
    out.key = (uint32_t)(sh.keys[place] >> 32);
    int first = -1;  // of the equal ones
    for (uint32_t i = tid; i <= place; i += THREADS)
      if ((uint32_t)(sh.keys[i] >> 32) == out.key && (i == 0 || (uint32_t)(sh.keys[i - 1] >> 32) != out.key))
        first = (int)i;
    out.ties = place - (uint32_t)tell(first, 0, 0, 0, 0) + 1;
  };
  static_assert(EACH == 4, "sums of four");
  // Radix passes over the tokens that `member` picks (neighbours in value), before
  // which `cnt` tokens of mass `msum` lie, with digits of 8 bits from the highest bit in
  // which they differ.  by_mass: the tokens that begin before `target` stay; else
  // `k` tokens do.
  auto radix = [&](auto&& member, bool by_mass, uint32_t cnt, unsigned long long msum, double target,
                   Border& out) {
    __syncthreads();
    if (tid == 0) {
      sh.kmin = 0xffffffffu;
      sh.kmax = 0;
    }
    __syncthreads();
    uint32_t lo = 0xffffffffu, hi = 0;
    each_token([&](float x, int) {
      if (!member(x)) return;
      const uint32_t key = ordered(x);
      lo = min(lo, key);
      hi = max(hi, key);
    });
    atomicMin(&sh.kmin, lo);
    atomicMax(&sh.kmax, hi);
    cl.sync();
    lo = __reduce_min_sync(0xffffffffu, lane < CL ? peer(lane)->kmin : 0xffffffffu);
    hi = __reduce_max_sync(0xffffffffu, lane < CL ? peer(lane)->kmax : 0u);
    cl.sync();  // all have read them
    int bits = 32 - __clz(lo ^ hi), buf = 0;
    uint32_t prefix = bits >= 32 ? 0 : (hi >> bits) << bits;
    uint32_t own = 0;               // tokens equal to the key so far
    unsigned long long own_mass = 0;
    if (tid < 256) {
      sh.radix.rmass[0][tid] = 0;
      sh.radix.rcount[0][tid] = 0;
    }
    __syncthreads();
    bool first = true;
    while (bits > 0 || first) {
      first = false;
      const int shift = max(0, bits - 8);
      const uint32_t dmask = bits > 0 ? ((bits >= 32 ? 0xffffffffu : (1u << bits) - 1u) >> shift) : 0u;
      const uint32_t high = bits >= 32 ? 0u : ~((1u << bits) - 1u);
      each_token([&](float x, int) {
        if (!member(x)) return;
        const uint32_t key = ordered(x);
        if ((key & high) != (prefix & high)) return;
        const uint32_t d = dmask - ((key >> shift) & dmask);  // largest first
        atomicAdd(&sh.radix.rcount[buf][d], 1u);
        if (by_mass) atomicAdd(&sh.radix.rmass[buf][d], (unsigned long long)rw.fixed(x));
      });
      cl.sync();
      unsigned long long m = 0;
      uint32_t n = 0;
      if (tid < 256) {
        for (int c = 0; c < CL; ++c) {
          m += peer(c)->radix.rmass[buf][tid];
          n += peer(c)->radix.rcount[buf][tid];
        }
        sh.radix.rmass[buf ^ 1][tid] = 0;  // its last readers passed the sync above
        sh.radix.rcount[buf ^ 1][tid] = 0;
      }
      unsigned long long pm, tm;
      uint32_t pn, tn;
      scan(m, n, pm, pn, tm, tn);
      pm += msum;
      pn += cnt;
      // the digit that holds the k-th token, or the last one that begins before the target
      const bool mine = n > 0 && (by_mass ? (double)pm < target && !((double)(pm + m) < target)
                                          : pn < k && pn + n >= k);
      const int d = max(tell(mine ? tid : -1, pn, pm, n, m), 0);
      cnt = sh.found_count;
      msum = sh.found_mass;
      own = sh.found_own;
      own_mass = sh.found_own_mass;
      prefix = (prefix & high) | ((dmask - (uint32_t)d) << shift);
      buf ^= 1;
      bits = shift;
    }
    cl.sync();  // the buffers are read: a later call may use their place
    out.key = prefix;
    out.ties = by_mass ? staying(own, own ? own_mass / own : 0, msum, target) : min(own, k - cnt);
  };

  int direct = -1;  // the kept tokens are the sorted list up to this one
  if (by_k || by_p) {
    // this thread's bin over the whole row: tokens, and the least that its sum can be
    // (count * 2^-((bin + 1) / 11), with room for roundings)
    uint32_t hc = 0, bc, total_c;
    unsigned long long bm, tm;
#pragma unroll
    for (int c = 0; c < MAX_CL; ++c)
      if (c < CL) hc += peer(c)->count[tid];
    const unsigned long long least = (unsigned long long)(
        hc * (double)exp2f(-((float)tid + 1.01f) / 11.f) * 0.9999 * rw.scale);
    scan(least, hc, bm, bc, tm, total_c);
    const bool cut_k = by_k && total_c > k;
    if (by_k && !cut_k && by_p) {  // fewer tokens than k: top-p over all of them
      sum_terms();
      cl.sync();
    }
    unsigned long long z = 0;  // mass that top-k leaves
    double target = 0.0;
    if (by_p && !cut_k) {
      if (warp == 0) {
#pragma unroll
        for (int i = 0; i < MAX_CL * WARPS / 32; ++i)
          if (32 * i + lane < CL * WARPS)
            z += peer((32 * i + lane) / WARPS)->wmass[(32 * i + lane) % WARPS];
        z = warp_sum64(z);
      }
      tell(tid == 0 ? 0 : -1, 0, z, 0, 0);
      z = sh.found_mass;
      target = fmax(p, 0.0) * (double)z;
    }
    // the bin down to which a border can lie that matters (min-p leaves nothing
    // below its own), and the tokens down to there
    int limit = -1;
    uint32_t through = 0;
    if (cut_k) {
      limit = tell(bc < k && bc + hc >= k ? tid : -1, bc, 0, bc + hc, 0);
      through = sh.found_own;
    } else if (by_p) {
      limit = tell((double)bm < target && !((double)(bm + least) < target) ? tid : -1, 0, 0, bc + hc, 0);
      through = sh.found_own;
      if (limit < 0) {
        limit = BINS - 2;
        through = total_c;
      }
    }
    const uint32_t k_before = sh.found_count;  // with cut_k: tokens of the bins before
    const int floor_bin = by_min ? (int)fmin(floor_y * 11.0 + 0.01, BINS - 2.0) : BINS - 2;
    // (top-p after top-k needs the mass of all k, though)
    bool k_border = cut_k;  // `limit` is the k-th token's bin: top-k has a border to find
    if (limit > floor_bin && !(cut_k && by_p)) {
      tell(tid == floor_bin ? tid : -1, 0, 0, bc + hc, 0);
      // worth it where it makes the list short.  All that min-p keeps then lies in bins
      // before the k-th token's, so that top-k takes nothing of it
      if (sh.found_own <= LIST) {
        limit = floor_bin;
        through = sh.found_own;
        k_border = false;
      }
    }
    if (limit >= 0) {
      uint32_t n = LIST + 1;
      if (through <= LIST) {
        // the value down to which to collect, a little too far rather than too short
        const float d = ((float)limit + 1.f) * 1.0001f / (11.f * cf);
        float thr = mx;
        if (mx < INFINITY) {
          thr = mx - d;
          if (thr > -INFINITY) thr -= fabsf(thr) * 3e-7f;
        }
        n = collect([&](float x) { return x >= thr && x > -INFINITY; });
      }
      if (n <= LIST) {
        sorted(n);
        const uint32_t nk = cut_k ? min(k, n) : n;  // (min-p may have made the list shorter than k)
        uint32_t place = nk - 1;
        if (by_p) {
          uint64_t f[EACH];
          unsigned long long pm, total;
          running(nk, f, pm, total);
          if (cut_k) target = fmax(p, 0.0) * (double)total;
          place = last_before(nk, f, pm, target);
        }
        if (place < DIRECT) {
          direct = (int)place;
        } else {
          border_at(place, border);
        }
      } else {
        // (a list shortened by min-p can be too long all the same: it reaches a little
        // past its bin, where many equal logits may lie)
        if (k_border) {
          n = collect([&](float x) { return bin_of(x) == limit; });
          if (n <= LIST) {
            sorted(n);
            border_at(k - k_before - 1, border);
          } else {
            radix([&](float x) { return bin_of(x) == limit; }, false, k_before, 0, 0.0, border);
          }
        }
        if (by_p) {
          const uint32_t above = cut_k ? border.key : 0u;
          const unsigned long long each = cut_k ? rw.fixed(from_ordered(border.key)) : 0;
          auto add_up = [&](uint64_t mine) {  // over the row
            mine = warp_sum64(mine);
            if (lane == 0) sh.wmass[warp] = mine;
            cl.sync();
            unsigned long long all = 0;
            if (warp == 0) {
#pragma unroll
              for (int i = 0; i < MAX_CL * WARPS / 32; ++i)
                if (32 * i + lane < CL * WARPS)
                  all += peer((32 * i + lane) / WARPS)->wmass[(32 * i + lane) % WARPS];
              all = warp_sum64(all);
            }
            tell(tid == 0 ? 0 : -1, 0, all, 0, 0);
            return sh.found_mass;
          };
          if (cut_k) {  // what top-k left
            uint64_t mine = 0;
            each_token([&](float x, int) {
              if (x > -INFINITY && ordered(x) > above) mine += rw.fixed(x);
            });
            target = fmax(p, 0.0) * (double)(add_up(mine) + border.ties * each);
          }
          cl.sync();  // wmass is read and may be written again
          // Where the border is likely to be: the bins' sums estimated halfway between
          // their bounds, a bin's tokens spread evenly; up and down from there 0.25 % of the
          // target, but at least 200 tokens and at most 800.  One pass adds up what lies
          // before and collects what lies there: a flat row of 128256 bf16 tokens takes 32
          // to 40 us, by the cells below 45 to 62.  Not found there, it is looked for so.
          bool found = false;
          if (!cut_k && rw.plain) {
            const unsigned long long most = (unsigned long long)(
                hc * (double)exp2f(-((float)tid - 0.01f) / 11.f) * 1.0001 * rw.scale);
            const unsigned long long half = least / 2 + most / 2;
            unsigned long long pe, te;
            uint32_t pn, tn;
            scan(half, 0, pe, pn, te, tn);
            const double ratio = (double)z / (double)te;
            const double b = (double)pe * ratio, e = (double)(pe + half) * ratio;
            auto place = [&](double t, float otherwise) {  // depth at which the sum should be t
              const bool mine = b < t && !(e < t);
              const int bin = tell(mine ? tid : -1, 0, mine ? (unsigned long long)__double_as_longlong((t - b) / (e - b)) : 0, 0, 0);
              return bin < 0 ? otherwise : (float)bin + (float)__longlong_as_double((long long)sh.found_mass);
            };
            const double about = exp2f(place(target, (float)(BINS - 1)) / -11.f) * rw.scale;  // a term there
            const double off = fmin(fmax(0.0025 * target, 200.0 * about), 800.0 * about);
            const float from = place(target - off, 0.f), to = place(target + off, (float)(BINS - 1));
            begin_list();
            uint64_t before = 0;
            each_unit([&](const float (&x)[VEC], int i) {
#pragma unroll
              for (int h = 0; h < VEC; h += 4) {
                float v[4];
                bool any = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float d = depth(x[h + e]);
                  v[e] = d < from ? x[h + e] : rw.low;
                  any |= d < from;
                  if (d >= from && d < to) list_token(x[h + e], i + h + e);
                }
                if (any) before += rw.sum4(v);
              }
            });
            const unsigned long long base = add_up(before);
            n = listed();
            if (n <= LIST) {
              sorted(n);
              uint64_t f[EACH];
              unsigned long long pm, total;
              running(n, f, pm, total);
              found = (double)base < target && !((double)(base + total) < target);
              if (found) border_at(last_before(n, f, pm + base, target), border);
              cl.sync();  // the lists are read, as is wmass
            }
          }
          if (!found) {
            // the first bin by whose end the sum can have reached the target: a bin's sum
            // is at most its count times its largest e
            const unsigned long long most = (unsigned long long)(
                hc * (double)exp2f(-((float)tid - 0.01f) / 11.f) * 1.0001 * rw.scale) + hc;
            unsigned long long pm;
            uint32_t pn, tn;
            scan(most, 0, pm, pn, tm, tn);
            const int low =
                max(tell((double)pm < target && !((double)(pm + most) < target) ? tid : -1, 0, 0, 0, 0), 0);
            // one pass: the sum of what lies before bin `low`, and of each of 512 cells
            // between there and bin `limit`
            const float split = (float)max(1, BINS / max(1, limit + 1 - min(low, limit)));
            const float first_depth = (float)min(low, limit), end_depth = (float)(limit + 1);
            auto cell = [&](float x) {  // -1 before, BINS behind
              const float d = depth(x);
              if (!(d < end_depth) || (cut_k && ordered(x) <= above)) return BINS;
              return d < first_depth ? -1 : min(BINS - 1, (int)((d - first_depth) * split));
            };
            uint64_t before = 0;
            each_unit([&](const float (&x)[VEC], int) {
#pragma unroll
              for (int h = 0; h < VEC; h += 4) {
                double y[4];
                bool have[4];
                int c[4];
                uint64_t f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  c[e] = cell(x[h + e]);
                  have[e] = c[e] < BINS && rw.distance(x[h + e], y[e]);
                  y[e] = have[e] ? y[e] : 0.0;
                }
                if (!(have[0] || have[1] || have[2] || have[3])) continue;
                rw.fixed(y, have, f);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if (!have[e]) continue;
                  if (c[e] < 0) {
                    before += f[e];
                  } else {  // (64-bit additions here took 5 times as long)
                    const uint32_t mask = (1u << a.limb) - 1u;
                    atomicAdd(&sh.mass[0][c[e]], (uint32_t)f[e] & mask);
                    atomicAdd(&sh.mass[1][c[e]], (uint32_t)(f[e] >> a.limb) & mask);
                    atomicAdd(&sh.mass[2][c[e]], (uint32_t)(f[e] >> 2 * a.limb));
                  }
                }
              }
            });
            const unsigned long long base = add_up(before);
            unsigned long long hm = 0;
#pragma unroll
            for (int c = 0; c < MAX_CL; ++c)
              if (c < CL) {
                const Shared* o = peer(c);
                hm += o->mass[0][tid] + ((unsigned long long)o->mass[1][tid] << a.limb) +
                      ((unsigned long long)o->mass[2][tid] << 2 * a.limb);
              }
            scan(hm, 0, pm, pn, tm, tn);
            pm += base;
            // the last cell that begins before the target
            const int fc = tell((double)pm < target && !((double)(pm + hm) < target) ? tid : -1, 0, pm, 0, 0);
            const unsigned long long msum = sh.found_mass;
            if (fc >= 0) {
              auto member = [&](float x) { return cell(x) == fc; };
              n = collect(member);
              if (n <= LIST) {
                sorted(n);
                uint64_t f[EACH];
                unsigned long long total;
                running(n, f, pm, total);
                border_at(last_before(n, f, pm + msum, target), border);
              } else {
                radix(member, true, 0, msum, target, border);
              }
            } else {
              if (cut_k) border.ties = staying(border.ties, each, base + tm, target);  // among equal ones
              cl.sync();  // as above
            }
          }
        }
      }
    }
    // p = 0, or sums that leave the first token alone
    if (by_p && !(target > 0.0)) {
      border = Border{ordered(mx), 1};
      direct = -1;
    }
  }

  // A short list of kept tokens is all that the draw needs: block 0 adds up, for
  // each of them, the terms of those with a smaller index.
  if (direct >= 0) {
    // nothing more is read from another block: one may leave when all are here
    auto here = cl.barrier_arrive();
    if (rank == 0) {
      const uint32_t n = (uint32_t)direct + 1;
      double y = 0.0;
      uint32_t index = 0;
      uint64_t f = 0;
      if (tid < n) {
        const float x = sorted_value(tid);
        index = ~(uint32_t)sh.keys[tid];
        if (rw.distance(x, y) && !(by_min && y > floor_y)) f = rw.fixed(x);
      }
      if (tid < DIRECT) {
        sh.term[tid] = f;
        sh.index[tid] = index;
      }
      __syncthreads();
      uint64_t before = 0, W = 0;
      uint32_t latest = 0;
      for (uint32_t j = 0; j < n; ++j) {
        const uint64_t t = sh.term[j];
        const uint32_t o = sh.index[j];
        W += t;
        before += o < index ? t : 0;
        if (t > 0) latest = max(latest, o);
      }
      const double want = u * (double)W;
      // the one that passes u W, or for u of 1 or more the last
      const bool passes = (before == 0 || !((double)before > want)) && (double)(before + f) > want;
      if (f > 0 && (passes || (index == latest && !((double)W > want)))) {
        a.tokens[r] = index;
        if (a.logprobs)
          a.logprobs[r] = (float)(-y * 0.69314718055994530942 - log((double)W / a.scale));
      }
    }
    cl.barrier_wait(std::move(here));
    return;
  }

  // ---- 4. what is kept, per warp
  const bool filtered = border.key != 0 || by_min || by_k;
  const float border_value = border.key != 0 ? from_ordered(border.key) : -INFINITY;
  auto kept = [&](float l, double& y, bool& tie) {
    tie = l == border_value;
    return l >= border_value && rw.distance(l, y) && !(by_min && y > floor_y);
  };
  if (filtered) {
    uint64_t sum = 0;
    uint32_t ties = 0;
    each_unit([&](const float (&x)[VEC], int) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < VEC; ++e) any |= x[e] >= border_value;
      if (!any) return;
      if (rw.plain && !by_min) {
#pragma unroll
        for (int h = 0; h < VEC; h += 4) {
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool tie = x[h + e] == border_value && border.key != 0;
            ties += tie;
            v[e] = x[h + e] >= border_value && !tie ? x[h + e] : rw.low;
          }
          sum += rw.sum4(v);
        }
        return;
      }
#pragma unroll
      for (int h = 0; h < VEC; h += 4) {
        double y[4];
        bool have[4];
        uint64_t f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          bool tie;
          have[e] = kept(x[h + e], y[e], tie);
          if (have[e] && tie && border.key != 0) {
            ++ties;
            have[e] = false;
          }
          y[e] = have[e] ? y[e] : 0.0;
        }
        if (!(have[0] || have[1] || have[2] || have[3])) continue;
        rw.fixed(y, have, f);
        sum += f[0] + f[1] + f[2] + f[3];
      }
    });
    sum = warp_sum64(sum);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) {
      sh.wmass[warp] = sum;
      sh.wties[warp] = ties;
    }
    cl.sync();
  }

  // ---- 5. the draw: warp 0 of every block finds which of the cluster's warps,
  // in order, passes u W (or is the last with any mass)
  uint64_t each = 0;  // term of a token equal to the border
  if (border.key != 0) each = rw.fixed(from_ordered(border.key));
  if (tid < CL * WARPS) {
    const Shared* o = cl.map_shared_rank(&sh, tid / WARPS);
    sh.all_mass[tid] = o->wmass[tid % WARPS];
    sh.all_ties[tid] = o->wties[tid % WARPS];
  }
  __syncthreads();
  if (warp == 0) {
    constexpr int PER = MAX_CL * WARPS / 32;
    uint32_t t[PER], nt = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = lane * PER + i;
      t[i] = at < CL * WARPS ? sh.all_ties[at] : 0;
      nt += t[i];
    }
    uint32_t it = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, it, o);
      if (lane >= o) it += v;
    }
    const uint32_t total_ties = __shfl_sync(0xffffffffu, it, 31);
    uint32_t tie_at = it - nt;
    uint64_t m[PER], nm = 0;
    uint32_t tb[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = lane * PER + i;
      tb[i] = tie_at;
      const uint32_t take = min(t[i], border.ties - min(border.ties, tie_at));
      tie_at += t[i];
      m[i] = at < CL * WARPS ? sh.all_mass[at] + take * each : 0;
      nm += m[i];
    }
    uint64_t im = nm;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t v = __shfl_up_sync(0xffffffffu, im, o);
      if (lane >= o) im += v;
    }
    const uint64_t W = __shfl_sync(0xffffffffu, im, 31);
    const double want = u * (double)W;
    uint64_t before = im - nm;
    int hit = -1, lst = -1;
    uint64_t bhit = 0, blst = 0;
    uint32_t thit = 0, tlst = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (m[i] > 0) {
        lst = lane * PER + i;
        blst = before;
        tlst = tb[i];
        if (hit < 0 && (double)(before + m[i]) > want) {
          hit = lst;
          bhit = before;
          thit = tb[i];
        }
      }
      before += m[i];
    }
    const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0);
    const uint32_t any = __ballot_sync(0xffffffffu, lst >= 0);
    if (lane == (hits ? __ffs(hits) - 1 : 31 - __clz(any))) {
      sh.pick_warp = hits ? hit : lst;
      sh.pick_before = hits ? bhit : blst;
      sh.pick_ties = hits ? thit : tlst;
      sh.pick_total = W;
      sh.pick_all_ties = total_ties;
    }
  }
  __syncthreads();
  const int target_warp = sh.pick_warp;
  const uint64_t mine_before = sh.pick_before, W = sh.pick_total;
  const uint32_t my_tie_base = sh.pick_ties;
  const double want = u * (double)W;
  // nothing more is read from another block: one may leave when all are here
  auto here = cl.barrier_arrive();
  // The block that has it: a thread per unit of that warp's part, in order.
  if (target_warp / WARPS == rank) {
    const int q0 = warp_begin(target_warp % WARPS), q1 = warp_begin(target_warp % WARPS + 1);
    uint64_t run = mine_before;
    uint32_t seen = my_tie_base;
    for (int qb = q0; qb < q1; qb += THREADS) {
      const int q = qb + tid;
      float x[VEC];
      uint64_t f[VEC];
      double ys[VEC];
      uint32_t tie_bits = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = __uint_as_float(0x7fc00000u);
      if (q < q1) un.values(unit(q), x);
#pragma unroll
      for (int h = 0; h < VEC; h += 4) {
        double y[4];
        bool have[4];
        uint64_t g[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          bool tie;
          have[e] = kept(x[h + e], ys[h + e], tie);
          y[e] = have[e] ? ys[h + e] : 0.0;
          if (have[e] && tie) tie_bits |= 1u << (h + e);
        }
        rw.fixed(y, have, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[h + e] = g[e];
      }
      unsigned long long pm, tm;
      uint32_t pn, tn;
      if (border.key != 0 && sh.pick_all_ties > border.ties) {
        // of the tokens equal to the border only the first stay
        scan(0, __popc(tie_bits), pm, pn, tm, tn);
        pn += seen;
        seen += tn;
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (tie_bits >> e & 1) {
            if (pn >= border.ties) f[e] = 0;
            ++pn;
          }
      }
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum += f[e];
      scan(sum, 0, pm, pn, tm, tn);
      uint64_t acc = run + pm;
      run += tm;
      int hit = -1, lst = -1;
      double yhit = 0.0, ylst = 0.0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (f[e] == 0) continue;
        acc += f[e];
        lst = q * VEC - un.shift + e;
        ylst = ys[e];
        if (hit < 0 && (double)acc > want) {
          hit = lst;
          yhit = ylst;
        }
      }
      // the first that passes u W: sums only grow, so it is the one whose
      // predecessor does not
      if (hit >= 0 && (acc == sum || !((double)(acc - sum) > want))) {
        sh.hit = hit;
        sh.hit_y = yhit;
      }
      const uint32_t any = __ballot_sync(0xffffffffu, lst >= 0);
      if (any && lane == 31 - __clz(any)) atomicMax(&sh.last, lst);
      __syncthreads();
      if (lst >= 0 && lst == sh.last) sh.last_y = ylst;
      __syncthreads();
      if (sh.hit >= 0) break;
    }
    if (tid == 0) {
      const bool have = sh.hit >= 0;  // u of 1 or more: the last kept token
      a.tokens[r] = have ? sh.hit : sh.last;
      if (a.logprobs) {
        // log of (e / W) with e from its exponent: no digits of a small term are lost
        const double lw = log((double)W / a.scale);
        a.logprobs[r] = (float)(-(have ? sh.hit_y : sh.last_y) * 0.69314718055994530942 - lw);
      }
    }
  }
  cl.barrier_wait(std::move(here));
}

template <typename T>
int run(const Args& a, cudaStream_t st) {
  // Blocks of a row: as many as leave each at least 2048 tokens while the row's
  // blocks do not fill half the slots (two to an SM); beyond that, as many as fill
  // them once, with at least 6144 tokens each: larger clusters spend their time in
  // the exchanges between blocks.  More only where the rows that run at once would
  // not stay in L2 for the second pass.  256 x 128256 bf16, top-k 50 and top-p 0.95:
  // 126 us by clusters of 8, 85 by 4, 75 by 2, 65 by 1; float32: 138, 110, 93, 118;
  // 48 rows bf16: 30, 23, 29, 29.  (And no block more than 131000: see a.limb.)
  int cluster = 1;
  const auto rows_at_once = [&] { return std::min<int64_t>(a.rows, 2 * sm_count() / cluster); };
  while (cluster < MAX_CL && a.vocab >= 4096 * cluster &&
         (a.vocab > 131000 * cluster || a.rows * cluster * 2 <= sm_count() ||
          (a.vocab >= 12288 * cluster && a.rows * cluster <= sm_count()) ||
          rows_at_once() * a.vocab * (int64_t)sizeof(T) > (96 << 20)))
    cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * cluster));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  // a block's part of the row, in units of 16 bytes (one more where they do not divide)
  const int64_t part = (ceil_div(ceil_div(a.vocab, (int64_t)(16 / sizeof(T))) + 1, cluster) + 1) * 16;
  cudaError_t e;
  if (part <= MAX_STAGE + 256) {
    static std::atomic<uint64_t> ready{0};  // devices on which the attribute is set
    int dev = 0;
    GQ_CHECK_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (dev > 63 || !(ready.load(std::memory_order_acquire) & bit)) {
      GQ_CHECK_CUDA(cudaFuncSetAttribute(sample_kernel<T, true>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_STAGE + 256));
      ready.fetch_or(bit, std::memory_order_release);
    }
    cfg.dynamicSmemBytes = (size_t)part;
    e = cudaLaunchKernelEx(&cfg, sample_kernel<T, true>, a);
  } else {
    e = cudaLaunchKernelEx(&cfg, sample_kernel<T, false>, a);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(GQ_ECUDA, "gq_sample: %s", cudaGetErrorString(e));
  }
  return check_launch("gq_sample");
}

}  // namespace samp
}  // namespace gq

extern "C" int gq_sample(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld,
                         const void* u, int u_kind, const void* temperature, int temperature_kind,
                         double temperature_value, const void* top_k, int top_k_kind,
                         double top_k_value, const void* top_p, int top_p_kind, double top_p_value,
                         const void* min_p, int min_p_kind, double min_p_value, int64_t* tokens,
                         float* logprobs, void* stream) {
  using namespace gq;
  GQ_REQUIRE(dtype >= 0 && dtype <= 2, "gq_sample: dtype must be 0 (float32), 1 (bf16) or 2 (fp16)");
  GQ_REQUIRE(rows >= 0 && vocab >= 1 && ld >= vocab, "gq_sample: bad shape");
  GQ_REQUIRE(vocab <= (1 << 20), "gq_sample: at most 2^20 tokens in the vocabulary");
  GQ_REQUIRE(rows < (1ll << 27), "gq_sample: too many rows");
  GQ_REQUIRE(u_kind == 1 || u_kind == 2, "gq_sample: u must be float32 or float64, one per row");
  samp::Args a;
  a.u = {u, u_kind, 0.0};
  a.temperature = {temperature, temperature_kind, temperature_value};
  a.top_k = {top_k, top_k_kind, top_k_value};
  a.top_p = {top_p, top_p_kind, top_p_value};
  a.min_p = {min_p, min_p_kind, min_p_value};
  for (const samp::RowParam* s : {&a.temperature, &a.top_k, &a.top_p, &a.min_p}) {
    GQ_REQUIRE(s->kind >= 0 && s->kind <= 4, "gq_sample: bad kind of a setting");
    GQ_REQUIRE(s->kind == 0 || s->rows != nullptr || rows == 0, "gq_sample: NULL setting");
  }
  if (rows == 0) return GQ_OK;
  GQ_REQUIRE(logits != nullptr && u != nullptr && tokens != nullptr, "gq_sample: NULL buffer");
  a.logits = logits;
  a.ld = ld;
  a.rows = rows;
  a.vocab = (int)vocab;
  a.tokens = tokens;
  a.logprobs = logprobs;
  int log2v = 0;
  while ((1ll << log2v) < vocab) ++log2v;
  const int bits = std::min(45, 62 - log2v);  // S: a term has S + 1 bits
  a.scale = (double)(1ll << bits);
  // The low limbs are below 2^limb, the high one at most 2^(S - 2 limb): 15 bits for S
  // from 43 to 45, at most 131000 tokens a block (run() sees to that); 14 for S = 42
  // (2^20 tokens in 8 blocks).  Either way a block's sum of one stays below 2^32.
  a.limb = (bits + 2) / 3;
  cudaStream_t st = as_stream(stream);
  if (dtype == 0) return samp::run<float>(a, st);
  if (dtype == 1) return samp::run<__nv_bfloat16>(a, st);
  return samp::run<__half>(a, st);
}
