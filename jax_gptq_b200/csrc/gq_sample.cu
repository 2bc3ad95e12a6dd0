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
// Temperature 0 (or below, or NaN) is the first largest logit.  A row without
// any token gives -1 and -inf.
//
// Sums.  The choice turns on sums that lie next to a border, so e is computed
// in float64 and held as a whole number of 2^-S (S = 45 for up to 2^17 tokens):
// sums of whole numbers do not depend on the order of additions, so the shared
// memory atomics and the split over threads and blocks never change a result,
// and a term's rounding (2^-46 of the largest) is far below what a float32
// uniform resolves.  Terms below 2^-(S+1) are zero: they can not be drawn.
//
// Split.  A cluster of blocks takes a row, each a contiguous part, each warp a
// contiguous part of that.  Passes over the row (it stays in L1 and L2):
//   1. the maximum;
//   2. each warp's sum of e, and with top-k or top-p a histogram (count and
//      sum) over 512 bins of log2 e;
//   3. only with a border: the bin it falls in is resolved exactly by radix
//      passes over the ordered bits of its members;
//   4. only with filters: each warp's sum of the kept e and its number of
//      tokens equal to the border;
//   5. the warp whose part holds u W finds the token.
#include "gq_common.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace gq {
namespace samp {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int BINS = 512;
constexpr int MAX_CL = 8;
constexpr int LIST = 1024;  // members of a border's bin kept per block

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

// 2^-y for 0 <= y < 1000, within 2^-48: y is split at the nearest whole number
// and 2^f, |f| <= 1/2, is the Taylor series of exp(f ln 2) to the 11th power
// (remainder below 7e-15).
__device__ __forceinline__ double exp2_neg(double y) {
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the whole part
  const double s = magic - y;
  const int n = __double2loint(s);
  const double x = ((magic - s) - y) * 0.69314718055994530942;
  double p = 2.505210838544172e-08;                // 1 / 11!
  p = fma(p, x, 2.755731922398589e-07);
  p = fma(p, x, 2.755731922398589e-06);
  p = fma(p, x, 2.48015873015873e-05);
  p = fma(p, x, 1.984126984126984e-04);
  p = fma(p, x, 1.388888888888889e-03);
  p = fma(p, x, 8.333333333333333e-03);
  p = fma(p, x, 4.1666666666666664e-02);
  p = fma(p, x, 1.6666666666666666e-01);
  p = fma(p, x, 0.5);
  p = fma(p, x, 1.0);
  p = fma(p, x, 1.0);
  return __hiloint2double(__double2hiint(p) + (n << 20), __double2loint(p));
}

struct Row {
  double mx, c;  // the maximum, log2(e) / temperature
  double limit;  // terms with log2 e below -limit are zero
  double scale;
  // distance below the maximum in powers of two; false where the term is zero
  __device__ __forceinline__ bool distance(float l, double& y) const {
    const double v = (double)l;
    y = v == mx ? 0.0 : (mx - v) * c;
    return y < limit;  // false for NaN
  }
  __device__ __forceinline__ uint64_t fixed(double y) const {
    const double t = fma(exp2_neg(y), scale, 4503599627370496.0);  // + 2^52: whole number in the low bits
    return (uint64_t)__double_as_longlong(t) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ int bin(double y) const {
    return min(BINS - 1, (int)((float)y * 11.f));  // 46.5 powers of two
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
  // NaN where there is no element
  __device__ __forceinline__ void load(int q, float (&x)[VEC]) const {
    const int i0 = q * VEC - shift;
    if (i0 >= 0 && i0 + VEC <= vocab) {
      struct alignas(16) Pack { T e[VEC]; };
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + i0));
      Pack p;
      memcpy(&p, &raw, 16);
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = to_f<T>(p.e[e]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        x[e] = (i0 + e >= 0 && i0 + e < vocab) ? to_f<T>(row[i0 + e]) : __uint_as_float(0x7fc00000u);
    }
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
  unsigned long long mass[BINS];       // histogram over log2 e
  uint32_t count[BINS];
  unsigned long long rmass[2][256];    // a radix pass, two buffers in turn
  uint32_t rcount[2][256];
  uint64_t wmass[WARPS];               // per warp: what the draw walks through
  uint32_t wties[WARPS];
  uint32_t list[LIST];
  uint32_t list_n, kmin, kmax;
  float mx[WARPS];
  uint32_t amax[WARPS];
  // scratch of the scans over bins and digits
  unsigned long long smass[WARPS];
  uint32_t scount[WARPS];
  float block_max;
  uint32_t block_arg;
  unsigned long long all_mass[MAX_CL * WARPS];  // every warp of the cluster
  uint32_t all_ties[MAX_CL * WARPS];
  int pick_warp;
  uint32_t pick_ties;
  unsigned long long pick_before, pick_total;
  int found;
  uint32_t found_count;
  unsigned long long found_mass;
  uint32_t found_own;
  unsigned long long found_own_mass;
};

template <typename T>
__global__ void __launch_bounds__(THREADS) sample_kernel(Args a) {
  constexpr int VEC = Units<T>::VEC;
  __shared__ Shared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int CL = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t r = blockIdx.x / CL;
  const T* row = static_cast<const T*>(a.logits) + r * a.ld;
  const Units<T> un(row, a.vocab);
  // this warp's units
  const int b0 = (int)((int64_t)un.count * rank / CL), b1 = (int)((int64_t)un.count * (rank + 1) / CL);
  const int w0 = b0 + (int)((int64_t)(b1 - b0) * warp / WARPS);
  const int w1 = b0 + (int)((int64_t)(b1 - b0) * (warp + 1) / WARPS);

  const double temp = row_value(a.temperature, r);
  const double kd = row_value(a.top_k, r);
  const double p = row_value(a.top_p, r);
  const double mp = row_value(a.min_p, r);
  const double u = row_value(a.u, r);

  // ---- 1. the maximum (and for temperature 0 its first index)
  float mx = -INFINITY;
  uint32_t arg = 0xffffffffu;
  for (int q = w0 + lane; q < w1; q += 32) {
    float x[VEC];
    un.load(q, x);
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (x[e] > mx) {  // indices grow along a lane's walk: the first one stays
        mx = x[e];
        arg = (uint32_t)(q * VEC - un.shift + e);
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
  for (int i = tid; i < BINS; i += THREADS) {
    sh.mass[i] = 0;
    sh.count[i] = 0;
  }
  if (tid < 256) {
    sh.rmass[0][tid] = 0;
    sh.rcount[0][tid] = 0;
  }
  if (tid == 0) {
    sh.list_n = 0;
    sh.kmin = 0xffffffffu;
    sh.kmax = 0;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < WARPS; ++w)
      if (sh.mx[w] > mx || (sh.mx[w] == mx && sh.amax[w] < arg)) {
        mx = sh.mx[w];
        arg = sh.amax[w];
      }
    sh.block_max = mx;
    sh.block_arg = arg;
  }
  cl.sync();
  mx = -INFINITY;
  arg = 0xffffffffu;
  for (int c = 0; c < CL; ++c) {
    const Shared* o = cl.map_shared_rank(&sh, c);
    const float om = o->block_max;
    const uint32_t oa = o->block_arg;
    if (om > mx || (om == mx && oa < arg)) {
      mx = om;
      arg = oa;
    }
  }
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
  rw.c = fmin(1.4426950408889634 / temp, 1e300);
  rw.scale = a.scale;
  rw.limit = (double)(((__double2hiint(a.scale) >> 20) & 0x7ff) - 1023) + 1.0;  // S + 1
  const bool by_k = kd >= 1.0 && kd < (double)a.vocab;
  const uint32_t k = by_k ? (uint32_t)kd : 0;
  const bool by_p = p < 1.0;
  const bool by_min = mp > 0.0;
  const double floor_e = fmin(mp, 1.0);  // the largest term stays whatever min_p is

  // ---- 2. sums and histogram
  {
    uint64_t sum = 0;
    const bool hist = by_k || by_p;
    for (int q = w0 + lane; q < w1; q += 32) {
      float x[VEC];
      un.load(q, x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        double y;
        if (!rw.distance(x[e], y)) continue;
        const uint64_t f = rw.fixed(y);
        sum += f;
        if (hist) {
          const int b = rw.bin(y);
          atomicAdd(&sh.mass[b], (unsigned long long)f);
          atomicAdd(&sh.count[b], 1u);
        }
      }
    }
    sum = warp_sum64(sum);
    if (lane == 0) {
      sh.wmass[warp] = sum;
      sh.wties[warp] = 0;
    }
  }
  cl.sync();

  // ---- 3. borders
  Border border{0, 0xffffffffu};  // everything
  if (by_k || by_p) {
    unsigned long long hm = 0;  // this thread's bin over the whole row
    uint32_t hc = 0;
    for (int c = 0; c < CL; ++c) {
      const Shared* o = cl.map_shared_rank(&sh, c);
      hm += o->mass[tid];
      hc += o->count[tid];
    }
    // exclusive prefixes over bins (the largest e first)
    auto scan = [&](unsigned long long m, uint32_t n, int width, unsigned long long& pm, uint32_t& pn) {
      unsigned long long im = m;
      uint32_t in = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long tm = __shfl_up_sync(0xffffffffu, im, o);
        const uint32_t tn = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) {
          im += tm;
          in += tn;
        }
      }
      __syncthreads();
      if (lane == 31) {
        sh.smass[warp] = im;
        sh.scount[warp] = in;
      }
      __syncthreads();
      pm = im - m;
      pn = in - n;
      for (int w = 0; w < warp; ++w) {
        pm += sh.smass[w];
        pn += sh.scount[w];
      }
    };
    unsigned long long bm, total_m = 0;
    uint32_t bc, total_c = 0;
    scan(hm, hc, BINS, bm, bc);
    for (int w = 0; w < WARPS; ++w) {
      total_m += sh.smass[w];
      total_c += sh.scount[w];
    }
    int buf = 0;
    // The key at which the border lies inside bin `fb`, before which `cnt`
    // tokens of mass `msum` lie.  by_mass: the first token whose preceding mass
    // reaches `target` is the first one out; else `k` tokens stay.
    auto resolve = [&](bool by_mass, int fb, uint32_t cnt, unsigned long long msum, double target,
                       Border& out, unsigned long long& kept_mass) {
      if (tid == 0) {
        sh.list_n = 0;
        sh.kmin = 0xffffffffu;
        sh.kmax = 0;
      }
      __syncthreads();
      uint32_t lo = 0xffffffffu, hi = 0;
      for (int q = w0 + lane; q < w1; q += 32) {
        float x[VEC];
        un.load(q, x);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          double y;
          if (!rw.distance(x[e], y) || rw.bin(y) != fb) continue;
          const uint32_t key = ordered(x[e]);
          lo = min(lo, key);
          hi = max(hi, key);
          const uint32_t at = atomicAdd(&sh.list_n, 1u);
          if (at < LIST) sh.list[at] = key;
        }
      }
      lo = __reduce_min_sync(0xffffffffu, lo);
      hi = __reduce_max_sync(0xffffffffu, hi);
      if (lane == 0) {
        atomicMin(&sh.kmin, lo);
        atomicMax(&sh.kmax, hi);
      }
      cl.sync();
      for (int c = 0; c < CL; ++c) {
        const Shared* o = cl.map_shared_rank(&sh, c);
        lo = min(lo, o->kmin);
        hi = max(hi, o->kmax);
      }
      const bool listed = sh.list_n <= LIST;
      const int members = listed ? (int)sh.list_n : 0;
      // digits of 8 bits from the highest bit in which the members differ
      int bits = 32 - __clz(lo ^ hi);
      uint32_t prefix = bits >= 32 ? 0 : (hi >> bits) << bits;
      uint32_t own = 0;               // tokens equal to the key so far
      unsigned long long own_mass = 0;
      bool first = true;
      while (bits > 0 || first) {
        first = false;
        const int shift = max(0, bits - 8);
        const uint32_t dmask = bits > 0 ? ((bits >= 32 ? 0xffffffffu : (1u << bits) - 1u) >> shift) : 0u;
        const uint32_t high = bits >= 32 ? 0u : ~((1u << bits) - 1u);
        auto put = [&](uint32_t key, uint64_t f) {
          const uint32_t d = dmask - ((key >> shift) & dmask);  // largest first
          atomicAdd(&sh.rcount[buf][d], 1u);
          atomicAdd(&sh.rmass[buf][d], (unsigned long long)f);
        };
        if (listed) {
          for (int i = tid; i < members; i += THREADS) {
            const uint32_t key = sh.list[i];
            if ((key & high) != (prefix & high)) continue;
            double y;
            rw.distance(from_ordered(key), y);
            put(key, rw.fixed(y));
          }
        } else {
          for (int q = w0 + lane; q < w1; q += 32) {
            float x[VEC];
            un.load(q, x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              double y;
              if (!rw.distance(x[e], y) || rw.bin(y) != fb) continue;
              const uint32_t key = ordered(x[e]);
              if ((key & high) == (prefix & high)) put(key, rw.fixed(y));
            }
          }
        }
        cl.sync();
        unsigned long long m = 0;
        uint32_t n = 0;
        if (tid < 256) {
          for (int c = 0; c < CL; ++c) {
            const Shared* o = cl.map_shared_rank(&sh, c);
            m += o->rmass[buf][tid];
            n += o->rcount[buf][tid];
          }
          sh.rmass[buf ^ 1][tid] = 0;  // the last readers of that buffer passed the sync above
          sh.rcount[buf ^ 1][tid] = 0;
        }
        unsigned long long pm;
        uint32_t pn;
        scan(m, n, 256, pm, pn);
        pm += msum;
        pn += cnt;
        // the digit that holds the border: for k the one with the k-th token,
        // for p the last one that begins before the target
        const bool mine = n > 0 && (by_mass ? (double)pm < target && !((double)(pm + m) < target)
                                            : pn < k && pn + n >= k);
        if (tid == 0) sh.found = -1;
        __syncthreads();
        if (mine) {
          sh.found = tid;
          sh.found_count = pn;
          sh.found_mass = pm;
          sh.found_own = n;
          sh.found_own_mass = m;
        }
        __syncthreads();
        const int d = max(sh.found, 0);
        cnt = sh.found_count;
        msum = sh.found_mass;
        own = sh.found_own;
        own_mass = sh.found_own_mass;
        prefix = (prefix & high) | ((dmask - (uint32_t)d) << shift);
        buf ^= 1;
        bits = shift;
        __syncthreads();
      }
      // `own` tokens share the key; their terms are equal
      const unsigned long long each = own ? own_mass / own : 0;
      uint32_t stay;
      if (by_mass) {
        // token number j of them stays while msum + j * each < target
        stay = own;
        if (each > 0) {
          const double room = (target - (double)msum) / (double)each;
          uint32_t j = room >= (double)own ? own : (uint32_t)room;
          while (j > 0 && !((double)(msum + (unsigned long long)(j - 1) * each) < target)) --j;
          while (j < own && (double)(msum + (unsigned long long)j * each) < target) ++j;
          stay = j;
        }
      } else {
        stay = min(own, k - cnt);
      }
      out.key = prefix;
      out.ties = stay;
      kept_mass = msum + (unsigned long long)stay * each;
    };

    unsigned long long zk = total_m;  // mass that top-k leaves
    bool cut_k = by_k && total_c > k;
    if (cut_k) {
      const bool mine = bc < k && bc + hc >= k;
      if (mine) {
        sh.found = tid;
        sh.found_count = bc;
        sh.found_mass = bm;
      }
      __syncthreads();
      const int fb = sh.found;
      const uint32_t cnt = sh.found_count;
      const unsigned long long msum = sh.found_mass;
      __syncthreads();
      resolve(false, fb, cnt, msum, 0.0, border, zk);
    }
    if (by_p) {
      const double target = fmax(p, 0.0) * (double)zk;
      // the last bin that begins before the target; the first token stays even at p = 0
      const bool mine = hc > 0 && (double)bm < target && !((double)(bm + hm) < target);
      if (tid == 0) sh.found = -1;
      __syncthreads();
      if (mine) {
        sh.found = tid;
        sh.found_count = bc;
        sh.found_mass = bm;
      }
      __syncthreads();
      const int fb = sh.found;
      const uint32_t cnt = sh.found_count;
      const unsigned long long msum = sh.found_mass;
      __syncthreads();
      Border bp{ordered(mx), 1};
      if (fb >= 0) {
        unsigned long long ignored;
        resolve(true, fb, cnt, msum, target, bp, ignored);
        if (bp.key > border.key || (bp.key == border.key && bp.ties < border.ties)) border = bp;
      } else if (!(target > 0.0)) {
        border = bp;
      }
    }
  }

  // ---- 4. what is kept, per warp
  const bool filtered = border.key != 0 || by_min;
  auto kept = [&](float l, double& y, uint64_t& f, bool& tie) {
    tie = false;
    if (!rw.distance(l, y)) return false;
    if (border.key != 0) {
      const uint32_t key = ordered(l);
      if (key < border.key) return false;
      tie = key == border.key;
    }
    if (by_min && y != 0.0 && exp2_neg(y) < floor_e) return false;
    f = rw.fixed(y);
    return true;
  };
  if (filtered) {
    uint64_t sum = 0;
    uint32_t ties = 0;
    for (int q = w0 + lane; q < w1; q += 32) {
      float x[VEC];
      un.load(q, x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        double y;
        uint64_t f;
        bool tie;
        if (!kept(x[e], y, f, tie)) continue;
        if (tie) ++ties;
        else sum += f;
      }
    }
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
  if (border.key != 0) {
    double y;
    if (rw.distance(from_ordered(border.key), y)) each = rw.fixed(y);
  }
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
    }
  }
  __syncthreads();
  const int target_warp = sh.pick_warp;
  const uint64_t mine_before = sh.pick_before, W = sh.pick_total;
  const uint32_t my_tie_base = sh.pick_ties;
  const double want = u * (double)W;
  if (target_warp == rank * WARPS + warp) {
    uint64_t run = mine_before;
    uint32_t seen = my_tie_base;
    int last = -1, token = -1;
    double ylast = 0.0, ytoken = 0.0;
    for (int qb = w0; qb < w1 && token < 0; qb += 32) {
      const int q = qb + lane;
      float x[VEC];
      uint64_t f[VEC];
      double ys[VEC];
      uint32_t tie_bits = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        f[e] = 0;
        x[e] = __uint_as_float(0x7fc00000u);
        ys[e] = 0.0;
      }
      if (q < w1) un.load(q, x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        bool tie;
        uint64_t v;
        if (!kept(x[e], ys[e], v, tie)) continue;
        f[e] = v;
        if (tie) tie_bits |= 1u << e;
      }
      // ties of earlier lanes, then the ones that still stay
      const uint32_t nt = __popc(tie_bits);
      uint32_t it = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, it, o);
        if (lane >= o) it += v;
      }
      uint32_t at = seen + it - nt;
      seen += __shfl_sync(0xffffffffu, it, 31);
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (tie_bits >> e & 1) {
          if (at >= border.ties) f[e] = 0;
          ++at;
        }
        sum += f[e];
      }
      uint64_t is = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t v = __shfl_up_sync(0xffffffffu, is, o);
        if (lane >= o) is += v;
      }
      const uint64_t step = __shfl_sync(0xffffffffu, is, 31);
      uint64_t acc = run + is - sum;
      int hit = -1, lst = -1;
      double yhit = 0.0, ylst = 0.0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        acc += f[e];
        if (f[e] > 0) {
          lst = q * VEC - un.shift + e;
          ylst = ys[e];
          if (hit < 0 && (double)acc > want) {
            hit = lst;
            yhit = ylst;
          }
        }
      }
      const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0);
      if (hits) {
        const int src = __ffs(hits) - 1;
        token = __shfl_sync(0xffffffffu, hit, src);
        ytoken = __shfl_sync(0xffffffffu, yhit, src);
      }
      const uint32_t any = __ballot_sync(0xffffffffu, lst >= 0);
      if (any) {
        const int src = 31 - __clz(any);
        last = __shfl_sync(0xffffffffu, lst, src);
        ylast = __shfl_sync(0xffffffffu, ylst, src);
      }
      run += step;
    }
    if (token < 0) {  // u of 1 or more: the last kept token
      token = last;
      ytoken = ylast;
    }
    if (lane == 0) {
      a.tokens[r] = token;
      if (a.logprobs) {
        // log of (e / W) with e from its exponent: no digits of a small term are lost
        const double lw = log((double)W / a.scale);
        a.logprobs[r] = (float)(-ytoken * 0.69314718055994530942 - lw);
      }
    }
  }
  cl.sync();  // no block leaves while another may read its shared memory
}

template <typename T>
int run(const Args& a, int cluster, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * cluster));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
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
  a.scale = (double)(1ll << std::min(45, 62 - log2v));
  // A row is split over as many blocks as leave each at least 4096 logits and
  // keep about two blocks per SM busy.
  int cluster = 1;
  while (cluster < samp::MAX_CL && rows * cluster * 2 <= 2 * sm_count() && vocab >= 4096 * 2 * cluster)
    cluster *= 2;
  cudaStream_t st = as_stream(stream);
  if (dtype == 0) return samp::run<float>(a, cluster, st);
  if (dtype == 1) return samp::run<__nv_bfloat16>(a, cluster, st);
  return samp::run<__half>(a, cluster, st);
}
