// Rotary positions: the first rotary_dim components of every head are taken in
// pairs, and pair i at position p is turned by the angle p * w_i and scaled:
//   a' = f (a cos - b sin),  b' = f (b cos + a sin);
// pairs are (i, i + rotary_dim / 2) (half layout) or (2 i, 2 i + 1)
// (interleaved).  Components past rotary_dim are copied.  `transpose` turns
// the other way (the transposed map, which is the gradient's).
//
// Angles.  w_i comes as a whole number of 2^-64 turns, so p * w_i modulo one
// turn is a 64-bit integer product that wraps: no digit of the angle is lost
// at far positions (or negative ones), where a float32 angle at position 10^6
// is off by 0.06.  The wrapped product, a signed fraction of half a turn,
// becomes a float32 argument of sincospif.
//
// Bound: HBM (or, for a few tokens, the launch).  Each block takes TOKENS
// positions of one batch entry, works out their cosines and sines once for all
// heads into shared memory, and reads and writes every head 16 bytes at a time;
// the first reads are issued before the angles are worked out.
#include "gq_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace gq {
namespace rot {

constexpr int THREADS = 256;
constexpr int AHEAD = 4;  // items a thread has in flight

struct Side {  // one of q and k
  const void* in;
  void* out;
  int64_t ib, ih, is;  // strides of the input: batch, head, position
  int64_t ob, oh, os;
  int heads;
};

struct Args {
  Side side[2];
  const void* positions;
  int64_t pos_b;
  int pos32;
  const uint64_t* turns;
  int64_t seq;
  int head_dim, half;  // half = rotary_dim / 2
  int heads;           // of both sides
  int heads_per_block;
  int tokens;          // positions per block
  float factor, sign;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// N consecutive components: one access where WIDE (the address is a multiple of
// its size), else one access each.
template <typename T, int N, bool WIDE>
struct alignas(WIDE ? sizeof(T) * N : sizeof(T)) Vec {
  T e[N];
};
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void get(Vec<T, N, WIDE>& v, const T* p) {
  if constexpr (WIDE) {
    v = *reinterpret_cast<const Vec<T, N, WIDE>*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v.e[i] = p[i];
  }
}
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void put(const Vec<T, N, WIDE>& v, T* p) {
  if constexpr (WIDE) {
    *reinterpret_cast<Vec<T, N, WIDE>*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = v.e[i];
  }
}

// One item = V pairs of a head (two vectors in the half layout, one vector of
// 2 V components in the interleaved one) or a vector (one component where not
// WIDE) to copy.
template <typename T, int V, bool INTER, bool WIDE>
__global__ void __launch_bounds__(THREADS) rotary_kernel(Args a) {
  extern __shared__ float2 cs[];  // [tokens][half]: f cos, f sin
  constexpr int VI = INTER ? 2 * V : V;
  constexpr int VC = WIDE ? VI : 1;
  using Val = Vec<T, VI, WIDE>;
  const int64_t s0 = (int64_t)blockIdx.x * a.tokens;
  const int ntok = (int)min((int64_t)a.tokens, a.seq - s0);
  const int64_t b = blockIdx.z;
  const int h0 = blockIdx.y * a.heads_per_block;
  const int nh = min(a.heads_per_block, a.heads - h0);
  const int turn_items = a.half / V;
  const int copy_items = (a.head_dim - 2 * a.half) / VC;
  const int per_head = turn_items + copy_items;
  const int total = ntok * nh * per_head;

  auto where = [&](int item, const T*& in, T*& out, int& tok, int& it) {
    it = item % per_head;
    const int rest = item / per_head;
    tok = rest / nh;
    int h = h0 + rest % nh;
    const Side& sd = a.side[h >= a.side[0].heads];
    if (h >= a.side[0].heads) h -= a.side[0].heads;
    in = static_cast<const T*>(sd.in) + b * sd.ib + h * sd.ih + (s0 + tok) * sd.is;
    out = static_cast<T*>(sd.out) + b * sd.ob + h * sd.oh + (s0 + tok) * sd.os;
  };
  auto load = [&](int item, Val& x, Val& y) {
    const T* in;
    T* out;
    int tok, it;
    where(item, in, out, tok, it);
    if (it >= turn_items) {
      const T* p = in + 2 * a.half + (it - turn_items) * VC;
      if constexpr (WIDE) get(x, p);
      else x.e[0] = *p;
    } else {
      get(x, in + it * VI);
      if constexpr (!INTER) get(y, in + a.half + it * VI);
    }
  };
  auto store = [&](int item, Val& x, Val& y) {
    const T* in;
    T* out;
    int tok, it;
    where(item, in, out, tok, it);
    if (it >= turn_items) {
      T* p = out + 2 * a.half + (it - turn_items) * VC;
      if constexpr (WIDE) put(x, p);
      else *p = x.e[0];
      return;
    }
    const float2* c = cs + tok * a.half + it * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      T& p = INTER ? x.e[2 * i] : x.e[i];
      T& q = INTER ? x.e[2 * i + 1] : y.e[i];
      const float u = to_f<T>(p), v = to_f<T>(q);
      const float2 t = c[i];
      p = from_f<T>(u * t.x - v * t.y);
      q = from_f<T>(v * t.x + u * t.y);
    }
    put(x, out + it * VI);
    if constexpr (!INTER) put(y, out + a.half + it * VI);
  };

  Val x[AHEAD], y[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int item = threadIdx.x + i * THREADS;
    if (item < total) load(item, x[i], y[i]);
  }
  for (int i = threadIdx.x; i < ntok * a.half; i += THREADS) {
    const int64_t at = b * a.pos_b + s0 + i / a.half;
    const int64_t pos = a.pos32 ? (int64_t)static_cast<const int32_t*>(a.positions)[at]
                                : static_cast<const int64_t*>(a.positions)[at];
    const int64_t frac = (int64_t)((uint64_t)pos * a.turns[i % a.half]);
    float s, c;
    sincospif((float)frac * 1.0842021724855044e-19f, &s, &c);  // 2^-63
    cs[i] = make_float2(c * a.factor, s * a.factor * a.sign);
  }
  __syncthreads();
  for (int base = 0; base < total; base += AHEAD * THREADS) {
    if (base > 0) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int item = base + threadIdx.x + i * THREADS;
        if (item < total) load(item, x[i], y[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int item = base + threadIdx.x + i * THREADS;
      if (item < total) store(item, x[i], y[i]);
    }
  }
}

template <typename T, int V, bool WIDE>
int run(const Args& a, int64_t batch, bool inter, cudaStream_t st) {
  for (int64_t b0 = 0; b0 < batch; b0 += 65535) {
    Args c = a;
    for (Side& s : c.side) {
      s.in = static_cast<const T*>(s.in) + b0 * s.ib;
      s.out = static_cast<T*>(s.out) + b0 * s.ob;
    }
    c.positions = static_cast<const char*>(c.positions) + b0 * c.pos_b * (c.pos32 ? 4 : 8);
    const dim3 grid((unsigned)ceil_div(c.seq, c.tokens),
                    (unsigned)ceil_div(c.heads, c.heads_per_block),
                    (unsigned)std::min<int64_t>(65535, batch - b0));
    const size_t smem = (size_t)c.tokens * c.half * sizeof(float2);
    if (inter)
      rotary_kernel<T, V, true, WIDE><<<grid, THREADS, smem, st>>>(c);
    else
      rotary_kernel<T, V, false, WIDE><<<grid, THREADS, smem, st>>>(c);
    GQ_TRY(check_launch("gq_rotary"));
  }
  return GQ_OK;
}

template <typename T>
int run_typed(const Args& a, int64_t batch, bool inter, int vec, cudaStream_t st) {
  constexpr int MAXV = 16 / sizeof(T);
  // in the interleaved layout an item of V pairs is one access of 2 V components
  if (vec >= MAXV) {
    if (inter) return run<T, MAXV / 2, true>(a, batch, inter, st);
    return run<T, MAXV, true>(a, batch, inter, st);
  }
  return run<T, 1, false>(a, batch, inter, st);
}

}  // namespace rot
}  // namespace gq

extern "C" int gq_rotary(const void* q, void* q_out, int64_t heads, const void* k, void* k_out,
                         int64_t kv_heads, const int64_t* strides, const void* positions,
                         int64_t position_stride, int positions_are_int32, const int64_t* turns,
                         int64_t batch, int64_t seq, int head_dim, int rotary_dim, int interleaved,
                         float factor, int transpose, int dtype, void* stream) {
  using namespace gq;
  GQ_REQUIRE(dtype >= 0 && dtype <= 2, "gq_rotary: dtype must be 0 (float32), 1 (bf16) or 2 (fp16)");
  GQ_REQUIRE(head_dim >= 1 && head_dim <= 4096 && rotary_dim >= 2 && rotary_dim <= head_dim &&
                 rotary_dim % 2 == 0,
             "gq_rotary: rotary_dim must be even, 2 .. head_dim, and head_dim at most 4096");
  GQ_REQUIRE(batch >= 0 && seq >= 0 && heads >= 0 && kv_heads >= 0 && seq < (1ll << 31) &&
                 heads + kv_heads < (1 << 20),
             "gq_rotary: bad shape");
  GQ_REQUIRE(kv_heads == 0 || (k != nullptr && k_out != nullptr) || batch == 0 || seq == 0,
             "gq_rotary: NULL k");
  if (batch == 0 || seq == 0 || heads + kv_heads == 0) return GQ_OK;
  GQ_REQUIRE(heads == 0 || (q != nullptr && q_out != nullptr), "gq_rotary: NULL q");
  GQ_REQUIRE(strides != nullptr && positions != nullptr && turns != nullptr, "gq_rotary: NULL input");
  const size_t size = dtype == 0 ? 4 : 2;
  rot::Args a;
  // 16-byte accesses where every row of both sides starts on such a boundary
  // and both the turned and the copied part are whole vectors
  const int maxv = (int)(16 / size);
  const int64_t unit = interleaved ? rotary_dim : rotary_dim / 2;
  bool wide = unit % maxv == 0 && (head_dim - rotary_dim) % maxv == 0;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = strides + 6 * i;
    rot::Side& d = a.side[i];
    d.in = i ? k : q;
    d.out = i ? k_out : q_out;
    d.ib = s[0]; d.ih = s[1]; d.is = s[2];
    d.ob = s[3]; d.oh = s[4]; d.os = s[5];
    d.heads = (int)(i ? kv_heads : heads);
    if (d.heads == 0) continue;
    for (int e = 0; e < 6; ++e) wide = wide && s[e] % maxv == 0;
    wide = wide && ((reinterpret_cast<uintptr_t>(d.in) | reinterpret_cast<uintptr_t>(d.out)) & 15) == 0;
  }
  a.positions = positions;
  a.pos_b = position_stride;
  a.pos32 = positions_are_int32;
  a.turns = reinterpret_cast<const uint64_t*>(turns);
  a.seq = seq;
  a.head_dim = head_dim;
  a.half = rotary_dim / 2;
  a.heads = (int)(heads + kv_heads);
  a.factor = factor;
  a.sign = transpose ? -1.f : 1.f;
  // A block gets about AHEAD items a thread: all heads of as many positions as
  // that takes (at most 32 KB of angles), or for few positions a part of the heads.
  const int64_t per_head = wide ? (interleaved ? head_dim / maxv
                                               : a.half / maxv + (head_dim - rotary_dim) / maxv)
                                : head_dim - a.half;
  const int64_t want = rot::THREADS * rot::AHEAD;
  const int64_t item_tok = per_head * a.heads;
  int64_t tokens = std::max<int64_t>(1, want / std::max<int64_t>(1, item_tok));
  tokens = std::min<int64_t>({tokens, seq, std::max<int64_t>(1, 32768 / (a.half * 8))});
  int64_t hpb = a.heads;
  if (tokens == 1) hpb = std::max<int64_t>(1, std::min<int64_t>(a.heads, want / per_head));
  while (hpb > 1 && ceil_div(seq, tokens) * ceil_div(a.heads, hpb) * batch < 148 &&
         tokens * hpb * per_head > rot::THREADS)
    hpb = (hpb + 1) / 2;
  a.tokens = (int)tokens;
  a.heads_per_block = (int)hpb;
  GQ_REQUIRE(ceil_div(a.heads, hpb) <= 65535, "gq_rotary: too many heads");
  cudaStream_t st = as_stream(stream);
  const int vec = wide ? maxv : 1;
  if (dtype == 0) return rot::run_typed<float>(a, batch, interleaved != 0, vec, st);
  if (dtype == 1) return rot::run_typed<__nv_bfloat16>(a, batch, interleaved != 0, vec, st);
  return rot::run_typed<__half>(a, batch, interleaved != 0, vec, st);
}
