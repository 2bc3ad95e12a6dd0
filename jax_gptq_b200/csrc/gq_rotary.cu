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
// is off by 0.06.  What the wrapped product lies from the nearest quarter turn
// is the argument of sincospif, so that its rounding to float32 is relative to
// at most an eighth of a turn, and cosines and sines next to 0 keep their digits
// (of the signed half turn it would be up to 9e-8 of any of them).
//
// Bound: HBM (or, for a few tokens, the launch).  Each block takes some
// positions of one batch entry, works out their cosines and sines once for all
// heads into shared memory, and reads and writes every head 16 bytes at a time;
// the first reads are issued before the angles are worked out.
#include "gq_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace gq {
namespace rot {

constexpr int THREADS = 128;

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
  int heads_per_block;
  int q_parts;         // blocks that the heads of q take; those of k follow
  int tokens;          // positions per block
  int per_head;        // items of a head
  int half_pad;        // half, to whole 16-byte pieces of floats
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

// W 32-bit words of components as one access, and as floats.
template <typename T, int W>
struct Wide {
  static constexpr int N = 4 * W / sizeof(T);
  struct alignas(4 * W) Raw {
    uint32_t w[W];
  } raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ void get(float (&f)[N]) const {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const uint32_t w = raw.w[i];
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      } else {
        f[2 * i] = __uint_as_float(w << 16);
        f[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
      }
    }
  }
  __device__ __forceinline__ void set(const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (sizeof(T) == 4) {
        raw.w[i] = __float_as_uint(f[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        raw.w[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        raw.w[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
  }
};
// One component at a time, for rows that are not made of whole words.
template <typename T>
struct Narrow {
  static constexpr int N = 1;
  T raw;
  __device__ __forceinline__ void load(const T* p) { raw = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = raw; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_f<T>(raw); }
  __device__ __forceinline__ void set(const float (&f)[1]) { raw = from_f<T>(f[0]); }
};

// An item of a head is one piece of each half of N pairs, or in the interleaved
// layout one piece of N / 2 pairs (two components where Narrow), or one piece to
// copy.  threadIdx.x is the item inside a head; along y the threads take `hg`
// heads of q or of k, of `tg` positions at a time.  Many warps with few
// registers each keep the loads in flight: 4 x 2048 positions of 64 + 8 heads of
// 128 in bf16 take 52 us (5.8 TB/s of the 302 MB read and written, a plain copy
// of them 49 us); reading two or four heads ahead in registers took 76 to 94 us.
template <typename T, typename P, bool INTER>
__global__ void __launch_bounds__(THREADS) rotary_kernel(Args a) {
  constexpr int N = P::N;
  constexpr bool SPLIT = !INTER || N == 1;  // a pair's components lie in two pieces
  constexpr int PAIRS = SPLIT ? N : N / 2;
  extern __shared__ float angles[];  // per position: f cos of every pair, then f sin
  const int64_t s0 = (int64_t)blockIdx.x * a.tokens;
  const int ntok = (int)min((int64_t)a.tokens, a.seq - s0);
  const int64_t b = blockIdx.z;
  const int second = blockIdx.y >= a.q_parts;
  const Side& sd = a.side[second];
  const int h0 = ((int)blockIdx.y - (second ? a.q_parts : 0)) * a.heads_per_block;
  const int nh = min(a.heads_per_block, sd.heads - h0);
  const int half = a.half, half_pad = a.half_pad;
  const int turn_items = half / PAIRS;
  const int per_head = a.per_head;
  const int threads = blockDim.x * blockDim.y, tid = threadIdx.y * blockDim.x + threadIdx.x;
  const int hg = min((int)blockDim.y, nh), tg = blockDim.y / hg;
  const int hh = threadIdx.y % hg, tt = threadIdx.y / hg;

  for (int i = tid; i < ntok * half; i += threads) {
    const int tok = i / half, pair = i - tok * half;
    const int64_t pi = b * a.pos_b + s0 + tok;
    const int64_t pos = a.pos32 ? (int64_t)static_cast<const int32_t*>(a.positions)[pi]
                                : static_cast<const int64_t*>(a.positions)[pi];
    const uint64_t turn = (uint64_t)pos * a.turns[pair];
    const uint32_t quarters = (uint32_t)((turn + (1ull << 61)) >> 62);  // to the nearest
    const int64_t rest = (int64_t)(turn - ((uint64_t)quarters << 62));
    float s, c;
    sincospif((float)rest * 1.0842021724855044e-19f, &s, &c);  // 2^-63
    if (quarters & 1) {  // a quarter further: (c, s) becomes (-s, c)
      const float t = c;
      c = -s;
      s = t;
    }
    const float f = (quarters & 2) ? -a.factor : a.factor;
    angles[tok * 2 * half_pad + pair] = c * f;
    angles[tok * 2 * half_pad + half_pad + pair] = s * f * a.sign;
  }
  __syncthreads();
  if (tt >= tg) return;
  const int64_t ig = sd.ih * hg, og = sd.oh * hg;
  for (int it = threadIdx.x; it < per_head; it += blockDim.x) {
    const bool turn = it < turn_items;
    // where the item's components begin, and how far its second piece lies
    const int at = !turn ? 2 * half + (it - turn_items) * N
                         : (INTER ? it * (SPLIT ? 2 : N) : it * N);
    const int next = INTER ? 1 : half;
    for (int tok = tt; tok < ntok; tok += tg) {
      const T* p = static_cast<const T*>(sd.in) + b * sd.ib + (s0 + tok) * sd.is + (h0 + hh) * sd.ih + at;
      T* o = static_cast<T*>(sd.out) + b * sd.ob + (s0 + tok) * sd.os + (h0 + hh) * sd.oh + at;
      float c[PAIRS], s[PAIRS];
      if (turn) {
        const float* t = angles + tok * 2 * half_pad + it * PAIRS;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          c[i] = t[i];
          s[i] = t[half_pad + i];
        }
      }
#pragma unroll 1
      for (int h = hh; h < nh; h += hg, p += ig, o += og) {
        P x, y;
        x.load(p);
        if (SPLIT && turn) y.load(p + next);
        if (turn) {
          float u[N], w[N];
          x.get(u);
          if constexpr (SPLIT) y.get(w);
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) {
            float& e = SPLIT ? u[i] : u[2 * i];
            float& f = SPLIT ? w[i] : u[2 * i + 1];
            const float m = e, n = f;
            e = m * c[i] - n * s[i];
            f = n * c[i] + m * s[i];
          }
          x.set(u);
          if constexpr (SPLIT) y.set(w);
        }
        x.store(o);
        if (SPLIT && turn) y.store(o + next);
      }
    }
  }
}

template <typename T, typename P>
int run(const Args& a, int64_t batch, bool inter, cudaStream_t st) {
  for (int64_t b0 = 0; b0 < batch; b0 += 65535) {
    Args c = a;
    for (Side& s : c.side) {
      if (s.heads == 0) continue;
      s.in = static_cast<const T*>(s.in) + b0 * s.ib;
      s.out = static_cast<T*>(s.out) + b0 * s.ob;
    }
    c.positions = static_cast<const char*>(c.positions) + b0 * c.pos_b * (c.pos32 ? 4 : 8);
    const dim3 grid((unsigned)ceil_div(c.seq, c.tokens),
                    (unsigned)(c.q_parts + ceil_div(c.side[1].heads, c.heads_per_block)),
                    (unsigned)std::min<int64_t>(65535, batch - b0));
    const size_t smem = (size_t)c.tokens * c.half_pad * 2 * sizeof(float);
    const int bx = std::min(c.per_head, THREADS);
    const dim3 block(bx, std::max(1, THREADS / bx));
    if (inter)
      rotary_kernel<T, P, true><<<grid, block, smem, st>>>(c);
    else
      rotary_kernel<T, P, false><<<grid, block, smem, st>>>(c);
    GQ_TRY(check_launch("gq_rotary"));
  }
  return GQ_OK;
}

template <typename T>
int run_typed(const Args& a, int64_t batch, bool inter, int words, cudaStream_t st) {
  if (words == 4) return run<T, Wide<T, 4>>(a, batch, inter, st);
  if (words == 2) return run<T, Wide<T, 2>>(a, batch, inter, st);
  if constexpr (sizeof(T) == 2) {
    if (words == 1) return run<T, Wide<T, 1>>(a, batch, inter, st);
  }
  return run<T, Narrow<T>>(a, batch, inter, st);
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
  const int size = dtype == 0 ? 4 : 2;
  rot::Args a;
  // The widest piece, 16 bytes down to one component, that every row of both
  // sides starts on and that both the turned and the copied part are made of:
  // all of these are multiples of it, in bytes.
  uint64_t all = (uint64_t)(interleaved ? rotary_dim : rotary_dim / 2) * size |
                 (uint64_t)(head_dim - rotary_dim) * size;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = strides + 6 * i;
    rot::Side& d = a.side[i];
    d.in = i ? k : q;
    d.out = i ? k_out : q_out;
    d.ib = s[0]; d.ih = s[1]; d.is = s[2];
    d.ob = s[3]; d.oh = s[4]; d.os = s[5];
    d.heads = (int)(i ? kv_heads : heads);
    if (d.heads == 0) continue;
    for (int e = 0; e < 6; ++e) all |= (uint64_t)s[e] * size;
    all |= reinterpret_cast<uintptr_t>(d.in) | reinterpret_cast<uintptr_t>(d.out);
  }
  a.positions = positions;
  a.pos_b = position_stride;
  a.pos32 = positions_are_int32;
  a.turns = reinterpret_cast<const uint64_t*>(turns);
  a.seq = seq;
  a.head_dim = head_dim;
  a.half = rotary_dim / 2;
  a.half_pad = (a.half + 3) & ~3;
  a.factor = factor;
  a.sign = transpose ? -1.f : 1.f;
  int piece = 16;
  while (piece > size && all % piece != 0) piece /= 2;
  const int words = piece > size ? piece / 4 : 0;
  const int n = words ? piece / size : 1;
  a.per_head = (interleaved && n > 1 ? rotary_dim / n : a.half / n) + (head_dim - rotary_dim) / n;
  // A block takes all heads of q or of k, of positions enough for about 8 items
  // a thread and at most one angle a thread (2 positions of 64 heads of 128: 52
  // us for 4 x 2048 of them, with 8 positions 57 us); while that leaves SMs
  // without a block, fewer positions, then fewer heads, down to one item a thread.
  int64_t hpb = std::max(heads, kv_heads);
  int64_t tokens = std::max<int64_t>(
      1, std::min<int64_t>({seq, rot::THREADS / a.half, 8 * rot::THREADS / (hpb * a.per_head)}));
  auto parts = [&] { return ceil_div(heads, hpb) + ceil_div(kv_heads, hpb); };
  auto blocks = [&] { return ceil_div(seq, tokens) * parts() * batch; };
  while (tokens > 1 && blocks() < 4 * sm_count()) tokens = (tokens + 1) / 2;
  while (hpb > 1 && blocks() < sm_count() && hpb * a.per_head > rot::THREADS) hpb = (hpb + 1) / 2;
  a.tokens = (int)tokens;
  a.heads_per_block = (int)hpb;
  a.q_parts = (int)ceil_div(heads, hpb);
  GQ_REQUIRE(parts() <= 65535, "gq_rotary: too many heads");
  cudaStream_t st = as_stream(stream);
  if (dtype == 0) return rot::run_typed<float>(a, batch, interleaved != 0, words, st);
  if (dtype == 1) return rot::run_typed<__nv_bfloat16>(a, batch, interleaved != 0, words, st);
  return rot::run_typed<__half>(a, batch, interleaved != 0, words, st);
}
