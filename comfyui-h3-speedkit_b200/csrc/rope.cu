// Rotary positions with several axes (time, height, width, ...) for Q and K, and
// the table of rotations that the QKV op takes.
//
// Token t has one position per axis.  Pair p belongs to axis(p) and turns by
//   angle = position[t, axis(p)] * frequency[p]
//   (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos)       (sin negated: the inverse)
// Split pairs are the channels (p, P + p) of a head, interleaved ones (2p, 2p + 1);
// the channels from 2 P on pass unchanged.  With a weight the head is normalised
// first: x * w / sqrt(mean(x^2) + eps).  FP32 throughout, one rounding at the end.
//
// Frequencies come in turns (angle / 2 pi) as doubles, and whole turns are dropped before
// anything is rounded to FP32, whose angle has no fraction left at positions of 2^31.  One
// CTA computes the sines of its tokens once, for all heads of Q and K.
//
// HBM bound: every value of Q and K is read and written once.  16384 tokens, 56 + 56 heads
// of 128, normalised, 48 pairs turned: 181 us, 5.2 TB/s, 0.79 of a copy's rate (issue slots
// 66 % busy: the rest is the norm and the rotation between the loads and the stores).  The
// table of 98304 tokens, 48 pairs: 14.1 to 15.4 us, where its bytes take 5.9: the rotations'
// 65 instructions bound it (without the stores still 13.9).  One token: 4.1 us, most of it the launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/h3sk_b200.h"
#include "host_util.h"
#include "wide_types.cuh"

namespace h3sk {
namespace rope {

constexpr int kMaxPairs = 128;
constexpr int kMaxDim = 256;
constexpr int kThreads = 256;
constexpr int kMaxTile = 16;   // tokens a tile

struct Tables {
  double turns[kMaxPairs];   // frequency / (2 pi)
  uint8_t axis[kMaxPairs];
};

struct Args {
  const void *q, *k;
  void *qo, *ko;
  const void *qw, *kw;
  const void* positions;
  int64_t q_token, q_head, k_token, k_head;       // strides in values
  int64_t qo_token, qo_head, ko_token, ko_head;
  int64_t tokens;
  int q_heads, k_heads, dim, pairs, axes;
  int tile, chunk;      // tokens per tile; heads (of Q and K together) per CTA
  int float_positions;
  float eps, sign;
};

// (cos, sin) of an angle of `quarter` quarter turns and r more turns, |r| <= 1/8:
// polynomials in r^2 for sin(2 pi r) / r and cos(2 pi r), of the least largest relative error
// (by Lawson's reweighted least squares, the cosine's 1 at 0 fixed), then rounded to FP32:
// 4.2e-8 and 8.3e-9 of the value (2 pi in FP32 alone is off by 2.8e-8), 1.4e-7 and 8e-8 as
// FP32 evaluates them.
__device__ __forceinline__ float2 cos_sin(int quarter, float r) {
  const float z = r * r;
  float s = fmaf(z, -75.39354705810547f, 81.59235382080078f);
  s = fmaf(s, z, -41.34165954589844f);
  s = r * fmaf(s, z, 6.2831854820251465f);
  float c = fmaf(z, 59.20278549194336f, -85.44229888916016f);
  c = fmaf(c, z, 64.9393081665039f);
  c = fmaf(c, z, -19.739208221435547f);
  c = fmaf(c, z, 1.0f);
  const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
  const uint32_t sx = uint32_t((quarter + 1) & 2) << 30, sy = uint32_t(quarter & 2) << 30;
  return make_float2(__uint_as_float(__float_as_uint(x) ^ sx), __uint_as_float(__float_as_uint(y) ^ sy));
}

// A pair's frequency: turns a position, and their fraction as a 64-bit binary one.  Whole
// positions multiply that and drop whole turns by overflow, which loses nothing; what is off is
// the frequency itself, a rounded double: up to 2^-56 turns at theta^0 / 2 pi = 0.159, so 2^-25
// turns (1.9e-7 of an angle) at a position of 2^31, as much as FP32 loses in the sine.
struct Frequency {
  double turns;
  uint64_t fraction;
  __device__ __forceinline__ explicit Frequency(double t) {
    turns = t;
    fraction = __double2ull_rn((t - floor(t)) * 18446744073709551616.0);
  }
  __device__ __forceinline__ float2 rotation(float position) const {
    const double t = double(position) * turns;
    const double f = t - rint(t), q = rint(4.0 * f);
    return cos_sin(int(q), float(f - 0.25 * q));
  }
  __device__ __forceinline__ float2 rotation(int position) const {
    const uint64_t f = uint64_t(int64_t(position)) * fraction;
    const uint32_t hi = uint32_t(f >> 32), q = (hi + (1u << 29)) >> 30;
    // the rest in two words: the upper one is whole in FP32 wherever the lower one counts
    const float upper = float(int(hi - (q << 30))) * 2.3283064365386963e-10f;   // 2^-32
    return cos_sin(int(q), fmaf(float(uint32_t(f)), 5.421010862427522e-20f, upper));   // 2^-64
  }
  __device__ __forceinline__ float2 rotation(const void* positions, int is_float, int64_t index) const {
    return is_float ? rotation(__ldg(static_cast<const float*>(positions) + index))
                    : rotation(__ldg(static_cast<const int*>(positions) + index));
  }
};

// A thread's pair of every tile: thread t below (kThreads / P) P computes pair t % P of
// tokens t / P, t / P + kThreads / P, ...  Each thread takes its entry of the tables once:
// the constant bank serves one address a warp and turn, so P threads read them there and
// the others in shared memory (every thread in the constant bank: 10,000 clocks an SM).
struct Pair {
  int tokens_at_once, token, pair, axis;
  Frequency frequency;
  static __device__ __forceinline__ void stage(const Args& a, const Tables& tb, Tables& shared) {
    if (int(threadIdx.x) < a.pairs) {
      shared.turns[threadIdx.x] = tb.turns[threadIdx.x];
      shared.axis[threadIdx.x] = tb.axis[threadIdx.x];
    }
    __syncthreads();
  }
  __device__ __forceinline__ Pair(const Args& a, const Tables& shared)
      : tokens_at_once(kThreads / a.pairs),
        token(int(threadIdx.x) / a.pairs),
        pair(int(threadIdx.x) - token * a.pairs),
        axis(shared.axis[pair]),
        frequency(shared.turns[pair]) {}
};

// cs[token][pair] of n tokens from token0 on; kByEight: pair 8 l + e of a token at
// e * eighths + l, so that the lanes of a row read consecutive words (in the pairs' order
// their bank conflicts bound the kernel: 188 us where this takes 180).
template <bool kByEight>
__device__ __forceinline__ void fill_rotations(float2* cs, const Args& a, const Pair& own, int64_t token0, int n) {
  if (own.token >= own.tokens_at_once) return;
  const int eighths = (a.pairs + 7) >> 3, size = kByEight ? 8 * eighths : a.pairs;
  const int at = kByEight ? (own.pair & 7) * eighths + (own.pair >> 3) : own.pair;
  for (int t = own.token; t < n; t += own.tokens_at_once) {
    float2 r = own.frequency.rotation(a.positions, a.float_positions, (token0 + t) * a.axes + own.axis);
    r.y *= a.sign;
    cs[t * size + at] = r;
  }
}

// BF16 squares can pass FP32: such a head is taken 2^100 smaller, its largest value then
// 2^-46 at least.  (FP16 squares stay below 2^40.)  rsqrt of the mean is 0 there, NaN or 0 in
// heads that are not finite.
constexpr float kDown = 0x1p-100f;
template <typename T, bool kNorm>
constexpr bool kSquaresPass = kNorm && std::is_same<T, __nv_bfloat16>::value;

// A lane's 16 channels of one head row.
template <typename T>
struct Chunk {
  uint4 u0, u1;
  T* dst;
  int t;
  bool is_q;
};

// kLanes threads a head row, 16 channels each; kUnroll rows in flight a thread (16384
// tokens, 56 + 56 heads, us with 1 / 2 / 4: 202 / 179 / 206).  Split
// pairs: a lane below P / 8 holds eight, the others 16 channels that pass.  Interleaved
// ones: a lane holds the pairs 8 lane .. 8 lane + 7, of which those below P turn.  CTAs
// take tiles of tokens in turn; a tile's sines are made while the one before is written.
template <typename T, typename W, bool kInterleaved, bool kNorm, int kLanes>
__global__ void __launch_bounds__(kThreads) rope_rows(const Args a, const __grid_constant__ Tables tb) {
  extern __shared__ float2 cs_buffers[];
  constexpr int kUnroll = 2, kStep = kThreads / kLanes;
  __shared__ Tables tables;
  Pair::stage(a, tb, tables);
  const Pair own(a, tables);
  const int64_t tiles = (a.tokens + a.tile - 1) / a.tile;
  const int head0 = int(blockIdx.y) * a.chunk, heads = min(a.chunk, a.q_heads + a.k_heads - head0);
  const int lane = threadIdx.x & (kLanes - 1), chunks = a.dim >> 4;
  const bool active = lane < chunks;
  const bool rotates = lane * 8 < a.pairs;
  // the lane's two 8-channel vectors
  const int c0 = kInterleaved || !rotates ? 16 * lane : 8 * lane;
  const int c1 = kInterleaved || !rotates ? c0 + 8 : a.pairs + c0;
  // the lane's norm weights of Q and K, as they are stored (16-bit ones stay in registers)
  constexpr bool kHeld = kNorm && sizeof(W) == 2;
  uint4 held[4];
  if (kHeld && active) {
    held[0] = *reinterpret_cast<const uint4*>(static_cast<const W*>(a.qw) + c0);
    held[1] = *reinterpret_cast<const uint4*>(static_cast<const W*>(a.qw) + c1);
    held[2] = *reinterpret_cast<const uint4*>(static_cast<const W*>(a.kw) + c0);
    held[3] = *reinterpret_cast<const uint4*>(static_cast<const W*>(a.kw) + c1);
  }
  const auto tokens_of = [&](int64_t tile) { return int(min(int64_t(a.tile), a.tokens - tile * a.tile)); };
  const int eighths = (a.pairs + 7) >> 3, token_size = 8 * eighths;
  if (blockIdx.x < tiles) fill_rotations<true>(cs_buffers, a, own, int64_t(blockIdx.x) * a.tile, tokens_of(blockIdx.x));
  int buffer = 0;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, buffer ^= 1) {
    __syncthreads();
    const float2* cs = cs_buffers + buffer * a.tile * token_size;
    const int64_t token0 = tile * a.tile, next = tile + gridDim.x;
    const int rows = tokens_of(tile) * heads;
    if (next < tiles)
      fill_rotations<true>(cs_buffers + (buffer ^ 1) * a.tile * token_size, a, own, next * a.tile, tokens_of(next));
    const auto load = [&](int row, Chunk<T>& ch) {
      const bool on = row < rows && active;
      ch.t = row / heads;
      const int head = head0 + row - ch.t * heads;
      ch.is_q = head < a.q_heads;
      const int h = ch.is_q ? head : head - a.q_heads;
      const int64_t token = token0 + ch.t;
      ch.dst = nullptr;
      ch.u0 = ch.u1 = make_uint4(0, 0, 0, 0);
      if (on) {
        const T* src = ch.is_q ? static_cast<const T*>(a.q) + token * a.q_token + h * a.q_head
                               : static_cast<const T*>(a.k) + token * a.k_token + h * a.k_head;
        ch.dst = ch.is_q ? static_cast<T*>(a.qo) + token * a.qo_token + h * a.qo_head
                         : static_cast<T*>(a.ko) + token * a.ko_token + h * a.ko_head;
        ch.u0 = *reinterpret_cast<const uint4*>(src + c0);
        ch.u1 = *reinterpret_cast<const uint4*>(src + c1);
      }
    };
    // false for a head whose squares pass FP32: it is not written.  `smaller` takes such heads.
    const auto turn = [&](const Chunk<T>& ch, auto smaller) -> bool {
      bool fine = true;
      float x[8], y[8];
      unpack8<T>(ch.u0, x);
      unpack8<T>(ch.u1, y);
      if constexpr (kNorm) {
        float sum = 0.0f, eps = a.eps;
        if constexpr (smaller) {
          eps = eps * kDown * kDown;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= kDown, y[e] *= kDown;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], fmaf(y[e], y[e], sum));
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (ch.dst) {
          const float r = rsqrtf(sum / float(a.dim) + eps);
          if (kSquaresPass<T, kNorm> && !smaller) fine = r > 0.0f;
          float w0[8], w1[8];
          if constexpr (kHeld) {
            unpack8<W>(ch.is_q ? held[0] : held[2], w0);
            unpack8<W>(ch.is_q ? held[1] : held[3], w1);
          } else {
            const W* w = static_cast<const W*>(ch.is_q ? a.qw : a.kw);
            load8<W>(w + c0, w0);
            load8<W>(w + c1, w1);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = x[e] * r * w0[e];
            y[e] = y[e] * r * w1[e];
          }
        }
      }
      if (ch.dst) {
        const float2* r = cs + ch.t * token_size + lane;   // pair 8 lane + e at r[e * eighths]
        if constexpr (kInterleaved) {
          const int left = a.pairs - 8 * lane;   // the lane's pairs that turn
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float* v = e < 4 ? x + 2 * e : y + 2 * e - 8;
            const float2 p = e < left ? r[e * eighths] : make_float2(1.0f, 0.0f);
            const float v0 = v[0], v1 = v[1];
            v[0] = v0 * p.x - v1 * p.y;
            v[1] = v0 * p.y + v1 * p.x;
          }
        } else if (rotates) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 p = r[e * eighths];
            const float x0 = x[e], x1 = y[e];
            x[e] = x0 * p.x - x1 * p.y;
            y[e] = x0 * p.y + x1 * p.x;
          }
        }
        if (fine) {
          *reinterpret_cast<uint4*>(ch.dst + c0) = pack8<T>(x);
          *reinterpret_cast<uint4*>(ch.dst + c1) = pack8<T>(y);
        }
      }
      return fine;
    };
    // whole warps iterate together: the row's sum is a shuffle
    uint32_t past = 0;   // a bit for each of the thread's rows, 16 at most
    for (int base = int(threadIdx.x) / kLanes; base - int(threadIdx.x) / kLanes < rows; base += kUnroll * kStep) {
      Chunk<T> ch[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) load(base + i * kStep, ch[i]);
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) past = 2 * past + !turn(ch[i], std::false_type());
    }
    // (a check of each pair of rows in the loop: 185 us where this takes 179)
    if (kSquaresPass<T, kNorm> && __any_sync(0xffffffffu, past != 0)) {
      const int turns = (rows + kUnroll * kStep - 1) / (kUnroll * kStep) * kUnroll;
#pragma unroll 1
      for (int i = 0; i < turns; ++i) {
        Chunk<T> ch;
        load(int(threadIdx.x) / kLanes + i * kStep, ch);
        if (!(past >> (turns - 1 - i) & 1u)) ch.dst = nullptr;
        turn(ch, std::true_type());
      }
    }
  }
}

// Any even width, pair count, stride and alignment: a warp a head row, one pair a
// lane and step.  The row is read twice with a norm.
template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) rope_rows_scalar(const Args a, const __grid_constant__ Tables tb,
                                                             const int interleaved) {
  extern __shared__ float2 cs[];
  __shared__ Tables tables;
  Pair::stage(a, tb, tables);
  const Pair own(a, tables);
  const int64_t tiles = (a.tokens + a.tile - 1) / a.tile;
  const int head0 = int(blockIdx.y) * a.chunk, heads = min(a.chunk, a.q_heads + a.k_heads - head0);
  const int lane = threadIdx.x & 31;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t token0 = tile * a.tile;
    const int n = int(min(int64_t(a.tile), a.tokens - token0)), rows = n * heads;
    __syncthreads();
    fill_rotations<false>(cs, a, own, token0, n);
    __syncthreads();
    // false for a head whose squares pass FP32: it is not written.  `smaller` takes such heads.
    const auto turn = [&](int row, auto smaller) -> bool {
      const int t = row / heads, head = head0 + row - t * heads;
      const bool is_q = head < a.q_heads;
      const int h = is_q ? head : head - a.q_heads;
      const int64_t token = token0 + t;
      const T* src = is_q ? static_cast<const T*>(a.q) + token * a.q_token + h * a.q_head
                          : static_cast<const T*>(a.k) + token * a.k_token + h * a.k_head;
      T* dst = is_q ? static_cast<T*>(a.qo) + token * a.qo_token + h * a.qo_head
                    : static_cast<T*>(a.ko) + token * a.ko_token + h * a.ko_head;
      const W* w = static_cast<const W*>(is_q ? a.qw : a.kw);
      float r = 1.0f;
      if (w) {
        float sum = 0.0f;
        for (int c = lane; c < a.dim; c += 32) {
          float x = to_float(src[c]);
          if constexpr (smaller) x *= kDown;
          sum = fmaf(x, x, sum);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        r = rsqrtf(sum / float(a.dim) + (smaller ? a.eps * kDown * kDown : a.eps));
        if (kSquaresPass<T, true> && !smaller && !(r > 0.0f)) return false;
      }
      // the pairs, then pairs of the channels that pass (a lane reads what it writes)
#pragma unroll 2
      for (int p = lane; p < a.dim / 2; p += 32) {
        const bool turns = p < a.pairs;
        const int i0 = interleaved || !turns ? 2 * p : p, i1 = interleaved || !turns ? i0 + 1 : a.pairs + p;
        float x0 = to_float(src[i0]), x1 = to_float(src[i1]);
        if (w) {
          if constexpr (smaller) x0 *= kDown, x1 *= kDown;
          x0 = x0 * r * to_float(w[i0]);
          x1 = x1 * r * to_float(w[i1]);
        }
        if (turns) {
          const float2 c = cs[t * a.pairs + p];
          const float y0 = x0 * c.x - x1 * c.y;
          x1 = x0 * c.y + x1 * c.x;
          x0 = y0;
        }
        dst[i0] = from_float<T>(x0);
        dst[i1] = from_float<T>(x1);
      }
      return true;
    };
    uint32_t past = 0;   // a bit for each of the warp's rows, 16 at most
    const int first = threadIdx.x >> 5, step = kThreads / 32;
    for (int row = first; row < rows; row += step) past = 2 * past + !turn(row, std::false_type());
    if (kSquaresPass<T, true> && past) {
      int row = first + (rows - 1 - first) / step * step;   // the warp's last, the lowest bit
#pragma unroll 1
      for (; past; past >>= 1, row -= step)
        if (past & 1u) turn(row, std::true_type());
    }
  }
}

// [tokens, P, 2, 2] BF16: ((cos, -sin), (sin, cos)) of every pair.
// A thread keeps its pair and goes through the tokens (see Pair), two at a time: their
// positions are on the way together (98304 tokens, 48 pairs, us: two 15.4, four 16.1).
// Index: 32 bits where the table's size allows.
template <typename P, typename Index>
__global__ void __launch_bounds__(kThreads) rope_table(const Args a, const __grid_constant__ Tables tb, uint2* out) {
  __shared__ Tables tables;
  Pair::stage(a, tb, tables);
  const Pair own(a, tables);
  if (own.token >= own.tokens_at_once) return;
  const Index step = Index(gridDim.x) * own.tokens_at_once, tokens = Index(a.tokens);
  Index t = Index(blockIdx.x) * own.tokens_at_once + own.token;
  const P* positions = static_cast<const P*>(a.positions) + own.axis;
  uint2* rows = out + own.pair;
  const Index in = step * a.axes, rows_step = step * a.pairs;
  Index at = t * a.axes, to = t * a.pairs;
  for (; t < tokens; t += 2 * step, at += 2 * in, to += 2 * rows_step) {
    P x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = t + i * step < tokens ? __ldg(positions + at + i * in) : P(0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 r = own.frequency.rotation(x[i]);
      const uint2 row = make_uint2(pack2<__nv_bfloat16>(r.x, -r.y), pack2<__nv_bfloat16>(r.y, r.x));
      if (t + i * step < tokens) rows[to + i * rows_step] = row;
    }
  }
}

template <typename T, typename W>
cudaError_t launch(const Args& a, const Tables& tb, int lanes, bool interleaved, cudaStream_t stream) {
  // as many CTAs as fit, sharing the tiles of every chunk of heads
  const int64_t tiles = (a.tokens + a.tile - 1) / a.tile;
  const int chunks = (a.q_heads + a.k_heads + a.chunk - 1) / a.chunk;
  const auto go = [&](auto* kernel, int buffers, auto... more) -> cudaError_t {
    const int smem = buffers * a.tile * ((a.pairs + 7) / 8 * 8) * int(sizeof(float2));
    int fit = 0;
    const cudaError_t e = rq_persistent_grid(reinterpret_cast<const void*>(kernel), kThreads, smem, INT_MAX, &fit);
    if (e != cudaSuccess) return e;
    const int64_t per_chunk = fit / chunks > 1 ? fit / chunks : 1;
    const dim3 grid(unsigned(tiles < per_chunk ? tiles : per_chunk), unsigned(chunks));
    kernel<<<grid, kThreads, smem, stream>>>(a, tb, more...);
    return cudaGetLastError();
  };
  const bool norm = a.qw != nullptr;
#define H3SK_ROPE(I, N) \
  (lanes == 4 ? go(rope_rows<T, W, I, N, 4>, 2) : lanes == 8 ? go(rope_rows<T, W, I, N, 8>, 2) : go(rope_rows<T, W, I, N, 16>, 2))
  if (lanes == 0) return go(rope_rows_scalar<T, W>, 1, int(interleaved));
  if (interleaved) return norm ? H3SK_ROPE(true, true) : H3SK_ROPE(true, false);
  return norm ? H3SK_ROPE(false, true) : H3SK_ROPE(false, false);
#undef H3SK_ROPE
}

bool misaligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

// The pairs' frequencies and axes from the caller's host arrays.
bool fill_tables(Tables* tb, const double* turns, const int* axis, int pairs, int axes) {
  for (int p = 0; p < pairs; ++p) {
    if (!std::isfinite(turns[p]) || axis[p] < 0 || axis[p] >= axes) return false;
    tb->turns[p] = turns[p];
    tb->axis[p] = uint8_t(axis[p]);
  }
  return true;
}

}  // namespace rope
}  // namespace h3sk

#define H3SK_EXPORT extern "C" __attribute__((visibility("default")))

H3SK_EXPORT size_t h3_rope_args_size(void) { return sizeof(H3RopeArgs); }

H3SK_EXPORT int h3_rope_axes_run(const H3RopeArgs* r, uintptr_t stream_ptr) {
  using namespace h3sk::rope;
  if (!r || r->tokens < 0 || r->q_heads < 0 || r->k_heads < 0 || r->q_heads > 65535 || r->k_heads > 65535)
    return cudaErrorInvalidValue;
  if (r->dim < 2 || r->dim > kMaxDim || r->dim % 2 || r->pairs < 1 || r->pairs > kMaxPairs || 2 * r->pairs > r->dim ||
      r->axes < 1 || r->axes > 255 || r->type < 0 || r->type > 1 || (r->weight_type != r->type && r->weight_type != 2))
    return cudaErrorInvalidValue;
  if (!(r->eps >= 1.17549435e-38f) || !std::isfinite(r->eps) || !r->turns || !r->axis) return cudaErrorInvalidValue;
  if (r->tokens == 0 || r->q_heads + r->k_heads == 0) return cudaSuccess;
  if (!r->positions || misaligned(r->positions, 4) || r->tokens > int64_t(0x7fffffff) * 8 ||
      (r->q_heads && (!r->q || !r->q_out)) || (r->k_heads && (!r->k || !r->k_out)))
    return cudaErrorInvalidValue;
  // a weight on one side only would leave the other without its norm
  const bool norm = r->q_weight || r->k_weight;
  if (norm && ((r->q_heads && !r->q_weight) || (r->k_heads && !r->k_weight))) return cudaErrorInvalidValue;
  const uintptr_t wa = r->weight_type == 2 ? 4 : 2;
  for (const void* p : {r->q, r->k, static_cast<const void*>(r->q_out), static_cast<const void*>(r->k_out)})
    if (misaligned(p, 2)) return cudaErrorInvalidValue;
  if (misaligned(r->q_weight, wa) || misaligned(r->k_weight, wa)) return cudaErrorInvalidValue;
  Tables tb;
  if (!fill_tables(&tb, r->turns, r->axis, r->pairs, r->axes)) return cudaErrorInvalidValue;

  bool vector = r->dim % 16 == 0 && (r->interleaved || r->pairs % 8 == 0) && !misaligned(r->q_weight, 16) && !misaligned(r->k_weight, 16);
  if (r->q_heads)
    vector = vector && !misaligned(r->q, 16) && !misaligned(r->q_out, 16) && r->q_stride_t % 8 == 0 && r->q_stride_h % 8 == 0 &&
             r->qo_stride_t % 8 == 0 && r->qo_stride_h % 8 == 0;
  if (r->k_heads)
    vector = vector && !misaligned(r->k, 16) && !misaligned(r->k_out, 16) && r->k_stride_t % 8 == 0 && r->k_stride_h % 8 == 0 &&
             r->ko_stride_t % 8 == 0 && r->ko_stride_h % 8 == 0;
  const int lanes = !vector ? 0 : r->dim <= 64 ? 4 : r->dim <= 128 ? 8 : 16;

  Args a{};
  a.q = r->q, a.k = r->k, a.qo = r->q_out, a.ko = r->k_out;
  a.qw = norm ? (r->q_weight ? r->q_weight : r->k_weight) : nullptr;
  a.kw = norm ? (r->k_weight ? r->k_weight : r->q_weight) : nullptr;
  a.positions = r->positions;
  a.q_token = r->q_stride_t, a.q_head = r->q_stride_h, a.k_token = r->k_stride_t, a.k_head = r->k_stride_h;
  a.qo_token = r->qo_stride_t, a.qo_head = r->qo_stride_h, a.ko_token = r->ko_stride_t, a.ko_head = r->ko_stride_h;
  a.tokens = r->tokens;
  a.q_heads = r->q_heads, a.k_heads = r->k_heads, a.dim = r->dim, a.pairs = r->pairs, a.axes = r->axes;
  a.float_positions = r->float_positions;
  a.eps = r->eps;
  a.sign = r->inverse ? -1.0f : 1.0f;
  // Rows (a token's head) that a CTA's threads take at once are a step; a tile is as many steps
  // as leave every SM work: 1, 2, 4, 8 or 16, by the steps that an SM has in all.  Longer
  // tiles share a token's sines and overlap more, shorter ones spread over the SMs.  Us with
  // 1 / 2 / 4 / 8 / 16 (heads of 128, normalised; steps an SM):
  //   64 tokens, 8 heads (0.1): 3.3 / 3.9 / 5.5 / 5.5 / 5.5;  1024, 8 (1.7): 3.9 / 4.2 / 5.8 / 5.7 / 5.6
  //   2048, 8 (3.5): 5.6 / 4.7 / 5.8 / 5.9 / 5.8;  256, 112 (6.1): 8.3 / 7.2 / 6.1 / 7.4 / 11.8
  //   1024, 112 (24): 21.9 / 15.6 / 14.9 / 15.3 / 14.9;  16384, 32 (111): 85.6 / 61.3 / 58.8 / 60.5 / 64.0
  //   8192, 112 (194): 163 / 111 / 103 / 97.1 / 98.5;  16384, 112 (387): 321 / 218 / 203 / 189 / 180
  // heads of 64: 2048, 112 (24): 20.8 / 15.1 / 14.4 / 14.8 / 16.3;  16384, 112 (194): 160 / 110 / 102 / 96.2 / 96.6
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return cudaErrorInvalidDevice;
  const int step = lanes ? kThreads / lanes : kThreads / 32, heads = r->q_heads + r->k_heads;
  const int64_t per_sm = r->tokens * heads / (int64_t(step) * sms);
  const int want = step * (per_sm < 2 ? 1 : per_sm < 6 ? 2 : per_sm < 144 ? 4 : per_sm < 288 ? 8 : 16);
  a.chunk = heads < want ? heads : want;
  a.tile = a.chunk == heads ? want / heads : 1;
  if (a.tile > kMaxTile) a.tile = kMaxTile;
  if (a.tile < 1) a.tile = 1;
  if (a.tile > r->tokens) a.tile = int(r->tokens);
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  if (r->type == 0)
    return r->weight_type == 2 ? launch<__nv_bfloat16, float>(a, tb, lanes, r->interleaved != 0, stream)
                               : launch<__nv_bfloat16, __nv_bfloat16>(a, tb, lanes, r->interleaved != 0, stream);
  return r->weight_type == 2 ? launch<__half, float>(a, tb, lanes, r->interleaved != 0, stream)
                             : launch<__half, __half>(a, tb, lanes, r->interleaved != 0, stream);
}

H3SK_EXPORT int h3_rope_table_run(const void* positions, const double* turns, const int* axis, void* out, int64_t tokens,
                                  int pairs, int axes, int float_positions, uintptr_t stream_ptr) {
  using namespace h3sk::rope;
  if (tokens < 0 || tokens > int64_t(1) << 40 || pairs < 1 || pairs > kMaxPairs || axes < 1 || axes > 255 || !turns || !axis)
    return cudaErrorInvalidValue;
  Tables tb;
  if (!fill_tables(&tb, turns, axis, pairs, axes)) return cudaErrorInvalidValue;
  if (tokens == 0) return cudaSuccess;
  if (!positions || !out || misaligned(positions, 4) || misaligned(out, 8)) return cudaErrorInvalidValue;
  Args a{};
  a.positions = positions;
  a.tokens = tokens;
  a.pairs = pairs, a.axes = axes;
  a.float_positions = float_positions;
  const int at_once = kThreads / pairs;
  int grid = 0;
  // (a step past the end must fit too: up to two grids of tokens)
  const bool narrow = (tokens + (int64_t(1) << 20)) * (4 * pairs > axes ? 4 * pairs : axes) <= INT_MAX;
  auto* const kernel = float_positions ? (narrow ? rope_table<float, int> : rope_table<float, int64_t>)
                                       : (narrow ? rope_table<int, int> : rope_table<int, int64_t>);
  const cudaError_t e = h3sk::rq_persistent_grid(reinterpret_cast<const void*>(kernel), kThreads, 0,
                                                 (tokens + at_once - 1) / at_once, &grid);
  if (e != cudaSuccess) return e;
  kernel<<<grid, kThreads, 0, reinterpret_cast<cudaStream_t>(stream_ptr)>>>(a, tb, static_cast<uint2*>(out));
  return cudaGetLastError();
}

H3SK_EXPORT const char* h3_rope_error(int code) { return cudaGetErrorString(static_cast<cudaError_t>(code)); }
