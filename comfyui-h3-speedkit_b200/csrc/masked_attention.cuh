// Attention under document, padding, causal and prefix masks, with scores capped by
// a tanh and a bias by distance, on B200 (sm_100a).
//
//   s_ij = scale * (q_i . k_j);  s_ij = cap * tanh(s_ij / cap);  s_ij -= slope_h * |pos_i - j|
//   out_i = sum_j exp(s_ij) v_j / sum_j exp(s_ij),  lse_i = ln sum_j exp(s_ij),  j in [lo_i, hi_i)
//
// Every mask is an interval of keys per query: a document's keys, the valid keys of
// a padded sequence, and under a causal mask the keys up to the query's own place or
// the document's prefix.  A row without a visible key gives zeros and lse = -inf;
// rows that belong to no sequence are left as they were.
//
// One pass over the keys (online softmax in the base-2 domain).  A stream is 128 query rows
// (a TMEM lane each); a step of it takes 64 keys: S = Q K^T (kind::f16, FP32 in TMEM), a
// warpgroup turns S into P, O += P V.
//   * pair form: a CTA runs two streams, two tiles of rows that share every 128-key block
//     of K and V;
//   * single form: a CTA runs one stream on 64-key blocks with half of an SM's shared
//     memory and TMEM, so that two CTAs hide each other's beginnings, ends and waits.
// Query heads that share a K/V head lie side by side in one tile (row = token x head), so
// a block is read once for all of them; a long key axis with few rows is also split over
// CTAs, whose partial results a second kernel joins in a fixed order.
//
// Arithmetic: scores, maxima, sums and O are FP32.  P is rounded to the inputs' type, which
// the second product wants: half a step of every weight, against a sum of the unrounded
// ones.  P refers to a row maximum that is only moved when it grew by more than 2^8 (P and
// the sums carry the factor, the end divides it out), so O is rescaled in the first steps
// and hardly ever after.  An eighth of the exponentials takes a polynomial (1.1e-7
// relative) beside the exp2 unit.
//
// Roles, warp by warp: four of softmax a stream (thread = query row), the TMA producer, an
// MMA issuer a stream (the first owns the TMEM), the V check: in a block that some row does
// not see whole, P is 0 in masked places but 0 * inf is not, so values that are not finite
// are cleared from the staged V there, and the epilogue adds them to the rows that do see
// them.
//
// What it runs into: by clocks of a timing copy a step's softmax takes 900 clocks alone
// and 1300 beside the other stream's, its two products 620 (128 x 64 x 16 reads both
// operands from shared memory at 54 clocks where 32 would compute it); the exp2 unit
// (16 a clock and SM) wants 380 of them and the FP32 pipe as many.  Runs of more than a few
// milliseconds meet the 1000 W cap, and the clock falls to 1.6 GHz: 16384 x 16384 tokens, 16
// heads of 128, take 1685 us after a pause (1305 TFLOP/s) and 1930 to 2000 in a row; 8192 x
// 8192, 24 heads 701 and 760 to 800.  Few rows are bound by reading K and V: 1 query, 56 over 8
// heads, 32768 keys, batch 2: 50 us, 5.4 TB/s.  Tried and slower:
// S of 128 keys with P over it (the products of a stream wait for its softmax: 2.1 us a
// block of a pair, then 2.0 and 1.9 in short runs), two threads a row (2.2), P handed on a
// step late, and exponentials before the maximum is known (both 2.0).
//
// Every wait is bounded and reports a status code.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "host_util.h"
#include "sm100.cuh"
#include "wide_types.cuh"

namespace h3sk {
namespace mattn {

using namespace sm100;

constexpr int kRows = 128;   // query rows per stream (TMEM lanes)
constexpr int kStep = 64;    // keys per step of a stream
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
enum { kCap = 1, kDistance = 2 };
// Of eight pairs of exponentials so many take the polynomial.  None / one / two, us, after
// pauses: 16384 x 16384, 16 heads (pairs of tiles) 1797 / 1685 / 1712; 8192 x 8192, 24 heads of
// 64 600 / 589 / 595; single tiles of 128 channels hardly care: 8192 x 8192, 24 heads 700 / 701 /
// 706, 16384 x 16384, 8 heads 901 / 904 / 914.  Under a cap, whose tanh wants the same pipe, none:
// causal 6000 x 6000 with a prefix, 8 over 2 heads 111, with one 123, with two 124.
constexpr int poly_of_8(int feat) { return feat & kCap ? 0 : 1; }
constexpr float kGrowth = 8.0f;   // the row maximum may lag this far (in powers of two)

struct Args {
  int batch, q_len, k_len;
  int groups, pack, tile_tokens;   // head groups, heads per group, tokens per 128-row tile
  int heads, groups_per_kv;        // query heads; groups that share a K/V head
  int tiles, q_tiles;              // CTAs along the rows; 128-row tiles
  int splits, causal;
  int q_bmul, k_bmul, k_hmul, v_bmul, v_hmul;   // 0 where a tensor is shared along that dimension
  int documents;
  const int *q_offsets, *k_offsets, *q_lengths, *k_lengths, *prefix;
  const float* slopes;
  float scale_log2;                // scale * log2(e); with a cap: scale / cap * 2 log2(e)
  float cap_log2, cap_y;           // cap * log2(e), scale / cap
  void* out;
  int64_t o_sb, o_ss, o_sh;
  float* lse;                      // [B, H, Sq] or null
  const void* v;
  int64_t v_sb, v_ss, v_sh;
  int fill;                        // rows of no sequence: 0 left as they are, 1 written as zeros
  float* part;                     // [splits][B, Sq, H, D], then [splits][B, Sq, H] (lse in base 2)
  float* part_lse;
  int* status;
};

// The two forms of a CTA.  Pair: two streams, blocks of 128 keys for both; 168 registers a
// thread (a thirteenth warp would leave 128).  Else one stream, blocks of 64 keys, half the
// shared memory and TMEM: two CTAs an SM.
template <bool kPair>
struct Form {
  static constexpr int kStreams = kPair ? 2 : 1, kCtas = kPair ? 1 : 2;
  static constexpr int kBlock = kPair ? 128 : 64;
  static constexpr int kSoftWarps = 4 * kStreams;
  static constexpr int kProducerWarp = kSoftWarps, kMmaWarp = kProducerWarp + 1, kCheckWarp = kMmaWarp + kStreams;
  static constexpr int kThreads = 32 * (kCheckWarp + 1);
  // TMEM columns: one S of 64 keys a stream (free again as soon as it is in registers), two
  // P of 32 columns a stream, O.  Nothing lies over anything else.
  static constexpr uint32_t kP = 64 * kStreams, kO = 128 * kStreams, kColumns = 256 * kStreams;
};

template <int D, bool kPair>
struct Smem {
  using F = Form<kPair>;
  static constexpr int kTileQ = kRows * D * 2, kTile = F::kBlock * D * 2;
  static constexpr int kKStages = D == 128 ? 2 : 4, kVStages = !kPair && D == 128 ? 2 : D == 128 ? 3 : 4;
  uint8_t q[F::kStreams][kTileQ];
  uint8_t k[kKStages][kTile];
  uint8_t v[kVStages][kTile];
  uint64_t q_full;
  uint64_t k_full[kKStages], k_empty[kKStages];
  uint64_t v_full[kVStages], v_ok[kVStages], v_empty[kVStages];
  uint64_t s_full[F::kStreams], s_empty[F::kStreams], p_full[F::kStreams][2], pv_done[F::kStreams], done;   // P: step & 1
  int4 seen[F::kSoftWarps];        // a softmax warp's lowest and highest ends: lo min, lo max, hi min, hi max
  int bad;                         // a V value that is not finite and that some row sees, in a partly seen block
  uint32_t tmem;
  int abort;
  // an output row of every softmax thread crosses over the operand tiles
  static constexpr int kStage = 32 * (D * 4 + 16);
};

// The MMA warp runs its loop converged, so that descriptors stay in uniform registers;
// one elected lane (`lead`) issues.  (A single-lane branch cost 80 to 100 clocks a
// tcgen05.mma on moves to uniform registers, more than the 64 that it computes for.)
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t lead;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(lead));
  return lead;
}
__device__ __forceinline__ void mma_f16_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void commit_led(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_addr(bar)),
      "r"(lead)
      : "memory");
}
// kind::f16 instruction descriptor, FP32 accumulator; bit 16: B is N-major.
template <typename T>
constexpr uint32_t idesc_f16(int m, int n, bool b_n_major) {
  const uint32_t t = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | (uint32_t(b_n_major) << 16) | (uint32_t(n >> 3) << 17) |
         (uint32_t(m >> 4) << 24);
}
// N-major B tile as TMA writes it: [keys][64 channels] boxes of 128-byte rows, 128-byte
// swizzle; 8-key groups 1024 bytes apart (stride offset), 64-channel boxes one box of
// kBlock keys apart (leading offset).
template <int kBlock>
__device__ __forceinline__ uint64_t smem_desc_n_sw128(const void* tile) {
  const uint64_t start = (smem_addr(tile) >> 4) & 0x3FFFu;
  return start | (uint64_t((kBlock * 128) >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w,
                                            int u) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(u)
      : "memory");
}

// The last document that begins at or before token i (0 if none does); by a whole warp,
// whose first lane has the smallest i.  32 offsets at a time, then on from there.
__device__ __forceinline__ int document_of(const Args& a, int i) {
  const int lane = threadIdx.x & 31, i0 = __shfl_sync(0xffffffffu, i, 0);
  int first = 0, n = a.documents;   // the document lies in [first, first + n)
  while (n > 1) {
    const int step = (n + 31) >> 5, at = first + lane * step;
    const uint32_t before = __ballot_sync(0xffffffffu, lane * step < n && __ldg(a.q_offsets + at) <= i0);
    const int last = max(31 - __clz(before), 0);
    first += last * step;
    n = min(step, n - last * step);
  }
  for (int steps = 0; first + 1 < a.documents && __ldg(a.q_offsets + first + 1) <= i; ++steps, ++first) {
    if (steps < 32) continue;
    // (a long run of empty documents: by halves)
    int last = a.documents;
    while (last - first > 1) {
      const int mid = first + (last - first) / 2;
      if (__ldg(a.q_offsets + mid) <= i)
        first = mid;
      else
        last = mid;
    }
    break;
  }
  return first;
}

// The keys [lo, hi) that query token i of batch b sees, and its place among them
// (for the distance); false for a token of no sequence.  By whole warps.
__device__ __forceinline__ bool visible(const Args& a, int b, int i, int& lo, int& hi, int& pos) {
  lo = hi = pos = 0;
  const int first = a.documents ? document_of(a, i) : 0;
  if (i >= a.q_len) return false;
  int local = i, qlen = a.q_len, klen = a.k_len, seq = b;
  if (a.documents) {
    const int begin = __ldg(a.q_offsets + first), end = __ldg(a.q_offsets + first + 1);
    if (i < begin || i >= end) return false;
    seq = first;
    local = i - begin;
    qlen = end - begin;
    lo = min(max(__ldg(a.k_offsets + first), 0), a.k_len);
    klen = min(max(__ldg(a.k_offsets + first + 1), lo), a.k_len) - lo;
  } else {
    if (a.q_lengths) qlen = min(max(__ldg(a.q_lengths + b), 0), a.q_len);
    if (a.k_lengths) klen = min(max(__ldg(a.k_lengths + b), 0), a.k_len);
    if (i >= qlen) return false;
  }
  pos = lo + local + klen - qlen;
  int seen = klen;
  if (a.causal) {
    const int prefix = a.prefix ? __ldg(a.prefix + seq) : 0;
    seen = min(klen, max(max(prefix, pos - lo + 1), 0));
  }
  hi = lo + seen;
  return true;
}

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* abort, int* status, int code) {
  return wait_sleep(bar, parity, reinterpret_cast<volatile int*>(abort), status, code);
}

// The same by a whole warp, with one verdict.
__device__ __forceinline__ bool all_wait(uint64_t* bar, uint32_t parity, int* abort, int* status, int code) {
  return __all_sync(0xffffffffu, wait(bar, parity, abort, status, code));
}

// The upper bits of a word's halves that are not finite values of the type.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t exponent = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t carry = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  return ((w & exponent) + carry) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ uint32_t not_finite(const uint4& w) {
  return not_finite<T>(w.x) | not_finite<T>(w.y) | not_finite<T>(w.z) | not_finite<T>(w.w);
}

// Clears a stage's values that are not finite, by a warp, and notes whether some row may see
// one: those behind the last that one does, padding most of all, hold anything.
template <typename T, int D, bool kPair>
__device__ __forceinline__ void clear_not_finite(Smem<D, kPair>& sm, int stage, int key0, int hi_max) {
  constexpr int kBlock = Form<kPair>::kBlock;
  uint4* tile_v = reinterpret_cast<uint4*>(sm.v[stage]);
#pragma unroll 1
  for (int c = threadIdx.x & 31; c < Smem<D, kPair>::kTile / 16; c += 32) {
    uint4 w = tile_v[c];
    if (!not_finite<T>(w)) continue;
    uint32_t* u = &w.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] &= ~((not_finite<T>(u[e]) >> 15) * 0xffffu);
    tile_v[c] = w;
    const int key = key0 + ((c >> 3) & (kBlock - 1));   // (boxes of 64 channels, 128 bytes a key)
    if (key < hi_max) sm.bad = 1;
  }
  fence_async_shared();
}

// FP16 probabilities are scaled by 2^7, away from that type's subnormals.
template <typename T>
__device__ constexpr float bias_of() {
  return std::is_same<T, __half>::value ? 7.0f : 0.0f;
}

// One warpgroup's thread: the softmax of its row's scores against each block, then
// the epilogue.
template <typename T, int D, int kFeat>
struct Softmax {
  static constexpr float kBias = bias_of<T>();

  // The terms of cap R(z), R(y^2) y = tanh(y) for |y| <= 1: six of the least largest relative
  // error (by Lawson's reweighted least squares), rounded to FP32, 6.1e-7 of the value, so that
  // small scores under a high cap keep their digits.
  struct Cap {
    uint64_t y, c[6];
    __device__ __forceinline__ explicit Cap(const Args& a) {
      const float terms[6] = {0.9999994039535522f,   -0.3332904279232025f,  0.13281433284282684f,
                              -0.051605671644210815f, 0.016743114218115807f, -0.0030670599080622196f};
      y = pkf(a.cap_y, a.cap_y);
#pragma unroll
      for (int i = 0; i < 6; ++i) c[i] = pkf(terms[i] * a.cap_log2, terms[i] * a.cap_log2);
    }
    // cap tanh + add of a pair of raw products
    __device__ __forceinline__ uint64_t operator()(uint64_t s, uint64_t add) const {
      const uint64_t t = mul2(s, y), z = mul2(t, t);
      uint64_t r = fma2(z, c[5], c[4]);
#pragma unroll
      for (int i = 3; i >= 0; --i) r = fma2(r, z, c[i]);
      return fma2(t, r, add);
    }
  };
  // Scores in base 2 of 32 keys from key0 on, from the raw products.  cap tanh(y) comes
  // without the exp2 unit where |y| are at most 1 (`small`); elsewhere as
  // cap - 2 cap / (1 + e^(2y)), whose absolute error is a few 2^-24 of the cap too.
  static __device__ __forceinline__ void transform(uint32_t (&u)[32], const Args& a, const Cap& cap, bool small, float slope,
                                                   int pos, int key0) {
    if constexpr (kFeat & kCap) {
      if (small) {
#pragma unroll
        for (int c = 0; c < 32; c += 2) upk(cap(pk(u[c], u[c + 1]), 0ull), u[c], u[c + 1]);
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float s = __uint_as_float(u[c]) * a.scale_log2;
          u[c] = __float_as_uint(fmaf(-2.0f * a.cap_log2, rcp(1.0f + ex2(s)), a.cap_log2));
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < 32; ++c) u[c] = __float_as_uint(__uint_as_float(u[c]) * a.scale_log2);
    }
    if constexpr (kFeat & kDistance) {
      const float d0 = float(pos - key0);
#pragma unroll
      for (int c = 0; c < 32; ++c) u[c] = __float_as_uint(fmaf(-slope, fabsf(d0 - float(c)), __uint_as_float(u[c])));
    }
  }
  // Whether the row's products stay within |y| <= 1 (NaN does not).  The choice moves last
  // bits, and masked places hold anything.  So in a block that some row does not see whole
  // each row chooses for itself, by what it sees; elsewhere the warp's rows, which see the
  // same keys, choose together, but for those of no sequence (`idle`: a bit each).
  template <bool kPart>
  static __device__ __forceinline__ bool is_small(const uint32_t (&x0)[32], const uint32_t (&x1)[32], const Args& a,
                                                   uint32_t idle, int from, int to) {
    const uint32_t seen0 = seen(from, to), seen1 = seen(from - 32, to - 32);
    const auto at = [](uint32_t x, uint32_t seen, int c) { return !kPart || (seen >> c) & 1u ? fabsf(__uint_as_float(x)) : 0.0f; };
    float m[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
      m[(c >> 1) & 1] = max3_nan(m[(c >> 1) & 1], at(x0[c], seen0, c), at(x0[c + 1], seen0, c + 1));
      m[2 + ((c >> 1) & 1)] = max3_nan(m[2 + ((c >> 1) & 1)], at(x1[c], seen1, c), at(x1[c + 1], seen1, c + 1));
    }
    const bool fits = max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3])) * a.cap_y <= 1.0f;
    return kPart ? fits : (__ballot_sync(0xffffffffu, fits) | idle) == 0xffffffffu;
  }
  // bits of the places [from, to) of 32 keys
  static __device__ __forceinline__ uint32_t seen(int from, int to) {
    const int f = min(max(from, 0), 32), e = min(max(to, 0), 32);
    const uint32_t below = e == 32 ? 0xffffffffu : (1u << e) - 1u, skip = f == 32 ? 0xffffffffu : (1u << f) - 1u;
    return below & ~skip;
  }
  // -inf in the places outside [from, to) of 32 keys
  static __device__ __forceinline__ void mask(uint32_t (&u)[32], int from, int to) {
    const uint32_t in = seen(from, to);
#pragma unroll
    for (int c = 0; c < 32; ++c) u[c] = (in >> c) & 1u ? u[c] : 0xff800000u;
  }
  // what is taken off the scores before the exponential, twice
  static __device__ __forceinline__ uint64_t reference(float m) {
    const float ref = kBias - (m == -INFINITY ? 0.0f : m);
    return pkf(ref, ref);
  }
  static __device__ __forceinline__ void scores(uint32_t (&u)[32], const Args& a, const Cap& cap, bool small, float slope,
                                                int pos, int key0, bool part, int from, int to) {
    if (kFeat) transform(u, a, cap, small, slope, pos, key0);
    if (part) mask(u, from, to);
  }
  // P of 32 keys, as the type's pairs in 16 words, and its sum before rounding; from scores
  // or, with kRaw, from raw products within the cap's polynomial
  template <bool kRaw = false>
  static __device__ __forceinline__ void probabilities(const uint32_t (&s)[32], uint64_t scale2, uint64_t ref2,
                                                       uint64_t (&sum2)[2], uint32_t (&p)[16], const Cap* cap = nullptr) {
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const uint64_t x = kRaw ? (*cap)(pk(s[2 * c], s[2 * c + 1]), ref2) : fma2(pk(s[2 * c], s[2 * c + 1]), scale2, ref2);
      float e0, e1;
      if ((c & 7) >= 8 - poly_of_8(kFeat)) {
        exp2_pair(x, e0, e1);
      } else {
        uint32_t x0, x1;
        upk(x, x0, x1);
        e0 = ex2(__uint_as_float(x0)), e1 = ex2(__uint_as_float(x1));
      }
      sum2[c & 1] = add2(sum2[c & 1], pkf(e0, e1));
      p[c] = pack2<T>(e0, e1);
    }
  }
  static __device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
  }
  static __device__ __forceinline__ void maximum(float (&m)[4], const uint32_t (&u)[32]) {
#pragma unroll
    for (int c = 0; c < 32; c += 8)
#pragma unroll
      for (int e = 0; e < 4; ++e) m[e] = max3_nan(m[e], __uint_as_float(u[c + 2 * e]), __uint_as_float(u[c + 2 * e + 1]));
  }
  // 2^x of a pair without the exp2 unit: x = n + f with |f| <= 1/2 (the sum with
  // 1.5 * 2^23 rounds), a polynomial for 2^f (degree 5, 1 at 0, of the least largest relative
  // error by Lawson's reweighted least squares, rounded to FP32: 1.1e-7)
  // and n added to its exponent.  x <= 16; from -127 down, -inf among it, the result is
  // exactly 0, as a masked key's has to be.  NaN is lost: the caller sees to it.
  static __device__ __forceinline__ void exp2_pair(uint64_t x, float& e0, float& e1) {
    uint32_t x0, x1, t0, t1, p0, p1;
    upk(x, x0, x1);
    x = pkf(fmaxf(__uint_as_float(x0), -127.0f), fmaxf(__uint_as_float(x1), -127.0f));
    const uint64_t magic = pkf(12582912.0f, 12582912.0f), unmagic = pkf(-12582912.0f, -12582912.0f);
    const uint64_t t = add2(x, magic);
    const uint64_t f = fma2(add2(t, unmagic), pkf(-1.0f, -1.0f), x);
    uint64_t p = pkf(0.0013264723820611835f, 0.0013264723820611835f);
    p = fma2(p, f, pkf(0.009671512991189957f, 0.009671512991189957f));
    p = fma2(p, f, pkf(0.05550733581185341f, 0.05550733581185341f));
    p = fma2(p, f, pkf(0.24022242426872253f, 0.24022242426872253f));
    p = fma2(p, f, pkf(0.6931470036506653f, 0.6931470036506653f));
    p = fma2(p, f, pkf(1.0f, 1.0f));
    upk(t, t0, t1);
    upk(p, p0, p1);
    e0 = __uint_as_float(p0 + (t0 << 23));
    e1 = __uint_as_float(p1 + (t1 << 23));
  }
};

// A thread's row and its keys; the CTA's split of the keys: where it begins, its blocks.
struct Row {
  int batch, token, head, kv_head, lo, hi;
  bool valid, blank;               // of a sequence; of none, to be written as zeros
  int split, first_key, blocks, lo_max, hi_min;
};

// The rows' results from O, the reference maximum and the sum.
template <typename T, int D, bool kPair>
__device__ __forceinline__ void epilogue(const Args& a, Smem<D, kPair>& sm, uint32_t tmem, const Row& at, float m, float l,
                                         bool ok) {
  using F = Form<kPair>;
  using Smem_ = Smem<D, kPair>;
  const int warp = int(threadIdx.x) >> 5, stream = warp >> 2;
  const int batch = at.batch, token = at.token, head = at.head, lo = at.lo, hi = at.hi, kv_head = at.kv_head;
  const int split = at.split, first_key = at.first_key, blocks = at.blocks;
  const bool valid = at.valid, blank = at.blank;
  const int lo_max = at.lo_max, hi_min = at.hi_min;
  const auto partial = [&](int j) {
    return first_key + j * F::kBlock < lo_max || first_key + (j + 1) * F::kBlock > hi_min;
  };
  if (!ok) return;
  tc_fence_after();
  const bool none = l == 0.0f;
  const float inv = none ? 0.0f : 1.0f / l;
  const float lse2 = blank ? 0.0f : none ? -INFINITY : m - bias_of<T>() + log2f(l);
  const int64_t row = (int64_t(batch) * a.q_len + token) * a.heads + head;
  if (a.splits > 1) {
    if (valid) a.part_lse[int64_t(split) * a.batch * a.q_len * a.heads + row] = lse2;
  } else if ((valid || blank) && a.lse) {
    a.lse[(int64_t(batch) * a.heads + head) * a.q_len + token] = lse2 * kLn2;
  }
  const bool bad = sm.bad != 0;
  // A thread has a row, a warp's stores want consecutive bytes: the warp's 32 rows cross in
  // shared memory (operand tiles are free now), 16 bytes apart more than a row for the
  // banks, and leave row by row.  (Stores straight from the rows' threads took 14,500
  // clocks a CTA.)
  static_assert(F::kSoftWarps * Smem<D, kPair>::kStage <= offsetof(Smem_, q_full), "output rows");
  const bool whole = a.splits == 1;                  // else FP32 partial results
  const int row_bytes = D * (whole ? 2 : 4), pitch = row_bytes + 16;
  uint8_t* stage = reinterpret_cast<uint8_t*>(&sm) + warp * Smem<D, kPair>::kStage;
  const int lane = threadIdx.x & 31;
  const uint32_t t_o = tmem + (uint32_t((warp & 3) * 32) << 16) + F::kO + uint32_t(D) * stream;
#pragma unroll 1
  for (int c = 0; c < D; c += 32) {
    uint32_t u[32];
    float f[32];
    // (without a block there is no O: its columns hold what was there before)
    if (blocks > 0) {
      tmem_load_32cols(t_o + c, u);
      tmem_load_wait();
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) f[e] = blocks > 0 && !none && valid ? __uint_as_float(u[e]) * inv : 0.0f;
    if (valid && bad) {
      // values that are not finite, cleared from partly seen blocks, where this row sees them
      const T* v = static_cast<const T*>(a.v) + int64_t(batch * a.v_bmul) * a.v_sb + int64_t(kv_head * a.v_hmul) * a.v_sh + c;
      const int end = min(hi, first_key + blocks * F::kBlock);
#pragma unroll 1
      for (int key = max(lo, first_key); key < end; ++key) {
        const int j = (key - first_key) / F::kBlock;
        if (!partial(j)) {   // on to the next block
          key = first_key + (j + 1) * F::kBlock - 1;
          continue;
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float y = to_float(v[int64_t(key) * a.v_ss + e]);
          if (!(fabsf(y) < INFINITY)) f[e] += y;
        }
      }
    }
    __syncwarp();
    if (whole) {
      uint4* dst = reinterpret_cast<uint4*>(stage + lane * pitch + c * 2);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        dst[e] = make_uint4(pack2<T>(f[8 * e], f[8 * e + 1]), pack2<T>(f[8 * e + 2], f[8 * e + 3]),
                            pack2<T>(f[8 * e + 4], f[8 * e + 5]), pack2<T>(f[8 * e + 6], f[8 * e + 7]));
    } else {
      float4* dst = reinterpret_cast<float4*>(stage + lane * pitch + c * 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
    }
  }
  __syncwarp();
  // where the row begins in the output, or null
  uint8_t* const to = !(valid || (blank && whole)) ? nullptr
                      : whole ? static_cast<uint8_t*>(a.out) +
                                    (int64_t(batch) * a.o_sb + int64_t(token) * a.o_ss + int64_t(head) * a.o_sh) * 2
                              : reinterpret_cast<uint8_t*>(a.part) +
                                    ((int64_t(split) * a.batch * a.q_len * a.heads + row) * D) * 4;
  const int lanes_a_row = row_bytes / 16, rows_at_once = 32 / lanes_a_row;   // 8 to 32 lanes
  const int lane_row = lane / lanes_a_row, lane_at = (lane % lanes_a_row) * 16;
#pragma unroll 8
  for (int rr = 0; rr < 32; rr += rows_at_once) {
    uint8_t* const dst = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), rr + lane_row));
    const uint4 x = *reinterpret_cast<const uint4*>(stage + (rr + lane_row) * pitch + lane_at);
    if (dst) *reinterpret_cast<uint4*>(dst + lane_at) = x;
  }
}

template <typename T, int D, int kFeat, bool kPair>
__global__ void __launch_bounds__(Form<kPair>::kThreads, Form<kPair>::kCtas)
    masked_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                            const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args a) {
  using F = Form<kPair>;
  using S = Smem<D, kPair>;
  using Soft = Softmax<T, D, kFeat>;
  extern __shared__ uint8_t smem_raw[];
  S& sm = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  // The CTA's tile, head group, batch and split.  Tiles of one head follow one another
  // and share its keys in L2, unless they differ in work: under a causal mask the
  // heaviest come first, and a long document's tiles of all heads start together (16
  // over 4 heads, 21 documents in 12288 tokens: 176 us by heads, 172 by tiles, then).
  int id = int(blockIdx.x), tile, group, rest;
  const int per_batch = a.groups * a.splits;
  if (a.causal || a.documents) {
    const int others = per_batch * a.batch;
    tile = id / others;
    rest = id - tile * others;
    if (!a.documents) tile = a.tiles - 1 - tile;
    group = rest % a.groups;
    rest /= a.groups;
  } else {
    tile = id % a.tiles;
    rest = id / a.tiles;
    group = rest % a.groups;
    rest /= a.groups;
  }
  const int split = rest % a.splits, batch = rest / a.splits;
  const int kv_head = group / a.groups_per_kv;

  if (threadIdx.x == F::kProducerWarp * 32) {
    mbar_init(&sm.q_full, 1);
    for (int s = 0; s < S::kKStages; ++s) {
      mbar_init(&sm.k_full[s], 1);
      mbar_init(&sm.k_empty[s], F::kStreams);
    }
    for (int s = 0; s < S::kVStages; ++s) {
      mbar_init(&sm.v_full[s], 1);
      mbar_init(&sm.v_ok[s], 1);
      mbar_init(&sm.v_empty[s], F::kStreams);
    }
    for (int t = 0; t < F::kStreams; ++t) {
      mbar_init(&sm.s_full[t], 1);
      mbar_init(&sm.s_empty[t], 4);
      mbar_init(&sm.p_full[t][0], 4);
      mbar_init(&sm.p_full[t][1], 4);
      mbar_init(&sm.pv_done[t], 1);
    }
    mbar_init(&sm.done, F::kStreams);
    sm.bad = sm.abort = 0;
    fence_mbar_init();
    tma_prefetch_map(&map_k);
    tma_prefetch_map(&map_v);
    fence_async_shared();
    // Q sets out before the CTA knows its keys
    const uint32_t q_bytes = uint32_t(a.tile_tokens * a.pack) * D * 2;
    const int q_first = F::kStreams * tile, q_count = min(F::kStreams, a.q_tiles - q_first);
    mbar_arrive_expect_tx(&sm.q_full, q_count * q_bytes);
    for (int t = 0; t < q_count; ++t)
      for (int x = 0; x < D / 64; ++x)
        tma_load_5d(sm.q[t] + x * 128 * 128, &map_q, &sm.q_full, 64 * x, 0, (q_first + t) * a.tile_tokens, group,
                    batch * a.q_bmul);
  }
  if (warp == F::kMmaWarp) {
    tmem_alloc(&sm.tmem, F::kColumns);
    tmem_relinquish();
  }
  // the row of a softmax thread and its keys
  const int stream = warp >> 2;
  const int r = threadIdx.x & 127;
  const int q_tile = F::kStreams * tile + stream;
  int token = 0, head = 0, lo = 0, hi = 0, pos = 0;
  bool valid = false, blank = false;
  if (warp < F::kProducerWarp) {
    token = q_tile * a.tile_tokens + r / a.pack;
    head = group * a.pack + r % a.pack;
    valid = visible(a, batch, token, lo, hi, pos);
    blank = a.fill && !valid && token < a.q_len && r < a.tile_tokens * a.pack;
    valid = valid && r < a.tile_tokens * a.pack;
    const bool some = valid && hi > lo;
    // a row that sees nothing makes every block a partly seen one
    const int lo_min = __reduce_min_sync(0xffffffffu, some ? lo : INT_MAX);
    const int hi_max = __reduce_max_sync(0xffffffffu, some ? hi : 0);
    const int lo_max = __reduce_max_sync(0xffffffffu, valid ? (some ? lo : INT_MAX) : 0);
    const int hi_min = __reduce_min_sync(0xffffffffu, valid ? hi : INT_MAX);
    if (lane == 0) sm.seen[warp] = make_int4(lo_min, lo_max, hi_min, hi_max);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  int lo_min = INT_MAX, lo_max = 0, hi_min = INT_MAX, hi_max = 0;
#pragma unroll
  for (int w = 0; w < F::kSoftWarps; ++w) {
    const int4 e = sm.seen[w];
    lo_min = min(lo_min, e.x), lo_max = max(lo_max, e.y), hi_min = min(hi_min, e.z), hi_max = max(hi_max, e.w);
  }
  // The CTA's key blocks, from the first key that a row of it sees (a document's tiles
  // need no mask then but at its end).
  int first_key = 0, blocks = 0, keys = 0;
  if (lo_min < hi_max) {
    const int n = (hi_max - lo_min + F::kBlock - 1) / F::kBlock, per = (n + a.splits - 1) / a.splits;
    first_key = lo_min + min(split * per, n) * F::kBlock;
    blocks = max(0, min(per, n - split * per));
    keys = max(0, min(hi_max - first_key, blocks * F::kBlock));
  }
  // a stream's steps: in pair form the halves of every block (but those behind the last
  // key)
  const int steps = (keys + kStep - 1) / kStep;
  const auto partial = [&](int j) {
    return first_key + j * F::kBlock < lo_max || first_key + (j + 1) * F::kBlock > hi_min;
  };

  if (warp >= F::kProducerWarp) {
    if (warp == F::kProducerWarp) {
      if (lane == 0) {
        // ---------------- TMA producer ----------------
        bool ok = true;
        int loaded_k = 0, loaded_v = 0;
        const auto load_k = [&](int j) {
          const int s = j % S::kKStages;
          if (j >= S::kKStages) ok = wait(&sm.k_empty[s], uint32_t(j / S::kKStages - 1) & 1u, &sm.abort, a.status, 81);
          if (!ok) return;
          mbar_arrive_expect_tx(&sm.k_full[s], S::kTile);
          for (int x = 0; x < D / 64; ++x)
            tma_load_4d(sm.k[s] + x * F::kBlock * 128, &map_k, &sm.k_full[s], 64 * x, first_key + j * F::kBlock, kv_head * a.k_hmul,
                        batch * a.k_bmul);
          loaded_k = j + 1;
        };
        const auto load_v = [&](int j) {
          const int s = j % S::kVStages;
          if (j >= S::kVStages) ok = wait(&sm.v_empty[s], uint32_t(j / S::kVStages - 1) & 1u, &sm.abort, a.status, 82);
          if (!ok) return;
          mbar_arrive_expect_tx(&sm.v_full[s], S::kTile);
          for (int x = 0; x < D / 64; ++x)
            tma_load_4d(sm.v[s] + x * F::kBlock * 128, &map_v, &sm.v_full[s], 64 * x, first_key + j * F::kBlock, kv_head * a.v_hmul,
                        batch * a.v_bmul);
          loaded_v = j + 1;
        };
        // in the order of use: K runs `ahead` blocks in front of V (S runs two steps
        // in front of P V)
        constexpr int ahead = kPair ? 1 : 2;
        for (int j = 0; ok && j < min(ahead, blocks); ++j) load_k(j);
        for (int j = 0; ok && j < blocks; ++j) {
          load_v(j);
          if (ok && j + ahead < blocks) load_k(j + ahead);
        }
        // every copy lands before the CTA exits
        mbar_wait_bounded(&sm.q_full, 0, nullptr, a.status, 83, kTimeoutNs);
        for (int j = max(0, loaded_k - S::kKStages); j < loaded_k; ++j)
          mbar_wait_bounded(&sm.k_full[j % S::kKStages], uint32_t(j / S::kKStages) & 1u, nullptr, a.status, 83, kTimeoutNs);
        for (int j = max(0, loaded_v - S::kVStages); j < loaded_v; ++j)
          mbar_wait_bounded(&sm.v_full[j % S::kVStages], uint32_t(j / S::kVStages) & 1u, nullptr, a.status, 83, kTimeoutNs);
      }
      __syncwarp();
    } else if (warp < F::kCheckWarp) {
      if (steps > 0) {
        // ---------------- MMA issuer of one stream ----------------
        // Per step: P V of the step before, then S of the step after, into columns that
        // the softmax has just emptied.  A warp of its own for each stream: the tensor
        // pipe queues hardly more than one MMA, so a wait for one stream would idle it.
        constexpr uint32_t kIdescS = idesc_f16<T>(kRows, kStep, false), kIdescO = idesc_f16<T>(kRows, D, true);
        const uint32_t lead = elect_lane();
        const int t = warp - F::kMmaWarp;
        bool ok = all_wait(&sm.q_full, 0, &sm.abort, a.status, 84);
        const uint64_t qd = smem_desc_k_sw128(sm.q[t]);
        // the block of a step, the half of it, and whether the step opens or closes it
        const auto block_of = [](int n) { return kPair ? n >> 1 : n; };
        const auto half_of = [](int n) { return kPair ? n & 1 : 0; };
        const auto opens = [](int n) { return !kPair || (n & 1) == 0; };
        const auto closes = [](int n) { return !kPair || (n & 1) == 1; };
        const auto issue_s = [&](int n) {
          const int j = block_of(n), s = j % S::kKStages;
          if (opens(n)) ok = all_wait(&sm.k_full[s], uint32_t(j / S::kKStages) & 1u, &sm.abort, a.status, 85);
          if (!ok) return;
          tc_fence_after();
          const uint64_t kd = smem_desc_k_sw128(sm.k[s]) + uint64_t(half_of(n) * ((kStep * 128) >> 4));
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t in_box = uint64_t(2 * (kk & 3));
            mma_f16_ss(lead, tmem + 64u * t, qd + uint64_t((kk >> 2) * ((kRows * 128) >> 4)) + in_box,
                       kd + uint64_t((kk >> 2) * ((F::kBlock * 128) >> 4)) + in_box, kIdescS, kk);
          }
          if (closes(n)) commit_led(lead, &sm.k_empty[s]);
          commit_led(lead, &sm.s_full[t]);
        };
        if (ok) issue_s(0);
        for (int n = 0; ok && n < steps; ++n) {
          if (n + 1 < steps) {
            ok = all_wait(&sm.s_empty[t], uint32_t(n) & 1u, &sm.abort, a.status, 92);
            if (ok) issue_s(n + 1);
            if (!ok) break;
          }
          const int j = block_of(n), s = j % S::kVStages;
          ok = (!opens(n) || all_wait(&sm.v_ok[s], uint32_t(j / S::kVStages) & 1u, &sm.abort, a.status, 86)) &&
               all_wait(&sm.p_full[t][n & 1], uint32_t(n >> 1) & 1u, &sm.abort, a.status, 87);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vd = smem_desc_n_sw128<F::kBlock>(sm.v[s]) + uint64_t(half_of(n) * ((kStep * 128) >> 4));
#pragma unroll
          for (int kk = 0; kk < kStep / 16; ++kk)
            mma_f16_ts(lead, tmem + F::kO + uint32_t(D) * t, tmem + F::kP + 64u * t + 32u * (n & 1) + 8u * kk,
                       vd + uint64_t(kk * (2048 >> 4)), kIdescO, uint32_t(n > 0 || kk > 0));
          if (closes(n)) commit_led(lead, &sm.v_empty[s]);
          commit_led(lead, &sm.pv_done[t]);
        }
        // every MMA completes before the epilogue and before TMEM is released
        commit_led(lead, &sm.done);
        mbar_wait_bounded(&sm.done, 0, nullptr, a.status, 88, kTimeoutNs);
      }
      __syncwarp();
    } else {
      // ---------------- V check ----------------
      bool ok = true;
      for (int j = 0; ok && j < blocks; ++j) {
        const int s = j % S::kVStages;
        ok = all_wait(&sm.v_full[s], uint32_t(j / S::kVStages) & 1u, &sm.abort, a.status, 89);
        if (!ok) break;
        if (partial(j)) {
          const uint4* tile_v = reinterpret_cast<const uint4*>(sm.v[s]);
          uint32_t hits = 0;
#pragma unroll 4
          for (int c = lane; c < S::kTile / 16; c += 32) hits |= not_finite<T>(tile_v[c]);
          if (__any_sync(0xffffffffu, hits != 0)) clear_not_finite<T, D, kPair>(sm, s, first_key + j * F::kBlock, hi_max);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.v_ok[s]);
      }
    }
  } else {
    // ---------------- softmax ----------------
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + 64u * stream, t_o = tmem + lanes + F::kO + uint32_t(D) * stream;
    const float scale = kFeat ? 1.0f : a.scale_log2;
    const uint64_t scale2 = pkf(scale, scale);
    const typename Soft::Cap cap(a);
    const float slope = (kFeat & kDistance) && valid ? a.slopes[head] * kLog2e : 0.0f;
    const uint32_t idle = (kFeat & kCap) ? __ballot_sync(0xffffffffu, !valid) : 0u;   // the warp's rows of no sequence
    float m = -INFINITY, l = 0.0f;   // the reference maximum (base 2) and the sum
    bool ok = true;
    for (int n = 0; n < steps; ++n) {
      const int key0 = first_key + n * kStep;
      ok = all_wait(&sm.s_full[stream], uint32_t(n) & 1u, &sm.abort, a.status, 90);
      if (!ok) break;
      tc_fence_after();
      uint32_t x0[32], x1[32];
      tmem_load_32cols(t_s, x0);
      tmem_load_32cols(t_s + 32, x1);
      tmem_load_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.s_empty[stream]);
      const bool part = key0 < lo_max || key0 + kStep > hi_min;
      // a cap alone grows with the product, so the largest product gives the maximum and
      // the rest of the cap's polynomial goes into the probabilities
      const bool small = (kFeat & kCap) && (part ? Soft::template is_small<true>(x0, x1, a, idle, lo - key0, hi - key0)
                                                  : Soft::template is_small<false>(x0, x1, a, idle, 0, 0));
      const bool raw = kFeat == kCap && small && !part;
      if ((kFeat || part) && !raw) {
        Soft::scores(x0, a, cap, small, slope, pos, key0, part, lo - key0, hi - key0);
        Soft::scores(x1, a, cap, small, slope, pos, key0 + 32, part, lo - key0 - 32, hi - key0 - 32);
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      Soft::maximum(mx, x0);
      Soft::maximum(mx, x1);
      float top = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])) * scale;
      if (raw) {
        uint32_t t0, t1;
        upk(cap(pkf(top, top), 0ull), t0, t1);
        top = __uint_as_float(t0);
      }
      const bool broken = !(top < INFINITY);   // a score of NaN or infinity: so is the row's result
      const bool grow = top > m + kGrowth || broken;
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? ex2(m - top) : 1.0f;
        const bool sums = l != 0.0f;   // without a sum, O of the row is zero (or not begun)
        if (grow) m = broken ? NAN : top;
        if (sums) l *= f;
        if (__any_sync(0xffffffffu, grow && sums)) {
          ok = all_wait(&sm.pv_done[stream], uint32_t(n - 1) & 1u, &sm.abort, a.status, 93);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_load_16cols(t_o + c, o);
            tmem_load_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_store_16cols(t_o + c, o);
          }
        }
      }
      // probabilities and their sum; this P was last read two steps before, complete
      // since S of this step was issued behind that product
      const uint64_t ref2 = Soft::reference(m);
      const uint32_t t_p = tmem + lanes + F::kP + 64u * stream + 32u * (n & 1);
      uint64_t sum2[2] = {0ull, 0ull};
      uint32_t p[16];
      if (raw) {
        Soft::template probabilities<true>(x0, scale2, ref2, sum2, p, &cap);
        tmem_store_16cols(t_p, p);
        Soft::template probabilities<true>(x1, scale2, ref2, sum2, p, &cap);
      } else {
        Soft::probabilities(x0, scale2, ref2, sum2, p);
        tmem_store_16cols(t_p, p);
        Soft::probabilities(x1, scale2, ref2, sum2, p);
      }
      tmem_store_16cols(t_p + 16, p);
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full[stream][n & 1]);
      uint32_t u0, u1;
      upk(add2(sum2[0], sum2[1]), u0, u1);
      l += __uint_as_float(u0) + __uint_as_float(u1);
    }
    // (without a step only Q was loaded: it has to land before the rows cross there)
    if (ok) ok = all_wait(steps > 0 ? &sm.done : &sm.q_full, 0, &sm.abort, a.status, 91);
    epilogue<T, D, kPair>(a, sm, tmem, Row{batch, token, head, kv_head, lo, hi, valid, blank, split, first_key, blocks, lo_max, hi_min}, m, l, ok);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == F::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, F::kColumns);
  }
}

// Joins the splits of every row, eight rows a CTA: a warp a row, or the CTA's eight warps a
// row where there are more than eight splits of few rows (a lone warp's loads of one split
// after another took 0.15 us each: 64 splits of 12 rows 9 us; the other way round 4096 rows
// of 9 splits take 14 us more).  The order of the sums is fixed.
__host__ __device__ inline int join_team(const Args& a) {
  return a.splits > 8 && int64_t(a.batch) * a.q_len * a.heads <= 1024 ? 8 : 1;
}
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args a) {
  constexpr int kOwn = D / 32, kAtOnce = 4;   // channels a lane, splits in flight
  __shared__ float shared[8][D + 1];
  const int team = join_team(a), warp = threadIdx.x >> 5, member = warp & (team - 1);
  const int64_t rows = int64_t(a.batch) * a.q_len * a.heads, row = (int64_t(blockIdx.x) * 8 + warp) / team;
  const int lane = threadIdx.x & 31;
  // launched beside the kernel above: its results are there from here on (every thread
  // waits, so that this grid does not end before that one)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row >= rows) return;
  const int head = int(row % a.heads);
  const int64_t bt = row / a.heads;
  const int token = int(bt % a.q_len), batch = int(bt / a.q_len);
  int lo, hi, pos;
  const bool valid = visible(a, batch, token, lo, hi, pos);
  if (!valid && !a.fill) return;
  const int splits = valid ? a.splits : 0;
  float m = -INFINITY;
  for (int s = lane; s < splits; s += 32) m = max_nan(m, a.part_lse[s * rows + row]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float ref = m == -INFINITY ? 0.0f : m;
  float total = 0.0f, f[kOwn];
#pragma unroll
  for (int e = 0; e < kOwn; ++e) f[e] = 0.0f;
  for (int s0 = member; s0 < splits; s0 += kAtOnce * team) {
    float w[kAtOnce], p[kAtOnce][kOwn];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int s = min(s0 + i * team, splits - 1);
      w[i] = a.part_lse[s * rows + row];
      const float* from = a.part + (s * rows + row) * D + lane * kOwn;
      if constexpr (kOwn == 4) {
        const float4 x = *reinterpret_cast<const float4*>(from);
        p[i][0] = x.x, p[i][1] = x.y, p[i][2] = x.z, p[i][3] = x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(from);
        p[i][0] = x.x, p[i][1] = x.y;
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const float x = s0 + i * team < splits ? ex2(w[i] - ref) : 0.0f;
      total += x;
#pragma unroll
      for (int e = 0; e < kOwn; ++e) f[e] = x == 0.0f ? f[e] : fmaf(x, p[i][e], f[e]);
    }
  }
  if (team > 1) {
#pragma unroll
    for (int e = 0; e < kOwn; ++e) shared[member][lane * kOwn + e] = f[e];
    if (lane == 0) shared[member][D] = total;
    __syncthreads();
    if (member) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) {
#pragma unroll
      for (int e = 0; e < kOwn; ++e) f[e] += shared[w][lane * kOwn + e];
      total += shared[w][D];
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  T* dst = static_cast<T*>(a.out) + int64_t(batch) * a.o_sb + int64_t(token) * a.o_ss + int64_t(head) * a.o_sh + lane * kOwn;
#pragma unroll
  for (int e = 0; e < kOwn; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack2<T>(f[e] * inv, f[e + 1] * inv);
  if (lane == 0 && a.lse)
    a.lse[(int64_t(batch) * a.heads + head) * a.q_len + token] = !valid ? 0.0f : total == 0.0f ? -INFINITY : (ref + log2f(total)) * kLn2;
}

template <typename T, int D, bool kPair>
cudaError_t launch_form(const Args& g, int feat, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                        unsigned grid, cudaStream_t stream) {
  constexpr int smem = int(sizeof(Smem<D, kPair>)) + 1024;
  // an SM has 228 KB for its CTAs, each with 1 KB that it does not see
  static_assert((smem + 1024) * Form<kPair>::kCtas <= 233472 && smem <= 232448, "shared memory");
  const auto go = [&](auto* kernel) -> cudaError_t {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    kernel<<<grid, Form<kPair>::kThreads, smem, stream>>>(mq, mk, mv, g);
    return cudaGetLastError();
  };
  return feat == 0          ? go(masked_attention_kernel<T, D, 0, kPair>)
         : feat == kCap     ? go(masked_attention_kernel<T, D, kCap, kPair>)
         : feat == kDistance ? go(masked_attention_kernel<T, D, kDistance, kPair>)
                             : go(masked_attention_kernel<T, D, kCap | kDistance, kPair>);
}

template <typename T, int D>
cudaError_t launch(const Args& g, bool pair, int feat, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                   unsigned grid, cudaStream_t stream) {
  const cudaError_t e = pair ? launch_form<T, D, true>(g, feat, mq, mk, mv, grid, stream)
                             : launch_form<T, D, false>(g, feat, mq, mk, mv, grid, stream);
  if (e != cudaSuccess || g.splits == 1) return e;
  const int64_t rows = int64_t(g.batch) * g.q_len * g.heads;
  // (programmatic launch: its CTAs come up while the last of the kernel's finish)
  cudaLaunchAttribute beside{};
  beside.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  beside.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned((rows * join_team(g) + 7) / 8));
  config.blockDim = dim3(256);
  config.stream = stream;
  config.attrs = &beside;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, join_kernel<T, D>, g);
}

}  // namespace mattn
}  // namespace h3sk
