// Host side of the attention under masks: argument checks, the cut of the work, tensor maps
// and launches of masked_attention.cuh's kernels, and the BF16 ones themselves.
#include "../../include/h3sk_b200.h"
#include "masked_attention.cuh"

namespace h3sk {
namespace mattn {

// FP16 is compiled in a unit of its own (masked_attention_fp16.cu).
extern template cudaError_t launch<__half, 128>(const Args&, bool, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                                unsigned, cudaStream_t);
extern template cudaError_t launch<__half, 64>(const Args&, bool, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                               unsigned, cudaStream_t);

bool misaligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

// A tensor map of 16-bit values; dims and byte strides innermost first, box of 64
// channels by box_rows.
bool encode(CUtensorMap* map, const void* base, bool bf16, int rank, const uint64_t* dims, const uint64_t* strides,
            const uint32_t* box) {
  auto fn = tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t d[5], st[4];
  cuuint32_t b[5], es[5];
  for (int i = 0; i < rank; ++i) d[i] = dims[i], b[i] = box[i], es[i] = 1;
  for (int i = 0; i + 1 < rank; ++i) st[i] = strides[i];
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, cuuint32_t(rank),
            const_cast<void*>(base), d, st, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace mattn
}  // namespace h3sk

#define H3SK_EXPORT extern "C" __attribute__((visibility("default")))

namespace h3sk {
namespace mattn {

struct Plan {
  int pack, tile_tokens, groups, q_tiles, tiles, pair, splits;
  uint64_t workspace;
};

// How the work is cut.
//
// Packing the g heads of a group into the rows of a tile needs ceil(S / floor(128 / g))
// tiles a group instead of ceil(S / 128) a head: the fewer tiles win.
//
// A CTA takes a pair of tiles (K and V blocks shared) or one tile, two CTAs an SM.  128 keys
// cost 2.0 us a pair, 2.06 a single tile beside another, 1.3 one that has its SM alone; a
// CTA's beginning and end 8.5 and 6.  The form with the shorter estimate runs: the longest
// CTA, or all of them shared out over the SMs, a last round counting half where pairs run and
// a quarter where single tiles do.  Measured pairs / single tiles in turn, at 1.6 to 1.7 GHz,
// us: 8192 x 8192, 24 heads 819 / 772; 4096 x 4096, 8 heads 67 / 64; 2048 x 2048, 74 heads 177 /
// 163; causal 6000 x 6000, 8 over 2 heads 94 / 78; 16384 x 16384, 8 heads 1074 / 1007, 16
// heads 1963 / 2000, 56 heads 6833 / 6977.  16 over 4 heads of 12288 tokens in 2 / 5 / 21 / 60 /
// 200 equal documents 615 / 288 / 116 / 74 / 61 against 568 / 269 / 104 / 65 / 50; in 21 ragged
// ones 165 / 151.  Under a cap 6000 x 6000, 8 over 2 heads 271 / 222; 4096 x 4096, 8 heads 95.6 /
// 96.6.
// CTAs of at most ten blocks are taken at 2.0 and 2.1 with 6 for either, which gives pairs
// where they fill whole rounds.  (Single tiles measured 4 to 10 % shorter there too: 1000 x
// 1000, 74 heads 44 / 42, causal 34 / 31; 256 x 20000, 8 heads in 18 splits 33.5 / 32.0.  Their
// plans stay as they were.)
//
// When the CTAs do not fill the SMs the keys are split beyond 512: at least 256 to a single
// tile's CTA, 128 where there is one tile of rows and the splits are at most 16, 512 to a
// pair's.  At least 128 / 256 / 512 / 1024, us: 1 query x 1000 keys, 12 over 3 heads 11.0 /
// 11.9 / 14.3 / 16.5; x 2048, batch 2, 24 over 4 10.7 / 11.8 / 13.7 / 18.9; x 8192, 28 over 4
// 13.5 / 12.1 / 14.2 / 19.7; 1000 x 1000, 6 heads 19.5 / 17.7 / 18.2 / 18.2; 1 query x 300 keys
// 9.9 / 9.5 unsplit.
struct Cut {
  int tiles, splits;
  double us;
};
Cut cut(const H3MaskedAttentionArgs& a, const Plan& p, bool pair, int sms) {
  Cut c{};
  c.tiles = pair ? (p.q_tiles + 1) / 2 : p.q_tiles;
  const int64_t ctas = int64_t(c.tiles) * p.groups * a.batch, room = pair ? sms : 2 * sms;
  const int blocks = (a.k_len + 127) / 128;   // in this estimate of 128 keys
  c.splits = 1;
  if (ctas < room && blocks > 4) {
    const int64_t by_room = room / ctas, by_keys = pair ? blocks / 4 : p.q_tiles == 1 && blocks <= 16 ? blocks : blocks / 2;
    c.splits = int(by_room < by_keys ? by_room : by_keys);
  }
  // blocks of an average CTA and of the longest: documents are taken to be equal but for
  // one three times as long, a causal mask hides a triangle
  double mean = blocks, most = blocks;
  if (a.documents > 1) {
    mean = double(blocks) / a.documents + 1.0;
    most = mean * 3.0 < blocks ? mean * 3.0 : blocks;
  }
  if (a.causal) mean *= 1.0 - 0.5 * (a.q_len < a.k_len ? a.q_len : a.k_len) / (a.k_len > 0 ? a.k_len : 1);
  const bool alone = ctas * c.splits <= sms;   // single tiles with an SM each
  const bool few = blocks <= 10 * c.splits;
  const auto cta = [&](double b, double block_us) { return (pair && !few ? 8.5 : 6.0) + block_us * b / c.splits; };
  const double turns = double(ctas) * c.splits / (alone ? sms : room);
  const double block_us = pair ? 2.0 : alone ? 1.3 : few ? 2.1 : 2.06;
  if (mean < most) {
    // (a long single tile is alone in the end)
    const double longest = cta(most, pair ? 2.0 : alone ? 1.3 : 1.6), shared = turns * cta(mean, block_us) + 0.1 * longest;
    c.us = longest > shared ? longest : shared;
  } else {
    const double rounds = turns <= 1.0 ? 1.0 : turns + (std::ceil(turns) - turns) * (pair ? 0.5 : 0.25);
    c.us = rounds * cta(most, block_us);
  }
  return c;
}

Plan plan(const H3MaskedAttentionArgs& a, int sms) {
  Plan p{};
  const int g = a.q_heads / a.k_heads;
  const int64_t plain = int64_t(a.q_heads) * ((a.q_len + kRows - 1) / kRows);
  p.pack = 1;
  if (g > 1 && g <= kRows) {
    const int tokens = kRows / g;
    if (int64_t(a.k_heads) * ((a.q_len + tokens - 1) / tokens) <= plain) p.pack = g;
  }
  p.tile_tokens = kRows / p.pack;
  p.groups = a.q_heads / p.pack;
  p.q_tiles = (a.q_len + p.tile_tokens - 1) / p.tile_tokens;
  const Cut single = cut(a, p, false, sms), pairs = cut(a, p, true, sms);
  p.pair = p.q_tiles > 1 && pairs.us <= single.us;
  p.tiles = p.pair ? pairs.tiles : single.tiles;
  p.splits = p.pair ? pairs.splits : single.splits;
  if (p.splits > 1)
    p.workspace = uint64_t(p.splits) * a.batch * a.q_len * a.q_heads * (a.dim + 1) * sizeof(float);
  return p;
}

int sm_count() {
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return 0;
  return sms;
}

bool args_ok(const H3MaskedAttentionArgs* a) {
  if (!a || a->batch < 0 || a->q_len < 0 || a->k_len < 0 || a->q_heads < 1 || a->k_heads < 1 || a->q_heads % a->k_heads ||
      (a->dim != 64 && a->dim != 128) || a->type < 0 || a->type > 1 || a->documents < 0)
    return false;
  if (a->batch > (1 << 20) || a->q_heads > 65535 || a->q_len > (1 << 30) || a->k_len > (1 << 30)) return false;
  if (!(a->scale > 0.0f) || !std::isfinite(a->scale) || !(a->softcap >= 0.0f) || !std::isfinite(a->softcap)) return false;
  if (!std::isfinite(a->scale * 3.0f) || (a->softcap > 0.0f && (!std::isfinite(a->scale / a->softcap * 3.0f) ||
                                                                !std::isfinite(a->softcap * 3.0f))))
    return false;   // their products with log2(e)
  if (a->documents && (a->batch != 1 || !a->q_offsets || !a->k_offsets || a->q_lengths || a->k_lengths)) return false;
  if (!a->documents && (a->q_offsets || a->k_offsets)) return false;
  if (a->prefix && !a->causal) return false;
  return true;
}

}  // namespace mattn
}  // namespace h3sk

H3SK_EXPORT size_t h3_masked_attention_args_size(void) { return sizeof(H3MaskedAttentionArgs); }
H3SK_EXPORT const char* h3_masked_attention_error(int code) { return cudaGetErrorString(static_cast<cudaError_t>(code)); }

H3SK_EXPORT int64_t h3_masked_attention_workspace(const H3MaskedAttentionArgs* a) {
  using namespace h3sk::mattn;
  if (!args_ok(a)) return -1;
  if (!a->batch || !a->q_len) return 0;
  const int sms = sm_count();
  return sms < 1 ? -1 : int64_t(plan(*a, sms).workspace);
}

// How a call is cut: tiles by pairs (1) or singly (0), heads of a group in a tile, splits
// of the keys.
H3SK_EXPORT int h3_masked_attention_plan(const H3MaskedAttentionArgs* a, int* out) {
  using namespace h3sk::mattn;
  if (!args_ok(a) || !out) return cudaErrorInvalidValue;
  const int sms = sm_count();
  if (sms < 1) return cudaErrorInvalidDevice;
  const Plan p = plan(*a, sms);
  out[0] = p.pair, out[1] = p.pack, out[2] = p.splits;
  return cudaSuccess;
}

H3SK_EXPORT int h3_masked_attention_run(const H3MaskedAttentionArgs* a, uintptr_t stream_ptr) {
  using namespace h3sk::mattn;
  if (!args_ok(a)) return cudaErrorInvalidValue;
  if (!a->batch || !a->q_len) return cudaSuccess;
  if (!a->q || !a->out || (a->k_len && (!a->k || !a->v))) return cudaErrorInvalidValue;
  const int64_t qs[3] = {a->q_stride_b, a->q_stride_s, a->q_stride_h}, ks[3] = {a->k_stride_b, a->k_stride_s, a->k_stride_h};
  const int64_t vs[3] = {a->v_stride_b, a->v_stride_s, a->v_stride_h}, os[3] = {a->o_stride_b, a->o_stride_s, a->o_stride_h};
  for (int i = 0; i < 3; ++i)
    for (const int64_t s : {qs[i], ks[i], vs[i], os[i]})
      if (s < 0 || s % 8 || s >= (int64_t(1) << 38)) return cudaErrorInvalidValue;
  if (misaligned(a->q, 16) || misaligned(a->out, 16) || misaligned(a->lse, 4) || misaligned(a->slopes, 4) ||
      misaligned(a->q_offsets, 4) || misaligned(a->k_offsets, 4) || misaligned(a->q_lengths, 4) || misaligned(a->k_lengths, 4) ||
      misaligned(a->prefix, 4) || (a->k_len && (misaligned(a->k, 16) || misaligned(a->v, 16))))
    return cudaErrorInvalidValue;
  // shared along a dimension: batches of every operand, heads of K and V
  const auto shared = [](int64_t stride, int n) { return stride == 0 && n > 1; };
  if (shared(qs[1], a->q_len) || shared(qs[2], a->q_heads) || shared(ks[1], a->k_len) || shared(vs[1], a->k_len) ||
      shared(os[0], a->batch) || shared(os[1], a->q_len) || shared(os[2], a->q_heads))
    return cudaErrorInvalidValue;
  const int sms = sm_count();
  if (sms < 1) return cudaErrorInvalidDevice;
  const Plan p = plan(*a, sms);
  if (p.workspace && (!a->workspace || misaligned(a->workspace, 16) || a->workspace_bytes < p.workspace))
    return cudaErrorInvalidValue;
  const int64_t ctas = int64_t(p.tiles) * p.groups * a->batch * p.splits;
  if (ctas > INT_MAX || int64_t(a->batch) * a->q_len * a->q_heads / 8 >= INT_MAX) return cudaErrorInvalidValue;

  // strides of dimensions of one element may be anything: a valid one stands in
  const auto bytes = [&](int64_t stride, int n) { return uint64_t(n > 1 && stride > 0 ? stride * 2 : a->dim * 2); };
  CUtensorMap mq, mk, mv;
  {
    const int qb = shared(qs[0], a->batch) ? 1 : a->batch;
    const uint64_t dims[5] = {uint64_t(a->dim), uint64_t(p.pack), uint64_t(a->q_len), uint64_t(p.groups), uint64_t(qb)};
    const uint64_t st[4] = {bytes(qs[2], p.pack), bytes(qs[1], a->q_len),
                            p.groups > 1 ? uint64_t(qs[2]) * p.pack * 2 : uint64_t(a->dim * 2), bytes(qs[0], qb)};
    const uint32_t box[5] = {64, uint32_t(p.pack), uint32_t(p.tile_tokens), 1, 1};
    if (!encode(&mq, a->q, a->type == 0, 5, dims, st, box)) return cudaErrorInvalidValue;
  }
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? vs : ks;
    const int n = a->k_len > 0 ? a->k_len : 1, h = shared(s[2], a->k_heads) ? 1 : a->k_heads, b = shared(s[0], a->batch) ? 1 : a->batch;
    const void* base = a->k_len > 0 ? (i ? a->v : a->k) : a->q;   // without keys nothing is loaded
    const uint64_t dims[4] = {uint64_t(a->dim), uint64_t(n), uint64_t(h), uint64_t(b)};
    const uint64_t st[3] = {bytes(s[1], n), bytes(s[2], h), bytes(s[0], b)};
    const uint32_t box[4] = {64, uint32_t(p.pair ? Form<true>::kBlock : Form<false>::kBlock), 1, 1};
    if (!encode(i ? &mv : &mk, base, a->type == 0, 4, dims, st, box)) return cudaErrorInvalidValue;
  }
  int* status = h3sk::status_device_ptr();
  if (!status) return cudaErrorInvalidSymbol;

  Args g{};
  g.batch = a->batch, g.q_len = a->q_len, g.k_len = a->k_len;
  g.groups = p.groups, g.pack = p.pack, g.tile_tokens = p.tile_tokens;
  g.heads = a->q_heads;
  g.groups_per_kv = p.groups / a->k_heads;
  g.tiles = p.tiles, g.q_tiles = p.q_tiles, g.splits = p.splits, g.causal = a->causal != 0;
  g.q_bmul = !shared(qs[0], a->batch), g.k_bmul = !shared(ks[0], a->batch), g.v_bmul = !shared(vs[0], a->batch);
  g.k_hmul = !shared(ks[2], a->k_heads), g.v_hmul = !shared(vs[2], a->k_heads);
  g.documents = a->documents;
  g.q_offsets = a->q_offsets, g.k_offsets = a->k_offsets, g.q_lengths = a->q_lengths, g.k_lengths = a->k_lengths;
  g.prefix = a->prefix;
  g.slopes = a->slopes;
  g.scale_log2 = a->softcap > 0.0f ? a->scale / a->softcap * 2.0f * kLog2e : a->scale * kLog2e;
  g.cap_log2 = a->softcap * kLog2e;
  g.cap_y = a->softcap > 0.0f ? a->scale / a->softcap : 0.0f;
  g.out = a->out, g.o_sb = os[0], g.o_ss = os[1], g.o_sh = os[2];
  g.lse = a->lse;
  g.fill = a->fill != 0;
  g.v = a->v, g.v_sb = vs[0], g.v_ss = vs[1], g.v_sh = vs[2];
  g.part = static_cast<float*>(a->workspace);
  g.part_lse = g.part ? g.part + uint64_t(p.splits) * a->batch * a->q_len * a->q_heads * a->dim : nullptr;
  g.status = status;
  const int feat = (a->softcap > 0.0f ? kCap : 0) | (a->slopes ? kDistance : 0);
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  const unsigned grid = unsigned(ctas);
  if (a->type == 0)
    return a->dim == 128 ? launch<__nv_bfloat16, 128>(g, p.pair, feat, mq, mk, mv, grid, stream)
                         : launch<__nv_bfloat16, 64>(g, p.pair, feat, mq, mk, mv, grid, stream);
  return a->dim == 128 ? launch<__half, 128>(g, p.pair, feat, mq, mk, mv, grid, stream)
                       : launch<__half, 64>(g, p.pair, feat, mq, mk, mv, grid, stream);
}
