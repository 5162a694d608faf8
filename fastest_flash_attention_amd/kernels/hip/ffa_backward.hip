// Attention backward launches for gfx950: which kernels of ffa_backward_kernels.h a call runs, and
// how its dK/dV sweeps are cut over workgroups.

#include "ffa_backward_kernels.h"

namespace ffa {
namespace {

int64_t sq_padded(int32_t seqlen_q) {
  return (static_cast<int64_t>(seqlen_q) + kQTile - 1) / kQTile * kQTile;
}

}  // namespace

size_t attn_bwd_workspace_bytes(int32_t batch, int32_t heads_q, int32_t seqlen_q) {
  return static_cast<size_t>(2) * batch * heads_q * sq_padded(seqlen_q) * sizeof(float);
}

namespace {

// Whether the dK/dV kernel runs with two halves (its comment has the rule and what it measured):
// calls with sinks, at most a workgroup per CU, sweeps (the longest: `most` tiles) long enough.
bool pair_waves(const BwdParams& p, int64_t units, int64_t most) {
  return p.sinks > 0 && p.D <= 128 && p.n_part_s == 1 && units * p.n_kt <= 256 && (p.D <= 64 || most >= 10);
}

// Cuts the dK/dV sweeps of a launch that its heaviest workgroup would hold up: sets n_part,
// part_len and the key tiles cut, returns the bytes of the partials (0: no sweep is cut). A part is 1.5 times
// an even share of the work over the chip's slots (two workgroups per CU up to head_dim
// 128), at least 16 tiles; sweeps are cut when the longest exceeds 2.5 parts, so that the
// partials (written and read once in fp32) cost less than the waiting. Measured on MI355X,
// whole backward, bf16, us uncut / cut (B, Hq/Hkv, S, D, causal unless said):
//   2, 32/8, 2011, 128    409 / 306      1, 40/8, 1024, 128, softcap   270 / 107
//   1, 32/8, 4096, 128    774 / 555      1, 28/4, 1500, 96             432 / 146
//   1, 8/8, 2048, 128     132 / 107      2, 8/1, 1000, 64              243 / 56
//   1, 24/8, 2000, 192    373 / 223      1, 8/8, 4096, 64              180 / 150
// with parts of one even share 1, 12/12, 2048, 128 not causal: 137 / 151, so it stays uncut.
//
// With sinks the same share counts all tiles; those of the sinks (n_skt of them, swept by every
// row) and the window's are cut apart. The sweeps of the sinks are few and come first, so they are
// cut from 1.5 parts on; us with 2.5 / 1.5, and with 1.5 at parts of one even share:
//   1, 16/16, 4096, 128, window 500, 1024 sinks   283 / 213, 246
//   2, 16/4, 3000, 128, window 500, 256 sinks     202 / 202, 218
//   4, 32/8, 4096, 64, window 256, 128 sinks      415 / 415, 333
size_t plan_dkv_parts(BwdParams& p, int32_t dtype) {
  p.pair = 0;
  p.n_part = p.n_part_s = 1;
  p.part_len = p.part_len_s = 0x7fffffff;
  const int64_t units = static_cast<int64_t>(p.B) * p.Hkv;
  const int64_t slots = p.D <= 128 ? 512 : 256;
  if (dtype == FFA_DTYPE_FP32 || p.D > kCutMaxDim || p.n_kt == 0) return 0;
  const bool few = units * p.n_kt < 1024;  // workgroups
  if (!few && p.n_skt == 0) return 0;
  const size_t tile_bytes = static_cast<size_t>(kDkvKeys) * (p.D + p.Dv) * sizeof(float);
  int64_t total = 0, most = 0, most_s = 0;
  for (int kt = 0; kt < p.n_kt; ++kt) {
    int first, n;
    dkv_rows(p, kt, first, n);
    const int64_t nit = static_cast<int64_t>(n) * p.ratio;
    total += nit;
    int64_t& m = kt < p.n_skt ? most_s : most;
    m = nit > m ? nit : m;
  }
  const int64_t even = (3 * total * units + 2 * slots - 1) / (2 * slots);
  size_t bytes = 0;
  int64_t len = even < 16 ? 16 : even;
  if (2 * most_s > 3 * len) {
    if (most_s > 16 * len) len = (most_s + 15) / 16;  // at most 16 parts
    p.n_part_s = static_cast<int>((most_s + len - 1) / len);
    p.part_len_s = static_cast<int>(len);
    bytes += static_cast<size_t>(units) * p.n_skt * p.n_part_s * tile_bytes;
  }
  len = even < 16 ? 16 : even;
  p.pair = pair_waves(p, units, most) ? 1 : 0;
  if (!few || 2 * most <= 5 * len) return bytes;
  if (most > 16 * len) len = (most + 15) / 16;  // at most 16 parts
  p.n_part = static_cast<int>((most + len - 1) / len);
  p.part_len = static_cast<int>(len);
  // Only the key tiles with longer sweeps than a part have partials. A sweep's length is a
  // concave function of the key tile (q_hi - q_lo of dkv_rows), so they follow one another
  // and average at least (len + most) / 2: with len at least 1.5 even shares that is at most
  // 4/3 slots partial tiles, 90 MB at head_dim 128 (683 of 128 KB), whatever the lengths
  // of the sequences. (Sweeps of sinks are equal, with at
  // most 4/3 parts for each `len` of them: at most 8/9 slots, 60 MB.)
  int end = 0;
  p.cut_first = p.n_kt;
  for (int kt = p.n_skt; kt < p.n_kt; ++kt) {
    int first, n;
    dkv_rows(p, kt, first, n);
    if (static_cast<int64_t>(n) * p.ratio <= len) continue;
    p.cut_first = kt < p.cut_first ? kt : p.cut_first;
    end = kt + 1;
  }
  p.n_cut = end - p.cut_first;
  return bytes + static_cast<size_t>(units) * p.n_cut * p.n_part * tile_bytes;
}

constexpr int kSinkGroups = 256;  // workgroups that the sinks' rows are split over

void fill_bwd_sizes(const ffa_attn_bwd_args& a, BwdParams& p) {
  p.B = a.batch;
  p.Hq = a.heads_q;
  p.Hkv = a.heads_kv;
  p.Sq = a.seqlen_q;
  p.Skv = a.seqlen_kv;
  p.D = a.head_dim;
  p.Dv = a.v_head_dim > 0 ? a.v_head_dim : a.head_dim;
  p.q_offset = a.q_offset;
  p.causal = a.causal ? 1 : 0;
  p.window = clamp_window(a.window, a.q_offset, a.seqlen_q);
  p.ratio = a.heads_q / a.heads_kv;
  p.sq_pad = static_cast<int>(sq_padded(a.seqlen_q));
  p.n_qt = p.sq_pad / kQTile;
  p.n_kt = (a.seqlen_kv + kDkvKeys - 1) / kDkvKeys;
  p.sinks = clamp_sinks(a.sinks, p.window, a.q_offset, a.seqlen_q);
  p.sinks = p.sinks < a.seqlen_kv ? p.sinks : a.seqlen_kv;
  // Whole key tiles of sinks: swept in the dK/dV kernel where it is compiled for cut sweeps, else
  // (fp32: 32-key workgroups) in blocks like the other sinks.
  p.n_skt = a.dtype == FFA_DTYPE_FP32 || p.D > kCutMaxDim ? 0 : p.sinks / kDkvKeys;
  p.sink0 = p.n_skt * kDkvKeys;
  p.n_skb = (p.sinks - p.sink0 + 31) / 32;
  p.n_part_k = 1;
  p.part_len_k = 0x7fffffff;
}

// Rows of the sinks' 32-key blocks over workgroups: sets n_part_k and part_len_k, returns the bytes
// of the partials. A part has at least two row tiles for each of its four waves; there are parts
// for about two workgroups per CU, and none (each block's rows stay whole) with 256 blocks and
// more, so at most 512 partial blocks of 32 keys (32 MB at head_dim 256).
size_t plan_sink_parts(BwdParams& p, int32_t dtype) {
  const int64_t blocks = static_cast<int64_t>(p.B) * p.Hkv * p.n_skb;
  if (blocks == 0 || blocks >= 256 || (dtype == FFA_DTYPE_FP32 && p.D > 128)) return 0;
  const int64_t items = static_cast<int64_t>(p.ratio) * ((p.Sq + kDkvRows - 1) / kDkvRows);
  int64_t parts = kSinkGroups / blocks;
  parts = parts < items / 8 ? parts : items / 8;
  if (parts < 2) return 0;
  p.part_len_k = static_cast<int>((items + parts - 1) / parts);
  p.n_part_k = static_cast<int>((items + p.part_len_k - 1) / p.part_len_k);
  return static_cast<size_t>(blocks) * p.n_part_k * 64 * p.D * sizeof(float);
}


}  // namespace

size_t attn_bwd_split_workspace_bytes(const ffa_attn_bwd_args& a) {
  BwdParams p{};
  fill_bwd_sizes(a, p);
  return attn_bwd_workspace_bytes(a.batch, a.heads_q, a.seqlen_q) + plan_dkv_parts(p, a.dtype) +
         plan_sink_parts(p, a.dtype);
}

int launch_attn_bwd(const ffa_attn_bwd_args& a, hipStream_t stream) {
  BwdParams p{};
  fill_bwd_sizes(a, p);
  p.q = static_cast<const uint16_t*>(a.q);
  p.k = static_cast<const uint16_t*>(a.k);
  p.v = static_cast<const uint16_t*>(a.v);
  p.o = static_cast<const uint16_t*>(a.o);
  p.dout = static_cast<const uint16_t*>(a.dout);
  p.lse = a.lse;
  p.dq = static_cast<uint16_t*>(a.dq);
  p.dk = static_cast<uint16_t*>(a.dk);
  p.dv = static_cast<uint16_t*>(a.dv);
  p.q_sb = a.q_stride[0];
  p.q_sh = a.q_stride[1];
  p.q_ss = a.q_stride[2];
  p.k_sb = a.k_stride[0];
  p.k_sh = a.k_stride[1];
  p.k_ss = a.k_stride[2];
  p.v_sb = a.v_stride[0];
  p.v_sh = a.v_stride[1];
  p.v_ss = a.v_stride[2];
  p.o_sb = a.o_stride[0];
  p.o_sh = a.o_stride[1];
  p.o_ss = a.o_stride[2];
  p.do_sb = a.do_stride[0];
  p.do_sh = a.do_stride[1];
  p.do_ss = a.do_stride[2];
  p.dq_sb = a.dq_stride[0];
  p.dq_sh = a.dq_stride[1];
  p.dq_ss = a.dq_stride[2];
  p.dk_sb = a.dk_stride[0];
  p.dk_sh = a.dk_stride[1];
  p.dk_ss = a.dk_stride[2];
  p.dv_sb = a.dv_stride[0];
  p.dv_sh = a.dv_stride[1];
  p.dv_ss = a.dv_stride[2];
  p.l_sb = a.lse_stride[0];
  p.l_sh = a.lse_stride[1];
  p.l_ss = a.lse_stride[2];
  const bool softcap = a.softcap > 0.0f;
  if (softcap) {
    p.score_mul = a.scale / a.softcap;
    p.cap_mul = a.softcap * kLog2e;
    p.tanh_mul = 2.0f * kLog2e * a.scale / a.softcap;
  } else {
    p.score_mul = a.scale * kLog2e;
    p.cap_mul = 0.0f;
    p.tanh_mul = 0.0f;
  }
  p.scale = a.scale;
  float* ws = static_cast<float*>(a.workspace);
  const int64_t rows = static_cast<int64_t>(a.batch) * a.heads_q * p.sq_pad;
  p.lse2 = ws;
  p.di = ws + rows;
  const size_t stats = attn_bwd_workspace_bytes(a.batch, a.heads_q, a.seqlen_q);
  const size_t sink_parts = plan_sink_parts(p, a.dtype);
  const size_t parts = plan_dkv_parts(p, a.dtype);
  // behind the statistics: the partials of the sinks' blocks, of the window's tiles, of the sinks'
  p.part_k = ws + stats / sizeof(float);
  p.part = p.part_k + sink_parts / sizeof(float);
  p.part_s = p.part;
  if (p.n_part > 1) {
    p.part_s += static_cast<int64_t>(a.batch) * a.heads_kv * p.n_cut * p.n_part * kDkvKeys * (p.D + p.Dv);
  }
  if (a.workspace_bytes < stats + sink_parts + parts) {  // whole sweeps need none
    p.n_part = p.n_part_s = p.n_part_k = 1;
    p.part_len = p.part_len_s = p.part_len_k = 0x7fffffff;
  }

  const int64_t grid_pre = rows / 32;
  const int64_t grid_dq = static_cast<int64_t>(p.n_qt) * a.batch * a.heads_q;
  const int64_t kv_units = static_cast<int64_t>(a.batch) * a.heads_kv;
  const int64_t grid_win = (p.n_kt - p.n_skt) * p.n_part * kv_units;  // workgroups of the window's tiles
  const int64_t grid_dkv = grid_win + static_cast<int64_t>(p.n_skt) * p.n_part_s * kv_units;
  if (grid_pre > 0x7fffffff || grid_dq > 0x7fffffff || grid_dkv > 0x7fffffff ||
      kv_units * p.n_skb * p.n_part_k > 0x7fffffff) {
    return FFA_ERR_TOO_LARGE;
  }
  if (grid_pre == 0 || grid_dq == 0) return FFA_OK;
  // the forward's grid order: each XCD runs its units one after another (their K / V,
  // or Q / dO, stay in its L2) and interleaves only its last ones. At the north-star
  // shape the step reads 0.53 GB less than with every pair interleaved (4.24 against
  // 4.78 GB per backward); time within +-0.5 %, +5 % at head_dim 64.
  prefill_grid_order(p.causal, static_cast<int64_t>(a.batch) * a.heads_q, grid_dq, p.xcd_group_dq,
                     p.xcd_remap_dq);
  prefill_grid_order(p.causal, kv_units, grid_win, p.xcd_group_dkv, p.xcd_remap_dkv);
  if (a.dtype == FFA_DTYPE_FP32) {
    // 32-row / 32-key workgroups
    const int64_t g32 = static_cast<int64_t>(a.batch) * a.heads_q * ((a.seqlen_q + 31) / 32) +
                        static_cast<int64_t>(a.batch) * a.heads_kv * ((a.seqlen_kv + 31) / 32);
    if (g32 > 0x7fffffff) return FFA_ERR_TOO_LARGE;
    if (p.sinks > 0) {
      launch_bwd_sinks(p, a.dtype, softcap, static_cast<int>(grid_pre), 0, 0, stream);
    } else {
      launch_f32<false>(p, softcap, static_cast<int>(grid_pre), stream);
    }
  } else if (p.sinks > 0) {
    launch_bwd_sinks(p, a.dtype, softcap, static_cast<int>(grid_pre), static_cast<int>(grid_dkv),
                     static_cast<int>(grid_dq), stream);
  } else if (a.dtype == FFA_DTYPE_BF16) {
    launch_tag<Bf16Tag>(p, softcap, static_cast<int>(grid_pre), static_cast<int>(grid_dkv),
                        static_cast<int>(grid_dq), stream);
  } else {
    launch_tag<F16Tag>(p, softcap, static_cast<int>(grid_pre), static_cast<int>(grid_dkv),
                       static_cast<int>(grid_dq), stream);
  }
  return hipGetLastError() == hipSuccess ? FFA_OK : FFA_ERR_LAUNCH;
}

}  // namespace ffa
