// Prefill launches for gfx950: which kernels of ffa_prefill_kernels.h a call runs, and how its
// keys are split over workgroups.

#include "ffa_prefill_kernels.h"

namespace ffa {
namespace {

// How a call's keys are split, or n_split = 0: one workgroup sweeps all of a row's keys.
//
// `base` workgroups (128-row tiles over all heads) times the ranges should fill the
// chip's slots (two workgroups per CU, one at head_dim above 192) once. Measured on
// MI355X, bf16, us per call (device time; unsplit figures of cached calls with the
// concatenation they need):
//   over a cache (B, Hq/Hkv, Sq + cached, D)       unsplit   split
//     8, 32/8, 1 + 4095, 128                          152     27.5  (4.9 TB/s of K/V)
//     32, 32/32, 1 + 2047, 128   (base 1024)          992      202
//     1, 32/8, 509 + 7683, 128   (base 128)           170       84
//     1, 32/8, 1024 + 15000, 128 (base 256)           334      237
//     4, 32/32, 512 + 512, 128   (base 512)           124       63
//     1, 32/8, 1024 + 64, 128    (base 256)            35       41  -> not split
//     4, 24/8, 1024 + 1000, 64   (base 768)            96       94  -> not split
//   no cache, causal
//     1, 4/4, 2048, 128 (base 64)                      33       24
//     1, 2/2, 8192, 128 (base 128)                    116       64
//     1, 8/8, 1024, 128 (base 64)                    20.4     20.3  -> not split
//     1, 16/16, 2048, 128 (base 256)                 35.5     48.3  -> not split
//     1, 8/8, 2048, 128, window 1024 (base 128)        25       34  -> not split
constexpr int kSplitLeast = 256;       // shortest range over a cache (keys)
constexpr int kSplitLeastOwn = 512;    // without one
constexpr int kSplitMinSweep = FFA_SPLIT_MIN_KEYS;  // without a cache, shorter sweeps stay whole ...
constexpr int kSplitMaxBase = 128;     // ... and so do launches of more workgroups
struct SplitPlan {
  int n_split = 0;
  int n_qt = 0, pack = 0;
  int lo0 = 0, lo1 = 0, len = 0, n0 = 0;
  int n_sink = 0, sink_end = 0;
  int64_t grid = 0;
  size_t bytes = 0;
};

SplitPlan plan_split(const ffa_prefill_args& a) {
  SplitPlan pl;
  if (a.dtype == FFA_DTYPE_FP32 || a.batch == 0 || a.seqlen_q == 0 ||
      (a.block_key_mask != nullptr && a.k_cache != nullptr) || (a.v_head_dim > 0 && a.v_head_dim < a.head_dim)) {
    return pl;
  }
  const int64_t ratio = a.heads_q / a.heads_kv;
  const int64_t sq = a.seqlen_q;
  const int64_t cache = a.k_cache != nullptr ? a.cache_len : 0;
  const int64_t own = a.seqlen_kv - cache;
  const int bn = a.head_dim <= 128 ? 64 : 32;
  const int64_t t1 = (sq + kBlockM - 1) / kBlockM;
  const int64_t tp = (sq * ratio + kBlockM - 1) / kBlockM;
  pl.pack = sq < kBlockM && tp < t1 * ratio;
  pl.n_qt = static_cast<int>(pl.pack ? tp : t1);
  const int64_t base = static_cast<int64_t>(a.batch) * a.heads_kv * (pl.pack ? tp : t1 * ratio);
  // the keys that any row sees, in each segment
  int64_t lo = 0, hi = a.seqlen_kv;
  const int window = clamp_window(a.window, a.q_offset, a.seqlen_q);
  if (window > 0) lo = a.q_offset - static_cast<int64_t>(window) + 1;
  if (a.causal) hi = a.q_offset + sq < hi ? a.q_offset + sq : hi;
  lo = lo < 0 ? 0 : lo;
  if (hi <= lo) return pl;
  const int64_t keys = hi - lo;
  const int64_t sinks = clamp_sinks(a.sinks, window, a.q_offset, a.seqlen_q);
  if (sinks > (cache > 0 ? cache : own)) return pl;  // sinks in both segments
  const int64_t lo1 = lo > cache ? lo - cache : 0;
  const int64_t end0 = cache < hi ? cache : hi;
  const int64_t end1 = hi - cache < own ? hi - cache : own;
  int64_t n_max = (a.head_dim <= 192 ? 512 : 256) / base;
  bool own_free = false;
  if (cache > 0) {
    // The partials (8 bytes written and read per row, dim and range) against the
    // concatenation (as much per key and dim of each KV head): a full launch splits only
    // to avoid the larger of the two, a half-empty one gains more than that.
    n_max = n_max < 3 ? 3 : n_max;
    if (base > kSplitMaxBase && ratio * sq * n_max > keys * (base > 512 ? 1 : 4)) return pl;
    // a few own keys take no slot's worth of time: one more range over the cache pays
    // unless the ranges are short already
    own_free = end1 - lo1 <= kSplitLeast && keys > 384 * n_max * (n_max - 1);
  } else {
    const int64_t sweep = window > 0 && window + kBlockM < keys ? window + kBlockM : keys;
    if (base > kSplitMaxBase || sweep < kSplitMinSweep) return pl;
  }
  pl.lo0 = static_cast<int>(lo / bn * bn);
  pl.lo1 = static_cast<int>(lo1 / bn * bn);
  const int64_t least = cache > 0 ? kSplitLeast : kSplitLeastOwn;
  int64_t len = keys / n_max;
  len = ((len < least ? least : len) + bn - 1) / bn * bn;
  int64_t n1;
  for (;;) {  // len grows by 1/16 or a tile: ends once both segments are one range each
    pl.n0 = static_cast<int>(lo < end0 ? (end0 - pl.lo0 + len - 1) / len : 0);
    n1 = end1 > lo1 ? (end1 - pl.lo1 + len - 1) / len : 0;
    if (pl.n0 + (own_free ? 0 : n1) <= n_max || len >= hi) break;
    len += (len / 16 + bn - 1) / bn * bn;
  }
  pl.len = static_cast<int>(len);
  int64_t n = pl.n0 + n1;
  if (n < 1 || (cache == 0 && n < 2)) return pl;
  if (sinks > 0) {  // those below the window's first tile (of a cache: or all of its sinks)
    const int64_t below = cache == 0 ? pl.lo1 : (lo < end0 ? pl.lo0 : cache);
    pl.sink_end = static_cast<int>(sinks < below ? sinks : below);
    pl.n_sink = static_cast<int>((pl.sink_end + len - 1) / len);
    n += pl.n_sink;
  }
  pl.grid = base * n;
  if (pl.grid > 0x7fffffff) return pl;
  pl.n_split = static_cast<int>(n);
  const int64_t rows = static_cast<int64_t>(a.batch) * a.heads_q * sq;
  pl.bytes = static_cast<size_t>(rows) * n * (static_cast<size_t>(a.head_dim) + 1) * sizeof(float);
  return pl;
}

}  // namespace

size_t prefill_workspace_bytes(const ffa_prefill_args& a) { return plan_split(a).bytes; }

int launch_prefill(const ffa_prefill_args& a, hipStream_t stream) {
  PrefillParams p{};
  p.q = static_cast<const uint16_t*>(a.q);
  p.k = static_cast<const uint16_t*>(a.k);
  p.v = static_cast<const uint16_t*>(a.v);
  p.o = static_cast<uint16_t*>(a.o);
  p.lse = a.lse;
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
  p.l_sb = a.lse_stride[0];
  p.l_sh = a.lse_stride[1];
  p.l_ss = a.lse_stride[2];
  p.B = a.batch;
  p.Hq = a.heads_q;
  p.Hkv = a.heads_kv;
  p.Sq = a.seqlen_q;
  p.Skv = a.seqlen_kv;
  p.D = a.head_dim;
  p.Dv = a.v_head_dim > 0 ? a.v_head_dim : a.head_dim;
  p.Do = a.o_head_dim > 0 ? a.o_head_dim : a.head_dim;
  p.q_offset = a.q_offset;
  p.causal = a.causal ? 1 : 0;
  p.window = clamp_window(a.window, a.q_offset, a.seqlen_q);
  p.sinks = clamp_sinks(a.sinks, p.window, a.q_offset, a.seqlen_q);
  p.ratio = a.heads_q / a.heads_kv;
  p.n_qt = (a.seqlen_q + kBlockM - 1) / kBlockM;
  const bool softcap = a.softcap > 0.0f;
  // Without softcap the kernels keep the running max of raw q.k, so their multiplier
  // must be positive: a negative scale flips Q's sign instead (q.k * scale =
  // (-q).k * |scale|), and a zero or tiny scale becomes 1e-30, which rounds every
  // exponent q.k * 1e-30 * log2 e (|q.k| < 1e20) to 0: the uniform softmax with
  // LSE = log(n) that scale 0 gives. With softcap the scores are tanh-transformed
  // before the max (tanh is odd), so any finite scale is used as it is.
  float scale = a.scale;
  p.q_neg = 0;
  if (!softcap) {
    if (scale < 0.0f) {
      scale = -scale;
      p.q_neg = 1;
    }
    scale = fmaxf(scale, 1e-30f);
  }
  if (softcap) {
    p.score_mul = scale / a.softcap;
    p.cap_mul = a.softcap * kLog2e;
  } else {
    p.score_mul = scale * kLog2e;
    p.cap_mul = 0.0f;
  }
  p.ref_bq = a.ref_block_q > 0 ? a.ref_block_q : 64;
  p.ref_bkv = a.ref_block_kv > 0 ? a.ref_block_kv : 64;
  p.masked_lse_mode = a.window > 0 && a.sinks > 0 ? 1 : a.masked_lse_mode;
  p.kmask = a.block_key_mask;
  p.kmask_words = a.block_key_mask_words;
  p.visited = a.block_visited;

  // The kernels move 16-byte chunks: callers guarantee 16-byte aligned bases, strides
  // that are multiples of 8 elements and head_dim % 8 == 0 (checked by ffa_prefill_fwd),
  // and per-tile byte offsets that fit 32 bits.
  const int64_t grid64 = static_cast<int64_t>(p.n_qt) * a.batch * a.heads_q;
  if (grid64 <= 0) return FFA_OK;
  if (grid64 > 0x7fffffff) return FFA_ERR_TOO_LARGE;
  const SplitPlan pl = plan_split(a);
  const bool cached = a.k_cache != nullptr && a.cache_len > 0;
  if (pl.n_split > 0 && a.workspace != nullptr && a.workspace_bytes >= pl.bytes) {
    SplitParams& sp = p.sp;
    sp.kc = static_cast<const uint16_t*>(a.k_cache);
    sp.vc = static_cast<const uint16_t*>(a.v_cache);
    sp.kc_sb = a.k_cache_stride[0];
    sp.kc_sh = a.k_cache_stride[1];
    sp.kc_ss = a.k_cache_stride[2];
    sp.vc_sb = a.v_cache_stride[0];
    sp.vc_sh = a.v_cache_stride[1];
    sp.vc_ss = a.v_cache_stride[2];
    sp.cache_len = cached ? a.cache_len : 0;
    sp.lo0 = pl.lo0;
    sp.lo1 = pl.lo1;
    sp.len = pl.len;
    sp.n0 = pl.n0;
    sp.n_split = pl.n_split;
    p.n_sink = pl.n_sink;
    p.sink_end = pl.sink_end;
    sp.pack = pl.pack;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.heads_q * a.seqlen_q;
    sp.ws_o = static_cast<float*>(a.workspace);
    sp.ws_lse = sp.ws_o + rows * pl.n_split * a.head_dim;
    p.n_qt = pl.n_qt;
    p.xcd_remap = pl.grid % 8 == 0 ? 1 : 0;
    const int grid_s = static_cast<int>(pl.grid);
    if (p.sinks > 0) {
      launch_split_sinks(p, a.dtype == FFA_DTYPE_BF16, softcap, grid_s, stream);
    } else if (a.dtype == FFA_DTYPE_BF16) {
      launch_split<Bf16Tag>(p, softcap, grid_s, stream);
    } else {
      launch_split<F16Tag>(p, softcap, grid_s, stream);
    }
    return hipGetLastError() == hipSuccess ? FFA_OK : FFA_ERR_LAUNCH;
  }
  if (cached) return FFA_ERR_WORKSPACE;  // only the split kernel reads a cache in place
  const int grid = static_cast<int>(grid64);
  prefill_grid_order(p.causal != 0, static_cast<int64_t>(a.batch) * a.heads_q, grid,
                     p.xcd_group, p.xcd_remap, prefill_pairs(a.head_dim, softcap, grid));

  if (p.sinks > 0) {
    launch_sinks(p, a.dtype, softcap, grid, stream);
  } else if (a.dtype == FFA_DTYPE_BF16) {
    launch_tag<Bf16Tag>(p, softcap, grid, stream);
  } else if (a.dtype == FFA_DTYPE_FP16) {
    launch_tag<F16Tag>(p, softcap, grid, stream);
  } else {
    launch_f32<false>(p, softcap, grid, stream);
  }
  return hipGetLastError() == hipSuccess ? FFA_OK : FFA_ERR_LAUNCH;
}

}  // namespace ffa
