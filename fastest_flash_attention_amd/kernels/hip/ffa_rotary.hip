// Rotary positions of queries and keys for gfx950, alone (ffa_rotary) or on the way of a
// batch's new tokens into the paged KV cache (ffa_paged_append_batch).
//
// Pair i of a row at position t turns by the angle t f_i (f = inv_freq):
//   (a, b) -> m (a cos - b sin, b cos + a sin)
// with a, b = dims i and i + R / 2 (halves) or 2i and 2i + 1 (interleaved), R = rotary_dim;
// dims past R pass through bit for bit. The gradient turns by the opposite angle.
//
// The angle is formed in 64 bits, as turns t f_i / (2 pi) less their nearest whole number:
// in 32 bits a position of 100000 loses 17 bits of a fast pair's angle. What is left, at most
// half a turn, is split into a float and a remainder d that turns the float's cos and sin by
// first order (d^2 < 2^-47), so that both are exact to about 2^-23 whatever the position.
// Products and sums are fp32, rounded once to the tensors' type.
//
// Bound by HBM: every element is read and written once. A thread owns P pairs (two vectors of
// P elements: 16 bytes each for P = 8 of 16 bits) of one token and walks over heads, so cos
// and sin are formed once for up to kHeadsMost heads; neighbouring threads take the chunks of
// a row, then the next token. Few tokens (a decode step) take fewer heads per thread instead,
// down to one, to have threads enough for the chip.
//
// Measured on MI355X (bf16 unless said; S tokens, Hq + Hk heads x D, R turned): 2 x 4096, 32 + 8 x
// 128, 128: 29 us, 5.7 TB/s; 2 x 4097, 24 + 8 x 80, 40: 17.3 us; 64 x 1, 32 + 8 x 128: 3.5 us.
//   rows loaded at once 1 / 2 / 4 / 8           29.1 / 29.4 / 29.9 / 31.2 us, fp32 7.5 / 7.2 / 7.2 / 7.2
//   at most 4 / 8 / 16 heads per thread         31.0 / 29.9 / 29.6 us, D 80 17.9 / 18.1 / 17.3
//   64 / 128 / 256 / 1024 k threads wanted      29.8 / 29.5 / 29.9 / 31.4 us, fp32 7.7 / 8.5 / 7.2 / 8.7
// With inputs and outputs both cold it takes 37 us. Nontemporal stores take 30 then, but the
// attention that reads the rows next loses more (rotary and attention together, 4 x 1024 tokens: 68 us
// against 64), and rows of 160 bytes take 32 us against 17. Nontemporal loads: 33 us cold, but 33
// against 29 warm and 31 against 17 with rows of 160 bytes.

#include <type_traits>

#include "ffa_common.h"
#include "ffa_internal.h"

namespace ffa {
namespace {

constexpr int kRotThreads = 256;
constexpr int kHeadsMost = 16;     // heads that share a thread's cos and sin
constexpr int kHeadsAtOnce = 2;   // rows whose loads are issued together
constexpr int64_t kThreadsWanted = 256 * 1024;  // four waves per SIMD

struct Rot32Tag {};

template <int BYTES>
struct RawOf;
template <>
struct RawOf<16> { using type = u32x4; };
template <>
struct RawOf<8> { using type = u32x2; };
template <>
struct RawOf<4> { using type = uint32_t; };
template <>
struct RawOf<2> { using type = uint16_t; };

template <typename Tag>
constexpr int kElemBytes = std::is_same_v<Tag, Rot32Tag> ? 4 : 2;

// P consecutive elements as loaded, and their values.
template <typename Tag, int P>
struct Piece {
  using Raw = typename RawOf<P * kElemBytes<Tag>>::type;
  __device__ static inline void get(const Raw& r, float (&x)[P]) {
    if constexpr (std::is_same_v<Tag, Rot32Tag>) {
      __builtin_memcpy(x, &r, sizeof(r));
    } else {
      uint16_t h[P];
      __builtin_memcpy(h, &r, sizeof(r));
#pragma unroll
      for (int e = 0; e < P; ++e) x[e] = Elem<Tag>::to_f32(h[e]);
    }
  }
  __device__ static inline Raw put(const float (&x)[P]) {
    Raw r;
    if constexpr (std::is_same_v<Tag, Rot32Tag>) {
      __builtin_memcpy(&r, x, sizeof(r));
    } else if constexpr (P == 1) {
      r = static_cast<uint16_t>(Elem<Tag>::pack2(x[0], x[0]) & 0xffffu);
    } else {
      uint32_t w[P / 2];
#pragma unroll
      for (int e = 0; e < P / 2; ++e) w[e] = Elem<Tag>::pack2(x[2 * e], x[2 * e + 1]);
      __builtin_memcpy(&r, w, sizeof(r));
    }
    return r;
  }
};

struct RotaryParams {
  const char* q;
  const char* k;
  const char* v;  // append only
  char* q_out;
  char* k_out;    // append: the K pool
  char* v_out;    // append: the V pool
  const double* inv_freq;
  const void* positions;     // or null
  const int32_t* tables;     // append: block tables
  const int32_t* counts;     // append: tokens of each sequence that count, or null
  // bytes between batches, heads and tokens
  int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;
  int64_t qo_sb, qo_sh, qo_ss, ko_sb, ko_sh, ko_ss;
  int64_t pos_sb, pos_ss;    // elements of `positions`
  int64_t offset;            // added to every position
  int pos_wide;              // positions are 64-bit
  int add_s;                 // the token's index is added to its position
  int S, Hq, Hk, D, R;
  int n_rot, n_it;           // items of a row that turn, and all of them
  int n_threads, hpt;
  float sign, magnitude;
  int table_stride, num_pages, page_size;
};

template <typename Tag, int P, bool IL, bool APPEND>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(const RotaryParams p) {
  using Pc = Piece<Tag, P>;
  using Raw = typename Pc::Raw;
  constexpr int EB = kElemBytes<Tag>;
  const int id = static_cast<int>(blockIdx.x) * kRotThreads + static_cast<int>(threadIdx.x);
  if (id >= p.n_threads) return;
  const int tok = id / p.n_it;
  const int it = id - tok * p.n_it;
  const int b = tok / p.S;
  const int s = tok - b * p.S;
  const int h0 = static_cast<int>(blockIdx.y) * p.hpt;
  const int n_turn = p.Hq + p.Hk;
  const int h1 = min(h0 + p.hpt, APPEND ? n_turn + p.Hk : n_turn);

  int64_t pos = p.offset + (p.add_s ? s : 0);
  if (p.positions != nullptr) {
    const int64_t at = b * p.pos_sb + s * p.pos_ss;
    pos += p.pos_wide ? static_cast<const int64_t*>(p.positions)[at]
                      : static_cast<const int32_t*>(p.positions)[at];
  }

  // this thread's two vectors: a turning item's, or two chunks that pass through
  const bool turns = it < p.n_rot;
  int da, db;
  if (turns) {
    da = IL ? 2 * P * it : P * it;
    db = IL ? da + P : da + (p.R >> 1);
  } else {
    da = p.R + 2 * P * (it - p.n_rot);
    db = da + P;
  }
  const bool has_b = db < p.D;

  float cs[P], sn[P];
  if (turns && h0 < n_turn) {
#pragma unroll
    for (int e = 0; e < P; ++e) {
      double t = static_cast<double>(pos) * (p.inv_freq[P * it + e] * 0.15915494309189535);
      t = 2.0 * (t - rint(t));  // half turns, in [-1, 1]
      const float x = static_cast<float>(t);
      const float d = static_cast<float>(t - static_cast<double>(x)) * 3.14159265f;
      float c0, s0;
      sincospif(x, &s0, &c0);
      cs[e] = fmaf(-d, s0, c0) * p.magnitude;
      sn[e] = fmaf(d, c0, s0) * p.magnitude * p.sign;
    }
  }

  // append: where this token's row of KV head 0 lies in the pools, if it has a place there
  int64_t slot_row = 0;
  bool placed = true;
  if constexpr (APPEND) {
    placed = pos >= 0 && (p.counts == nullptr || s < p.counts[b]);
    if (placed) {
      const int64_t at = pos / p.page_size;
      placed = at < p.table_stride;
      if (placed) {
        const int page = p.tables[static_cast<int64_t>(b) * p.table_stride + at];
        placed = page >= 0 && page < p.num_pages;
        slot_row = static_cast<int64_t>(page) * p.Hk * p.page_size + (pos - at * p.page_size);
      }
    }
  }

  for (int hh = h0; hh < h1; hh += kHeadsAtOnce) {
    Raw a[kHeadsAtOnce], c[kHeadsAtOnce];
#pragma unroll
    for (int u = 0; u < kHeadsAtOnce; ++u) {
      const int h = hh + u;
      if (h < h1) {
        const char* src;
        if (h < p.Hq) {
          src = p.q + b * p.q_sb + h * p.q_sh + s * p.q_ss;
        } else if (h < n_turn) {
          src = p.k + b * p.k_sb + (h - p.Hq) * p.k_sh + s * p.k_ss;
        } else {
          src = p.v + b * p.v_sb + (h - n_turn) * p.v_sh + s * p.v_ss;
        }
        a[u] = *reinterpret_cast<const Raw*>(src + da * EB);
        if (has_b) c[u] = *reinterpret_cast<const Raw*>(src + db * EB);
      }
    }
#pragma unroll
    for (int u = 0; u < kHeadsAtOnce; ++u) {
      const int h = hh + u;
      if (h >= h1) break;
      if (turns && h < n_turn) {
        float x[P], y[P];
        Pc::get(a[u], x);
        Pc::get(c[u], y);
        float lo[2 * P];  // the item's pairs: (lo[2 e], lo[2 e + 1]) = pair e
#pragma unroll
        for (int e = 0; e < P; ++e) {
          if constexpr (IL && P > 1) {
            lo[e] = x[e];
            lo[P + e] = y[e];
          } else {
            lo[2 * e] = x[e];
            lo[2 * e + 1] = y[e];
          }
        }
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const float va = lo[2 * e];
          const float vb = lo[2 * e + 1];
          lo[2 * e] = fmaf(va, cs[e], -(vb * sn[e]));
          lo[2 * e + 1] = fmaf(vb, cs[e], va * sn[e]);
        }
#pragma unroll
        for (int e = 0; e < P; ++e) {
          x[e] = IL && P > 1 ? lo[e] : lo[2 * e];
          y[e] = IL && P > 1 ? lo[P + e] : lo[2 * e + 1];
        }
        a[u] = Pc::put(x);
        c[u] = Pc::put(y);
      }
      char* dst;
      if (h < p.Hq) {
        dst = p.q_out + b * p.qo_sb + h * p.qo_sh + s * p.qo_ss;
      } else if constexpr (APPEND) {
        if (!placed) continue;
        const bool is_k = h < n_turn;
        const int hk = is_k ? h - p.Hq : h - n_turn;
        dst = (is_k ? p.k_out : p.v_out) +
              (slot_row + static_cast<int64_t>(hk) * p.page_size) * p.D * EB;
      } else {
        dst = p.k_out + b * p.ko_sb + (h - p.Hq) * p.ko_sh + s * p.ko_ss;
      }
      *reinterpret_cast<Raw*>(dst + da * EB) = a[u];
      if (has_b) *reinterpret_cast<Raw*>(dst + db * EB) = c[u];
    }
  }
}

// The most pairs of an item (as asked, or fewer) that rows, strides and addresses allow: both
// vectors whole and aligned. `bits` is the OR of every address and byte stride.
int piece_pairs(int most, int elem_bytes, bool interleaved, int D, int R, uint64_t bits) {
  for (int P = most; P > 1; P /= 2) {
    const int unit = interleaved ? 2 * P : P;
    const int turn = interleaved ? R : R / 2;
    if (turn % unit == 0 && (D - R) % P == 0 && R % P == 0 &&
        bits % static_cast<uint64_t>(P * elem_bytes) == 0) {
      return P;
    }
  }
  return 1;
}

template <typename Tag, int P, bool APPEND>
void run_rotary(const RotaryParams& p, bool il, dim3 grid, hipStream_t s) {
  if (il) {
    hipLaunchKernelGGL((rotary_kernel<Tag, P, true, APPEND>), grid, dim3(kRotThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL((rotary_kernel<Tag, P, false, APPEND>), grid, dim3(kRotThreads), 0, s, p);
  }
}

// Sizes the grid and launches. p.n_rot, n_it, n_threads and hpt are set here.
template <bool APPEND>
int launch_items(RotaryParams& p, int64_t tokens, int dtype, bool il, uint64_t bits, hipStream_t s) {
  const int eb = dtype == FFA_DTYPE_FP32 ? 4 : 2;
  const int P = piece_pairs(16 / eb, eb, il, p.D, p.R, bits);
  p.n_rot = p.R / 2 / P;
  p.n_it = p.n_rot + (p.D - p.R + 2 * P - 1) / (2 * P);
  const int64_t heads = static_cast<int64_t>(p.Hq) + (APPEND ? 2 : 1) * static_cast<int64_t>(p.Hk);
  const int64_t threads = tokens * p.n_it;
  if (threads > 0x7fffff00) return FFA_ERR_TOO_LARGE;
  if (threads == 0 || heads == 0) return FFA_OK;
  int64_t hpt = (threads * heads + kThreadsWanted - 1) / kThreadsWanted;
  hpt = hpt < 1 ? 1 : (hpt > kHeadsMost ? kHeadsMost : hpt);
  if ((heads + hpt - 1) / hpt > 65535) return FFA_ERR_TOO_LARGE;
  p.hpt = static_cast<int>(hpt);
  p.n_threads = static_cast<int>(threads);
  const dim3 grid(static_cast<unsigned>((threads + kRotThreads - 1) / kRotThreads),
                  static_cast<unsigned>((heads + hpt - 1) / hpt));
  auto run = [&](auto tag) {
    using Tag = decltype(tag);
    switch (P) {
      case 8:
        if constexpr (kElemBytes<Tag> == 2) run_rotary<Tag, 8, APPEND>(p, il, grid, s);
        break;
      case 4: run_rotary<Tag, 4, APPEND>(p, il, grid, s); break;
      case 2: run_rotary<Tag, 2, APPEND>(p, il, grid, s); break;
      default: run_rotary<Tag, 1, APPEND>(p, il, grid, s); break;
    }
  };
  if (dtype == FFA_DTYPE_BF16) {
    run(Bf16Tag{});
  } else if (dtype == FFA_DTYPE_FP16) {
    run(F16Tag{});
  } else {
    run(Rot32Tag{});
  }
  return hipGetLastError() == hipSuccess ? FFA_OK : FFA_ERR_LAUNCH;
}

// One tensor's address and byte strides into the parameters, and into the alignment bits.
// A stride that is never stepped over (one batch, head or token) does not count.
void set_view(const void* base, const int64_t (&st)[3], const int (&n)[3], int eb, int64_t& sb,
              int64_t& sh, int64_t& ss, uint64_t& bits) {
  int64_t* out[3] = {&sb, &sh, &ss};
  bits |= reinterpret_cast<uintptr_t>(base);
  for (int i = 0; i < 3; ++i) {
    *out[i] = n[i] > 1 ? st[i] * eb : 0;
    bits |= static_cast<uint64_t>(*out[i]);
  }
}

}  // namespace

int launch_rotary(const ffa_rotary_args& a, hipStream_t stream) {
  RotaryParams p{};
  const int eb = a.dtype == FFA_DTYPE_FP32 ? 4 : 2;
  uint64_t bits = 0;
  if (a.heads_q > 0) {
    const int n[3] = {a.batch, a.heads_q, a.seqlen};
    p.q = static_cast<const char*>(a.q);
    p.q_out = static_cast<char*>(a.q_out);
    set_view(a.q, a.q_stride, n, eb, p.q_sb, p.q_sh, p.q_ss, bits);
    set_view(a.q_out, a.q_out_stride, n, eb, p.qo_sb, p.qo_sh, p.qo_ss, bits);
  }
  if (a.heads_k > 0) {
    const int n[3] = {a.batch, a.heads_k, a.seqlen};
    p.k = static_cast<const char*>(a.k);
    p.k_out = static_cast<char*>(a.k_out);
    set_view(a.k, a.k_stride, n, eb, p.k_sb, p.k_sh, p.k_ss, bits);
    set_view(a.k_out, a.k_out_stride, n, eb, p.ko_sb, p.ko_sh, p.ko_ss, bits);
  }
  p.inv_freq = a.inv_freq;
  p.positions = a.positions;
  p.pos_sb = a.position_stride[0];
  p.pos_ss = a.position_stride[1];
  p.pos_wide = a.position_bytes == 8;
  p.offset = a.positions != nullptr ? 0 : a.q_offset;
  p.add_s = a.positions == nullptr;
  p.S = a.seqlen;
  p.Hq = a.heads_q;
  p.Hk = a.heads_k;
  p.D = a.head_dim;
  p.R = a.rotary_dim;
  p.sign = a.inverse ? -1.0f : 1.0f;
  p.magnitude = a.magnitude;
  return launch_items<false>(p, static_cast<int64_t>(a.batch) * a.seqlen, a.dtype, a.interleaved != 0,
                             bits, stream);
}

int launch_paged_append_batch(const ffa_paged_append_batch_args& a, hipStream_t stream) {
  RotaryParams p{};
  const int eb = a.dtype == FFA_DTYPE_FP32 ? 4 : 2;
  uint64_t bits = reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages) |
                  static_cast<uint64_t>(a.head_dim) * eb;
  if (a.heads_q > 0) {
    const int n[3] = {a.batch, a.heads_q, a.n_tokens};
    p.q = static_cast<const char*>(a.q);
    p.q_out = static_cast<char*>(a.q_out);
    set_view(a.q, a.q_stride, n, eb, p.q_sb, p.q_sh, p.q_ss, bits);
    set_view(a.q_out, a.q_out_stride, n, eb, p.qo_sb, p.qo_sh, p.qo_ss, bits);
  }
  const int n[3] = {a.batch, a.heads_kv, a.n_tokens};
  p.k = static_cast<const char*>(a.k_new);
  p.v = static_cast<const char*>(a.v_new);
  set_view(a.k_new, a.k_new_stride, n, eb, p.k_sb, p.k_sh, p.k_ss, bits);
  set_view(a.v_new, a.v_new_stride, n, eb, p.v_sb, p.v_sh, p.v_ss, bits);
  p.k_out = static_cast<char*>(a.k_pages);
  p.v_out = static_cast<char*>(a.v_pages);
  p.inv_freq = a.inv_freq;
  p.positions = a.positions;
  p.tables = a.block_tables;
  p.counts = a.counts;
  p.pos_sb = 1;
  p.pos_ss = 0;
  p.pos_wide = 0;
  p.add_s = 1;
  p.S = a.n_tokens;
  p.Hq = a.heads_q;
  p.Hk = a.heads_kv;
  p.D = a.head_dim;
  p.R = a.rotary_dim;
  p.sign = 1.0f;
  p.magnitude = a.magnitude;
  p.table_stride = a.block_table_stride;
  p.num_pages = a.num_pages;
  p.page_size = a.page_size;
  return launch_items<true>(p, static_cast<int64_t>(a.batch) * a.n_tokens, a.dtype, a.interleaved != 0,
                            bits, stream);
}

}  // namespace ffa
