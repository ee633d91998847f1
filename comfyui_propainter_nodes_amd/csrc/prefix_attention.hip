// prefix_attention.hip -- attention of a batch whose sequences share a prefix and have own keys behind it.
// Contract: include/propainter_mi355.h (pp_prefix_attention); the inner loop: tile_attention.h.
//
// All B L G rows of a key / value head (G = H / KH query heads share it) meet the same prefix keys: they are tiled 128 at a time, so a
// prefix of P keys is staged ceil(B L G / 128) times (its keys twice that for f32 above 128 channels) instead of B times, and the two products run at matrix speed.  The prefix is
// cut into pieces so that few rows still fill the chip; the own keys of a sequence (its L G rows) are work-groups of the same launch.  Every piece
// leaves (maximum, sum, sum of weighted values) in fp32; a second launch joins them in piece order.
//
// 128 tokens behind 32768 keys, 64 / 8 heads of 128, f16: 176-200 us (138 GF; the prefix part at the rate of a long prompt, one wave of four in
// the own part); 32 tokens behind 8192 keys, 32 / 8 heads, bf16: 25 us, 20 + 5 for the join -- 8-10 steps per work-group, each waits for memory.
#include "attention_parts.h"

#include <math.h>

#include <initializer_list>

namespace pp {

struct PrefixK {
  const void *q, *kp, *vp, *ko, *vo;
  const int* own_len;
  PartsK parts;
  int64_t q_seq, q_row, q_head, kp_row, kp_head, vp_row, vp_head, ko_seq, ko_row, ko_head, vo_seq, vo_row, vo_head;
  int64_t P, S;
  int B, L, H, KH, G, D, prefix_splits, own_splits;
  int prefix_tiles, own_tiles;  // 128-row tiles of all B L G rows / of one sequence's L G rows
  int64_t prefix_items;         // work-groups of the prefix part; those of the own part follow
  float sc;
};

template <typename Tile>
__global__ void __launch_bounds__(Tile::kThreads, Tile::kWaves) prefix_attention_kernel(const PrefixK a) {
  typedef typename Tile::type T;
  constexpr int kRows = Tile::kRows;
  const int lane = lane_id(), wave = wave_uniform((int)threadIdx.x >> 6), q32 = lane & 31, h = lane >> 5;
  const int d0 = (int)blockIdx.x % Tile::kHalves * Tile::kDV;  // the value channels from d0 on
  const int DV = a.D - d0 < Tile::kDV ? a.D - d0 : Tile::kDV;
  int64_t id = (int64_t)blockIdx.x / Tile::kHalves;
  const bool shared = id < a.prefix_items;
  if (!shared) id -= a.prefix_items;
  const int kh = (int)(id % a.KH);
  id /= a.KH;
  const int lg = a.L * a.G;
  int seq = 0, part;
  int64_t row0, rows, n0, n1;  // rows of the item's tile space; its keys
  const T *k, *v;
  int64_t k_row, v_row, visible = 0;
  if (shared) {
    const int tile = (int)(id % a.prefix_tiles);
    part = (int)(id / a.prefix_tiles);
    rows = (int64_t)a.B * lg;
    row0 = (int64_t)tile * kRows;
    n0 = a.P * part / a.prefix_splits;
    n1 = a.P * (part + 1) / a.prefix_splits;
    k = (const T*)a.kp + kh * a.kp_head;
    v = (const T*)a.vp + kh * a.vp_head + d0;
    k_row = a.kp_row;
    v_row = a.vp_row;
  } else {
    const int tile = (int)(id % a.own_tiles);
    id /= a.own_tiles;
    const int sp = (int)(id % a.own_splits);
    seq = (int)(id / a.own_splits);
    part = a.prefix_splits + sp;
    rows = lg;
    row0 = (int64_t)tile * kRows;
    const int64_t len = a.own_len[seq];
    visible = len < 0 ? 0 : len > a.S ? a.S : len;
    n0 = visible * sp / a.own_splits;
    n1 = visible * (sp + 1) / a.own_splits;
    k = (const T*)a.ko + seq * a.ko_seq + kh * a.ko_head;
    v = (const T*)a.vo + seq * a.vo_seq + kh * a.vo_head + d0;
    k_row = a.ko_row;
    v_row = a.vo_row;
  }
  // keys of [n0, n1) that a row sees
  auto limit_of = [&](int64_t row) __attribute__((always_inline)) -> int {
    const int64_t c = shared ? n1 - n0 : visible - a.L + row / a.G + 1 - n0;
    return (int)(c < 0 ? 0 : c > n1 - n0 ? n1 - n0 : c);
  };
  const int64_t last = rows - 1, wrow = row0 + 32 * wave, row = wrow + q32;
  AttnLimits lim;
  lim.wave_max = wrow <= last ? limit_of(wrow + 31 < last ? wrow + 31 : last) : 0;
  lim.group_min = limit_of(row0);
  lim.nkeys = limit_of(row0 + kRows - 1 < last ? row0 + kRows - 1 : last);
  Tile t;
  AttnState<Tile> st;
  t.init(PP_DYN_SMEM);
  const bool live = row <= last;
  lim.row = live ? limit_of(row) : 0;
  {
    const int64_t b = shared ? row / lg : seq;
    const int in_seq = (int)(shared ? row % lg : row);
    t.load_q(live ? (const T*)a.q + b * a.q_seq + (in_seq / a.G) * a.q_row + (kh * a.G + in_seq % a.G) * a.q_head : nullptr, a.D);
  }
  attend(t, st, k + n0 * k_row, v + n0 * v_row, k_row, v_row, lim, a.D, DV, a.sc);
  if (st.not_finite) add_not_finite(t, st, v + n0 * v_row, v_row, lim, DV);
  if (!live) return;
  const int64_t b = shared ? row / lg : seq;
  const int in_seq = (int)(shared ? row % lg : row);
  store_part(a.parts, t, st, (b * a.L + in_seq / a.G) * a.H + kh * a.G + in_seq % a.G, part, lim.row > 0, d0, DV);
}

}  // namespace pp

template <typename Tile>
static int launch_prefix(void* stream, pp::PrefixK& a) {
  using namespace pp;
  const int64_t rows = (int64_t)a.B * a.L * a.G;
  a.prefix_tiles = (int)((rows + Tile::kRows - 1) / Tile::kRows);
  a.own_tiles = (a.L * a.G + Tile::kRows - 1) / Tile::kRows;
  a.prefix_items = (int64_t)a.prefix_splits * a.prefix_tiles * a.KH;
  const int64_t items = a.prefix_items + (int64_t)a.own_splits * a.B * a.own_tiles * a.KH;
  if (items * Tile::kHalves * 256 >= ((int64_t)1 << 32)) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prefix_attention: the launch needs 2^32 threads or more");
  PP_ALLOW_BIG_LDS((&prefix_attention_kernel<Tile>), Tile::kSmem);
  if (items > 0) PP_LAUNCH((prefix_attention_kernel<Tile>), dim3((unsigned)(items * Tile::kHalves)), dim3(Tile::kThreads), Tile::kSmem, stream, a);
  const int rc = pp_check_launch("pp_prefix_attention");
  if (rc != PP_OK) return rc;
  return launch_join<Tile>(stream, a.parts, "pp_prefix_attention(join)");
}

template <typename T>
static int launch_prefix_d(void* stream, pp::PrefixK& a) {
  using namespace pp;
  if constexpr (sizeof(T) == 2) {
    if (a.D <= 32) return launch_prefix<AttnTile<T, 32, 4, 2>>(stream, a);
    if (a.D <= 64) return launch_prefix<AttnTile<T, 64, 4, 2>>(stream, a);
    if (a.D <= 96) return launch_prefix<AttnTile<T, 96, 4, 1>>(stream, a);
    if (a.D <= 128) return launch_prefix<AttnTile<T, 128, 4, 1>>(stream, a);
    return launch_prefix<AttnTile<T, 256, 4, 1>>(stream, a);
  } else {
    if (a.D <= 32) return launch_prefix<AttnTile<T, 32, 4, 1>>(stream, a);
    if (a.D <= 64) return launch_prefix<AttnTile<T, 64, 4, 1>>(stream, a);
    if (a.D <= 96) return launch_prefix<AttnTile<T, 96, 4, 1>>(stream, a);
    if (a.D <= 128) return launch_prefix<AttnTile<T, 128, 4, 1>>(stream, a);
    return launch_prefix<AttnTile<T, 256, 4, 1>>(stream, a);
  }
}

extern "C" int32_t pp_prefix_attention(void* stream, const pp_prefix_attention_params* p) {
  using namespace pp;
  if (!p || !p->q || !p->out || !p->own_len || !p->scratch) return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: null argument");
  if (p->dtype != PP_F32 && p->dtype != PP_F16 && p->dtype != PP_BF16) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prefix_attention: dtype");
  if (p->KH < 1 || p->H < 1 || p->H % p->KH || p->H > (1 << 20))
    return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: H must be a multiple of KH");
  const int e = p->dtype == PP_F32 ? 4 : 8;  // elements of 16 bytes
  if (p->D < 1 || p->D > 256 || p->D % e) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prefix_attention: D must be a multiple of 8 (fp32: 4) up to 256");
  if (p->B < 0 || p->L < 0 || p->P < 0 || p->S < 0 || p->B > (1 << 24) || p->L > (1 << 20))
    return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: B, L, P, S out of range");
  if (p->P > kMostKeys || p->S > kMostKeys) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prefix_attention: P or S above 2^31 - 1024");
  if ((p->P > 0 && (!p->kp || !p->vp)) || (p->S > 0 && (!p->ko || !p->vo))) return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: null keys or values");
  if (p->prefix_splits < 0 || p->own_splits < 0 || p->prefix_splits > 65536 || p->own_splits > 65536 || (p->P > 0 && p->prefix_splits < 1) ||
      (p->S > 0 && p->own_splits < 1) || p->prefix_splits + p->own_splits < 1)
    return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: splits must be in [0, 65536], and at least 1 for a part with keys");
  if (!(p->scale > 0.f) || !(p->scale * kLog2e < INFINITY)) return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: scale must be positive and finite");
  const int64_t strides[16] = {p->q_seq, p->q_row, p->q_head, p->kp_row, p->kp_head, p->vp_row, p->vp_head, p->ko_seq,
                               p->ko_row, p->ko_head, p->vo_seq, p->vo_row, p->vo_head, p->out_seq, p->out_row, p->out_head};
  for (int i = 0; i < 16; ++i)
    if (strides[i] < 0 || strides[i] % e) return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: strides must be >= 0 and keep rows 16-byte aligned");
  // (a block of keys is addressed with 32-bit byte offsets)
  for (const int64_t row : {p->kp_row, p->vp_row, p->ko_row, p->vo_row})
    if (row >= 1 << 24) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prefix_attention: a key or value row stride must be below 2^24 elements");
  if (((uintptr_t)p->q | (uintptr_t)p->kp | (uintptr_t)p->vp | (uintptr_t)p->ko | (uintptr_t)p->vo | (uintptr_t)p->out | (uintptr_t)p->scratch) % 16)
    return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: tensors must be 16-byte aligned");
  if (p->B == 0 || p->L == 0) return PP_OK;  // no row to write
  PrefixK a;
  a.q = p->q; a.kp = p->kp; a.vp = p->vp; a.ko = p->ko; a.vo = p->vo; a.own_len = (const int*)p->own_len;
  a.q_seq = p->q_seq; a.q_row = p->q_row; a.q_head = p->q_head;
  a.kp_row = p->kp_row; a.kp_head = p->kp_head; a.vp_row = p->vp_row; a.vp_head = p->vp_head;
  a.ko_seq = p->ko_seq; a.ko_row = p->ko_row; a.ko_head = p->ko_head;
  a.vo_seq = p->vo_seq; a.vo_row = p->vo_row; a.vo_head = p->vo_head;
  a.P = p->P; a.S = p->S;
  a.B = (int)p->B; a.L = (int)p->L; a.H = (int)p->H; a.KH = (int)p->KH; a.G = (int)(p->H / p->KH); a.D = (int)p->D;
  a.prefix_splits = p->P > 0 ? p->prefix_splits : 0;
  a.own_splits = p->S > 0 ? p->own_splits : 0;
  a.sc = p->scale * kLog2e;
  // (the products below stay inside 64 bits: B L and H are at most 2^24 and 2^20)
  if (p->B * p->L > (1 << 24) || p->B * p->L * p->H > (1 << 24))
    return pp_fail(PP_ERR_UNSUPPORTED, "pp_prefix_attention: more than 2^24 rows (B * L * H)");
  const int64_t rows = p->B * p->L * p->H;
  if (p->scratch_bytes < rows * (p->prefix_splits + p->own_splits) * (p->D + 4) * 4)
    return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: scratch smaller than B * L * H * (prefix_splits + own_splits) * (D + 4) floats");
  PartsK& pt = a.parts;
  pt.parts = a.prefix_splits + a.own_splits;
  pt.o = (float*)p->scratch;
  pt.ml = pt.o + rows * pt.parts * p->D;
  pt.out = p->out; pt.out_seq = p->out_seq; pt.out_row = p->out_row; pt.out_head = p->out_head;
  pt.lse = nullptr; pt.cu_q = nullptr; pt.ncu = 0;
  pt.rows = rows; pt.L = a.L; pt.H = a.H; pt.D = a.D; pt.sc = a.sc; pt.scale = p->scale;
  if (p->dtype == PP_F32) return launch_prefix_d<float>(stream, a);
  if (p->dtype == PP_F16) return launch_prefix_d<half_t>(stream, a);
  return launch_prefix_d<bf16_t>(stream, a);
}
