// prefix_attention.hip -- attention of a batch whose sequences share a prefix and have own keys behind it.
// Contract: include/propainter_mi355.h (pp_prefix_attention); the inner loop: tile_attention.h.
//
// All B L G rows of a key / value head (G = H / KH query heads share it) meet the same prefix keys: they are tiled 128 at a time, so a
// prefix of P keys is staged ceil(B L G / 128) times instead of B times, and the two products run at matrix speed.  The prefix is
// cut into pieces so that few rows still fill the chip; the own keys of a sequence (its L G rows) are work-groups of the same launch.  Every piece
// leaves (maximum, sum, sum of weighted values) in fp32; a second launch joins them in piece order.
#include "tile_attention.h"
#include "pp_host.h"

#include <math.h>

#include <initializer_list>

namespace pp {

struct PrefixK {
  const void *q, *kp, *vp, *ko, *vo;
  void* out;
  const int* own_len;
  float* part_o;   // [row][part][D]
  float* part_ml;  // [row][part][2]
  int64_t q_seq, q_row, q_head, kp_row, kp_head, vp_row, vp_head, ko_seq, ko_row, ko_head, vo_seq, vo_row, vo_head, out_seq, out_row, out_head;
  int64_t P, S;
  int B, L, H, KH, G, D, prefix_splits, own_splits, parts;
  int prefix_tiles, own_tiles;  // 128-row tiles of all B L G rows / of one sequence's L G rows
  int64_t prefix_items;         // work-groups of the prefix part; those of the own part follow
  float sc;
};

template <typename Tile>
__global__ void __launch_bounds__(Tile::kThreads, Tile::kWaves) prefix_attention_kernel(const PrefixK a) {
  typedef typename Tile::type T;
  constexpr int kRows = Tile::kRows, RB = Tile::RB;
  const int lane = lane_id(), wave = wave_uniform((int)threadIdx.x >> 6), q32 = lane & 31, h = lane >> 5;
  const bool shared = (int64_t)blockIdx.x < a.prefix_items;
  int64_t id = shared ? (int64_t)blockIdx.x : (int64_t)blockIdx.x - a.prefix_items;
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
    v = (const T*)a.vp + kh * a.vp_head;
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
    v = (const T*)a.vo + seq * a.vo_seq + kh * a.vo_head;
    k_row = a.ko_row;
    v_row = a.vo_row;
  }
  // keys of [n0, n1) that a row sees
  auto limit_of = [&](int64_t row) __attribute__((always_inline)) -> int {
    const int64_t c = shared ? n1 - n0 : visible - a.L + row / a.G + 1 - n0;
    return (int)(c < 0 ? 0 : c > n1 - n0 ? n1 - n0 : c);
  };
  const int64_t last = rows - 1, wrow = row0 + 32 * RB * wave;
  AttnLimits<RB> lim;
  lim.wave_min = wrow <= last ? limit_of(wrow) : 0;
  lim.wave_max = wrow <= last ? limit_of(wrow + 32 * RB - 1 < last ? wrow + 32 * RB - 1 : last) : 0;
  lim.group_min = limit_of(row0);
  lim.nkeys = limit_of(row0 + kRows - 1 < last ? row0 + kRows - 1 : last);
  Tile t;
  AttnState<Tile> st;
  t.init(PP_DYN_SMEM);
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int64_t row = wrow + 32 * rb + q32;
    const bool live = row <= last;
    lim.row[rb] = live ? limit_of(row) : 0;
    const int64_t b = shared ? row / lg : seq;
    const int in_seq = (int)(shared ? row % lg : row);
    t.load_q(rb, live ? (const T*)a.q + b * a.q_seq + (in_seq / a.G) * a.q_row + (kh * a.G + in_seq % a.G) * a.q_head : nullptr, a.D);
  }
  attend(t, st, k + n0 * k_row, v + n0 * v_row, k_row, v_row, lim, a.D, a.sc);
  if (st.not_finite) add_not_finite(t, st, v + n0 * v_row, v_row, lim, a.D);
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int64_t row = wrow + 32 * rb + q32;
    if (row > last) continue;
    const int64_t b = shared ? row / lg : seq;
    const int in_seq = (int)(shared ? row % lg : row);
    const int64_t at = ((b * a.L + in_seq / a.G) * a.H + kh * a.G + in_seq % a.G) * a.parts + part;
    float* dst = a.part_o + at * a.D;
#pragma unroll
    for (int db = 0; db < Tile::kDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * db + 8 * g + 4 * h;
        const f16v& o = st.o[rb][db];
        if (d < a.D) *reinterpret_cast<f4*>(dst + d) = f4{o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]};
      }
    if (h == 0) {
      a.part_ml[2 * at] = st.m[rb];
      a.part_ml[2 * at + 1] = st.l[rb];
    }
  }
}

// Joins the parts of a row: a row's D values are DL threads of 4, and PG groups of such threads take every PG-th part each, four parts'
// loads in flight; then the groups' results are joined in LDS.  (One thread per 4 values walking all parts took 17 us for 33 parts of 1024 rows.)
template <typename Tile, int DL>
__global__ void __launch_bounds__(256) prefix_join_kernel(const PrefixK a, int pg_log2) {
  typedef typename Tile::type T;
  __shared__ f4 so[256];
  __shared__ float sm[256], sl[256];
  const int tid = (int)threadIdx.x, dl = tid % DL, PG = 1 << pg_log2, pg = tid / DL % PG, slot = tid / (DL * PG);
  const int64_t row = (int64_t)blockIdx.x * (256 / (DL * PG)) + slot, rows = (int64_t)a.B * a.L * a.H;
  const bool live = row < rows && 4 * dl < a.D;
  float m = neg_inf(), l = 0.f;
  f4 o = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    const float* ml = a.part_ml + row * a.parts * 2;
    const float* po = a.part_o + row * a.parts * a.D + 4 * dl;
    for (int p0 = pg; p0 < a.parts; p0 += 4 * PG) {
      float pm[4], pl[4];
      f4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int p = p0 + u * PG;
        const bool in = p < a.parts;
        pm[u] = in ? ml[2 * p] : neg_inf();
        pl[u] = in ? ml[2 * p + 1] : 0.f;
        v[u] = in ? *reinterpret_cast<const f4*>(po + (int64_t)p * a.D) : f4{0.f, 0.f, 0.f, 0.f};
      }
      const float top = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), m);
      const float w = m == top ? 1.f : fast_exp2((m - top) * a.sc);
      m = top;
      l *= w;
      o *= w;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float x = pm[u] == top ? 1.f : fast_exp2((pm[u] - top) * a.sc);
        l += x * pl[u];
        o += x * v[u];
      }
    }
  }
  so[tid] = o;
  sm[tid] = m;
  sl[tid] = l;
  __syncthreads();
  if (!live || pg != 0) return;
  float top = m;
  for (int g = 1; g < PG; ++g) top = fmaxf(top, sm[tid + g * DL]);
  const float w = m == top ? 1.f : fast_exp2((m - top) * a.sc);
  l *= w;
  o *= w;
  for (int g = 1; g < PG; ++g) {
    const float x = sm[tid + g * DL] == top ? 1.f : fast_exp2((sm[tid + g * DL] - top) * a.sc);
    l += x * sl[tid + g * DL];
    o += x * so[tid + g * DL];
  }
  const int64_t bl = row / a.H, head = row - bl * a.H, b = bl / a.L, tok = bl - b * a.L;
  // no key at all: 0; keys whose scores are all -inf: 0 / 0, as the formula says
  const int64_t own = a.own_len[b] > a.S ? a.S : a.own_len[b];
  const float inv = a.P > 0 || own - a.L + tok + 1 > 0 ? 1.f / l : 0.f;
  Tile::store4((T*)a.out + b * a.out_seq + tok * a.out_row + head * a.out_head + 4 * dl, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
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
  if (items * 256 >= ((int64_t)1 << 32)) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prefix_attention: the launch needs 2^32 threads or more");
  PP_ALLOW_BIG_LDS((&prefix_attention_kernel<Tile>), Tile::kSmem);
  if (items > 0) PP_LAUNCH((prefix_attention_kernel<Tile>), dim3((unsigned)items), dim3(Tile::kThreads), Tile::kSmem, stream, a);
  const int rc = pp_check_launch("pp_prefix_attention");
  if (rc != PP_OK) return rc;
  constexpr int DL = Tile::kDB <= 1 ? 8 : Tile::kDB <= 2 ? 16 : Tile::kDB <= 4 ? 32 : 64;
  int pg = 0;  // a part group gets up to 4 parts before there is another
  while ((4 << pg) < a.parts && (2 << pg) * DL <= 256) ++pg;
  const int64_t per = 256 / (DL << pg), blocks = ((int64_t)a.B * a.L * a.H + per - 1) / per;
  if (blocks * 256 >= ((int64_t)1 << 32)) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prefix_attention: the join needs 2^32 threads or more");
  PP_LAUNCH((prefix_join_kernel<Tile, DL>), dim3((unsigned)blocks), dim3(256), 0, stream, a, pg);
  return pp_check_launch("pp_prefix_attention(join)");
}

template <typename T>
static int launch_prefix_d(void* stream, pp::PrefixK& a) {
  using namespace pp;
  if constexpr (sizeof(T) == 2) {
    if (a.D <= 32) return launch_prefix<AttnTile<T, 32, 4, 1, 2>>(stream, a);
    if (a.D <= 64) return launch_prefix<AttnTile<T, 64, 4, 1, 2>>(stream, a);
    if (a.D <= 96) return launch_prefix<AttnTile<T, 96, 4, 1, 1>>(stream, a);
    if (a.D <= 128) return launch_prefix<AttnTile<T, 128, 4, 1, 1>>(stream, a);
    return launch_prefix<AttnTile<T, 256, 4, 1, 1>>(stream, a);
  } else {
    if (a.D <= 32) return launch_prefix<AttnTile<T, 32, 4, 1, 1>>(stream, a);
    if (a.D <= 64) return launch_prefix<AttnTile<T, 64, 4, 1, 1>>(stream, a);
    if (a.D <= 96) return launch_prefix<AttnTile<T, 96, 4, 1, 1>>(stream, a);
    if (a.D <= 128) return launch_prefix<AttnTile<T, 128, 4, 1, 1>>(stream, a);
    return launch_prefix<AttnTile<T, 256, 4, 1, 1>>(stream, a);
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
  if (p->B < 0 || p->L < 0 || p->P < 0 || p->S < 0 || p->B > (1 << 24) || p->L > (1 << 20) || p->P > INT32_MAX || p->S > INT32_MAX)
    return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: B, L, P, S out of range");
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
  a.q = p->q; a.kp = p->kp; a.vp = p->vp; a.ko = p->ko; a.vo = p->vo; a.out = p->out; a.own_len = (const int*)p->own_len;
  a.q_seq = p->q_seq; a.q_row = p->q_row; a.q_head = p->q_head;
  a.kp_row = p->kp_row; a.kp_head = p->kp_head; a.vp_row = p->vp_row; a.vp_head = p->vp_head;
  a.ko_seq = p->ko_seq; a.ko_row = p->ko_row; a.ko_head = p->ko_head;
  a.vo_seq = p->vo_seq; a.vo_row = p->vo_row; a.vo_head = p->vo_head;
  a.out_seq = p->out_seq; a.out_row = p->out_row; a.out_head = p->out_head;
  a.P = p->P; a.S = p->S;
  a.B = (int)p->B; a.L = (int)p->L; a.H = (int)p->H; a.KH = (int)p->KH; a.G = (int)(p->H / p->KH); a.D = (int)p->D;
  a.prefix_splits = p->P > 0 ? p->prefix_splits : 0;
  a.own_splits = p->S > 0 ? p->own_splits : 0;
  a.parts = a.prefix_splits + a.own_splits;
  a.sc = p->scale * kLog2e;
  const int64_t rows = p->B * p->L * p->H;
  if (rows > ((int64_t)1 << 40) / 65536 || p->L * a.G > INT32_MAX / 2) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prefix_attention: too many rows");
  if (p->scratch_bytes < rows * (p->prefix_splits + p->own_splits) * (p->D + 4) * 4)
    return pp_fail(PP_ERR_BAD_ARG, "pp_prefix_attention: scratch smaller than B * L * H * (prefix_splits + own_splits) * (D + 4) floats");
  a.part_o = (float*)p->scratch;
  a.part_ml = a.part_o + rows * a.parts * p->D;
  if (p->dtype == PP_F32) return launch_prefix_d<float>(stream, a);
  if (p->dtype == PP_F16) return launch_prefix_d<half_t>(stream, a);
  return launch_prefix_d<bf16_t>(stream, a);
}
