// prompt_attention.hip -- attention over packed sequences of different lengths, grouped heads, causal or not.
// Contract: include/propainter_mi355.h (pp_prompt_attention); the inner loop: tile_attention.h.
//
// The n query tokens of a sequence and the G = H / KH query heads of a key / value head make n * G rows, row = token * G + head in the group:
// a work-group takes kRows of them, so short prompts fill its tiles with heads, and the keys of a group are staged once for all of its heads.
// Tiles are numbered without knowing a length on the host: sequence s starts at tile floor(cu_q[s] G / kRows) + s, which leaves each at
// least ceil(n G / kRows) numbers; a work-group finds its sequence by a 64-ary search over cu_q and returns if its number is spare.
// Later tiles of a causal sequence see more keys and are launched first.  (Ordering the tiles of all sequences by their keys was slower, 16 ragged
// prompts of up to 2048 tokens: 130 -> 139 us -- neighbouring tiles of a sequence share its keys in the L2.)  The key / value head is the fastest index of the grid, so with 8 (or a
// multiple or divisor of 8) of them a head's keys stay in the L2 of its XCDs.
// Few tiles with many keys leave most of the chip idle: with `splits` > 1 a tile's keys go to that many work-groups, whose parts a second
// launch joins (attention_parts.h).
// The search needs offsets that do not decrease.  Others hit no memory but the tensors': a tile is then taken for the wrong sequence and
// returns, or takes rows of a sequence that it found, and with splits nothing is joined.
#include "attention_parts.h"

#include <math.h>

#include <initializer_list>

namespace pp {

struct PromptK {
  const void *q, *k, *v;
  void* out;
  float* lse;
  const int *cu_q, *cu_k;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head, Tq, Tk;
  int B, H, KH, G, D, causal, ntiles, splits;
  float scale, sc;
  PartsK parts;
};

template <typename Tile>
__global__ void __launch_bounds__(Tile::kThreads, Tile::kWaves) prompt_attention_kernel(const PromptK a) {
  typedef typename Tile::type T;
  constexpr int kRows = Tile::kRows;
  const int id = (int)blockIdx.x / Tile::kHalves, d0 = (int)blockIdx.x % Tile::kHalves * Tile::kDV;  // the value channels from d0 on
  const int DV = a.D - d0 < Tile::kDV ? a.D - d0 : Tile::kDV;
  const int kh = id % a.KH, split = id / a.KH % a.splits;
  const int lane = lane_id(), wave = wave_uniform((int)threadIdx.x >> 6), q32 = lane & 31, h = lane >> 5;

  // ---- the sequence that owns this tile: the last s with first_tile(s) <= tile
  const int64_t tile = a.ntiles - 1 - id / a.KH / a.splits;
  int s = 0;
  for (int n = a.B; n > 1;) {
    const int step = (n + 63) / 64, i = s + lane * step;
    const bool below = lane * step < n && (lane == 0 || clamped(a.cu_q, i, a.Tq) * a.G / kRows + i <= tile);
    const int count = wave_count(below);
    s += (count - 1) * step;
    n = n - (count - 1) * step < step ? n - (count - 1) * step : step;
  }
  const int64_t q0 = clamped(a.cu_q, s, a.Tq), q1 = clamped(a.cu_q, s + 1, a.Tq);
  const int64_t k0 = clamped(a.cu_k, s, a.Tk), k1 = clamped(a.cu_k, s + 1, a.Tk);
  const int64_t n = q1 - q0, m = k1 > k0 ? k1 - k0 : 0, rows = n * a.G;
  const int64_t row0 = (tile - (q0 * a.G / kRows + s)) * kRows;
  if (row0 < 0 || row0 >= rows) return;

  // ---- what the rows see of the keys [first, first + most)
  int first = 0;
  int64_t most = m;
  auto limit_of = [&](int64_t row) __attribute__((always_inline)) -> int {
    const int64_t c = (a.causal ? row / a.G + 1 + m - n : m) - first;
    return (int)(c < 0 ? 0 : c > most ? most : c);
  };
  const int64_t last = rows - 1, wrow = row0 + 32 * wave, row = wrow + q32;
  if (a.splits > 1) {
    const int all = limit_of(row0 + kRows - 1 < last ? row0 + kRows - 1 : last);
    const int per = ((all + a.splits - 1) / a.splits + 63) / 64 * 64;
    first = split * per < all ? split * per : all;
    most = all - first < per ? all - first : per;
  }
  AttnLimits lim;
  lim.wave_max = wrow <= last ? limit_of(wrow + 31 < last ? wrow + 31 : last) : 0;
  lim.group_min = limit_of(row0);
  lim.nkeys = limit_of(row0 + kRows - 1 < last ? row0 + kRows - 1 : last);
  Tile t;
  AttnState<Tile> st;
  t.init(PP_DYN_SMEM);
  const bool live = row <= last;
  lim.row = live ? limit_of(row) : 0;
  t.load_q(live ? (const T*)a.q + (q0 + row / a.G) * a.q_row + (kh * a.G + row % a.G) * a.q_head : nullptr, a.D);
  const T* k = (const T*)a.k + (k0 + first) * a.k_row + kh * a.k_head;
  const T* v = (const T*)a.v + (k0 + first) * a.v_row + kh * a.v_head + d0;
  attend(t, st, k, v, a.k_row, a.v_row, lim, a.D, DV, a.sc);
  if (st.not_finite) add_not_finite(t, st, v, a.v_row, lim, DV);
  if (!live) return;
  const int64_t token = q0 + row / a.G;
  const int head = kh * a.G + (int)(row % a.G);
  if (a.splits > 1) {
    store_part(a.parts, t, st, token * a.H + head, split, lim.row > 0, d0, DV);
    return;
  }
  // no key at all: 0; keys whose scores are all -inf: 0 / 0, as the formula says
  const float inv = lim.row > 0 ? 1.f / st.l : 0.f;
  T* dst = (T*)a.out + token * a.out_row + head * a.out_head + d0;
#pragma unroll
  for (int db = 0; db < Tile::kDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * db + 8 * g + 4 * h;
      const f16v& o = st.o[db];
      if (d < DV) Tile::store4(dst + d, o[4 * g] * inv, o[4 * g + 1] * inv, o[4 * g + 2] * inv, o[4 * g + 3] * inv);
    }
  if (a.lse && h == 0 && d0 == 0) a.lse[token * a.H + head] = lim.row > 0 ? st.m * a.scale + logf(st.l) : neg_inf();
}

}  // namespace pp

template <typename Tile>
static int launch_prompt(void* stream, pp::PromptK& a) {
  using namespace pp;
  const int64_t ntiles = a.Tq * a.G / Tile::kRows + a.B;
  if (ntiles * a.KH * a.splits * Tile::kHalves * 256 >= ((int64_t)1 << 32)) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prompt_attention: the launch needs 2^32 threads or more");
  a.ntiles = (int)ntiles;
  PP_ALLOW_BIG_LDS((&prompt_attention_kernel<Tile>), Tile::kSmem);
  PP_LAUNCH((prompt_attention_kernel<Tile>), dim3((unsigned)(a.ntiles * a.KH * a.splits * Tile::kHalves)), dim3(Tile::kThreads), Tile::kSmem, stream, a);
  const int rc = pp_check_launch("pp_prompt_attention");
  return rc != PP_OK || a.splits == 1 ? rc : launch_join<Tile>(stream, a.parts, "pp_prompt_attention(join)");
}

template <typename T>
static int launch_prompt_d(void* stream, pp::PromptK& a) {
  using namespace pp;
  if constexpr (sizeof(T) == 2) {
    if (a.D <= 32) return launch_prompt<AttnTile<T, 32, 4, 2>>(stream, a);
    if (a.D <= 64) return launch_prompt<AttnTile<T, 64, 4, 2>>(stream, a);
    if (a.D <= 96) return launch_prompt<AttnTile<T, 96, 4, 1>>(stream, a);
    if (a.D <= 128) return launch_prompt<AttnTile<T, 128, 4, 1>>(stream, a);
    return launch_prompt<AttnTile<T, 256, 4, 1>>(stream, a);
  } else {
    // Rows of a sequence that fit one 64-row work-group of 2 waves: with 4 waves half of them would idle (45 rows and keys, 128 channels: 121
    // -> 99 us for 2592 sequences and heads).  Long sequences share the staging of 4 waves (2048 tokens, 16 / 4 heads: 281 us against 294).
    if (a.Tq * a.G <= 64 * (int64_t)a.B) {
      if (a.D <= 32) return launch_prompt<AttnTile<T, 32, 2, 1>>(stream, a);
      if (a.D <= 64) return launch_prompt<AttnTile<T, 64, 2, 1>>(stream, a);
      if (a.D <= 96) return launch_prompt<AttnTile<T, 96, 2, 1>>(stream, a);
      if (a.D <= 128) return launch_prompt<AttnTile<T, 128, 2, 1>>(stream, a);
    }
    if (a.D <= 32) return launch_prompt<AttnTile<T, 32, 4, 1>>(stream, a);
    if (a.D <= 64) return launch_prompt<AttnTile<T, 64, 4, 1>>(stream, a);
    if (a.D <= 96) return launch_prompt<AttnTile<T, 96, 4, 1>>(stream, a);
    if (a.D <= 128) return launch_prompt<AttnTile<T, 128, 4, 1>>(stream, a);
    return launch_prompt<AttnTile<T, 256, 4, 1>>(stream, a);
  }
}

extern "C" int32_t pp_prompt_attention(void* stream, const pp_prompt_attention_params* p) {
  using namespace pp;
  if (!p || !p->q || !p->k || !p->v || !p->out || !p->cu_q || !p->cu_k) return pp_fail(PP_ERR_BAD_ARG, "pp_prompt_attention: null argument");
  if (p->dtype != PP_F32 && p->dtype != PP_F16 && p->dtype != PP_BF16) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prompt_attention: dtype");
  if (p->KH < 1 || p->H < 1 || p->H % p->KH || p->H > (1 << 20))
    return pp_fail(PP_ERR_BAD_ARG, "pp_prompt_attention: H must be a multiple of KH");
  const int e = p->dtype == PP_F32 ? 4 : 8;  // elements of 16 bytes
  if (p->D < 1 || p->D > 256 || p->D % e) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prompt_attention: D must be a multiple of 8 (fp32: 4) up to 256");
  if (p->B < 0 || p->Tq < 0 || p->Tk < 0 || p->B > INT32_MAX / 2 || p->Tq > INT32_MAX)
    return pp_fail(PP_ERR_BAD_ARG, "pp_prompt_attention: B, Tq, Tk must be in [0, 2^31)");
  if (p->Tk > kMostKeys) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prompt_attention: Tk above 2^31 - 1024");
  if (p->Tq * p->H > (int64_t)1 << 40 || p->B * p->KH > (int64_t)1 << 32)  // (what is computed from them stays inside 64 bits)
    return pp_fail(PP_ERR_UNSUPPORTED, "pp_prompt_attention: Tq * H or B * KH too large");
  if (!(p->scale > 0.f) || !(p->scale * kLog2e < INFINITY)) return pp_fail(PP_ERR_BAD_ARG, "pp_prompt_attention: scale must be positive and finite");
  const int64_t strides[8] = {p->q_row, p->q_head, p->k_row, p->k_head, p->v_row, p->v_head, p->out_row, p->out_head};
  for (int i = 0; i < 8; ++i)
    if (strides[i] < 0 || strides[i] % e) return pp_fail(PP_ERR_BAD_ARG, "pp_prompt_attention: strides must be >= 0 and keep rows 16-byte aligned");
  // (a block of keys is addressed with 32-bit byte offsets)
  for (const int64_t row : {p->k_row, p->v_row})
    if (row >= 1 << 24) return pp_fail(PP_ERR_UNSUPPORTED, "pp_prompt_attention: a key or value row stride must be below 2^24 elements");
  if (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->out) % 16)
    return pp_fail(PP_ERR_BAD_ARG, "pp_prompt_attention: tensors must be 16-byte aligned");
  if (p->out == p->q && p->dtype == PP_F32 && p->D > 128)  // two work-groups read a row's query, either may be done first
    return pp_fail(PP_ERR_UNSUPPORTED, "pp_prompt_attention: out cannot be q for fp32 heads of more than 128 channels");
  const int splits = p->splits ? p->splits : 1;
  if (splits < 1 || splits > 64) return pp_fail(PP_ERR_BAD_ARG, "pp_prompt_attention: splits must be in [0, 64]");
  if (splits > 1 && (!p->scratch || (uintptr_t)p->scratch % 16 || p->scratch_bytes / (splits * (p->D + 4) * 4) < p->Tq * p->H))
    return pp_fail(PP_ERR_BAD_ARG, "pp_prompt_attention: splits need a 16-byte aligned scratch of Tq * H * splits * (D + 4) floats");
  if (p->B == 0 || p->Tq == 0) return PP_OK;  // no row to write
  PromptK a;
  a.q = p->q; a.k = p->k; a.v = p->v; a.out = p->out; a.lse = (float*)p->lse;
  a.cu_q = (const int*)p->cu_q; a.cu_k = (const int*)p->cu_k;
  a.q_row = p->q_row; a.q_head = p->q_head; a.k_row = p->k_row; a.k_head = p->k_head;
  a.v_row = p->v_row; a.v_head = p->v_head; a.out_row = p->out_row; a.out_head = p->out_head;
  a.Tq = p->Tq; a.Tk = p->Tk;
  a.B = (int)p->B; a.H = (int)p->H; a.KH = (int)p->KH; a.G = (int)(p->H / p->KH); a.D = (int)p->D; a.causal = p->causal != 0;
  a.scale = p->scale; a.sc = p->scale * kLog2e;
  a.splits = p->B <= kSharedSequences ? splits : 1;
  if (a.splits > 1) {
    PartsK& pt = a.parts;
    pt.rows = p->Tq * p->H; pt.L = (int)p->Tq; pt.H = a.H; pt.D = a.D; pt.parts = splits;
    pt.o = (float*)p->scratch;
    pt.ml = pt.o + pt.rows * splits * p->D;
    pt.out = p->out; pt.out_seq = 0; pt.out_row = p->out_row; pt.out_head = p->out_head;
    pt.lse = a.lse; pt.cu_q = a.cu_q; pt.ncu = a.B; pt.sc = a.sc; pt.scale = a.scale;
  }
  if (p->dtype == PP_F32) return launch_prompt_d<float>(stream, a);
  if (p->dtype == PP_F16) return launch_prompt_d<half_t>(stream, a);
  return launch_prompt_d<bf16_t>(stream, a);
}
