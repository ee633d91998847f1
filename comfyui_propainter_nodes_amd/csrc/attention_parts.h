// attention_parts.h -- attention whose keys are dealt to several work-groups: what each leaves behind, and how it is joined.
//
// A part of a row is (m, l, o): the maximum that it refers to, the sum of its weights 2^((s - m) sc), the weighted sum of its values, all fp32; a
// part without a visible key has l = -1.  The row is sum_p w_p o_p / sum_p w_p l_p with w_p = 2^((m_p - max m) sc), in part order.
#pragma once
#include "tile_attention.h"
#include "pp_host.h"

namespace pp {

// Sequences up to which keys are shared: each wave of the joining launch looks over their offsets.
constexpr int kSharedSequences = 4096;

// an offset, inside [0, most]
__device__ __forceinline__ int64_t clamped(const int* cu, int i, int64_t most) {
  const int64_t v = cu[i];
  return v < 0 ? 0 : v > most ? most : v;
}

struct PartsK {
  float* o;   // [row][part][D]
  float* ml;  // [row][part][2]
  void* out;  // [b][L][H][D] by strides; row = (b L + token) H + head
  float* lse; // [row] or null
  const int* cu_q;  // or null: rows of the tokens before cu_q[0] and from cu_q[ncu] on are left as they were, all rows if an offset decreases
  int64_t rows, out_seq, out_row, out_head;
  int L, H, D, parts, ncu;
  float sc, scale;
};

template <typename Tile>
__device__ __forceinline__ void store_part(const PartsK& a, const Tile& t, const AttnState<Tile>& st, int64_t row, int part, bool any, int d0,
                                           int DV) {  // channels d0 .. d0 + DV - 1
  const int64_t at = row * a.parts + part;
  float* dst = a.o + at * a.D + d0;
#pragma unroll
  for (int db = 0; db < Tile::kDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * db + 8 * g + 4 * t.h;
      const f16v& o = st.o[db];
      if (d < DV) *reinterpret_cast<f4*>(dst + d) = f4{o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]};
    }
  if (t.h == 0 && d0 == 0) {
    a.ml[2 * at] = st.m;
    a.ml[2 * at + 1] = any ? st.l : -1.f;
  }
}

// A row's D values are DL threads of 4, and PG groups of such threads take every PG-th part each, four parts' loads in flight; then the groups'
// results are joined in LDS.  (One thread per 4 values walking all parts: 31 us for 32 tokens behind 8192 keys in all, this 26.)
template <typename Tile, int DL>
__global__ void __launch_bounds__(256) attention_join_kernel(const PartsK a, int pg_log2) {
  typedef typename Tile::type T;
  __shared__ f4 so[256];
  __shared__ float sm[256], sl[256], sany[256];
  const int tid = (int)threadIdx.x, dl = tid % DL, PG = 1 << pg_log2, pg = tid / DL % PG, slot = tid / (DL * PG);
  const int64_t row = (int64_t)blockIdx.x * (256 / (DL * PG)) + slot;
  bool live = row < a.rows && 4 * dl < a.D;
  if (live && a.cu_q) {
    const int64_t token = row / a.H;
    live = token >= a.cu_q[0] && token < a.cu_q[a.ncu];
  }
  float m = neg_inf(), l = 0.f, any = 0.f;
  f4 o = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    const float* ml = a.ml + row * a.parts * 2;
    const float* po = a.o + row * a.parts * a.D + 4 * dl;
    for (int p0 = pg; p0 < a.parts; p0 += 4 * PG) {
      float pm[4], pl[4];
      f4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int p = p0 + u * PG;
        const bool in = p < a.parts;
        pm[u] = in ? ml[2 * p] : neg_inf();
        pl[u] = in ? ml[2 * p + 1] : -1.f;
        v[u] = in ? *reinterpret_cast<const f4*>(po + (int64_t)p * a.D) : f4{0.f, 0.f, 0.f, 0.f};
      }
      const float top = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), m);
      const float w = m == top ? 1.f : fast_exp2((m - top) * a.sc);
      m = top;
      l *= w;
      o *= w;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (pl[u] == -1.f) continue;  // no key: nothing to add (and its maximum is -inf)
        any = 1.f;
        const float x = pm[u] == top ? 1.f : fast_exp2((pm[u] - top) * a.sc);
        l += x * pl[u];
        o += x * v[u];
      }
    }
  }
  so[tid] = o;
  sm[tid] = m;
  sl[tid] = l;
  sany[tid] = any;
  // Every row between the offsets has its parts stored only if they do not decrease (the search for a tile's sequence needs the order); else
  // scratch that nobody wrote could be among them.
  bool down = false;
  if (a.cu_q)
    for (int i = lane_id(); i < a.ncu; i += 64) down |= clamped(a.cu_q, i, a.L) > clamped(a.cu_q, i + 1, a.L);
  down = wave_any(down);
  __syncthreads();
  if (!live || pg != 0 || down) return;
  float top = m;
  for (int g = 1; g < PG; ++g) top = fmaxf(top, sm[tid + g * DL]);
  const float w = m == top ? 1.f : fast_exp2((m - top) * a.sc);
  l *= w;
  o *= w;
  for (int g = 1; g < PG; ++g) {
    const float x = sm[tid + g * DL] == top ? 1.f : fast_exp2((sm[tid + g * DL] - top) * a.sc);
    l += x * sl[tid + g * DL];
    o += x * so[tid + g * DL];
    any += sany[tid + g * DL];
  }
  const int64_t bl = row / a.H, head = row - bl * a.H, b = bl / a.L, tok = bl - b * a.L;
  // no key at all: 0; keys whose scores are all -inf: 0 / 0, as the formula says
  const float inv = any > 0.f ? 1.f / l : 0.f;
  Tile::store4((T*)a.out + b * a.out_seq + tok * a.out_row + head * a.out_head + 4 * dl, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (a.lse && dl == 0) a.lse[row] = any > 0.f ? top * a.scale + logf(l) : neg_inf();
}

template <typename Tile>
int launch_join(void* stream, const PartsK& a, const char* who) {
  constexpr int DP = Tile::kDB * 32 * Tile::kHalves, DL = DP <= 32 ? 8 : DP <= 64 ? 16 : DP <= 128 ? 32 : 64;
  int pg = 0;  // a part group gets up to 4 parts before there is another
  while ((4 << pg) < a.parts && (2 << pg) * DL <= 256) ++pg;
  const int64_t per = 256 / (DL << pg), blocks = (a.rows + per - 1) / per;
  if (blocks * 256 >= ((int64_t)1 << 32)) return pp_fail(PP_ERR_UNSUPPORTED, "attention: the join of the parts needs 2^32 threads or more");
  PP_LAUNCH((attention_join_kernel<Tile, DL>), dim3((unsigned)blocks), dim3(256), 0, stream, a, pg);
  return pp_check_launch(who);
}

}  // namespace pp
