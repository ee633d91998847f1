// tile_attention.h -- one work-group's attention over a run of keys: the part that pp_prompt_attention and pp_prefix_attention share.
//
// A work-group of 4 waves takes 128 query rows, 32 per wave, of ONE key / value head (the query heads of a group are rows of the
// same tile, so their keys are staged once).  Keys are walked in tiles through LDS:
//   S^T = K . Q^T     32x32 MFMA; lane l holds the scores of query l & 31 against keys (r & 3) + 8 (r >> 2) + 4 (l >> 5), r = 0..15
//   online softmax    lane-local, one exchange between lanes l and l ^ 32; fp32 maxima, sums and accumulators
//   O^T += V^T . P^T  the lane's own probabilities are the B operand, V^T fragments come out of LDS transposed (f16 / bf16:
//                     ds_read_b64_tr_b16; f32: one value per lane)
// The running maximum that the probabilities refer to moves only when a score of the wave passes it by more than kDefer in the
// exponent of 2, so most tiles rescale nothing.  A probability is then at most 2^kDefer, far inside f16 and exact in relative terms.
//
// Rows that see different numbers of keys: `limit` is the row's own count, scores at or past it become -inf before the softmax.  Their
// probability is 0, but 0 x V is NaN for a V that is not finite.  Keys past the last one that any row of the work-group sees are staged as
// zeros; a sub-tile in which only some rows see a key whose V is not finite goes through pv_guarded(), which multiplies
// the finite part and adds infinities and NaN to the rows that see them and to no others.
#pragma once
#include "attn_device.h"
#include "bf16_device.h"

namespace pp {

constexpr float kDefer = 8.f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

#ifdef PP_EMU
inline float neg_inf() { return -INFINITY; }
#else
__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }
#endif

// 16-bit operand types travel as h8 bit patterns
template <typename T>
struct Op;
template <>
struct Op<half_t> {
  static constexpr unsigned kExp = 0x7c007c00u, kCarry = 0x04000400u, kOne = 0x3c00u;
  static __device__ __forceinline__ f16v mfma(h8 a, h8 b, f16v c) { return mfma_32x32x16_f16(a, b, c); }
  static __device__ __forceinline__ unsigned pack(float a, float b) { return __builtin_bit_cast(unsigned, h2{(half_t)a, (half_t)b}); }
};
template <>
struct Op<bf16_t> {
  static constexpr unsigned kExp = 0x7f807f80u, kCarry = 0x00800080u, kOne = 0x3f80u;
#ifndef PP_EMU
  typedef __bf16 hw8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f16v mfma(h8 a, h8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(hw8, a), __builtin_bit_cast(hw8, b), c, 0, 0, 0);
  }
#else
  static f16v mfma(h8 a, h8 b, f16v c) {
    struct Slot {
      h8 a, b;
      unsigned char pad[32];
    };
    Slot* s = reinterpret_cast<Slot*>(pp_emu::wave_scratch());
    const int l = pp_emu::cur->lane;
    s[l].a = a;
    s[l].b = b;
    pp_emu::wave_sync();
    auto f = [](half_t v) { return __builtin_bit_cast(float, (unsigned)__builtin_bit_cast(unsigned short, v) << 16); };
    f16v d = c;
    for (int r = 0; r < 16; ++r) {
      const int row = (r & 3) + 8 * (r >> 2) + 4 * (l >> 5);
      float acc = 0.f;
      for (int g = 0; g < 2; ++g)
        for (int j = 0; j < 8; ++j) acc += f(s[row + 32 * g].a[j]) * f(s[(l & 31) + 32 * g].b[j]);
      d[r] += acc;
    }
    pp_emu::wave_sync();
    return d;
  }
#endif
  static __device__ __forceinline__ unsigned pack(float a, float b) { return pack_bf16(a, b); }
};

// key index of score register r inside its 32-key sub-tile
__device__ __forceinline__ int score_key(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

// ----------------------------------------------------------------------------------------
// 16-bit storage.  K and V tiles of kBN keys lie in LDS row by row, kPitch bytes a row, their 16-byte pieces XOR-swizzled so that the
// K reads (16 bytes of 32 rows at once) and the transposing V reads (64 bytes of 4 rows at once) touch every bank once.
// ----------------------------------------------------------------------------------------
template <typename T, int DP>
struct AttnTile {
  typedef T type;
  static constexpr int kBN = DP > 128 ? 32 : 64;
  static constexpr int kPitch = DP <= 32 ? 64 : DP <= 64 ? 128 : DP <= 128 ? 256 : 512;
  static constexpr int kPieces = DP / 8, kStage = kBN * kPieces / 256, kDB = DP / 32, kQF = DP / 16;
  static constexpr int kSmem = 2 * kBN * kPitch;
  static_assert(kBN * kPieces % 256 == 0, "a tile is dealt to 256 threads");

  h8 q[kQF];
  u4 ks[kStage], vs[kStage];  // the next tile on its way
  unsigned char* smem;
  int q32, h;

  static __device__ __forceinline__ int k_slot(int row, int piece) {
    constexpr int m = kPitch >= 256 ? 15 : kPitch / 16 - 1, sh = kPitch >= 256 ? 0 : kPitch == 128 ? 1 : 2;
    return row * kPitch + ((piece ^ ((row >> sh) & m)) << 4);
  }
  static __device__ __forceinline__ int v_slot(int row, int piece) {
    constexpr int m = kPitch >= 256 ? 3 : kPitch == 128 ? 1 : 0, sh = kPitch >= 256 ? 0 : 1;
    return kBN * kPitch + row * kPitch + ((piece ^ (((row >> sh) & m) << 2)) << 4);
  }
  __device__ __forceinline__ void init(unsigned char* lds) {
    smem = lds;
    q32 = (int)threadIdx.x & 31;
    h = ((int)threadIdx.x >> 5) & 1;
  }
  // row: this lane's query, or null
  __device__ __forceinline__ void load_q(const T* row, int D) {
#pragma unroll
    for (int c = 0; c < kQF; ++c) {
      const int d = 16 * c + 8 * h;
      u4 v = {0u, 0u, 0u, 0u};
      if (row && d < D) v = *reinterpret_cast<const u4*>(row + d);
      q[c] = __builtin_bit_cast(h8, v);
    }
  }
  __device__ __forceinline__ void load_tile(const T* k, const T* v, int64_t k_row, int64_t v_row, int64_t kt, int64_t nkeys, int D) {
#pragma unroll
    for (int i = 0; i < kStage; ++i) {
      const int at = (int)threadIdx.x + 256 * i, row = at / kPieces, piece = at - row * kPieces;
      ks[i] = vs[i] = u4{0u, 0u, 0u, 0u};
      if (kt + row < nkeys && 8 * piece < D) {
        ks[i] = *reinterpret_cast<const u4*>(k + (kt + row) * k_row + 8 * piece);
        vs[i] = *reinterpret_cast<const u4*>(v + (kt + row) * v_row + 8 * piece);
      }
    }
  }
  __device__ __forceinline__ void store_tile() {
#pragma unroll
    for (int i = 0; i < kStage; ++i) {
      const int at = (int)threadIdx.x + 256 * i, row = at / kPieces, piece = at - row * kPieces;
      *reinterpret_cast<u4*>(smem + k_slot(row, piece)) = ks[i];
      *reinterpret_cast<u4*>(smem + v_slot(row, piece)) = vs[i];
    }
  }
  __device__ __forceinline__ f16v qk(int sub) const {
    f16v s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int c = 0; c < kQF; ++c) {
      const h8 a = *reinterpret_cast<const h8*>(smem + k_slot(32 * sub + q32, 2 * c + h));
      s = Op<T>::mfma(a, q[c], s);
    }
    return s;
  }
  static __device__ __forceinline__ void pack_p(const float* p, h8* pf) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      u4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = Op<T>::pack(p[8 * m + 2 * j], p[8 * m + 2 * j + 1]);
      pf[m] = __builtin_bit_cast(h8, w);
    }
  }
  // V^T fragment of head-dim block db, 16-key group m of sub-tile `sub`: rows d = 32 db + (lane & 31), keys in score order
  __device__ __forceinline__ h8 v_frag(int sub, int db, int m) const {
    const int lane = lane_id(), i = lane & 15, ir = i >> 2, g16 = lane >> 4;
    const int row = 32 * sub + 16 * m + 4 * h + ir, piece = 4 * db + 2 * (g16 & 1) + ((i & 3) >> 1);
    const h4 lo = lds_read_tr16(reinterpret_cast<const half_t*>(smem + v_slot(row, piece) + (i & 1) * 8));
    const h4 hi = lds_read_tr16(reinterpret_cast<const half_t*>(smem + v_slot(row + 8, piece) + (i & 1) * 8));
    return h8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
  __device__ __forceinline__ void pv(int sub, const float* p, f16v* o) const {
    h8 pf[2];
    pack_p(p, pf);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[db] = Op<T>::mfma(v_frag(sub, db, m), pf[m], o[db]);
  }
  // does the sub-tile's V hold a value that is not finite?  (exponent all ones: adding one to it carries out of the field)
  __device__ __forceinline__ bool v_not_finite(int sub) const {
    unsigned any = 0;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        const u4 w = __builtin_bit_cast(u4, v_frag(sub, db, m));
#pragma unroll
        for (int j = 0; j < 4; ++j) any |= ((w[j] & Op<T>::kExp) + Op<T>::kCarry) & 0x80008000u;
      }
    return wave_any(any != 0);
  }
  __device__ __forceinline__ void pv_guarded(int sub, const float* p, const bool* seen, f16v* o) const {
    h8 pf[2], sf[2];
    float sv[16];
    pack_p(p, pf);
#pragma unroll
    for (int r = 0; r < 16; ++r) sv[r] = seen[r] ? 1.f : 0.f;
    pack_p(sv, sf);
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      f16v pos, neg, nan;
#pragma unroll
      for (int r = 0; r < 16; ++r) pos[r] = neg[r] = nan[r] = 0.f;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        u4 w = __builtin_bit_cast(u4, v_frag(sub, db, m)), wp = {0, 0, 0, 0}, wn = wp, wx = wp;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int s = 0; s < 32; s += 16) {
            const unsigned x = (w[j] >> s) & 0xffffu, e = Op<T>::kExp & 0xffffu;
            if ((x & e) != e) continue;
            if (x & 0x7fffu & ~e) wx[j] |= Op<T>::kOne << s;
            else if (x & 0x8000u) wn[j] |= Op<T>::kOne << s;
            else wp[j] |= Op<T>::kOne << s;
            w[j] &= ~(0xffffu << s);
          }
        o[db] = Op<T>::mfma(__builtin_bit_cast(h8, w), pf[m], o[db]);
        pos = Op<T>::mfma(__builtin_bit_cast(h8, wp), sf[m], pos);
        neg = Op<T>::mfma(__builtin_bit_cast(h8, wn), sf[m], neg);
        nan = Op<T>::mfma(__builtin_bit_cast(h8, wx), sf[m], nan);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (pos[r] > 0.f) o[db][r] -= neg_inf();
        if (neg[r] > 0.f) o[db][r] += neg_inf();
        if (nan[r] > 0.f) o[db][r] = __builtin_nanf("");
      }
    }
  }
  // 4 consecutive head-dim values of a row
  static __device__ __forceinline__ void store4(T* dst, float a, float b, float c, float d) {
    *reinterpret_cast<u2*>(dst) = u2{Op<T>::pack(a, b), Op<T>::pack(c, d)};
  }
};

// ----------------------------------------------------------------------------------------
// f32 storage: both products on v_mfma_f32_32x32x2_f32 (64 cycles for 2 keys or channels: the matrix pipe is the bound by far, LDS and
// the vector ALU have slack).  Rows have a pitch of DP + 4 floats.
// ----------------------------------------------------------------------------------------
template <int DP>
struct AttnTile<float, DP> {
  typedef float type;
  static constexpr int kBN = 32;
  static constexpr int kP = DP + 4;
  static constexpr int kPieces = DP / 4, kStage = kBN * kPieces / 256, kDB = DP / 32, kQF = DP / 8;
  static constexpr int kSmem = 2 * kBN * kP * 4;

  f4 q[kQF];
  f4 ks[kStage], vs[kStage];
  float* smem;
  int q32, h;

  __device__ __forceinline__ void init(unsigned char* lds) {
    smem = reinterpret_cast<float*>(lds);
    q32 = (int)threadIdx.x & 31;
    h = ((int)threadIdx.x >> 5) & 1;
  }
  __device__ __forceinline__ void load_q(const float* row, int D) {
#pragma unroll
    for (int c = 0; c < kQF; ++c) {
      const int d = 8 * c + 4 * h;
      q[c] = f4{0.f, 0.f, 0.f, 0.f};
      if (row && d < D) q[c] = *reinterpret_cast<const f4*>(row + d);
    }
  }
  __device__ __forceinline__ void load_tile(const float* k, const float* v, int64_t k_row, int64_t v_row, int64_t kt, int64_t nkeys, int D) {
#pragma unroll
    for (int i = 0; i < kStage; ++i) {
      const int at = (int)threadIdx.x + 256 * i, row = at / kPieces, piece = at - row * kPieces;
      ks[i] = vs[i] = f4{0.f, 0.f, 0.f, 0.f};
      if (kt + row < nkeys && 4 * piece < D) {
        ks[i] = *reinterpret_cast<const f4*>(k + (kt + row) * k_row + 4 * piece);
        vs[i] = *reinterpret_cast<const f4*>(v + (kt + row) * v_row + 4 * piece);
      }
    }
  }
  __device__ __forceinline__ void store_tile() {
#pragma unroll
    for (int i = 0; i < kStage; ++i) {
      const int at = (int)threadIdx.x + 256 * i, row = at / kPieces, piece = at - row * kPieces;
      *reinterpret_cast<f4*>(smem + row * kP + 4 * piece) = ks[i];
      *reinterpret_cast<f4*>(smem + kBN * kP + row * kP + 4 * piece) = vs[i];
    }
  }
  // channels are taken in the order (8c + 4h + j): any order serves a dot product as long as both operands share it
  __device__ __forceinline__ f16v qk(int) const {
    f16v s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int c = 0; c < kQF; ++c) {
      const f4 a = *reinterpret_cast<const f4*>(smem + q32 * kP + 8 * c + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = mfma_32x32x2_f32(a[j], q[c][j], s);
    }
    return s;
  }
  __device__ __forceinline__ float v_at(int r, int db) const { return smem[kBN * kP + score_key(r, h) * kP + 32 * db + q32]; }
  __device__ __forceinline__ void pv(int, const float* p, f16v* o) const {
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[db] = mfma_32x32x2_f32(v_at(r, db), p[r], o[db]);
  }
  __device__ __forceinline__ bool v_not_finite(int) const {
    bool any = false;
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int db = 0; db < kDB; ++db) any |= (__builtin_bit_cast(unsigned, v_at(r, db)) & 0x7f800000u) == 0x7f800000u;
    return wave_any(any);
  }
  __device__ __forceinline__ void pv_guarded(int, const float* p, const bool* seen, f16v* o) const {
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      f16v pos, neg, nan;
#pragma unroll
      for (int r = 0; r < 16; ++r) pos[r] = neg[r] = nan[r] = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float v = v_at(r, db), w = seen[r] ? 1.f : 0.f;
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const bool bad = (u & 0x7f800000u) == 0x7f800000u, isnan = bad && (u & 0x7fffffu);
        o[db] = mfma_32x32x2_f32(bad ? 0.f : v, p[r], o[db]);
        pos = mfma_32x32x2_f32(bad && !isnan && !(u >> 31) ? 1.f : 0.f, w, pos);
        neg = mfma_32x32x2_f32(bad && !isnan && (u >> 31) ? 1.f : 0.f, w, neg);
        nan = mfma_32x32x2_f32(isnan ? 1.f : 0.f, w, nan);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (pos[r] > 0.f) o[db][r] -= neg_inf();
        if (neg[r] > 0.f) o[db][r] += neg_inf();
        if (nan[r] > 0.f) o[db][r] = __builtin_nanf("");
      }
    }
  }
  static __device__ __forceinline__ void store4(float* dst, float a, float b, float c, float d) {
    *reinterpret_cast<f4*>(dst) = f4{a, b, c, d};
  }
};

// ----------------------------------------------------------------------------------------
// the walk over the keys
// ----------------------------------------------------------------------------------------
template <typename Tile>
struct AttnState {
  f16v o[Tile::kDB];  // O^T: row d = 32 db + score_key(r, h), column = the lane's query
  float m, l;         // running maximum (of the raw scores; -inf before the first visible key) and this lane's part of the sum
};

// Keys [0, nkeys) at k, v.  limit: keys that this lane's row sees (<= nkeys).  wave_min / wave_max: the smallest and largest limit among
// the wave's live rows (wave-uniform; wave_max = 0: no live row, the wave only helps staging).  sc = scale * log2(e) > 0.
template <typename Tile>
__device__ __forceinline__ void attend(Tile& t, AttnState<Tile>& st, const typename Tile::type* k, const typename Tile::type* v,
                                       int64_t k_row, int64_t v_row, int64_t nkeys, int64_t limit, int64_t wave_min, int64_t wave_max,
                                       int D, float sc) {
#pragma unroll
  for (int db = 0; db < Tile::kDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.o[db][r] = 0.f;
  st.m = neg_inf();
  st.l = 0.f;
  if (nkeys <= 0) return;
  t.load_tile(k, v, k_row, v_row, 0, nkeys, D);
  for (int64_t kt = 0; kt < nkeys; kt += Tile::kBN) {
    t.store_tile();
    __syncthreads();
    if (kt + Tile::kBN < nkeys) t.load_tile(k, v, k_row, v_row, kt + Tile::kBN, nkeys, D);
#pragma unroll
    for (int sub = 0; sub < Tile::kBN / 32; ++sub) {
      const int64_t k0 = kt + 32 * sub;
      if (k0 >= wave_max) break;
      f16v s = t.qk(sub);
      const bool masked = k0 + 32 > wave_min;
      const int left = (int)(limit - k0 < 32 ? limit - k0 : 32);  // keys of this sub-tile that the row sees (may be negative)
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = score_key(r, t.h) < left ? s[r] : neg_inf();
      }
      float mt = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[r]);
      mt = fmaxf(st.m, pair32_max(mt));
      // (-inf) - (-inf) is NaN and compares false: a row that has seen nothing yet moves nothing
      if (wave_any((mt - st.m) * sc > kDefer)) {
        const float alpha = mt == st.m ? 1.f : fast_exp2((st.m - mt) * sc);
        st.l *= alpha;
#pragma unroll
        for (int db = 0; db < Tile::kDB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) st.o[db][r] *= alpha;
        st.m = mt;
      }
      const float nm = st.m == neg_inf() ? 0.f : -st.m * sc;
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = fast_exp2(__builtin_fmaf(s[r], sc, nm));
        st.l += p[r];
      }
      bool guarded = false;
      if (masked && wave_min < (nkeys < k0 + 32 ? nkeys : k0 + 32)) guarded = t.v_not_finite(sub);
      if (guarded) {
        bool seen[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) seen[r] = score_key(r, t.h) < left;
        t.pv_guarded(sub, p, seen, st.o);
      } else {
        t.pv(sub, p, st.o);
      }
    }
    __syncthreads();
  }
  st.l = pair32_sum(st.l);
}

}  // namespace pp
