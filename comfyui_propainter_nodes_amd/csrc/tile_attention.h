// tile_attention.h -- one work-group's attention over a run of keys: the part that pp_prompt_attention and pp_prefix_attention share.
//
// A work-group of NW waves takes 32 NW query rows, 32 per wave, of ONE key / value head (the query heads of a group are rows of the
// same tile, so their keys are staged once).  Keys are walked in steps of 32 NS through LDS:
//   S^T = K . Q^T     32x32 MFMA; lane l holds the scores of query l & 31 against keys (r & 3) + 8 (r >> 2) + 4 (l >> 5), r = 0..15
//   online softmax    lane-local, one exchange between lanes l and l ^ 32; fp32 maxima, sums and accumulators
//   O^T += V^T . P^T  the lane's own probabilities are the B operand, V^T fragments come out of LDS transposed (f16 / bf16:
//                     ds_read_b64_tr_b16; f32: one value per lane)
// A 16-bit product takes 16-bit operands: a probability is rounded to the storage type once, half a step of its own size, before it meets V (its f32
// value goes into the sum).  The error against 64 bits is 1.1 to 1.4 times that of f32 probabilities with the result rounded once (f16 2.5e-4 against
// 1.9e-4 on the long prompt, bf16 2.3e-3 against 1.7e-3 behind a prefix); f32 operands would run at a seventh of the rate.
// Step i works on three key blocks at once -- the softmax of block i, the second product of block i - 1 and the first of block i + 1 -- so
// every MFMA of a step is independent of its exponentials.  K and V pass through two LDS slots each; their loads are issued a step
// before they are stored, one barrier a step.
// The maximum m that the probabilities 2^(s sc - m sc) refer to is a true one, but not the newest: a block is taken against the m it
// finds, and only if a lane's sum over the block comes out above kMost (any probability would be then, or NaN) is m moved, what was summed
// up rescaled and the block taken again.  Otherwise a maximum is only computed where a lane has no m to go by: rows that see no key yet (rows behind
// the last one of a tile among them, in every block that masks them) and the far scores below.
// A probability is at most kMost, inside f16 and as exact as any other relative to its own size, and the sum of a row is 1 or more, the weight
// of the key that m came from.  That rests on 2^((s - m) sc), where the difference is exact near m: m sc rounded to f32 is half a unit in
// its last place off, which nothing cancels -- 2^-13 of a power of two below kFar, less than a 16-bit probability's own rounding, and whole powers
// of two from 2^24 on.  So 16-bit blocks are weighed by one fma with the rounded -m sc while |m sc| < kFar, and every block by the difference
// beyond it; f32 storage and the blocks that move m always take the difference.
//
// Bound by the matrix pipes: one causal prompt of 8192 tokens, 32 query heads over 8 key heads of 128, f16: 533-590 us by card, 0.93-1.03 PF/s, MFMA busy
// 50-52 % of the cycles at the 1.8-1.9 GHz that the card holds under it, LDS 38 %, no bank conflict; 800-830 TF/s at 64 channels, 920 at 256; f32 129,
// 135 and 66 TF/s at 64, 128 and 256 channels (a library product: 152).  On a card where it takes 570 us it took 565 before differences were kept exact
// for far scores, 640 with a maximum per block and per-lane addresses, 672 with the MFMAs left to the compiler's order besides.  64 rows a wave
// would halve the LDS reads, but left one wave per SIMD and cost register moves.
//
// Rows that see different numbers of keys: `limit` is the row's own count, scores at or past it become -inf before the softmax.  Their
// probability is 0, but 0 x V is NaN for a V that is not finite.  Keys past the last one that any row of the work-group sees are staged as
// zeros, or as they are where rows overlap; in blocks that only some rows see, and in such a last block, V values that are not finite are staged
// as zeros too, and if there were any, add_not_finite() goes over those blocks once more at the end and adds them to the rows that do see them.
#pragma once
#include "attn_device.h"
#include "bf16_device.h"

#include <type_traits>

namespace pp {

constexpr float kMost = 4096.f;
constexpr float kFar = 4096.f;  // |m sc| from which a block is not weighed by 2^(s sc - m sc)
// Keys of one walk: its counters are 32 bits wide and run up to three blocks past the last key.
constexpr int64_t kMostKeys = ((int64_t)1 << 31) - 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

#ifdef PP_EMU
inline float neg_inf() { return -INFINITY; }
#else
__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }
#endif

#ifdef PP_EMU
inline void keep_branch() {}
template <int N>
inline void wave_priority() {}
inline void pin(float&) {}
inline void pin(unsigned&) {}
#else
__device__ __forceinline__ void pin(float& v) { asm volatile("" : "+v"(v)); }  // the value is computed by here
__device__ __forceinline__ void pin(unsigned& v) { asm volatile("" : "+v"(v)); }
template <int N>
__device__ __forceinline__ void wave_priority() {
  __builtin_amdgcn_s_setprio(N);
}
__device__ __forceinline__ void keep_branch() { asm volatile(""); }  // what follows is not computed ahead of its condition
#endif
// A block of rows that is read 16 bytes at a time; what starts behind its last byte reads as zeros.  The base is wave-uniform, a lane's
// byte offset the same in every block: no address arithmetic on the vector ALU.
#ifdef PP_EMU
struct Rows16 {
  const char* base;
  unsigned bytes;
};
inline Rows16 rows16(const void* base, unsigned bytes) { return Rows16{static_cast<const char*>(base), bytes}; }
inline u4 load_row16(const Rows16& r, unsigned off) {
  return (uint64_t)off + 16 <= r.bytes ? *reinterpret_cast<const u4*>(r.base + off) : u4{0u, 0u, 0u, 0u};
}
#else
typedef __amdgpu_buffer_rsrc_t Rows16;
__device__ __forceinline__ Rows16 rows16(const void* base, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00027000);
}
__device__ __forceinline__ u4 load_row16(Rows16 r, unsigned off) {
  return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}
#endif

// 16-bit operand types travel as h8 bit patterns
template <typename T>
struct Op;
template <>
struct Op<half_t> {
  static constexpr unsigned kExp = 0x7c007c00u, kCarry = 0x04000400u;
  static __device__ __forceinline__ f16v mfma(h8 a, h8 b, f16v c) { return mfma_32x32x16_f16(a, b, c); }
  static __device__ __forceinline__ unsigned pack(float a, float b) { return __builtin_bit_cast(unsigned, h2{(half_t)a, (half_t)b}); }
};
template <>
struct Op<bf16_t> {
  static constexpr unsigned kExp = 0x7f807f80u, kCarry = 0x00800080u;
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
// 16-bit storage.  The two K and two V slots of 32 NS keys lie in LDS row by row, kPitch bytes a row, their 16-byte pieces XOR-swizzled so
// that the K reads (16 bytes of 32 rows at once) and the transposing V reads (64 bytes of 4 rows at once) touch every bank once.
// ----------------------------------------------------------------------------------------
template <typename T, int DP, int NW_, int NS_>
struct AttnTile {
  typedef T type;
  static constexpr int NW = NW_, NS = NS_, kThreads = 64 * NW, kBN = 32 * NS, kRows = 32 * NW;
  static constexpr bool kSteady = true;  // has products(): the pipelined step
  static constexpr int kWaves = DP > 128 ? 1 : 2;  // per SIMD
  static constexpr int kPitch = DP <= 32 ? 64 : DP <= 64 ? 128 : DP <= 128 ? 256 : 512;
  static constexpr int kPieces = DP / 8, kPer = 8, kAll = kBN * kPieces, kStage = (kAll + kThreads - 1) / kThreads, kDB = DP / 32, kQF = DP / 16;
  static constexpr int kHalves = 1, kDV = DP, kPiecesV = kPieces, kAllV = kAll, kStageV = kStage;
  static constexpr int kSlot = kBN * kPitch, kFlag = 4 * kSlot, kSmem = kFlag + 16;
  struct P {
    h8 f[2];
  };

  h8 q[kQF];
  u4 ks[kStage], vs[kStageV];  // blocks on their way
  unsigned char* smem;
  int q32, h;

  static __device__ __forceinline__ int k_at(int slot, int row, int piece) {
    constexpr int m = kPitch >= 256 ? 15 : kPitch / 16 - 1, sh = kPitch >= 256 ? 0 : kPitch == 128 ? 1 : 2;
    return slot * kSlot + row * kPitch + ((piece ^ ((row >> sh) & m)) << 4);
  }
  static __device__ __forceinline__ int v_at(int slot, int row, int piece) {
    constexpr int m = kPitch >= 256 ? 3 : kPitch == 128 ? 1 : 0, sh = kPitch >= 256 ? 0 : 1;
    return (2 + slot) * kSlot + row * kPitch + ((piece ^ (((row >> sh) & m) << 2)) << 4);
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
  __device__ __forceinline__ void store_k(int slot, int i, int row, int piece) const { *reinterpret_cast<u4*>(smem + k_at(slot, row, piece)) = ks[i]; }
  __device__ __forceinline__ void store_v(int slot, int i, int row, int piece) const { *reinterpret_cast<u4*>(smem + v_at(slot, row, piece)) = vs[i]; }
  __device__ __forceinline__ void qk(int slot, f16v* s) const {
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[sub][r] = 0.f;
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
#pragma unroll
      for (int c = 0; c < kQF; ++c) {
        const h8 a = *reinterpret_cast<const h8*>(smem + k_at(slot, 32 * sub + q32, 2 * c + h));
        s[sub] = Op<T>::mfma(a, q[c], s[sub]);
      }
  }
  static __device__ __forceinline__ P pack_p(const float* p) {
    P f;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      u4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = Op<T>::pack(p[8 * m + 2 * j], p[8 * m + 2 * j + 1]);
      f.f[m] = __builtin_bit_cast(h8, w);
    }
    return f;
  }
  // V^T fragment of head-dim block db, 16-key group m of sub-tile `sub`: rows d = 32 db + (lane & 31), keys in score order
  __device__ __forceinline__ h8 v_frag(int slot, int sub, int db, int m) const {
    const int lane = lane_id(), i = lane & 15, ir = i >> 2, g16 = lane >> 4;
    const int row = 32 * sub + 16 * m + 4 * h + ir, piece = 4 * db + 2 * (g16 & 1) + ((i & 3) >> 1);
    const h4 lo = lds_read_tr16(reinterpret_cast<const half_t*>(smem + v_at(slot, row, piece) + (i & 1) * 8));
    const h4 hi = lds_read_tr16(reinterpret_cast<const half_t*>(smem + v_at(slot, row + 8, piece) + (i & 1) * 8));
    return h8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
  // keys: wave-uniform; sub-tiles behind the last one that any row sees are left out
  __device__ __forceinline__ void pv(int slot, const P* p, f16v* o, int keys) const {
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
      if (sub > 0 && 32 * sub >= keys) break;
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int db = 0; db < kDB; ++db) o[db] = Op<T>::mfma(v_frag(slot, sub, db, m), p[sub].f[m], o[db]);
    }
  }
  // A whole step: w = K Q^T, o += V^T z, y = exp2(x sc + nm) with its sums in bs.  The MFMAs are laid out one fragment at a time, each
  // followed by its share of the exponentials, and the LDS reads run kAhead fragments ahead: left to itself the compiler puts all the vector
  // work behind the last MFMA, and waits for each read.
  __device__ __forceinline__ void products(int slot, f16v (&w)[NS], const P (&z)[NS], f16v* o, const f16v (&x)[NS], P (&y)[NS], float nm, float sc,
                                           float& bs) const {
    constexpr int n1 = NS * kQF, n2 = NS * 2 * kDB, n = n1 + n2, kAhead = 3, kRing = kAhead + 1;
    constexpr int kEl = NS * 16;
    h8 ring[kRing];
    auto fragment = [&](int j) __attribute__((always_inline)) -> h8 {
      if (j < n1) return *reinterpret_cast<const h8*>(smem + k_at(slot, 32 * (j / kQF) + q32, 2 * (j % kQF) + h));
      const int i = j - n1;
      return v_frag(slot, i / (2 * kDB), i % kDB, i / kDB % 2);
    };
    u4 yw[NS][2];
    float v[kEl];
    auto take = [&](int e) __attribute__((always_inline)) {  // one exponential behind: its result is not waited for
      const int sub = e / 16, r = e % 16;
      bs = e == 0 ? v[e] : bs + v[e];
      pin(bs);
      if (r % 2) {
        unsigned two = Op<T>::pack(v[e - 1], v[e]);
        pin(two);
        yw[sub][r / 8][r % 8 / 2] = two;
      }
    };
#pragma unroll
    for (int j = 0; j < kAhead; ++j) ring[j] = fragment(j);
#pragma unroll
    for (int j = 0; j < n; ++j) {
      if (j + kAhead < n) ring[(j + kAhead) % kRing] = fragment(j + kAhead);
      const h8 a = ring[j % kRing];
      if (j < n1) {
        const f16v zero = {};
        w[j / kQF] = Op<T>::mfma(a, q[j % kQF], j % kQF == 0 ? zero : w[j / kQF]);
      } else {
        const int i = j - n1;
        o[i % kDB] = Op<T>::mfma(a, z[i / (2 * kDB)].f[i / kDB % 2], o[i % kDB]);
      }
#pragma unroll
      for (int e = kEl * j / n; e < kEl * (j + 1) / n; ++e) {
        v[e] = fast_exp2(__builtin_fmaf(x[e / 16][e % 16], sc, nm));
        if (e > 0) take(e - 1);
      }
      pp_sched_fence();
    }
    take(kEl - 1);
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
#pragma unroll
      for (int m = 0; m < 2; ++m) y[sub].f[m] = __builtin_bit_cast(h8, yw[sub][m]);
  }
  // zeroes what is not finite (exponent all ones: adding one to it carries out of the field); was there any?
  static __device__ __forceinline__ bool scrub(u4& w) {
    unsigned any = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned bad = ((w[j] & Op<T>::kExp) + Op<T>::kCarry) & 0x80008000u;  // the top bit of each bad half
      any |= bad;
      w[j] &= ~((bad >> 15) * 0xffffu);
    }
    return any != 0;
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
template <int DP, int NW_, int NS_>
struct AttnTile<float, DP, NW_, NS_> {
  typedef float type;
  static_assert(NS_ == 1, "f32: 32 keys a step");
  static constexpr int NW = NW_, NS = 1, kThreads = 64 * NW, kBN = 32, kRows = 32 * NW;
  static constexpr bool kSteady = false;  // (the vector work is a twentieth of the matrix work: nothing to overlap by hand)
  static constexpr int kWaves = DP > 128 || (DP > 96 && NW == 2) ? 1 : 2;  // per SIMD; LDS holds no more
  static constexpr int kP = DP + 4;
  // Queries of 256 channels and the sums of 256 do not fit the registers together (they spill: 25 TF/s, against 60): two work-groups take half of the
  // value channels each and both compute the scores, 3/2 of the work at more than three times the rate.
  static constexpr int kHalves = DP > 128 ? 2 : 1, kDV = DP / kHalves;
  static constexpr int kPieces = DP / 4, kPer = 4, kAll = kBN * kPieces, kStage = (kAll + kThreads - 1) / kThreads, kDB = kDV / 32, kQF = DP / 8;
  static constexpr int kPiecesV = kDV / 4, kAllV = kBN * kPiecesV, kStageV = (kAllV + kThreads - 1) / kThreads;
  static constexpr int kPV = kDV + 4, kSlot = kBN * kP, kSlotV = kBN * kPV, kFlag = (2 * kSlot + 2 * kSlotV) * 4, kSmem = kFlag + 16;
  struct P {
    float f[16];
  };

  f4 q[kQF];
  u4 ks[kStage], vs[kStageV];
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
  __device__ __forceinline__ void store_k(int slot, int i, int row, int piece) const {
    *reinterpret_cast<u4*>(smem + slot * kSlot + row * kP + 4 * piece) = ks[i];
  }
  __device__ __forceinline__ void store_v(int slot, int i, int row, int piece) const {
    *reinterpret_cast<u4*>(smem + 2 * kSlot + slot * kSlotV + row * kPV + 4 * piece) = vs[i];
  }
  // channels are taken in the order (8c + 4h + j): any order serves a dot product as long as both operands share it
  __device__ __forceinline__ void qk(int slot, f16v* s) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
#pragma unroll
    for (int c = 0; c < kQF; ++c) {
      const f4 a = *reinterpret_cast<const f4*>(smem + slot * kSlot + q32 * kP + 8 * c + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[0] = mfma_32x32x2_f32(a[j], q[c][j], s[0]);
    }
  }
  static __device__ __forceinline__ P pack_p(const float* p) {
    P f;
#pragma unroll
    for (int r = 0; r < 16; ++r) f.f[r] = p[r];
    return f;
  }
  __device__ __forceinline__ float v_val(int slot, int r, int db) const { return smem[2 * kSlot + slot * kSlotV + score_key(r, h) * kPV + 32 * db + q32]; }
  // keys: wave-uniform; groups of 8 keys behind the last one that any row sees are left out
  __device__ __forceinline__ void pv(int slot, const P* p, f16v* o, int keys) const {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (8 * g < keys) {
#pragma unroll
        for (int r = 4 * g; r < 4 * g + 4; ++r)
#pragma unroll
          for (int db = 0; db < kDB; ++db) o[db] = mfma_32x32x2_f32(v_val(slot, r, db), p[0].f[r], o[db]);
      }
  }
  static __device__ __forceinline__ bool scrub(u4& w) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool bad = (w[j] & 0x7f800000u) == 0x7f800000u;
      any |= bad;
      w[j] = bad ? 0u : w[j];
    }
    return any;
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
  float m, l;         // running maximum (of the raw scores; -inf before the first visible key) and the sum
  bool not_finite;    // values of V were left out: add_not_finite()
};

// What the rows of a work-group see of its nkeys keys: this lane's row, the largest count among the wave's live rows (0 without one) and the
// smallest among the work-group's.
struct AttnLimits {
  int row, wave_max, group_min, nkeys;
};

// The key from whose block on V is staged without values that are not finite: the first one that not every row sees -- or, where rows
// lie closer together than their channels (a single row, an expanded or overlapping view), the first of a last block with rows left: such a row
// starts before the block's last byte, so it is not read as zeros, and its weight of 0 does not make an infinity go away.
template <typename Tile>
__device__ __forceinline__ int mixed_key(const AttnLimits& lim, int64_t v_row, int DV) {
  const int whole = lim.nkeys / Tile::kBN * Tile::kBN;
  return v_row < DV && whole < lim.group_min ? whole : lim.group_min;
}

// k, v: the first key; D, DV: their channels (of v: those from the pointer on that this work-group sums).  sc = scale * log2(e) > 0.
template <typename Tile>
__device__ __forceinline__ void attend(Tile& t, AttnState<Tile>& st, const typename Tile::type* k, const typename Tile::type* v,
                                       int64_t k_row, int64_t v_row, const AttnLimits& lim, int D, int DV, float sc) {
  typedef typename Tile::type T;
  typedef typename Tile::P P;
  constexpr int NS = Tile::NS, BN = Tile::kBN;
#pragma unroll
  for (int db = 0; db < Tile::kDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.o[db][r] = 0.f;
  st.m = neg_inf();
  st.l = 0.f;
  st.not_finite = false;
  const int nsteps = (lim.nkeys + BN - 1) / BN;
  if (nsteps <= 0) return;

  // ---- staging: thread -> 16-byte pieces of a block; a piece past the head dim has an offset that no block reaches
  unsigned koff[Tile::kStage], voff[Tile::kStageV];
#pragma unroll
  for (int i = 0; i < Tile::kStage; ++i) {
    const int at = (int)threadIdx.x + Tile::kThreads * i, row = at / Tile::kPieces, piece = at - row * Tile::kPieces;
    koff[i] = piece * Tile::kPer < D && row < BN ? (unsigned)(row * k_row + piece * Tile::kPer) * sizeof(T) : ~0u << 5;
  }
#pragma unroll
  for (int i = 0; i < Tile::kStageV; ++i) {
    const int at = (int)threadIdx.x + Tile::kThreads * i, row = at / Tile::kPiecesV, piece = at - row * Tile::kPiecesV;
    voff[i] = piece * Tile::kPer < DV && row < BN ? (unsigned)(row * v_row + piece * Tile::kPer) * sizeof(T) : ~0u << 5;
  }
  const int mixed_from = mixed_key<Tile>(lim, v_row, DV);
  volatile int* const flag = reinterpret_cast<volatile int*>(reinterpret_cast<unsigned char*>(t.smem) + Tile::kFlag);
  if (threadIdx.x == 0) *flag = 0;
  auto block_of = [&](const T* base, int64_t stride, int i, int channels) __attribute__((always_inline)) -> Rows16 {
    const int left = lim.nkeys - i * BN < BN ? lim.nkeys - i * BN : BN;
    return rows16(base + (int64_t)i * BN * stride, left > 0 ? (unsigned)((left - 1) * stride + channels) * (unsigned)sizeof(T) : 0u);
  };
  auto load_k = [&](u4* dst, int i) __attribute__((always_inline)) {
    const Rows16 block = block_of(k, k_row, i, D);
#pragma unroll
    for (int j = 0; j < Tile::kStage; ++j) dst[j] = load_row16(block, koff[j]);
  };
  auto load_v = [&](int i) __attribute__((always_inline)) {
    const Rows16 block = block_of(v, v_row, i, DV);
#pragma unroll
    for (int j = 0; j < Tile::kStageV; ++j) t.vs[j] = load_row16(block, voff[j]);
  };
  auto store_k = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < Tile::kStage; ++j) {
      const int at = (int)threadIdx.x + Tile::kThreads * j, row = at / Tile::kPieces;
      if (Tile::kAll % Tile::kThreads == 0 || at < Tile::kAll) t.store_k(slot, j, row, at - row * Tile::kPieces);
    }
  };
  auto store_v = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < Tile::kStageV; ++j) {
      const int at = (int)threadIdx.x + Tile::kThreads * j, row = at / Tile::kPiecesV;
      if (Tile::kAllV % Tile::kThreads == 0 || at < Tile::kAllV) t.store_v(slot, j, row, at - row * Tile::kPiecesV);
    }
  };

  typedef f16v Scores[NS];
  typedef P Probs[NS];
  // scores of the block whose softmax is next; probabilities of the block before it.  The second pair takes turns in the fast steps, so
  // that nothing is copied.
  Scores s, s2;
  Probs p, p2;
  // -m sc (NaN before the first visible key and from kFar on: whatever a block holds, it is taken again by its differences from the
  // maximum); sums over the block
  float nm = __builtin_nanf(""), bs;
  auto softmax = [&](const Scores& x, Probs& y) __attribute__((always_inline)) -> bool {  // x -> y, bs; did a sum come out too large?
    bs = 0.f;
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
      float e[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if constexpr (Tile::kSteady) e[r] = fast_exp2(__builtin_fmaf(x[sub][r], sc, nm));
        else e[r] = fast_exp2((x[sub][r] - st.m) * sc);  // (no maximum yet: infinite or NaN, taken again)
        bs += e[r];
      }
      y[sub] = Tile::pack_p(e);
    }
    return wave_any(!(bs <= kMost));
  };
  // moves the maximum to that of x and what was summed up with it; x -> y, bs
  auto move_max = [&](const Scores& x, Probs& y) __attribute__((always_inline)) {
    keep_branch();
    float top = x[0][0];
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, x[sub][r]);
    top = fmaxf(st.m, pair32_max(top));
    const float alpha = top == st.m ? 1.f : fast_exp2((st.m - top) * sc);
    const float base = top == neg_inf() ? 0.f : top;
    st.m = top;
    st.l *= alpha;
    nm = fabsf(top * sc) < kFar ? -top * sc : __builtin_nanf("");
#pragma unroll
    for (int db = 0; db < Tile::kDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) st.o[db][r] *= alpha;
    bs = 0.f;
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
      float e[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        e[r] = fast_exp2((x[sub][r] - base) * sc);
        bs += e[r];
      }
      y[sub] = Tile::pack_p(e);
    }
  };
  auto stage = [&](int i, int slot) __attribute__((always_inline)) {
    store_k(slot);  // block i + 2
    store_v(slot);  // block i
    load_k(t.ks, i + 3);
    load_v(i + 1);
  };
  // softmax of block i (x -> y), second product of block i - 1 (z), first product of block i + 1 (-> w); every live row of the work-group
  // sees all of block i
  [[maybe_unused]] auto fast_step = [&](int i, auto slot, const Scores& x, Scores& w, const Probs& z, Probs& y) __attribute__((always_inline)) {
    constexpr int S0 = decltype(slot)::value, S1 = 1 - S0;
    stage(i, S0);
    if (lim.wave_max > 0) {
      // a wave that is in its products goes before one that stages (prompt of 8192, 128 channels: 581 -> 571 us, 1131 -> 1103 without a
      // mask; 64: 338 either way, so not there)
      if constexpr (Tile::kDB > 2) wave_priority<1>();
      if constexpr (Tile::kSteady) t.products(S1, w, z, st.o, x, y, nm, sc, bs);
      if constexpr (Tile::kDB > 2) wave_priority<0>();
      if (wave_any(!(bs <= kMost))) move_max(x, y);
      st.l += bs;
    }
    pp_barrier();
  };
  // the same for any block: rows that see a part of it, waves that see none of it, no block before or behind it
  auto any_step = [&](int i) __attribute__((always_inline)) {
    const int s0 = i & 1, s1 = 1 - s0;
    if (mixed_from < lim.nkeys && (i + 1) * BN > mixed_from) {
#pragma unroll
      for (int j = 0; j < Tile::kStageV; ++j)
        if (Tile::scrub(t.vs[j])) *flag = 1;
    }
    stage(i, s0);
    if (i > 0 && (i - 1) * BN < lim.wave_max) t.pv(s1, p, st.o, lim.wave_max - (i - 1) * BN);
    if (i * BN < lim.wave_max) {
#pragma unroll
      for (int sub = 0; sub < NS; ++sub) {
        const int left = lim.row - i * BN - 32 * sub;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[sub][r] = score_key(r, t.h) < left ? s[sub][r] : neg_inf();
      }
      if (softmax(s, p)) move_max(s, p);
      st.l += bs;
      if ((i + 1) * BN < lim.wave_max) t.qk(s1, s);
    }
    pp_barrier();
  };

  // ---- before step 0: K of blocks 0 and 1 in LDS, block 2 and V of block 0 on their way, scores of block 0
  u4 k1[Tile::kStage];
  load_k(t.ks, 0);
  load_k(k1, 1);
  load_v(0);
  store_k(0);
  load_k(t.ks, 2);
#pragma unroll
  for (int j = 0; j < Tile::kStage; ++j) {
    const u4 two = t.ks[j];
    t.ks[j] = k1[j];
    k1[j] = two;
  }
  store_k(1);
#pragma unroll
  for (int j = 0; j < Tile::kStage; ++j) t.ks[j] = k1[j];
  pp_barrier();
  t.qk(0, s);
  pp_barrier();
  const int nfast = mixed_from / BN;
  for (int i = 0; i < nsteps;) {
    any_step(i);
    ++i;
    if constexpr (Tile::kSteady)
      if (i == 1)
        for (; i + 2 <= nfast; i += 2) {
          fast_step(i, std::integral_constant<int, 1>{}, s, s2, p, p2);
          fast_step(i + 1, std::integral_constant<int, 0>{}, s2, s, p2, p);
        }
  }
  if ((nsteps - 1) * BN < lim.wave_max) t.pv((nsteps - 1) & 1, p, st.o, lim.wave_max - (nsteps - 1) * BN);
  st.l = pair32_sum(st.l);
  st.not_finite = *flag != 0;
}

// Adds to o (weighted sums, normalised or not) what attend() left out: infinities and NaN of the keys that a row sees, from the block of
// mixed_key() on.
template <typename Tile>
__device__ __forceinline__ void add_not_finite(const Tile& t, AttnState<Tile>& st, const typename Tile::type* v, int64_t v_row,
                                               const AttnLimits& lim, int DV) {
#pragma unroll 1
  for (int key = mixed_key<Tile>(lim, v_row, DV) / Tile::kBN * Tile::kBN; key < lim.nkeys; ++key) {
    const typename Tile::type* row = v + key * v_row;
#pragma unroll
    for (int db = 0; db < Tile::kDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 32 * db + score_key(r, t.h);
        const float x = d < DV ? to_f32(row[d]) : 0.f;
        if ((__builtin_bit_cast(unsigned, x) & 0x7f800000u) == 0x7f800000u && key < lim.row) st.o[db][r] += x;
      }
  }
}

}  // namespace pp
