// Attention of the encoder layer (reference models/multiway_transformer.py:99-132) and its gradient, gfx950.
//
//   s_ij = scale q_i . k_j,   p_ij = keep_j exp(s_ij - m_i) / sum_j,   o_i = sum_j p_ij v_j
// in one pass over the keys with a running maximum and sum; the forward keeps L_i = m_i + log2 sum (base 2), from which the
// backward recomputes p_ij = 2^(s_ij c - L_i), c = scale log2 e:
//   delta_i = do_i . o_i,   ds_ij = p_ij (do_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij do_i.
//
// Rows.  The query heads that share a key/value head are rows of ONE problem: row i of (sample, kv head) is query i / G of head
// kvhead * G + i % G, G = H / Hkv.  A key tile is then read once for all of them, and one query of G heads fills G columns of a
// matrix instruction instead of one.
//
// Operand layout.  v_mfma_f32_32x32x16_bf16 (and, per 4 of them, v_mfma_f32_32x32x2_f32) leave in lane l column l & 31 and rows
// (r & 3) + 8 (r >> 2) + 4 (l >> 5).  Every product is oriented so that the softmax index is the COLUMN (query in the forward and
// dq kernels, key in the dk/dv kernel): maxima and sums are then register reductions plus one exchange between the wave's halves,
// and the probabilities are, as they lie, the B operand of the next product: its contraction index may be taken in any order as
// long as the A operand follows, so chunk c of a 32-row accumulator supplies rows 16c + 4h + {0..3} and 16c + 8 + 4h + {0..3} (bf16)
// and the A operand is read from LDS in that order (ds_read_b64_tr_b16: four rows of one column each).
//
// LDS.  Tiles go from memory to LDS directly (buffer_load ... lds, 1 KiB a wave instruction) into a ring of stages, one tile
// ahead of the one that is worked on.  A masked row is an offset outside the descriptor, for which the hardware delivers zeros.
// The 16-byte chunks of a row are permuted (AttnCfg::swizzle) -- on the source side, since the transfer writes LDS in lane order --
// so that both ways of reading, row fragments and transposed ones, spread over all banks.
// No atomics: dq and dk/dv have a kernel each (7 products instead of 5), or one workgroup has a head's whole backward, so results do
// not depend on the order of execution.
#include <math.h>

#include <type_traits>

#include "common.h"

namespace eve {

typedef __attribute__((ext_vector_type(8))) __bf16 at_bf16x8;
typedef __attribute__((ext_vector_type(4))) short at_s16x4;
typedef __attribute__((ext_vector_type(8))) short at_s16x8;
typedef __attribute__((ext_vector_type(16))) float at_f32x16;
typedef __attribute__((ext_vector_type(4))) float at_f32x4;
typedef __attribute__((ext_vector_type(2))) float at_f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 at_bf16x2;

struct AttnArgs {
  const void *q, *k, *v, *o, *dout;
  const uint8_t* mask;  // [B, Nk], nonzero = visible; may be null
  void *out, *dq, *dk, *dv;
  float* lse;                 // [B * Hkv, rows]
  uint4* stats;               // [B * Hkv, rows]: -L / c and -delta, as the dk/dv kernel wants them
  float *part_o, *part_ml;    // forward splits: [B * Hkv, nsplit, rows, D] and [..., 2]
  float *part_a, *part_b;     // backward splits: dq | dk, and dv: [B * Hkv, nsplit, rows or keys, D]
  eve_attn_layout in, grad;   // element strides of q, k, v and of their gradients
  int Nq, Nk, Hkv, G, D, rows;
  int heads;                  // B * Hkv
  int nblk, nsplit;           // row (or key) blocks of a head, splits of its key tiles
  int tiles_per_split;
  int by_xcd;                 // blocks of a head on one XCD (block_coord)
  float scale, c, inv_c;      // c = scale log2 e
};

// ---- operand traits: a fragment is 16 bytes a lane for either type
template <typename T> struct AT;
template <> struct AT<bf16_t> { static constexpr int E = 8; };
template <> struct AT<float> { static constexpr int E = 4; };

template <typename T, int DP, bool LONG = false> struct AttnCfg {
  static constexpr int E = AT<T>::E;
  static constexpr int NKS = DP / (2 * E);              // contraction steps over the head width
  static constexpr int CPR = DP / E;                    // 16-byte chunks of a row
  static constexpr int RB = DP * (int)sizeof(T);        // bytes of a row: 128, 256 or 512
  static constexpr int KT = RB == 128 || LONG ? 64 : 32;  // rows of a staged tile
  static constexpr uint64_t kFull = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;
  static constexpr int TILE = KT * RB;
  static constexpr int STAGE = 2 * TILE;                // keys and values, or queries and gradients
  static constexpr int NST = 2;                         // stages of the ring: NST - 1 tiles ahead
  static constexpr int PC = 32 / (2 * E);               // fragments of a 32-row accumulator
  static constexpr int ND = DP / 32;
  static constexpr int NJ = KT / 32;
  // Chunk c of a row lies at c ^ swizzle(row).  The banks are 256 bytes wide: 16 rows' fragments (a chunk each) take different ones,
  // as do four rows' 64 bytes (bf16 columns) or a row's 128 bytes and those of the row four further on (fp32 columns).
  static constexpr int swizzle(int row) {
    return RB == 128 ? (row >> 1 & 1) << 2 | (row >> 2 & 1) << 1 | (row >> 3 & 1)
           : sizeof(T) == 2 ? (row & 3) << 2 | (row >> 2 & 3)
                            : (row >> 2 & 1) << 3 | (row & 3) << 1 | (row >> 3 & 1);
  }
};

constexpr float kLowest = -3.4028234663852886e38f;  // the lowest finite number
constexpr int kBitTiles = 64;  // tiles whose mask words a workgroup holds

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ at_f32x16 mma(const uint4& a, const uint4& b, at_f32x16 acc, bf16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(at_bf16x8, a), __builtin_bit_cast(at_bf16x8, b), acc, 0, 0, 0);
}
__device__ __forceinline__ at_f32x16 mma(const uint4& a, const uint4& b, at_f32x16 acc, float) {
  acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), acc, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), acc, 0, 0, 0);
}

// 16 bytes from LDS.  (An access of a vector type keeps its type information; without it the compiler takes it for one that may
// meet what a transfer in flight writes, and waits for all of them.)
typedef uint32_t at_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t at_u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint4 lds16(const char* p) {
  const at_u32x4 w = *reinterpret_cast<const at_u32x4*>(p);
  return make_uint4(w.x, w.y, w.z, w.w);
}
__device__ __forceinline__ uint32_t lds_offset(const char* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }

// A lane's place in the row fragments of a tile (at smem + tile, a multiple of 128 bytes): row lane & 31 of 32-row block j, step ks.
template <typename C> struct RowReader {
  uint32_t base;
  __device__ __forceinline__ explicit RowReader(int lane) {
    const int row = lane & 31;
    base = row * C::RB + (((lane >> 5) ^ C::swizzle(row)) << 4);
  }
  __device__ __forceinline__ uint4 get(const char* smem, uint32_t tile, int j, int ks) const {
    constexpr int W = C::RB == 128 ? 4 : 8;  // steps whose chunks are permuted among themselves
    return lds16(smem + (((tile + base) ^ ((ks % W) << 5)) + ks / W * 256 + j * 32 * C::RB));
  }
};

// Transposed fragments, bf16: column d0 + (lane & 31), rows of 16-row chunk rc in the order of an accumulator's registers (rows
// 4 h + {0..3}, then 8 + 4 h + {0..3}).  Fragments -- of the two 16-row chunks of 32 rows, two column blocks -- are read and
// waited for in one block: through the builtin the compiler would also wait for the tiles in flight, which it cannot tell apart
// from what is read.
template <typename C> __device__ __forceinline__ void tr_frags4(const char* smem, uint32_t a0, uint32_t a1, uint4 (&f)[4]) {  // f[2 chunk + column block]
  constexpr int RB = C::RB, X = (C::swizzle(8) ^ C::swizzle(0)) << 4;  // eight rows on
  const uint32_t at = lds_offset(smem);
  at_s16x4 v[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %10 offset:%12\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %11 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %8 offset:%13\n\tds_read_b64_tr_b16 %5, %10 offset:%14\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:%13\n\tds_read_b64_tr_b16 %7, %11 offset:%14\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(at + a0), "v"(at + a1), "v"(at + (a0 ^ X)), "v"(at + (a1 ^ X)), "n"(8 * RB), "n"(16 * RB), "n"(24 * RB)
      : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const at_s16x8 w = __builtin_shufflevector(v[2 * i], v[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    f[i] = __builtin_bit_cast(uint4, w);
  }
}
// A lane's place in them: column blocks 0 and 1 (those of pair p: 128 p bytes on, permuted)
template <typename C> struct ColReader {
  uint32_t base[2];
  __device__ __forceinline__ explicit ColReader(int lane) {
    const int i = lane & 15, q = i >> 2, p = i & 3, h = lane >> 5;
    const int c = 2 * ((lane >> 4) & 1) + (p >> 1);
    base[0] = (4 * h + q) * C::RB + ((c ^ C::swizzle(4 * h + q)) << 4) + (p & 1) * 8;
    base[1] = base[0] ^ 64;
  }
};
// fp32: chunk c (8 rows) of the 32 rows from r0, column d0 + (lane & 31)
template <typename C> __device__ __forceinline__ uint4 col_frag_f32(const char* smem, uint32_t tile, int r0, int c, int d0, int lane) {
  const int h = lane >> 5, col = d0 + (lane & 31);
  uint32_t w[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int row = r0 + 8 * c + 4 * h + t;
    w[t] = *reinterpret_cast<const uint32_t*>(smem + (tile + row * C::RB + (((col >> 2) ^ C::swizzle(row)) << 4) + (col & 3) * 4));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The column fragments of 32-row block j of a tile: f[c ND + i]
template <typename T, typename C> struct ColFrags {
  uint4 f[C::PC * C::ND];
  // bf16: of column blocks 2 pair and 2 pair + 1, g[2 chunk + block]
  static __device__ __forceinline__ void read_pair(const char* smem, uint32_t at, int j, int pair, const ColReader<C>& r, uint4 (&g)[4]) {
    const uint32_t tile = at + j * 32 * C::RB;
    tr_frags4<C>(smem, (tile + r.base[0]) ^ pair * 128, (tile + r.base[1]) ^ pair * 128, g);
  }
  __device__ __forceinline__ void read(const char* smem, uint32_t at, int j, const ColReader<C>& r, int lane) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int pair = 0; pair < C::ND / 2; ++pair) {
        uint4 g[4];
        read_pair(smem, at, j, pair, r, g);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) f[c * C::ND + 2 * pair + i] = g[2 * c + i];
      }
    } else {
#pragma unroll
      for (int c = 0; c < C::PC; ++c)
#pragma unroll
        for (int i = 0; i < C::ND; ++i) f[c * C::ND + i] = col_frag_f32<C>(smem, at, 32 * j, c, 32 * i, lane);
    }
  }
};
__device__ __forceinline__ uint32_t at_pack(float lo, float hi) {
  const at_f32x2 t = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(t, at_bf16x2));
}
// chunk c of an accumulator as the B operand.  bf16: the probabilities (or ds) are rounded to the operands' type for the matrix
// unit, by at most half a step each (2^-8 relative); the sums over them stay in fp32.
__device__ __forceinline__ uint4 acc_frag(const at_f32x16& s, int c, bf16_t) {
  return make_uint4(at_pack(s[8 * c], s[8 * c + 1]), at_pack(s[8 * c + 2], s[8 * c + 3]), at_pack(s[8 * c + 4], s[8 * c + 5]),
                    at_pack(s[8 * c + 6], s[8 * c + 7]));
}
__device__ __forceinline__ uint4 acc_frag(const at_f32x16& s, int c, float) {
  return make_uint4(__float_as_uint(s[4 * c]), __float_as_uint(s[4 * c + 1]), __float_as_uint(s[4 * c + 2]), __float_as_uint(s[4 * c + 3]));
}
__device__ __forceinline__ at_f32x16 acc_zero() {
  at_f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}
// the two halves of a wave hold the same columns: combine lane l with lane l ^ 32
__device__ __forceinline__ void halves(float x, float& a, float& b) {
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  a = __uint_as_float(w[0]);
  b = __uint_as_float(w[1]);
}
__device__ __forceinline__ float halves_max(float x) { float a, b; halves(x, a, b); return fmaxf(a, b); }
__device__ __forceinline__ float halves_sum(float x) { float a, b; halves(x, a, b); return a + b; }

template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d);
template <> __device__ __forceinline__ void store4<float>(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
template <> __device__ __forceinline__ void store4<bf16_t>(bf16_t* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(at_pack(a, b), at_pack(c, d));
}
template <typename T> __device__ __forceinline__ float dot16(const uint4& a, const uint4& b) {
  Vec16<T> x, y;
  x.raw = __builtin_bit_cast(decltype(x.raw), a);
  y.raw = __builtin_bit_cast(decltype(y.raw), b);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < Vec16<T>::N; ++i) s = fmaf(x.get(i), y.get(i), s);
  return s;
}

// Workgroups are dealt round-robin over the 8 XCDs, each with an L2 of its own: with by_xcd all blocks of a head (which read the
// same keys) run on one of them.  Only where every XCD gets work (the host decides); otherwise heads follow each other.
__device__ __forceinline__ bool block_coord(const AttnArgs& a, int& head, int& blk, int& split) {
  const int per = a.nblk * a.nsplit;
  int r;
  if (a.by_xcd) {
    const int local = blockIdx.x >> 3;
    head = (local / per) * 8 + (blockIdx.x & 7);
    r = local % per;
  } else {
    head = blockIdx.x / per;
    r = blockIdx.x % per;
  }
  blk = r / a.nsplit;
  split = r % a.nsplit;
  return head < a.heads;
}

constexpr uint32_t kNowhere = 0xfffffff0u, kReach = 0x80000000u;  // an offset outside every descriptor, and their extent

// Which of the KT keys of a tile are visible, bit by bit.  A mask is turned into words in LDS, kBitTiles tiles at a time: were its
// bytes loaded tile by tile, their wait would also be one for the tiles in flight, which the same counter counts.
template <int KT, int NW> struct KeyBits {
  const uint8_t* mask;
  uint64_t* words;
  int Nk, t0, t1, wave, lane;
  // called by all waves, with t0, t0 + 1, ... one after the other
  __device__ __forceinline__ uint64_t of(int t) const {
    if (t >= t1) return 0;
    if (!mask) {
      const int n = Nk - t * KT;
      return n >= KT ? (KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1) : (1ull << n) - 1;
    }
    const int at = (t - t0) % kBitTiles;
    if (at == 0) {
      __syncthreads();
#pragma unroll 4
      for (int j = wave; j < kBitTiles; j += NW) {
        const int key = (t + j) * KT + lane;
        const uint64_t w = __ballot(t + j < t1 && lane < KT && key < Nk && mask[key] != 0);
        if (lane == 0) words[j] = w;
      }
      __syncthreads();
    }
    const uint64_t w = words[at];
    return (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(w >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)w);
  }
};

// Whether a sample sees so few keys that the backward forms delta as sum p dp: do . o sees the rounding of the stored result, which
// is large next to what is left of the ds of a few keys (bf16, 5 keys, width 112: dq 1.8 % off; 2 keys of width 64: 0.4 % instead of
// 0.2).  It goes by the keys that are seen, so that a sample's gradients do not depend on its padding.
constexpr int kFewKeys = 64;
// The same answer in all threads of NW waves; `scratch`: NW ints of LDS.  1024 keys and more a round, until enough are seen.
template <int NW> struct FewKeys {
  static constexpr int PER = 4;  // keys a thread and round
  const uint8_t* mask;
  int Nk, tid;
  uint8_t first[PER];  // of the first round, requested early
  __device__ __forceinline__ bool in(int key) const { return key < Nk && mask[key] != 0; }
  __device__ __forceinline__ FewKeys(const uint8_t* mask, int Nk, int tid) : mask(mask), Nk(Nk), tid(tid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) first[i] = mask && Nk > kFewKeys ? in(i * NW * 64 + tid) : 0;
  }
  __device__ __forceinline__ bool operator()(int* scratch) const {
    if (Nk <= kFewKeys) return true;
    if (!mask) return false;
    int seen = 0;
    for (int k0 = 0; k0 < Nk && seen <= kFewKeys; k0 += PER * NW * 64) {
      int mine = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) mine += __popcll(__ballot(k0 == 0 ? first[i] : in(k0 + i * NW * 64 + tid)));
      if (NW > 1) {
        if ((tid & 63) == 0) scratch[tid >> 6] = mine;
        __syncthreads();
        mine = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) mine += scratch[w];
        __syncthreads();
      }
      seen += mine;
    }
    return __builtin_amdgcn_readfirstlane(seen) <= kFewKeys;
  }
};

// Pieces of 1 KiB of a tile, dealt to the NW waves; lane l of piece p holds chunk l % CPR of row p (64 / CPR) + l / CPR.
template <typename C, int NW> struct TileLoader {
  static constexpr int N = C::TILE / 1024 / NW;  // a wave's transfers for a tile
  uint32_t off[N];
  int row[N];
  __device__ __forceinline__ TileLoader(int64_t stride, int D, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      row[i] = (i * NW + wave) * (64 / C::CPR) + lane / C::CPR;
      const int c = (lane % C::CPR) ^ C::swizzle(row[i]);
      off[i] = c * C::E < D ? (uint32_t)row[i] * ((uint32_t)stride * (16 / C::E)) + c * 16 : kNowhere;
    }
  }
  __device__ __forceinline__ void load(const void* p, char* tile, int wave, uint64_t bits) const {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, kReach, 0x00020000);
    auto to_lds = [&](int i, uint32_t o) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(tile + (i * NW + wave) * 1024), 16, o, 0, 0, 0);
    };
    if (bits == C::kFull) {
#pragma unroll
      for (int i = 0; i < N; ++i) to_lds(i, off[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) to_lds(i, (bits >> row[i]) & 1 ? off[i] : kNowhere);
    }
  }
};
// Waits until this wave's transfers of a tile have landed while the NEWER ones of later tiles may be in flight (loads between them
// only make the wait stricter), then for the other waves, which also have read what the next transfer overwrites.
template <int NEWER> __device__ __forceinline__ void tile_ready() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(NEWER) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// What the waves have written to LDS is seen by all of them (tiles on their way stay so).
__device__ __forceinline__ void lds_exchange() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// No transfer may be on its way into LDS when the workgroup ends.
__device__ __forceinline__ void tiles_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
#endif  // __HIP_DEVICE_COMPILE__

// ---------------------------------------------------------------------------------------------------------- forward
// Block: NW waves of 32 rows each; the key tiles are staged for all of them.
// Bound: the vector unit, busy for 74 % of a CU's cycles (250 instructions a wave and 64-key tile, the exponentials foremost; the
// matrix unit 33 %).  64 x 12 heads of 617 x 617: 123 us (610 TFLOP/s); 2 x 16 heads of 4096 x 4096: 171 to 187 us (740 to 800; 72 % and
// 42 %).  One query of 4 x 16 heads on 4 over 16384 keys (NW = 1, 47 splits): 25 us, 5.3 TB/s, the memory's rate.
// The bounds on waves keep the register budget at 256, where the compiler holds accumulators in plain registers: in the larger
// budget it moves them to and from accumulation registers, a third of the instructions of the loop.
// (bf16 of width 65 to 128: tiles of 64 keys, half as many waits: 36 us instead of 41 for 3 x 16 heads on 4, 1001 x 1001.  The
// gradients' kernels gain nothing by them, float32 loses its splits, one wave a workgroup its place for three in a CU.)
template <typename T, int DP, int NW> using FwdCfg = AttnCfg<T, DP, NW == 4 && sizeof(T) == 2 && DP == 128>;
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW == 1 ? 1 : DP == 128 ? 2 : sizeof(T) == 2 ? 4 : 3) void attn_fwd_kernel(AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using C = FwdCfg<T, DP, NW>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, wave_u = __builtin_amdgcn_readfirstlane(wave);
  int head, blk, split;
  if (!block_coord(a, head, blk, split)) return;
  const int b = head / a.Hkv, hk = head % a.Hkv;
  const T* kb = static_cast<const T*>(a.k) + b * a.in.k_b + hk * a.in.k_h;
  const T* vb = static_cast<const T*>(a.v) + b * a.in.v_b + hk * a.in.v_h;
  const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.Nk : nullptr;
  const int row = blk * (NW * 32) + wave * 32 + (lane & 31);
  const bool row_ok = row < a.rows;
  const int qi = row / a.G, qh = hk * a.G + row % a.G;

  uint4 qf[C::NKS];
  {
    const T* qp = static_cast<const T*>(a.q) + b * a.in.q_b + (int64_t)qi * a.in.q_n + qh * a.in.q_h;
#pragma unroll
    for (int ks = 0; ks < C::NKS; ++ks) {
      const int d = (2 * ks + half) * C::E;
      qf[ks] = make_uint4(0, 0, 0, 0);
      if (row_ok && d < a.D) qf[ks] = *reinterpret_cast<const uint4*>(qp + d);
    }
  }
  at_f32x16 o[C::ND];
#pragma unroll
  for (int i = 0; i < C::ND; ++i) o[i] = acc_zero();
  float m = -INFINITY, l = 0.f;
  bool any = false;  // key seen so far

  const int ntiles = (a.Nk + C::KT - 1) / C::KT;
  const int t0 = split * a.tiles_per_split, t1 = min(ntiles, t0 + a.tiles_per_split);
  const TileLoader<C, NW> kl(a.in.k_n, a.D, wave, lane), vl(a.in.v_n, a.D, wave, lane);
  const RowReader<C> rows(lane);
  const ColReader<C> cols(lane);
  const KeyBits<C::KT, NW> keys{mask, reinterpret_cast<uint64_t*>(smem + C::NST * C::STAGE), a.Nk, t0, t1, wave, lane};
  auto fetch = [&](int t, uint64_t b) {  // past the last tile: nothing is read
    char* stage = smem + (t - t0) % C::NST * C::STAGE;
    kl.load(kb + (int64_t)t * C::KT * a.in.k_n, stage, wave_u, b);
    vl.load(vb + (int64_t)t * C::KT * a.in.v_n, stage + C::TILE, wave_u, b);
  };
  uint64_t bits = keys.of(t0);
  fetch(t0, bits);
  for (int t = t0; t < t1; ++t) {
    const uint32_t ks_ = (t - t0) % C::NST * C::STAGE, vs_ = ks_ + C::TILE;
    tile_ready<0>();
    const uint64_t bits_next = keys.of(t + 1);
    fetch(t + 1, bits_next);
    if (bits) {
      any = true;
      at_f32x16 s[C::NJ];
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) {
        s[j] = acc_zero();
#pragma unroll
        for (int ks = 0; ks < C::NKS; ++ks) s[j] = mma(rows.get(smem, ks_, j, ks), qf[ks], s[j], T());
      }
      ColFrags<T, C> vf;  // read while the matrix unit works on the scores
      vf.read(smem, vs_, 0, cols, lane);
      if (bits != C::kFull) {
        const uint64_t mine = bits >> (4 * half);
#pragma unroll
        for (int j = 0; j < C::NJ; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!((mine >> (32 * j + (r & 3) + 8 * (r >> 2))) & 1)) s[j][r] = -INFINITY;
      }
      float mt = s[0][0];
#pragma unroll
      for (int j = 0; j < C::NJ; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[j][r]);
      // m is any number that keeps the sums in range: it follows the maximum only where that is 2^8 ahead, so that rows rarely rescale
      const float mx = halves_max(mt) * a.c;
      if (__any(mx > m + 8.f)) {
        const float m_new = fmaxf(m, mx), alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < C::ND; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
      }
      const float ms = m == -INFINITY ? 0.f : m;  // only scores of -inf so far: 2^(-inf - 0) = 0, should others follow
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < C::NJ; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[j][r] = __builtin_amdgcn_exp2f(fmaf(s[j][r], a.c, -ms));
          sum += s[j][r];
        }
      l += sum;
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) {
        if (j > 0) vf.read(smem, vs_, j, cols, lane);
#pragma unroll
        for (int cc = 0; cc < C::PC; ++cc) {
          const uint4 p = acc_frag(s[j], cc, T());
#pragma unroll
          for (int i = 0; i < C::ND; ++i) o[i] = mma(vf.f[cc * C::ND + i], p, o[i], T());
        }
      }
    }
    bits = bits_next;
  }
  tiles_landed();
  l = halves_sum(l);
  if (!row_ok) return;
  if (a.nsplit == 1) {
    const float none = any ? NAN : 0.f;  // no visible key: zeros; visible keys whose scores are all -inf: NaN, as -inf - (-inf) is
    const float inv = l == 0.f ? none : 1.f / l;
    T* op = static_cast<T*>(a.out) + (((int64_t)b * a.Nq + qi) * (a.Hkv * a.G) + qh) * a.D;
#pragma unroll
    for (int i = 0; i < C::ND; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * i + 8 * g + 4 * half;
        if (d < a.D) store4<T>(op + d, o[i][4 * g] * inv, o[i][4 * g + 1] * inv, o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv);
      }
    if (a.lse && half == 0) a.lse[(int64_t)head * a.rows + row] = l == 0.f ? (any ? NAN : INFINITY) : m + __builtin_amdgcn_logf(l);
  } else {
    const int64_t at = ((int64_t)head * a.nsplit + split) * a.rows + row;
    float* op = a.part_o + at * a.D;
#pragma unroll
    for (int i = 0; i < C::ND; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * i + 8 * g + 4 * half;
        if (d < a.D) store4<float>(op + d, o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
      }
    if (half == 0) {
      a.part_ml[2 * at] = any ? fmaxf(m, kLowest) : m;  // -inf tells the join that nothing was visible
      a.part_ml[2 * at + 1] = l;
    }
  }
#endif
}

// Joins the splits of a row, in a fixed order: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  A block a row: 8 splits of 32
// chunks of 4 columns at a time, then the 8 are added.
constexpr int kMaxSplit = 256;
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ float weight[kMaxSplit], red[8];
  __shared__ float4 sums[8][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int head = blockIdx.x / a.rows, row = blockIdx.x % a.rows;
  const int64_t at0 = (int64_t)head * a.nsplit * a.rows + row;
  float m = -INFINITY, l = 0.f;
  if (tid < a.nsplit) {
    m = a.part_ml[2 * (at0 + (int64_t)tid * a.rows)];
    l = a.part_ml[2 * (at0 + (int64_t)tid * a.rows) + 1];
  }
  float top = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  if (lane == 0) red[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float w = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
  weight[tid] = w;
  l = wave_sum(w * l);
  if (lane == 0) red[4 + wave] = l;
  __syncthreads();
  l = (red[4] + red[5]) + (red[6] + red[7]);
  const int d = (tid & 31) * 4;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d < a.D) {
#pragma unroll 4
    for (int s = tid >> 5; s < a.nsplit; s += 8) {
      const float4 y = *reinterpret_cast<const float4*>(a.part_o + (at0 + (int64_t)s * a.rows) * a.D + d);
      const float ws = weight[s];
      x.x = fmaf(ws, y.x, x.x);
      x.y = fmaf(ws, y.y, x.y);
      x.z = fmaf(ws, y.z, x.z);
      x.w = fmaf(ws, y.w, x.w);
    }
  }
  sums[tid >> 5][tid & 31] = x;
  __syncthreads();
  if (tid >= 32 || d >= a.D) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    const float4 y = sums[i][tid];
    x.x += y.x;
    x.y += y.y;
    x.z += y.z;
    x.w += y.w;
  }
  const bool any = top != -INFINITY;
  const float inv = l == 0.f ? (any ? NAN : 0.f) : 1.f / l;
  const int b = head / a.Hkv, hk = head % a.Hkv;
  T* op = static_cast<T*>(a.out) + (((int64_t)b * a.Nq + row / a.G) * (a.Hkv * a.G) + hk * a.G + row % a.G) * a.D;
  store4<T>(op + d, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
  if (a.lse && tid == 0) a.lse[(int64_t)head * a.rows + row] = l == 0.f ? (any ? NAN : INFINITY) : top + __builtin_amdgcn_logf(l);
#endif
}

// Adds the splits of a gradient in their order: g = factor * sum_s part[head, s, row].  Four columns a thread; for dq a row is
// query row / G of query head (key head) G + row % G, for dk and dv (G = 1) a key.
struct AttnSum { const float* part; void* g; int64_t g_b, g_n, g_h; int64_t total; int Hkv, G, D, rows, nsplit; float factor; };
struct AttnSums { AttnSum s[2]; };  // by blockIdx.y
template <typename T>
__global__ __launch_bounds__(256) void attn_sum_kernel(AttnSums sums) {
#if defined(__HIP_DEVICE_COMPILE__)
  const AttnSum a = sums.s[blockIdx.y];
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.total) return;
  const int cols = a.D / 4, d = (int)(i % cols) * 4;
  const int64_t hr = i / cols;
  const int row = (int)(hr % a.rows), head = (int)(hr / a.rows);
  const float* p = a.part + ((int64_t)head * a.nsplit * a.rows + row) * a.D + d;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < a.nsplit; ++s) {
    const float4 y = *reinterpret_cast<const float4*>(p + (int64_t)s * a.rows * a.D);
    x.x += y.x;
    x.y += y.y;
    x.z += y.z;
    x.w += y.w;
  }
  T* g = static_cast<T*>(a.g) + (head / a.Hkv) * a.g_b + (int64_t)(row / a.G) * a.g_n + ((head % a.Hkv) * a.G + row % a.G) * a.g_h + d;
  store4<T>(g, x.x * a.factor, x.y * a.factor, x.z * a.factor, x.w * a.factor);
#endif
}

// ---------------------------------------------------------------------------------------------------------- dq
#if defined(__HIP_DEVICE_COMPILE__)
// x = hi + mid + lo exactly, eight bits of the significand each
__device__ __forceinline__ void split3(float x, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffff0000u;
  const float r = x - __uint_as_float(hi);
  mid = __float_as_uint(r) & 0xffff0000u;
  lo = __float_as_uint(r - __uint_as_float(mid)) & 0xffff0000u;
}
// -L / c and -delta as three bf16 each (a row that sees nothing: p = 2^(-1e30) = 0; NaN stays).  The matrix unit multiplies what it does
// not add by zero, so that a delta that is no number would spoil p too: it is left out, as do . v is no number either in such a row.
__device__ __forceinline__ uint4 with_delta(const uint4& stats, float delta) {
  uint32_t d0, d1, d2;
  split3(__builtin_fabsf(delta) < INFINITY ? -delta : 0.f, d0, d1, d2);
  return make_uint4(stats.x, (stats.y & 0xffffu) | d0, (d1 >> 16) | d2, 0);
}
__device__ __forceinline__ uint4 row_stats(float L, float delta, float inv_c) {
  uint32_t l0, l1, l2;
  split3((L > 1e30f ? 1e30f : L) * -inv_c, l0, l1, l2);
  return with_delta(make_uint4((l0 >> 16) | l1, l2 >> 16, 0, 0), delta);
}
#endif

// The forward's shape: columns are query rows, the key tiles pass by (or a split of them).  Also forms delta_i for the dk/dv
// kernel.  -delta is the accumulator that the product do v^T starts from.
// Bound: matrix and vector unit, 43 and 47 % busy, and a barrier a tile between them.  2 x 16 heads of 4096 x 4096: 245 to 265 us
// (780 to 840 TFLOP/s).
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW == 1 || (sizeof(T) == 4 && DP == 128) ? 1 : sizeof(T) == 2 && DP == 64 ? 3 : 2) void attn_dq_kernel(AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using C = AttnCfg<T, DP>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, wave_u = __builtin_amdgcn_readfirstlane(wave);
  int head, blk, split;
  if (!block_coord(a, head, blk, split)) return;
  const int b = head / a.Hkv, hk = head % a.Hkv;
  const T* kb = static_cast<const T*>(a.k) + b * a.in.k_b + hk * a.in.k_h;
  const T* vb = static_cast<const T*>(a.v) + b * a.in.v_b + hk * a.in.v_h;
  const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.Nk : nullptr;
  const int row = blk * (NW * 32) + wave * 32 + (lane & 31);
  const bool row_ok = row < a.rows;
  const int qi = row / a.G, qh = hk * a.G + row % a.G;
  const int64_t lrow = (int64_t)head * a.rows + row;

  const FewKeys<NW> few_keys(sizeof(T) == 2 ? mask : nullptr, a.Nk, tid);
  uint4 qf[C::NKS], gf[C::NKS];  // q and do
  float L = INFINITY, delta = 0.f;
  {
    const T* qp = static_cast<const T*>(a.q) + b * a.in.q_b + (int64_t)qi * a.in.q_n + qh * a.in.q_h;
    const int64_t oo = (((int64_t)b * a.Nq + qi) * (a.Hkv * a.G) + qh) * a.D;
    const T *gp = static_cast<const T*>(a.dout) + oo, *op = static_cast<const T*>(a.o) + oo;
#pragma unroll
    for (int ks = 0; ks < C::NKS; ++ks) {
      const int d = (2 * ks + half) * C::E;
      qf[ks] = gf[ks] = make_uint4(0, 0, 0, 0);
      if (row_ok && d < a.D) {
        qf[ks] = *reinterpret_cast<const uint4*>(qp + d);
        gf[ks] = *reinterpret_cast<const uint4*>(gp + d);
        delta += dot16<T>(gf[ks], *reinterpret_cast<const uint4*>(op + d));
      }
    }
    delta = halves_sum(delta);
    if (row_ok) L = a.lse[lrow];
  }
  const bool few = sizeof(T) == 2 && few_keys(reinterpret_cast<int*>(smem));

  const int ntiles = (a.Nk + C::KT - 1) / C::KT;
  const int t0 = split * a.tiles_per_split, t1 = min(ntiles, t0 + a.tiles_per_split);
  const TileLoader<C, NW> kl(a.in.k_n, a.D, wave, lane), vl(a.in.v_n, a.D, wave, lane);
  const RowReader<C> rows(lane);
  const ColReader<C> cols(lane);
  const KeyBits<C::KT, NW> keys{mask, reinterpret_cast<uint64_t*>(smem + C::NST * C::STAGE), a.Nk, t0, t1, wave, lane};
  auto fetch = [&](int t, uint64_t b) {  // past the last tile: nothing is read
    char* stage = smem + (t - t0) % C::NST * C::STAGE;
    kl.load(kb + (int64_t)t * C::KT * a.in.k_n, stage, wave_u, b);
    vl.load(vb + (int64_t)t * C::KT * a.in.v_n, stage + C::TILE, wave_u, b);
  };
  uint64_t bits = keys.of(t0);
  fetch(t0, bits);
  if constexpr (sizeof(T) == 2) {
    if (few) {  // FewKeys: all of the sample's tiles, whatever the split; this split's first is on its way already
      const KeyBits<C::KT, NW> all{mask, keys.words + kBitTiles, a.Nk, 0, ntiles, wave, lane};
      float sum = 0.f;
      for (int t = 0; t < ntiles; ++t) {
        const uint64_t b = all.of(t);
        if (!b) continue;
        const uint32_t at = t == t0 ? 0 : C::STAGE;
        if (t != t0) {
          __syncthreads();  // the stage's last tile has been read
          kl.load(kb + (int64_t)t * C::KT * a.in.k_n, smem + at, wave_u, b);
          vl.load(vb + (int64_t)t * C::KT * a.in.v_n, smem + at + C::TILE, wave_u, b);
        }
        tile_ready<0>();
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) {
          at_f32x16 s = acc_zero(), dp = acc_zero();
#pragma unroll
          for (int ks = 0; ks < C::NKS; ++ks) {
            s = mma(rows.get(smem, at, j, ks), qf[ks], s, T());
            dp = mma(rows.get(smem, at + C::TILE, j, ks), gf[ks], dp, T());
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -L)) * dp[r];
            sum += (b >> (32 * j + (r & 3) + 8 * (r >> 2) + 4 * half)) & 1 ? x : 0.f;
          }
        }
      }
      delta = halves_sum(sum);
    }
  }
  if (row_ok && half == 0 && split == 0) a.stats[lrow] = row_stats(L, delta, a.inv_c);
  at_f32x16 minus_delta;
#pragma unroll
  for (int r = 0; r < 16; ++r) minus_delta[r] = -delta;
  at_f32x16 dq[C::ND];
#pragma unroll
  for (int i = 0; i < C::ND; ++i) dq[i] = acc_zero();
  for (int t = t0; t < t1; ++t) {
    const uint32_t ks_ = (t - t0) % C::NST * C::STAGE, vs_ = ks_ + C::TILE;
    tile_ready<0>();
    const uint64_t bits_next = keys.of(t + 1);
    fetch(t + 1, bits_next);
    if (bits) {
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) {
        at_f32x16 s = acc_zero(), dp = minus_delta;
#pragma unroll
        for (int ks = 0; ks < C::NKS; ++ks) {
          s = mma(rows.get(smem, ks_, j, ks), qf[ks], s, T());
          dp = mma(rows.get(smem, vs_, j, ks), gf[ks], dp, T());
        }
        ColFrags<T, C> kf;  // read while the matrix unit works
        kf.read(smem, ks_, j, cols, lane);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -L)) * dp[r];
        if (bits != C::kFull) {
          const uint64_t mine = bits >> (4 * half);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!((mine >> (32 * j + (r & 3) + 8 * (r >> 2))) & 1)) s[r] = 0.f;
        }
#pragma unroll
        for (int cc = 0; cc < C::PC; ++cc) {
          const uint4 p = acc_frag(s, cc, T());
#pragma unroll
          for (int i = 0; i < C::ND; ++i) dq[i] = mma(kf.f[cc * C::ND + i], p, dq[i], T());
        }
      }
    }
    bits = bits_next;
  }
  tiles_landed();
  if (!row_ok) return;
  if (a.nsplit > 1) {
    float* p = a.part_a + (((int64_t)head * a.nsplit + split) * a.rows + row) * a.D;
#pragma unroll
    for (int i = 0; i < C::ND; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * i + 8 * g + 4 * half;
        if (d < a.D) store4<float>(p + d, dq[i][4 * g], dq[i][4 * g + 1], dq[i][4 * g + 2], dq[i][4 * g + 3]);
      }
    return;
  }
  T* dqp = static_cast<T*>(a.dq) + b * a.grad.q_b + (int64_t)qi * a.grad.q_n + qh * a.grad.q_h;
#pragma unroll
  for (int i = 0; i < C::ND; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * i + 8 * g + 4 * half;
      if (d < a.D)
        store4<T>(dqp + d, dq[i][4 * g] * a.scale, dq[i][4 * g + 1] * a.scale, dq[i][4 * g + 2] * a.scale, dq[i][4 * g + 3] * a.scale);
    }
#endif
}

// ---------------------------------------------------------------------------------------------------------- dk, dv
// Columns are keys, held in registers; tiles of query rows (head after head of those that share the keys) pass by.
//
// Here L_i and delta_i belong to a row, that is, to a register, the same in 32 lanes.  The products are given -L_i / c and -delta_i on top:
// p = 2^(c acc), ds = p acc'.  These terms are themselves a matrix product: a row's 16 bytes hold both values as three bf16 each
// (exactly, 24 bits), which multiply ones; read as values, four at a time, they would be a third of the loop's LDS traffic.
// A row past the end is all zeros: p = 1 there, and its q and do, which p and ds multiply, are zero.
// Bound: matrix and vector unit, 51 and 44 % busy.  2 x 16 heads of 4096 x 4096: 312 to 339 us (810 to 880 TFLOP/s); three
// waves a SIMD instead of two change nothing.  Few live blocks (3 samples of 0 to 1001 keys, 16 heads on 4, width 128: 78 us; the units
// 23 and 19 % busy) are bound by a tile's way through the CU, 2.2 us.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 4 && DP == 128 ? 1 : 2) void attn_dkv_kernel(AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using C = AttnCfg<T, DP>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* stats = smem + C::NST * C::STAGE;  // [NST][64] of 16 bytes
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, wave_u = __builtin_amdgcn_readfirstlane(wave);
  int head, blk, split;
  if (!block_coord(a, head, blk, split)) return;
  const int b = head / a.Hkv, hk = head % a.Hkv;
  const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.Nk : nullptr;
  const int key = blk * (NW * 32) + wave * 32 + (lane & 31);
  const bool key_ok = key < a.Nk, see = key_ok && (!mask || mask[key] != 0);
  const int64_t o_n = (int64_t)a.Hkv * a.G * a.D;
  const T* qb = static_cast<const T*>(a.q) + b * a.in.q_b + (int64_t)hk * a.G * a.in.q_h;
  const T* gb = static_cast<const T*>(a.dout) + (int64_t)b * a.Nq * o_n + (int64_t)hk * a.G * a.D;

  uint4 kf[C::NKS], vf[C::NKS];
  {
    const T* kp = static_cast<const T*>(a.k) + b * a.in.k_b + hk * a.in.k_h + (int64_t)key * a.in.k_n;
    const T* vp = static_cast<const T*>(a.v) + b * a.in.v_b + hk * a.in.v_h + (int64_t)key * a.in.v_n;
#pragma unroll
    for (int ks = 0; ks < C::NKS; ++ks) {
      const int d = (2 * ks + half) * C::E;
      kf[ks] = vf[ks] = make_uint4(0, 0, 0, 0);
      if (see && d < a.D) {
        kf[ks] = *reinterpret_cast<const uint4*>(kp + d);
        vf[ks] = *reinterpret_cast<const uint4*>(vp + d);
      }
    }
  }
  at_f32x16 dk[C::ND], dv[C::ND];
#pragma unroll
  for (int i = 0; i < C::ND; ++i) dk[i] = dv[i] = acc_zero();
  // ones (bf16 0x3f80) against the three parts of -L / c, and of -delta
  const uint4 one_L = half ? make_uint4(0, 0, 0, 0) : make_uint4(0x3f803f80u, 0x00003f80u, 0, 0);
  const uint4 one_d = half ? make_uint4(0, 0, 0, 0) : make_uint4(0, 0x3f800000u, 0x3f803f80u, 0);

  const bool wave_sees = __any(see);
  const int tq = (a.Nq + C::KT - 1) / C::KT;
  // a block without a visible key has nothing to add up (the same decision in all its waves)
  const int t0 = split * a.tiles_per_split, t1 = __syncthreads_or(see) ? min(tq * a.G, t0 + a.tiles_per_split) : t0;
  const TileLoader<C, NW> ql(a.in.q_n, a.D, wave, lane), gl(o_n, a.D, wave, lane);
  const RowReader<C> rows(lane);
  const ColReader<C> cols(lane);
  // tile t: head t / tq of the group, rows from (t % tq) KT on; past the last one nothing is read
  auto fetch = [&](int t) {
    const int g = t < t1 ? t / tq : 0, r0 = t < t1 ? (t - g * tq) * C::KT : 0, n = t < t1 ? a.Nq - r0 : 0;
    const uint64_t bits = n >= C::KT ? C::kFull : (1ull << n) - 1;
    const int slot = (t - t0) % C::NST;
    char* stage = smem + slot * C::STAGE;
    if (wave_u == 0) {
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(a.stats + (int64_t)head * a.rows + (int64_t)r0 * a.G + g, 0, kReach, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(stats + slot * 1024), 16,
                                               lane < n && lane < C::KT ? (uint32_t)lane * a.G * 16 : kNowhere, 0, 0, 0);
    }
    ql.load(qb + g * a.in.q_h + r0 * a.in.q_n, stage, wave_u, bits);
    gl.load(gb + (int64_t)g * a.D + r0 * o_n, stage + C::TILE, wave_u, bits);
  };
#pragma unroll
  for (int i = 0; i < C::NST - 1; ++i) fetch(t0 + i);
  for (int t = t0; t < t1; ++t) {
    const uint32_t qs_ = (t - t0) % C::NST * C::STAGE, gs_ = qs_ + C::TILE;
    const char* st_ = stats + (t - t0) % C::NST * 1024;
    tile_ready<2 * TileLoader<C, NW>::N * (C::NST - 2)>();  // (wave 0 has one transfer more a tile, ahead of the others)
    fetch(t + C::NST - 1);
    if (wave_sees) {
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) {
        const uint4 both = lds16(st_ + (32 * j + (lane & 31)) * 16);
        at_f32x16 s = acc_zero(), dp = acc_zero();
        if constexpr (sizeof(T) == 2 && DP == 128) {  // one after the other, a pair of column blocks at a time: all at once spills
#pragma unroll
          for (int ks = 0; ks < C::NKS; ++ks) s = mma(rows.get(smem, qs_, j, ks), kf[ks], s, T());
          s = mma(both, one_L, s, bf16_t());
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] * a.c);
          uint4 x[2] = {acc_frag(s, 0, T()), acc_frag(s, 1, T())}, f[4];
#pragma unroll
          for (int i = 0; i < C::ND; ++i) {
            if (i % 2 == 0) ColFrags<T, C>::read_pair(smem, gs_, j, i / 2, cols, f);
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) dv[i] = mma(f[2 * cc + i % 2], x[cc], dv[i], T());
          }
#pragma unroll
          for (int ks = 0; ks < C::NKS; ++ks) dp = mma(rows.get(smem, gs_, j, ks), vf[ks], dp, T());
          dp = mma(both, one_d, dp, bf16_t());
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] *= s[r];
          x[0] = acc_frag(dp, 0, T());
          x[1] = acc_frag(dp, 1, T());
#pragma unroll
          for (int i = 0; i < C::ND; ++i) {
            if (i % 2 == 0) ColFrags<T, C>::read_pair(smem, qs_, j, i / 2, cols, f);
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) dk[i] = mma(f[2 * cc + i % 2], x[cc], dk[i], T());
          }
          continue;
        }
#pragma unroll
        for (int ks = 0; ks < C::NKS; ++ks) {
          s = mma(rows.get(smem, qs_, j, ks), kf[ks], s, T());
          dp = mma(rows.get(smem, gs_, j, ks), vf[ks], dp, T());
        }
        s = mma(both, one_L, s, bf16_t());  // last: L / c is large, and every term added to it would be rounded at its size
        dp = mma(both, one_d, dp, bf16_t());
        ColFrags<T, C> f;  // of do, read while the matrix unit works
        f.read(smem, gs_, j, cols, lane);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = __builtin_amdgcn_exp2f(s[r] * a.c);
          dp[r] *= s[r];
        }
#pragma unroll
        for (int cc = 0; cc < C::PC; ++cc) {
          const uint4 p = acc_frag(s, cc, T());
#pragma unroll
          for (int i = 0; i < C::ND; ++i) dv[i] = mma(f.f[cc * C::ND + i], p, dv[i], T());
        }
        f.read(smem, qs_, j, cols, lane);
#pragma unroll
        for (int cc = 0; cc < C::PC; ++cc) {
          const uint4 ds = acc_frag(dp, cc, T());
#pragma unroll
          for (int i = 0; i < C::ND; ++i) dk[i] = mma(f.f[cc * C::ND + i], ds, dk[i], T());
        }
      }
    }
  }
  tiles_landed();
  if (!key_ok) return;
  // a column's sums are its own: a masked key's are dropped here
  if (a.nsplit > 1) {
    const int64_t at = (((int64_t)head * a.nsplit + split) * a.Nk + key) * a.D;
#pragma unroll
    for (int i = 0; i < C::ND; ++i)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        const int d = 32 * i + 8 * gq + 4 * half;
        float x[4], y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[r] = see ? dk[i][4 * gq + r] : 0.f;
          y[r] = see ? dv[i][4 * gq + r] : 0.f;
        }
        if (d < a.D) {
          store4<float>(a.part_a + at + d, x[0], x[1], x[2], x[3]);
          store4<float>(a.part_b + at + d, y[0], y[1], y[2], y[3]);
        }
      }
    return;
  }
  T* dkp = static_cast<T*>(a.dk) + b * a.grad.k_b + hk * a.grad.k_h + (int64_t)key * a.grad.k_n;
  T* dvp = static_cast<T*>(a.dv) + b * a.grad.v_b + hk * a.grad.v_h + (int64_t)key * a.grad.v_n;
#pragma unroll
  for (int i = 0; i < C::ND; ++i)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const int d = 32 * i + 8 * gq + 4 * half;
      float x[4], y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = see ? dk[i][4 * gq + r] * a.scale : 0.f;
        y[r] = see ? dv[i][4 * gq + r] : 0.f;
      }
      if (d < a.D) {
        store4<T>(dkp + d, x[0], x[1], x[2], x[3]);
        store4<T>(dvp + d, y[0], y[1], y[2], y[3]);
      }
    }
#endif
}

// ---------------------------------------------------------------------------------------------------------- whole backward
// Up to 256 keys of up to 64 columns, bf16: a workgroup of 8 waves holds a head's keys and values, 32 keys a wave, and has all of
// a query row's scores at hand, so that dq is finished here too: 5 products instead of 7, one exponential instead of two, every
// operand read once.  ds is exchanged between the waves through LDS as [key][64 rows]; a wave then multiplies one 32 x 32 block of
// dq^T = k^T ds^T over half of the keys, and the two halves are added in a fixed order.  delta is formed from do and o by the
// threads that a tile's rows are dealt to, one tile ahead.
// Bound: latency.  64 x 12 heads of 237 x 237 take 82 us, the matrix unit is busy for 19 % of it, the vector unit for 27: with 116 KiB
// and 243 registers a CU holds one workgroup, and a head costs 11 k cycles before its first tile, then four times 7 k between two
// barriers each.  A sample of few visible keys (FewKeys) takes three more barriers a tile: 87 us instead of 70 if all see 40 keys.
__global__ __launch_bounds__(512) void attn_bwd_whole_kernel(AttnArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef bf16_t T;
  using C = AttnCfg<T, 64>;
  constexpr int NW = 8, KEYS = NW * 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr uint32_t kKeys = 0, kRing = KEYS * 128, kDs = kRing + 2 * C::STAGE, kHalf = kDs + KEYS * 128, kStats = kHalf + 4 * 4096, kDelta = kStats + 2 * 1024;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, wave_u = __builtin_amdgcn_readfirstlane(wave);
  int head, blk, split;
  if (!block_coord(a, head, blk, split)) return;
  const int b = head / a.Hkv, hk = head % a.Hkv;
  const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.Nk : nullptr;
  const int key = wave * 32 + (lane & 31);
  const bool key_ok = key < a.Nk;
  const int64_t o_n = (int64_t)a.Hkv * a.G * a.D;
  const T* qb = static_cast<const T*>(a.q) + b * a.in.q_b + (int64_t)hk * a.G * a.in.q_h;
  const T* gb = static_cast<const T*>(a.dout) + (int64_t)b * a.Nq * o_n + (int64_t)hk * a.G * a.D;
  const T* ob = static_cast<const T*>(a.o) + (int64_t)b * a.Nq * o_n + (int64_t)hk * a.G * a.D;
  const int tq = (a.Nq + C::KT - 1) / C::KT, nt = tq * a.G;
  const uint8_t mine = !key_ok ? 0 : mask ? mask[key] : 1;
  const TileLoader<C, NW> ql(a.in.q_n, a.D, wave, lane), gl(o_n, a.D, wave, lane), kl(a.in.k_n, a.D, wave, lane);
  const RowReader<C> rows(lane);
  const ColReader<C> cols(lane);

  auto fetch = [&](int t) {  // past the last tile: nothing is read
    const int g = t < nt ? t / tq : 0, r0 = t < nt ? (t - g * tq) * C::KT : 0, n = t < nt ? a.Nq - r0 : 0;
    const uint64_t bits = n >= C::KT ? C::kFull : (1ull << n) - 1;
    char* stage = smem + kRing + (t & 1) * C::STAGE;
    ql.load(qb + g * a.in.q_h + r0 * a.in.q_n, stage, wave_u, bits);
    gl.load(gb + (int64_t)g * a.D + r0 * o_n, stage + C::TILE, wave_u, bits);
  };
  // thread -> row tid / 8 of a tile, chunk tid % 8 of do and o
  const uint32_t st_off = (tid & 7) * 8 < a.D ? (uint32_t)(tid >> 3) * ((uint32_t)o_n * 2) + (tid & 7) * 16 : kNowhere;
  at_u32x4 st_g, st_o;
  float st_L;
  auto stats_request = [&](int t) {
    const int g = t < nt ? t / tq : 0, r0 = t < nt ? (t - g * tq) * C::KT : 0, n = t < nt ? a.Nq - r0 : 0;
    const bool in = (tid >> 3) < n;
    const int64_t at = (int64_t)g * a.D + r0 * o_n;
    const __amdgpu_buffer_rsrc_t rg = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(gb + at), 0, kReach, 0x00020000);
    const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(ob + at), 0, kReach, 0x00020000);
    const __amdgpu_buffer_rsrc_t rl = __builtin_amdgcn_make_buffer_rsrc(a.lse + (int64_t)head * a.rows + (int64_t)r0 * a.G + g, 0, kReach, 0x00020000);
    st_g = __builtin_amdgcn_raw_buffer_load_b128(rg, in ? st_off : kNowhere, 0, 0);
    st_o = __builtin_amdgcn_raw_buffer_load_b128(ro, in ? st_off : kNowhere, 0, 0);
    st_L = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rl, in ? (uint32_t)(tid >> 3) * a.G * 4 : kNowhere, 0, 0));
  };
  auto stats_store = [&](int t) {
    float delta = dot16<T>(__builtin_bit_cast(uint4, st_g), __builtin_bit_cast(uint4, st_o));
    auto from = [&](auto pattern) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(delta), decltype(pattern)::value, 0xf, 0xf, true)); };
    delta += from(std::integral_constant<int, 0xb1>());   // lane ^ 1
    delta += from(std::integral_constant<int, 0x4e>());   // lane ^ 2
    delta += from(std::integral_constant<int, 0x141>());  // 7 - lane of the eight
    if ((tid & 7) == 0) *reinterpret_cast<uint4*>(smem + kStats + (t & 1) * 1024 + (tid >> 3) * 16) = row_stats(st_L, delta, a.inv_c);
  };

  stats_request(0);
  fetch(0);
  {  // the keys that dq multiplies, 64 of them in a step
    const T* kb = static_cast<const T*>(a.k) + b * a.in.k_b + hk * a.in.k_h;
#pragma unroll
    for (int i = 0; i < KEYS / C::KT; ++i) {
      const int n = a.Nk - i * C::KT;
      kl.load(kb + (int64_t)i * C::KT * a.in.k_n, smem + kKeys + i * C::TILE, wave_u, n >= C::KT ? C::kFull : n > 0 ? (1ull << n) - 1 : 0);
    }
  }
  uint4 kf[C::NKS], vf[C::NKS];
  {
    const T* kp = static_cast<const T*>(a.k) + b * a.in.k_b + hk * a.in.k_h + (int64_t)key * a.in.k_n;
    const T* vp = static_cast<const T*>(a.v) + b * a.in.v_b + hk * a.in.v_h + (int64_t)key * a.in.v_n;
#pragma unroll
    for (int ks = 0; ks < C::NKS; ++ks) {
      const int d = (2 * ks + half) * C::E;
      kf[ks] = vf[ks] = make_uint4(0, 0, 0, 0);
      if (key_ok && d < a.D) {
        kf[ks] = *reinterpret_cast<const uint4*>(kp + d);
        vf[ks] = *reinterpret_cast<const uint4*>(vp + d);
      }
    }
  }
  const bool see = mine != 0, wave_sees = __any(see), wave_full = __all(see);
  if (!wave_sees) {  // its part of ds stays zero
    for (int i = lane; i < 32 * 8; i += 64) *reinterpret_cast<uint4*>(smem + kDs + wave * 4096 + i * 16) = make_uint4(0, 0, 0, 0);
  }
  float* part_delta = reinterpret_cast<float*>(smem + kDelta) + wave * 64;  // [wave][64 rows]; before the first tile: the wave's visible keys
  const uint32_t wave_bits = (uint32_t)__ballot(see);  // (the other half holds the same keys)
  if (lane == 0) *part_delta = (float)__popc(wave_bits);
  at_f32x16 dk[2], dv[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) dk[i] = dv[i] = acc_zero();
  const uint4 one_L = half ? make_uint4(0, 0, 0, 0) : make_uint4(0x3f803f80u, 0x00003f80u, 0, 0);
  const uint4 one_d = half ? make_uint4(0, 0, 0, 0) : make_uint4(0, 0x3f800000u, 0x3f803f80u, 0);
  stats_store(0);
  stats_request(1);
  lds_exchange();
  int seen = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) seen += (int)reinterpret_cast<const float*>(smem + kDelta)[w * 64];
  seen = __builtin_amdgcn_readfirstlane(seen);

  const int qblk = wave & 1, dblk = (wave >> 1) & 1, upper = wave_u >> 2;  // my block of dq^T, my half of the keys
  char* ds_at = smem + kDs + key * 128 + half * 8;
  const int ds_swz = C::swizzle(key);
  char* part = smem + kHalf + (wave & 3) * 4096 + lane * 16;
  at_f32x16 dq = acc_zero();
  auto dq_store = [&](int t) {  // tile t: the upper half's part was written before the last barrier
    const int g = t / tq, row = (t - g * tq) * C::KT + 32 * qblk + (lane & 31);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const at_f32x4 x = *reinterpret_cast<const at_f32x4*>(part + i * 1024);
#pragma unroll
      for (int r = 0; r < 4; ++r) dq[4 * i + r] += x[r];
    }
    if (row < a.Nq) {
      T* p = static_cast<T*>(a.dq) + b * a.grad.q_b + (int64_t)row * a.grad.q_n + (hk * a.G + g) * a.grad.q_h;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * dblk + 8 * i + 4 * half;
        if (d < a.D) store4<T>(p + d, dq[4 * i] * a.scale, dq[4 * i + 1] * a.scale, dq[4 * i + 2] * a.scale, dq[4 * i + 3] * a.scale);
      }
    }
  };
  auto tile = [&](int t, auto few) __attribute__((always_inline)) {
    const uint32_t qs_ = kRing + (t & 1) * C::STAGE, gs_ = qs_ + C::TILE;
    const char* st_ = smem + kStats + (t & 1) * 1024;
    tile_ready<0>();
    fetch(t + 1);
    if (t == 0 && !see) {  // a masked key, which may hold anything: its ds is zero
#pragma unroll
      for (int c = 0; c < 4; ++c) *reinterpret_cast<at_u32x4*>(smem + kKeys + key * C::RB + half * 64 + c * 16) = at_u32x4{0, 0, 0, 0};
    }
    if constexpr (decltype(few)::value) {  // FewKeys: delta of the tile's rows as sum p dp; operands swapped, so that a row is a lane and its keys are registers
      if (wave_sees) {
        const uint32_t bits = wave_bits >> (4 * half);
#pragma unroll 1
        for (int j = 0; j < 2; ++j) {
          const uint4 both = lds16(st_ + (32 * j + (lane & 31)) * 16);
          at_f32x16 s = acc_zero(), dp = acc_zero();
#pragma unroll
          for (int ks = 0; ks < C::NKS; ++ks) {
            s = mma(kf[ks], rows.get(smem, qs_, j, ks), s, T());
            dp = mma(vf[ks], rows.get(smem, gs_, j, ks), dp, T());
          }
          s = mma(one_L, both, s, T());
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float x = __builtin_amdgcn_exp2f(s[r] * a.c) * dp[r];
            sum += (bits >> ((r & 3) + 8 * (r >> 2))) & 1 ? x : 0.f;
          }
          sum = halves_sum(sum);
          if (half == 0) part_delta[32 * j + lane] = sum;
        }
      } else {
        part_delta[lane] = 0.f;
      }
      lds_exchange();
      if (tid < 64) {
        float delta = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) delta += reinterpret_cast<const float*>(smem + kDelta)[w * 64 + tid];
        uint4* st = reinterpret_cast<uint4*>(smem + kStats + (t & 1) * 1024) + tid;
        *st = with_delta(*st, delta);
      }
      lds_exchange();
    }
    stats_store(t + 1);
    stats_request(t + 2);
    if (t > 0 && !upper) dq_store(t - 1);
    if (wave_sees) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint4 both = lds16(st_ + (32 * j + (lane & 31)) * 16);
        at_f32x16 s = acc_zero(), dp = acc_zero();
#pragma unroll
        for (int ks = 0; ks < C::NKS; ++ks) {
          s = mma(rows.get(smem, qs_, j, ks), kf[ks], s, T());
          dp = mma(rows.get(smem, gs_, j, ks), vf[ks], dp, T());
        }
        s = mma(both, one_L, s, T());  // last, as in attn_dkv_kernel
        dp = mma(both, one_d, dp, T());
        ColFrags<T, C> f;  // of do, read while the matrix unit works
        f.read(smem, gs_, j, cols, lane);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = __builtin_amdgcn_exp2f(s[r] * a.c);
          dp[r] *= s[r];
        }
        if (!wave_full) {
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] = see ? dp[r] : 0.f;
        }
        uint4 ds[2];
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          ds[cc] = acc_frag(dp, cc, T());
          const uint4 p = acc_frag(s, cc, T());
          // rows 32 j + 8 (2 cc) + 4 half + {0..3}, and 8 on: half a chunk each
          *reinterpret_cast<at_u32x2*>(ds_at + (((4 * j + 2 * cc) ^ ds_swz) << 4)) = at_u32x2{ds[cc].x, ds[cc].y};
          *reinterpret_cast<at_u32x2*>(ds_at + (((4 * j + 2 * cc + 1) ^ ds_swz) << 4)) = at_u32x2{ds[cc].z, ds[cc].w};
#pragma unroll
          for (int i = 0; i < 2; ++i) dv[i] = mma(f.f[cc * 2 + i], p, dv[i], T());
        }
        f.read(smem, qs_, j, cols, lane);
#pragma unroll
        for (int cc = 0; cc < 2; ++cc)
#pragma unroll
          for (int i = 0; i < 2; ++i) dk[i] = mma(f.f[cc * 2 + i], ds[cc], dk[i], T());
      }
    }
    lds_exchange();  // ds is whole
    dq = acc_zero();
    const uint32_t ka = kKeys + upper * (KEYS / 2 * 128) + (cols.base[0] ^ (dblk << 6));
    const uint32_t da = kDs + upper * (KEYS / 2 * 128) + (cols.base[0] ^ (qblk << 6));
#pragma unroll
    for (int i = 0; i < KEYS / 64; ++i) {
      uint4 f[4];  // 32 keys: of the keys' block, of ds, twice
      tr_frags4<C>(smem, ka + i * 4096, da + i * 4096, f);
      dq = mma(f[0], f[1], dq, T());
      dq = mma(f[2], f[3], dq, T());
    }
    if (upper) {
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<at_f32x4*>(part + i * 1024) = at_f32x4{dq[4 * i], dq[4 * i + 1], dq[4 * i + 2], dq[4 * i + 3]};
    }
  };
  if (seen <= kFewKeys) {
    for (int t = 0; t < nt; ++t) tile(t, std::true_type());
  } else {
    for (int t = 0; t < nt; ++t) tile(t, std::false_type());
  }
  tile_ready<0>();
  if (nt > 0 && !upper) dq_store(nt - 1);
  if (!key_ok) return;
  T* dkp = static_cast<T*>(a.dk) + b * a.grad.k_b + hk * a.grad.k_h + (int64_t)key * a.grad.k_n;
  T* dvp = static_cast<T*>(a.dv) + b * a.grad.v_b + hk * a.grad.v_h + (int64_t)key * a.grad.v_n;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const int d = 32 * i + 8 * gq + 4 * half;
      float x[4], y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {  // a column's sums are its own: a masked key's are dropped here
        x[r] = see ? dk[i][4 * gq + r] * a.scale : 0.f;
        y[r] = see ? dv[i][4 * gq + r] : 0.f;
      }
      if (d < a.D) {
        store4<T>(dkp + d, x[0], x[1], x[2], x[3]);
        store4<T>(dvp + d, y[0], y[1], y[2], y[3]);
      }
    }
#endif
}
constexpr int kWholeLds = 256 * 128 + 2 * AttnCfg<bf16_t, 64>::STAGE + 256 * 128 + 4 * 4096 + 2 * 1024 + 8 * 256;

// ---------------------------------------------------------------------------------------------------------- host
namespace {

int attn_cus() {
  static thread_local int cached_dev = -1, cached = 0;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  if (dev != cached_dev) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cached = n;
    cached_dev = dev;
  }
  return cached;
}

// How a kernel's rows (or keys) are cut into blocks, and the tiles that pass by them into splits.
struct AttnPlan { int nw, nblk, tiles_per_split, nsplit; };

// A split has four tiles at least.  Fewer would win where the whole launch is small and long (12 heads, one query, 1000 keys: 11.0 us, 8.1
// with one tile; float32 6 heads, 129 on 333: 25 us, 19 with two) and lose where the join costs as much as a tile (12 heads of 237 x 237:
// 8.0 us, 11.8 with two; 2 x 12 heads of 617, backward: 44 us, 48 with two, 39 with eight).
AttnPlan plan_of(int64_t rows, int nw, int64_t heads, int64_t tiles, int64_t want_blocks, int64_t least_tiles) {
  AttnPlan p;
  p.nw = nw;
  p.nblk = (int)((rows + nw * 32 - 1) / (nw * 32));
  const int64_t blocks = heads * p.nblk;
  int64_t split = blocks > 0 ? want_blocks / blocks : 1;
  if (split > tiles / least_tiles) split = tiles / least_tiles;
  if (split > kMaxSplit) split = kMaxSplit;
  if (split < 1) split = 1;
  p.tiles_per_split = (int)((tiles + split - 1) / split);
  if (p.tiles_per_split < 1) p.tiles_per_split = 1;
  p.nsplit = tiles > 0 ? (int)((tiles + p.tiles_per_split - 1) / p.tiles_per_split) : 1;
  return p;
}

int64_t q_rows(const eve_attn_shape& s) { return (int64_t)s.Nq * (s.H / s.Hkv); }
int tile_rows(const eve_attn_shape& s) { return s.dtype == EVE_BF16 && s.D <= 64 ? 64 : 32; }
int64_t tiles_of(int n, int rows) { return ((int64_t)n + rows - 1) / rows; }

// Few rows against many keys: the key tiles are split until the launch fills the CUs, and the parts are joined.  Up to 64 rows a
// head go to blocks of one wave, of which three fit a CU.
AttnPlan fwd_plan(const eve_attn_shape& s, int cus) {
  const int nw = q_rows(s) <= 64 ? 1 : 4;
  const int kt = nw == 4 && s.dtype == EVE_BF16 ? 64 : tile_rows(s);  // FwdCfg
  return plan_of(q_rows(s), nw, (int64_t)s.B * s.Hkv, tiles_of(s.Nk, kt), (int64_t)cus * (nw == 4 ? 2 : 3), 4);
}
AttnPlan dq_plan(const eve_attn_shape& s, int cus) {
  const int nw = q_rows(s) <= 64 ? 1 : 4;
  return plan_of(q_rows(s), nw, (int64_t)s.B * s.Hkv, tiles_of(s.Nk, tile_rows(s)), (int64_t)cus * (nw == 4 ? 2 : 3), 4);
}
// The row tiles are counted head by head of a group, as the kernel walks them.
AttnPlan dkv_plan(const eve_attn_shape& s, int cus) {
  return plan_of(s.Nk, 4, (int64_t)s.B * s.Hkv, tiles_of(s.Nq, tile_rows(s)) * (s.H / s.Hkv), (int64_t)cus * 2, 4);
}

// The backward of whole heads, a workgroup each: where there is one for every other CU at least and their waves have keys.  Times in us
// of both ways, unmasked, width 64, heads x keys (whole | two kernels):
//   32 x 237   20.7 | 21.0    128 x 237  23.2 | 24.3    256 x 237  27.6 | 35.1    768 x 237  75.3 | 92.4
//   32 x 129   15.8 | 18.2    128 x 129  17.0 | 19.4    256 x 129  18.6 | 27.8    768 x 129  53.8 | 72.0
//   32 x 64    15.4 | 11.9    128 x 100  12.7 | 15.9    256 x 100  13.9 | 17.6    768 x 100  39.3 | 38.9
// (On fewer heads than cus / 2 it gains little.)
bool whole_heads(const eve_attn_shape& s, int cus) {
  return s.dtype == EVE_BF16 && s.D <= 64 && s.Nk > 128 && s.Nk <= 256 && (int64_t)s.B * s.Hkv >= cus / 2;
}

size_t fwd_ws(const eve_attn_shape& s, const AttnPlan& p) {
  if (p.nsplit == 1) return 0;
  const size_t rows = (size_t)s.B * s.Hkv * p.nsplit * q_rows(s);
  return align_up(rows * s.D * 4, 256) + align_up(rows * 8, 256);
}
// the rows' statistics, then the parts of dq, and in their place afterwards those of dk and dv
struct BwdWs { size_t stats, part, dv, bytes; };
BwdWs bwd_ws(const eve_attn_shape& s, const AttnPlan& pq, const AttnPlan& pk) {
  BwdWs w;
  const size_t heads = (size_t)s.B * s.Hkv;
  w.stats = 0;
  w.part = align_up(heads * q_rows(s) * 16, 256);
  const size_t dq = pq.nsplit > 1 ? align_up(heads * pq.nsplit * q_rows(s) * s.D * 4, 256) : 0;
  const size_t dk = pk.nsplit > 1 ? align_up(heads * pk.nsplit * s.Nk * s.D * 4, 256) : 0;
  w.dv = w.part + dk;
  w.bytes = w.part + (dq > 2 * dk ? dq : 2 * dk);
  return w;
}

constexpr float kLeastScale = 0x1p-100f;

int check_shape(const eve_attn_shape* s) {
  EVE_REQUIRE(s, EVE_ERR_ARG, "eve_attn: null shape");
  EVE_REQUIRE(s->dtype == EVE_F32 || s->dtype == EVE_BF16, EVE_ERR_ARG, "eve_attn: dtype %d", s->dtype);
  EVE_REQUIRE(s->B >= 0 && s->Nq >= 0 && s->Nk >= 0, EVE_ERR_ARG, "eve_attn: negative size");
  EVE_REQUIRE(s->H >= 1 && s->Hkv >= 1 && s->H % s->Hkv == 0, EVE_ERR_ARG, "eve_attn: %d query heads do not share %d key heads", s->H, s->Hkv);
  EVE_REQUIRE((int64_t)s->H * s->D <= (1 << 22), EVE_ERR_UNSUPPORTED, "eve_attn: %d heads of %d", s->H, s->D);
  EVE_REQUIRE(s->D >= 8 && s->D <= 128 && s->D % 8 == 0, EVE_ERR_UNSUPPORTED, "eve_attn: head width %d (a multiple of 8 up to 128)", s->D);
  // the backward works with L / c, c = scale log2 e: both it and 1 / c have to be normal numbers of 32 bits
  EVE_REQUIRE(s->scale >= kLeastScale && s->scale <= 1.f / kLeastScale, EVE_ERR_ARG, "eve_attn: scale must lie between 2^-100 and 2^100");
  EVE_REQUIRE((int64_t)s->Nq * (s->H / s->Hkv) <= 0x7fff0000LL && s->Nk <= 0x7fff0000, EVE_ERR_UNSUPPORTED, "eve_attn: too many rows");
  EVE_REQUIRE((int64_t)s->B * s->Hkv <= 0x7fff0000LL && (int64_t)s->B * s->Nq <= 0x7fff0000LL, EVE_ERR_UNSUPPORTED, "eve_attn: batch too large");
  return EVE_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_layout(const eve_attn_layout* l, int dtype, const char* what) {
  EVE_REQUIRE(l, EVE_ERR_ARG, "eve_attn: null %s layout", what);
  const int64_t e = dtype == EVE_BF16 ? 8 : 4;
  const int64_t st[9] = {l->q_b, l->q_n, l->q_h, l->k_b, l->k_n, l->k_h, l->v_b, l->v_n, l->v_h};
  for (int64_t x : st) EVE_REQUIRE(x >= 0 && x % e == 0, EVE_ERR_ARG, "eve_attn: %s strides must be multiples of 16 bytes", what);
  // a tile of 64 rows is reached by 32-bit offsets from its first row (64-bit from tile to tile)
  for (int i = 1; i < 9; i += 3)
    EVE_REQUIRE(st[i] <= (1 << 22), EVE_ERR_UNSUPPORTED, "eve_attn: %s rows more than 2^22 elements apart", what);
  return EVE_OK;
}

AttnArgs base_args(const eve_attn_shape& s) {
  AttnArgs a = {};
  a.Nq = s.Nq; a.Nk = s.Nk; a.Hkv = s.Hkv; a.G = s.H / s.Hkv; a.D = s.D;
  a.rows = s.Nq * a.G;
  a.heads = s.B * s.Hkv;
  a.nsplit = 1;
  a.scale = s.scale;
  a.c = (float)((double)s.scale * 1.4426950408889634);
  a.inv_c = (float)(1.0 / ((double)s.scale * 1.4426950408889634));
  return a;
}

// the ring, and behind it the mask's words or the rows' statistics
template <typename C> constexpr int attn_lds() { return C::NST * C::STAGE + kBitTiles * 8; }
template <typename C> constexpr int dq_lds() { return attn_lds<C>() + kBitTiles * 8; }  // and the words of the pass for delta
template <typename T, int DP> constexpr int dkv_lds() { return AttnCfg<T, DP>::NST * (AttnCfg<T, DP>::STAGE + 1024); }

int launch_attn(void (*kern)(AttnArgs), AttnArgs& a, int nw, int lds, hipStream_t st, const char* name) {
  const int64_t per = (int64_t)a.nblk * a.nsplit;
  a.by_xcd = a.heads % 8 == 0 || a.heads >= 64;
  const int64_t grid = (a.by_xcd ? ((int64_t)a.heads + 7) / 8 * 8 : a.heads) * per;
  EVE_REQUIRE(grid <= kMaxThreads / (nw * 64) && per <= 0x7fffffffLL, EVE_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    EVE_REQUIRE(e == hipSuccess, EVE_ERR_LAUNCH, "%s: %d bytes of LDS: %s", name, lds, hipGetErrorString(e));
  }
  kern<<<dim3((unsigned)grid), dim3(nw * 64), lds, st>>>(a);
  EVE_CHECK_LAUNCH(name);
  return EVE_OK;
}

void use_plan(AttnArgs& a, const AttnPlan& p) {
  a.nblk = p.nblk;
  a.nsplit = p.nsplit;
  a.tiles_per_split = p.tiles_per_split;
}

template <typename T, int DP>
int fwd_typed(AttnArgs& a, const AttnPlan& p, hipStream_t st) {
  use_plan(a, p);
  const int rc = launch_attn(p.nw == 1 ? attn_fwd_kernel<T, DP, 1> : attn_fwd_kernel<T, DP, 4>, a, p.nw,
                             p.nw == 1 ? attn_lds<FwdCfg<T, DP, 1>>() : attn_lds<FwdCfg<T, DP, 4>>(), st, "eve_attn_fwd");
  if (rc != EVE_OK || a.nsplit == 1) return rc;
  EVE_REQUIRE((int64_t)a.heads * a.rows <= kMaxThreads / 256, EVE_ERR_UNSUPPORTED, "eve_attn_fwd: too many rows");
  attn_join_kernel<T><<<dim3((unsigned)(a.heads * a.rows)), dim3(256), 0, st>>>(a);
  EVE_CHECK_LAUNCH("eve_attn_fwd (join)");
  return EVE_OK;
}

AttnSum sum_of(const AttnArgs& a, const float* part, void* g, int64_t g_b, int64_t g_n, int64_t g_h, int G, int rows, float factor) {
  return {part, g, g_b, g_n, g_h, (int64_t)a.heads * rows * (a.D / 4), a.Hkv, G, a.D, rows, a.nsplit, factor};
}
template <typename T>
int sum_parts(const AttnSums& s, int n, hipStream_t st) {  // n of one size
  const int64_t grid = (s.s[0].total + 255) / 256;
  EVE_REQUIRE(grid <= kMaxThreads / 256, EVE_ERR_UNSUPPORTED, "eve_attn_bwd: too many rows");
  attn_sum_kernel<T><<<dim3((unsigned)grid, n), dim3(256), 0, st>>>(s);
  EVE_CHECK_LAUNCH("eve_attn_bwd (sum of the splits)");
  return EVE_OK;
}

template <typename T, int DP>
int bwd_typed(AttnArgs& a, bool whole, const AttnPlan& pq, const AttnPlan& pk, hipStream_t st) {
  if constexpr (sizeof(T) == 2 && DP == 64) {
    if (whole) {
      a.nblk = 1;
      return launch_attn(attn_bwd_whole_kernel, a, 8, kWholeLds, st, "eve_attn_bwd");
    }
  }
  if (a.rows > 0) {
    use_plan(a, pq);
    int rc = launch_attn(pq.nw == 1 ? attn_dq_kernel<T, DP, 1> : attn_dq_kernel<T, DP, 4>, a, pq.nw, dq_lds<AttnCfg<T, DP>>(), st, "eve_attn_bwd (dq)");
    if (rc == EVE_OK && a.nsplit > 1)
      rc = sum_parts<T>({{sum_of(a, a.part_a, a.dq, a.grad.q_b, a.grad.q_n, a.grad.q_h, a.G, a.rows, a.scale)}}, 1, st);
    if (rc != EVE_OK) return rc;
  }
  if (a.Nk == 0) return EVE_OK;
  use_plan(a, pk);
  int rc = launch_attn(attn_dkv_kernel<T, DP, 4>, a, pk.nw, dkv_lds<T, DP>(), st, "eve_attn_bwd (dk, dv)");
  if (rc == EVE_OK && a.nsplit > 1)
    rc = sum_parts<T>({{sum_of(a, a.part_a, a.dk, a.grad.k_b, a.grad.k_n, a.grad.k_h, 1, a.Nk, a.scale),
                        sum_of(a, a.part_b, a.dv, a.grad.v_b, a.grad.v_n, a.grad.v_h, 1, a.Nk, 1.f)}}, 2, st);
  return rc;
}

}  // namespace
}  // namespace eve

using namespace eve;

extern "C" size_t eve_attn_fwd_workspace_bytes(const eve_attn_shape* s) {
  if (check_shape(s) != EVE_OK) return 0;
  return fwd_ws(*s, fwd_plan(*s, attn_cus()));
}

extern "C" int eve_attn_fwd(const eve_attn_shape* s, const eve_attn_layout* in, const void* q, const void* k, const void* v,
                            const uint8_t* key_mask, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_shape(s);
  if (rc != EVE_OK) return rc;
  rc = check_layout(in, s->dtype, "input");
  if (rc != EVE_OK) return rc;
  if (s->B == 0 || s->Nq == 0) return EVE_OK;
  EVE_REQUIRE(q && out && (s->Nk == 0 || (k && v)), EVE_ERR_ARG, "eve_attn_fwd: null pointer");
  EVE_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), EVE_ERR_ARG, "eve_attn_fwd: pointers must be 16-byte aligned");
  const AttnPlan p = fwd_plan(*s, attn_cus());
  AttnArgs a = base_args(*s);
  a.q = q; a.k = k; a.v = v; a.mask = key_mask; a.out = out; a.lse = lse; a.in = *in;
  if (p.nsplit > 1) {
    EVE_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= fwd_ws(*s, p), EVE_ERR_WORKSPACE, "eve_attn_fwd: workspace of %zu bytes, %zu needed",
                workspace_bytes, fwd_ws(*s, p));
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                         align_up((size_t)a.heads * p.nsplit * a.rows * a.D * 4, 256));
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (s->dtype == EVE_BF16) return s->D <= 64 ? fwd_typed<bf16_t, 64>(a, p, st) : fwd_typed<bf16_t, 128>(a, p, st);
  return s->D <= 64 ? fwd_typed<float, 64>(a, p, st) : fwd_typed<float, 128>(a, p, st);
}

extern "C" size_t eve_attn_bwd_workspace_bytes(const eve_attn_shape* s) {
  if (check_shape(s) != EVE_OK) return 0;
  return bwd_ws(*s, dq_plan(*s, attn_cus()), dkv_plan(*s, attn_cus())).bytes;
}

extern "C" int eve_attn_bwd(const eve_attn_shape* s, const eve_attn_layout* in, const eve_attn_layout* grad, const void* q,
                            const void* k, const void* v, const uint8_t* key_mask, const void* out, const float* lse,
                            const void* dout, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_shape(s);
  if (rc != EVE_OK) return rc;
  rc = check_layout(in, s->dtype, "input");
  if (rc != EVE_OK) return rc;
  rc = check_layout(grad, s->dtype, "gradient");
  if (rc != EVE_OK) return rc;
  if (s->B == 0 || (s->Nq == 0 && s->Nk == 0)) return EVE_OK;
  EVE_REQUIRE(s->Nq == 0 || (q && out && lse && dout && dq), EVE_ERR_ARG, "eve_attn_bwd: null pointer");
  EVE_REQUIRE(s->Nk == 0 || (k && v && dk && dv), EVE_ERR_ARG, "eve_attn_bwd: null pointer");
  const void* ptrs[8] = {q, k, v, out, dout, dq, dk, dv};
  for (const void* x : ptrs) EVE_REQUIRE(aligned16(x), EVE_ERR_ARG, "eve_attn_bwd: pointers must be 16-byte aligned");
  const AttnPlan pq = dq_plan(*s, attn_cus()), pk = dkv_plan(*s, attn_cus());
  const bool whole = whole_heads(*s, attn_cus());
  const BwdWs ws = bwd_ws(*s, pq, pk);
  EVE_REQUIRE(ws.bytes == 0 || (workspace && aligned16(workspace) && workspace_bytes >= ws.bytes), EVE_ERR_WORKSPACE,
              "eve_attn_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, ws.bytes);
  AttnArgs a = base_args(*s);
  a.q = q; a.k = k; a.v = v; a.mask = key_mask; a.o = out; a.dout = dout; a.dq = dq; a.dk = dk; a.dv = dv;
  a.lse = const_cast<float*>(lse); a.in = *in; a.grad = *grad;
  char* base = static_cast<char*>(workspace);
  a.stats = reinterpret_cast<uint4*>(base + ws.stats);
  a.part_a = reinterpret_cast<float*>(base + ws.part);
  a.part_b = reinterpret_cast<float*>(base + ws.dv);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (s->dtype == EVE_BF16) return s->D <= 64 ? bwd_typed<bf16_t, 64>(a, whole, pq, pk, st) : bwd_typed<bf16_t, 128>(a, false, pq, pk, st);
  return s->D <= 64 ? bwd_typed<float, 64>(a, false, pq, pk, st) : bwd_typed<float, 128>(a, false, pq, pk, st);
}
