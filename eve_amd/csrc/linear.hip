// The matrix products around the encoder's attention (reference models/multiway_transformer.py:104-106, :129-130, :341), gfx950:
//   z = x W^T + bias,   u = act(z),   y = residual + row_scale[row / T] gamma u
// with everything after the product done on the fp32 accumulator in the epilogue, and the gradient
//   dz = dy row_scale gamma act'(z)   (one pass, with the column sums dbias = sum dz, dgamma = sum dy row_scale u)
//   dx = dz W,   dW = dz^T x.
//
// An operand is row-major (its contraction index is contiguous in memory: x, W in the forward, dz in dx) or k-major (the
// contraction index is the row: W in dx, dz and x in dW).  Row-major tiles lie in LDS row by row and are read as 16-byte fragments;
// k-major tiles lie as in memory, [k][columns], and are transposed on the way to the matrix unit (bf16: ds_read_b64_tr_b16).
// Chunks of 16 bytes are XOR-permuted so that either read spreads over the banks.
//
// linear_stream_kernel: rows on 16-byte boundaries.  Tiles of 192 x 128 (256 x 128 of a k-major A, 128 x 128 of smaller problems),
// 4 waves, each half the rows and half the columns, so that five fragments feed six matrix instructions; steps of 64 bytes of the
// contraction go from memory to LDS directly, two or three steps ahead: two workgroups a CU, one of which computes while the other
// waits.  Bound: instruction issue.  39488 x 1024 -> 4096 with quick_gelu, gamma and residual takes 438 us at best, 505 in the mean of
// ten launches from a cold start (660 to 760 TFLOP/s; the vendor library's product alone 270 us); the matrix unit is busy for 40 % of the cycles.
// Reading fragments half a step ahead and 256-row tiles gained nothing.
// linear_tile_kernel: any size and alignment, and small problems; tiles of 128 or 64, staged through registers with every element
// outside an operand replaced by zero.  Bound: latency and the matrix unit, a half each (float32, 1899 x 750 -> 1001: 46 us, 62 of
// 138 TFLOP/s; the vendor library's product 35).
// linear_few_kernel (up to 4 rows) and linear_shared_kernel (few tiles, a long contraction): bound by a launch and the weight's way.
// dW has few tiles and a long contraction (the rows of the batch): it is split, with fp32 parts added in order.
#include "act.h"
#include "common.h"

namespace eve {

typedef __attribute__((ext_vector_type(8))) __bf16 li_bf16x8;
typedef __attribute__((ext_vector_type(4))) short li_s16x4;
typedef __attribute__((ext_vector_type(8))) short li_s16x8;
typedef __attribute__((ext_vector_type(16))) float li_f32x16;
typedef __attribute__((ext_vector_type(4))) float li_f32x4;

enum { LIN_FWD = 0, LIN_PLAIN = 1, LIN_PART = 2 };
constexpr int kActRuntime = -1;  // the activation is LinArgs::act

struct LinArgs {
  const void *A, *B;       // operands; rows of the result come from A, columns from B
  void* C;                 // [M, N] of the type
  float* part;             // LIN_PART: [nsplit][M][N]
  int M, N, K, lda, ldb;
  int nsplit, kspan;       // LIN_PART: splits of the contraction, its length in each
  float* part_bias;        // dW, may be null: [nsplit][M] column sums of A
  int ngroup;              // linear_stream_kernel: columns of tiles that are walked before the next row of tiles
  const void *bias, *gamma, *row_scale, *residual;  // LIN_FWD, each may be null
  void* z;                 // LIN_FWD: x W^T + bias, or null
  int rows_per_scale, act;
};

template <typename T> struct LT;
template <> struct LT<bf16_t> { static constexpr int E = 8, BK = 64; };
template <> struct LT<float> { static constexpr int E = 4, BK = 32; };

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ li_f32x16 lmma(const uint4& a, const uint4& b, li_f32x16 acc, bf16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(li_bf16x8, a), __builtin_bit_cast(li_bf16x8, b), acc, 0, 0, 0);
}
__device__ __forceinline__ li_f32x16 lmma(const uint4& a, const uint4& b, li_f32x16 acc, float) {
  acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), acc, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), acc, 0, 0, 0);
}

// byte offset of 16-byte chunk c of row (row-major tile) / k-row (k-major tile of W columns)
__device__ __forceinline__ int row_off(int row, int c) { return row * 128 + ((c ^ ((row >> 1) & 7)) << 4); }
template <typename T, int W> __device__ __forceinline__ int col_off(int k, int c) {
  constexpr int CPR = W / LT<T>::E;
  if constexpr (sizeof(T) == 2) return k * (CPR * 16) + ((c ^ (((k & 3) << 2) & (CPR - 1))) << 4);
  else return k * (CPR * 16) + (c << 4);
}
// fragment of the 32 rows / columns from r0, contraction step ks: lane l holds row r0 + (l & 31) and the E elements of the
// contraction from (2 ks + (l >> 5)) E on
template <typename T, bool COL, int W> __device__ __forceinline__ uint4 lfrag(const char* tile, int r0, int ks, int lane) {
  if constexpr (!COL) {
    return *reinterpret_cast<const uint4*>(tile + row_off(r0 + (lane & 31), 2 * ks + (lane >> 5)));
  } else if constexpr (sizeof(T) == 2) {
    const int i = lane & 15, q = i >> 2, p = i & 3, h = lane >> 5, e = r0 + 16 * ((lane >> 4) & 1) + 4 * p;
    li_s16x4 v[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int k = ks * 16 + 8 * h + 4 * r + q;
      char* a = const_cast<char*>(tile) + col_off<T, W>(k, e >> 3) + ((e & 7) << 1);
      v[r] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) li_s16x4*)(__attribute__((address_space(3))) char*)a);
    }
    const li_s16x8 w = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(uint4, w);
  } else {
    const int col = r0 + (lane & 31), k = ks * 8 + 4 * (lane >> 5);
    const char* a = tile + col_off<T, W>(k, col >> 2) + ((col & 3) << 2);
    constexpr int P = W * 4;
    uint4 w;
    w.x = *reinterpret_cast<const uint32_t*>(a);
    w.y = *reinterpret_cast<const uint32_t*>(a + P);
    w.z = *reinterpret_cast<const uint32_t*>(a + 2 * P);
    w.w = *reinterpret_cast<const uint32_t*>(a + 3 * P);
    return w;
  }
}

// n elements (of E) from p on, zeros behind them; p needs no alignment
template <typename T> __device__ __forceinline__ uint4 load_some(const T* p, int n) {
  uint4 w = make_uint4(0, 0, 0, 0);
  if (n >= LT<T>::E) {
    __builtin_memcpy(&w, p, 16);
  } else if (n > 0) {
    T e[LT<T>::E];
#pragma unroll
    for (int i = 0; i < LT<T>::E; ++i) e[i] = i < n ? p[i] : T(0.f);
    __builtin_memcpy(&w, e, 16);
  }
  return w;
}
template <typename T> __device__ __forceinline__ void store_some(T* p, const uint4& w, int n) {
  if (n >= LT<T>::E) {
    __builtin_memcpy(p, &w, 16);
  } else if (n > 0) {
    T e[LT<T>::E];
    __builtin_memcpy(e, &w, 16);
#pragma unroll
    for (int i = 0; i < LT<T>::E; ++i)
      if (i < n) p[i] = e[i];
  }
}

// a tile on its way to LDS through registers
template <typename T, bool COL, int W, int TH> struct LinTile {
  static constexpr int E = LT<T>::E, BK = LT<T>::BK;
  static constexpr int BYTES = W * 128;
  static constexpr int N = BYTES / 16 / TH;
  uint4 w[N];
  // ext: rows (columns) of the operand from the tile's first on; kext: contraction indices from the step's first on
  __device__ __forceinline__ void load(const T* p, int64_t ld, int ext, int kext, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * TH;
      if constexpr (!COL) {
        const int r = idx >> 3, c = (idx & 7) * E;
        w[i] = r < ext ? load_some<T>(p + r * ld + c, kext - c) : make_uint4(0, 0, 0, 0);
      } else {
        constexpr int CPR = W / E;
        const int k = idx / CPR, c = (idx % CPR) * E;
        w[i] = k < kext ? load_some<T>(p + k * ld + c, ext - c) : make_uint4(0, 0, 0, 0);
      }
    }
  }
  __device__ __forceinline__ void store(char* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * TH;
      if constexpr (!COL) {
        *reinterpret_cast<uint4*>(tile + row_off(idx >> 3, idx & 7)) = w[i];
      } else {
        constexpr int CPR = W / E;
        *reinterpret_cast<uint4*>(tile + col_off<T, W>(idx / CPR, idx % CPR)) = w[i];
      }
    }
  }
};

template <typename T> __device__ __forceinline__ float act_of(float z, int act) {
  constexpr bool F = sizeof(T) == 2;
  switch (act) {
    case EVE_ACT_QUICK_GELU: return act_fwd<EVE_ACT_QUICK_GELU, F>(z);
    case EVE_ACT_GELU: return act_fwd<EVE_ACT_GELU, F>(z);
    case EVE_ACT_RELU: return act_fwd<EVE_ACT_RELU, F>(z);
    default: return z;
  }
}
template <typename T> __device__ __forceinline__ float act_slope(float z, int act) {
  constexpr bool F = sizeof(T) == 2;
  switch (act) {
    case EVE_ACT_QUICK_GELU: return act_bwd<EVE_ACT_QUICK_GELU, F>(z);
    case EVE_ACT_GELU: return act_bwd<EVE_ACT_GELU, F>(z);
    case EVE_ACT_RELU: return act_bwd<EVE_ACT_RELU, F>(z);
    default: return 1.f;
  }
}
template <typename T> __device__ __forceinline__ uint4 pack16(const float* v) {
  Vec16<T> o;
  float t[Vec16<T>::N];
#pragma unroll
  for (int i = 0; i < Vec16<T>::N; ++i) t[i] = v[i];
  o.set_all(t);
  return __builtin_bit_cast(uint4, o.raw);
}
template <typename T> __device__ __forceinline__ void unpack16(const uint4& w, float* v) {
  Vec16<T> o;
  o.raw = __builtin_bit_cast(decltype(o.raw), w);
#pragma unroll
  for (int i = 0; i < Vec16<T>::N; ++i) v[i] = o.get(i);
}
#endif  // __HIP_DEVICE_COMPILE__

#if defined(__HIP_DEVICE_COMPILE__)
// The wave's block of the result, rows from m0 and WN columns from n0 on: 32 rows at a time through the wave's own image in LDS,
// then 8 columns of a row a lane.  The accumulators are those of the transposed product (B first): a lane holds row lane & 31 and
// four consecutive columns at a time, one 16-byte store into the image instead of four of 4 bytes.
//
// VEC (rows on 16-byte boundaries): all accesses go through buffer descriptors, where a lane outside the result has an offset
// outside, without a branch.  Behind a branch around a store the compiler cannot count it and waits for its completion before the
// next value that it has loaded: 2000 cycles a pass, twelve times a tile.  For bf16 the residual and the row factors of the whole
// block are requested before the first store.
typedef uint32_t li_u32x4 __attribute__((ext_vector_type(4)));
constexpr uint32_t kLinNowhere = 0xfffffff0u, kLinReach = 0x80000000u;  // an offset outside every descriptor, and their extent
template <typename T, int WN, int NTM, int NTN, int MODE, int ACT, bool VEC>
__device__ __forceinline__ void lin_epilogue(const li_f32x16 (&acc)[NTM][NTN], char* smem, const LinArgs& a, int split, int m0, int n0,
                                             int wave, int lane) {
  constexpr int E = LT<T>::E, EP = WN + 4;             // floats of an image row
  constexpr int CH = WN / 8, RPI = 64 / CH;            // chunks of 8 columns of an image row; rows a pass
  constexpr int PASS = 32 / RPI;
  constexpr bool AHEAD = VEC && MODE == LIN_FWD && sizeof(T) == 2;
  constexpr int OSIZE = MODE == LIN_PART ? 4 : (int)sizeof(T);
  float* img = reinterpret_cast<float*>(smem) + wave * 32 * EP;
  const int ch = lane % CH, n = n0 + ch * 8, nn = a.N - n;
  // VEC: descriptors from the block's first element on, a lane's offset for row r of the block
  auto rsrc = [&](const void* p, int64_t size) {
    const uint64_t x = reinterpret_cast<uint64_t>(p) + ((int64_t)m0 * a.N + n0) * size;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), 0, p ? kLinReach : 0u, 0x00020000);
  };
  auto offset = [&](int r, int e, int size) {
    return m0 + r < a.M && e < nn ? ((uint32_t)r * (uint32_t)a.N + ch * 8 + e) * size : kLinNowhere;
  };
  __amdgpu_buffer_rsrc_t to, to_z, from;
  if constexpr (VEC) {
    to = rsrc(MODE == LIN_PART ? a.part + (int64_t)split * a.M * a.N : a.C, OSIZE);
    to_z = rsrc(a.z, sizeof(T));
    from = rsrc(a.residual, sizeof(T));
  }
  li_u32x4 res[AHEAD ? NTM * PASS : 1];
  float rs[AHEAD ? NTM * PASS : 1];
  if constexpr (AHEAD) {
#pragma unroll
    for (int i = 0; i < NTM * PASS; ++i) {
      const int r = i * RPI + lane / CH;
      res[i] = __builtin_amdgcn_raw_buffer_load_b128(from, offset(r, 0, sizeof(T)), 0, 0);
      rs[i] = 1.f;
    }
    if (a.row_scale) {
#pragma unroll
      for (int i = 0; i < NTM * PASS; ++i)
        rs[i] = to_f32<T>(static_cast<const T*>(a.row_scale)[min(m0 + i * RPI + lane / CH, a.M - 1) / a.rows_per_scale]);
    }
  }
  float bias[8], gamma[8];
  if constexpr (MODE == LIN_FWD) {
#pragma unroll
    for (int e = 0; e < 8; e += E) {
      uint4 b = make_uint4(0, 0, 0, 0), g = make_uint4(0, 0, 0, 0);
      if constexpr (VEC) {
        const uint32_t o = e < nn ? (uint32_t)(n + e) * (uint32_t)sizeof(T) : kLinNowhere;
        const li_u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(
            __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(a.bias), 0, a.bias ? kLinReach : 0u, 0x00020000), o, 0, 0);
        const li_u32x4 y = __builtin_amdgcn_raw_buffer_load_b128(
            __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(a.gamma), 0, a.gamma ? kLinReach : 0u, 0x00020000), o, 0, 0);
        b = make_uint4(x.x, x.y, x.z, x.w);
        g = make_uint4(y.x, y.y, y.z, y.w);
      } else {
        if (a.bias) b = load_some<T>(static_cast<const T*>(a.bias) + n + e, nn - e);
        if (a.gamma) g = load_some<T>(static_cast<const T*>(a.gamma) + n + e, nn - e);
      }
      unpack16<T>(b, bias + e);
      unpack16<T>(g, gamma + e);
    }
    if (!a.gamma) {
#pragma unroll
      for (int e = 0; e < 8; ++e) gamma[e] = 1.f;
    }
  }
#pragma unroll
  for (int i = 0; i < NTM; ++i) {
#pragma unroll
    for (int j = 0; j < NTN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(img + (lane & 31) * EP + 32 * j + 8 * g + 4 * (lane >> 5)) =
            make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the image is the wave's own: no barrier, but its lanes exchange through it
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int it = 0; it < PASS; ++it) {
      const int rr = it * RPI + lane / CH, r = 32 * i + rr, m = m0 + r;
      float v[8];
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(img + rr * EP + ch * 8);
      *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(img + rr * EP + ch * 8 + 4);
      const int64_t at = (int64_t)m * a.N + n;
      const bool in = m < a.M && nn > 0;
      auto put = [&](const __amdgpu_buffer_rsrc_t& d, void* p, int e, const uint4& w) {  // 16 bytes from column e of the eight on
        if constexpr (VEC) __builtin_amdgcn_raw_buffer_store_b128(li_u32x4{w.x, w.y, w.z, w.w}, d, offset(r, e, OSIZE), 0, 0);
        else if (in) store_some<T>(static_cast<T*>(p) + at + e, w, nn - e);
      };
      if constexpr (MODE == LIN_PART) {
        float* p = a.part + (int64_t)split * a.M * a.N + at;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const uint4 w = __builtin_bit_cast(uint4, *reinterpret_cast<float4*>(v + e));
          if constexpr (VEC) put(to, nullptr, e, w);
          else if (in) store_some<float>(p + e, w, nn - e);
        }
      } else {
        if constexpr (MODE == LIN_FWD) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += bias[e];
          if (a.z) {
#pragma unroll
            for (int e = 0; e < 8; e += E) put(to_z, a.z, e, pack16<T>(v + e));
          }
          if constexpr (ACT == kActRuntime) {
            if (a.act != EVE_ACT_IDENTITY) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = act_of<T>(v[e], a.act);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = act_fwd<ACT, sizeof(T) == 2>(v[e]);
          }
          if (a.gamma || a.row_scale) {
            float f = 1.f;
            if constexpr (AHEAD) f = rs[i * PASS + it];
            else if (a.row_scale && in) f = to_f32<T>(static_cast<const T*>(a.row_scale)[m / a.rows_per_scale]);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= gamma[e] * f;
          }
          if (a.residual) {
#pragma unroll
            for (int e = 0; e < 8; e += E) {
              uint4 w = make_uint4(0, 0, 0, 0);
              if constexpr (AHEAD) {
                const li_u32x4 x = res[i * PASS + it];
                w = make_uint4(x.x, x.y, x.z, x.w);
              } else if constexpr (VEC) {
                const li_u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(from, offset(r, e, sizeof(T)), 0, 0);
                w = make_uint4(x.x, x.y, x.z, x.w);
              } else if (in) {
                w = load_some<T>(static_cast<const T*>(a.residual) + at + e, nn - e);
              }
              float x[E];
              unpack16<T>(w, x);
#pragma unroll
              for (int f = 0; f < E; ++f) v[e + f] += x[f];
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e += E) put(to, a.C, e, pack16<T>(v + e));
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}
#endif

// BT x BT tile, 4 waves of (BT/2) x (BT/2); two LDS stages, the next two steps' tiles in registers meanwhile.  BT = 64: twice the
// waves, half of a step's contraction each, added at the end (float32, 1899 x 750 -> 1001: 46 us instead of 48; bf16, 617 x
// 4096 -> 1024: 31 instead of 35).
template <int BT> constexpr int tile_threads() { return BT == 64 ? 512 : 256; }
template <typename T, int BT, bool ACOL, bool BCOL, int MODE>
__global__ __launch_bounds__(tile_threads<BT>()) void linear_tile_kernel(LinArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BK = LT<T>::BK, E = LT<T>::E, NT = BT / 64, TH = tile_threads<BT>(), SHARE = TH / 256, NKS = BK / (2 * E) / SHARE;
  constexpr int STAGE = 2 * BT * 128;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = (tid >> 6) & 3, share = tid >> 8, wm = wave >> 1, wn = wave & 1;
  // Workgroups go round-robin over the 8 XCDs: each of them gets a run of tiles, columns fastest, so that the tiles it works on
  // at a time share a few row panels of A through its L2.
  const int tm = (a.M + BT - 1) / BT, tn = (a.N + BT - 1) / BT, total = tm * tn * a.nsplit;
  const int per = (total + 7) >> 3;
  const int item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || item >= total) return;
  const int split = item / (tm * tn), tile = item % (tm * tn);
  const int m0 = (tile / tn) * BT, n0 = (tile % tn) * BT;
  const int k0 = MODE == LIN_PART ? split * a.kspan : 0;
  const int k1 = MODE == LIN_PART ? min(a.K, k0 + a.kspan) : a.K;

  const T* Ap = static_cast<const T*>(a.A) + (ACOL ? (int64_t)k0 * a.lda + m0 : (int64_t)m0 * a.lda + k0);
  const T* Bp = static_cast<const T*>(a.B) + (BCOL ? (int64_t)k0 * a.ldb + n0 : (int64_t)n0 * a.ldb + k0);
  const int64_t sa = ACOL ? (int64_t)BK * a.lda : BK, sb = BCOL ? (int64_t)BK * a.ldb : BK;

  li_f32x16 acc[NT][NT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  LinTile<T, ACOL, BT, TH> ta[2];
  LinTile<T, BCOL, BT, TH> tb[2];
  const int steps = (k1 - k0 + BK - 1) / BK;
  auto fetch = [&](int t, int i) {  // past the last step: zeros
    ta[i].load(Ap + t * sa, a.lda, a.M - m0, k1 - k0 - t * BK, tid);
    tb[i].load(Bp + t * sb, a.ldb, a.N - n0, k1 - k0 - t * BK, tid);
  };
  fetch(0, 0);
  fetch(1, 1);
  for (int t = 0; t < steps; t += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      char* as = smem + u * STAGE;
      char* bs = as + BT * 128;
      ta[u].store(as, tid);
      tb[u].store(bs, tid);
      __syncthreads();
      fetch(t + u + 2, u);
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        uint4 fa[NT], fb[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) fa[i] = lfrag<T, ACOL, BT>(as, wm * (BT / 2) + 32 * i, share * NKS + ks, lane);
#pragma unroll
        for (int j = 0; j < NT; ++j) fb[j] = lfrag<T, BCOL, BT>(bs, wn * (BT / 2) + 32 * j, share * NKS + ks, lane);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = lmma(fb[j], fa[i], acc[i][j], T());
      }
    }
  }
  __syncthreads();  // the stages become the waves' epilogue images
  if constexpr (SHARE == 2) {
    static_assert(NT == 1, "one accumulator");
    li_f32x4* part = reinterpret_cast<li_f32x4*>(smem) + (wave * 4) * 64 + lane;
    if (share == 1) {
#pragma unroll
      for (int g = 0; g < 4; ++g) part[g * 64] = li_f32x4{acc[0][0][4 * g], acc[0][0][4 * g + 1], acc[0][0][4 * g + 2], acc[0][0][4 * g + 3]};
    }
    __syncthreads();
    if (share == 0) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[0][0][4 * g + r] += part[g * 64][r];
    }
    __syncthreads();
    if (share == 1) return;
  }
  lin_epilogue<T, BT / 2, NT, NT, MODE, kActRuntime, false>(acc, smem, a, split, m0 + wm * (BT / 2), n0 + wn * (BT / 2), wave, lane);
#endif
}

#if defined(__HIP_DEVICE_COMPILE__)
// One operand's tile of W rows (columns) by 64 bytes of the contraction.
template <typename T, bool COL, int W> struct StreamTile {
  static constexpr int E = LT<T>::E, BK = 4 * E;        // contraction indices of a step
  static constexpr int BYTES = W * 64, N = BYTES / 1024 / 4;  // a wave's transfers of 1 KiB
  static constexpr int CPR = COL ? W / E : 4;           // chunks of a row of the tile in LDS
  static constexpr int RB = CPR * 16;
  uint32_t off[N];
  int k_of[N];  // the contraction index (COL: the row; else the chunk's first) a lane's chunk belongs to
  // permutation of the chunks of a row
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (!COL) return (row >> 2) & 3;              // 16 rows of 64 bytes: one chunk each of every 256 bytes
    else if constexpr (sizeof(T) == 2) return (row & 3) << 2;  // 4 rows: 64 bytes each of every 256
    else return ((row >> 2) & 1) << 3;                       // rows 4 apart: 128 bytes each
  }
  __device__ __forceinline__ StreamTile(int64_t ld, int ext, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = (i * 4 + wave) * 64 + lane, row = p / CPR, c = (p % CPR) ^ swizzle(row);
      k_of[i] = COL ? row : c * E;
      const bool in = COL ? c * E < ext : row < ext;
      off[i] = in ? (uint32_t)row * ((uint32_t)ld * sizeof(T)) + c * 16 : kLinNowhere;
    }
  }
  // the wave's transfer i; from the end of the contraction on (krem indices left) zeros
  __device__ __forceinline__ void piece(int i, __amdgpu_buffer_rsrc_t r, char* tile, int wave, int krem) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(tile + (i * 4 + wave) * 1024), 16,
                                             k_of[i] < krem ? off[i] : kLinNowhere, 0, 0, 0);
  }
};

__device__ __forceinline__ uint32_t lin_lds(const char* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }

// Four transposed fragments, read and waited for in one block (through the builtin the compiler would also wait for the
// transfers in flight): at p0 + D0, p1 + D1, p2 + D2, p3 + D3, their second halves 4 rows on.
template <int RB, int D0, int D1, int D2, int D3>
__device__ __forceinline__ void lin_tr4(uint32_t p0, uint32_t p1, uint32_t p2, uint32_t p3, uint4 (&f)[4]) {
  li_s16x4 v[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %2, %9 offset:%14\n\tds_read_b64_tr_b16 %3, %9 offset:%15\n\t"
      "ds_read_b64_tr_b16 %4, %10 offset:%16\n\tds_read_b64_tr_b16 %5, %10 offset:%17\n\t"
      "ds_read_b64_tr_b16 %6, %11 offset:%18\n\tds_read_b64_tr_b16 %7, %11 offset:%19\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(p0), "v"(p1), "v"(p2), "v"(p3), "n"(D0), "n"(D0 + 4 * RB), "n"(D1), "n"(D1 + 4 * RB), "n"(D2), "n"(D2 + 4 * RB), "n"(D3),
        "n"(D3 + 4 * RB)
      : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const li_s16x8 w = __builtin_shufflevector(v[2 * i], v[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    f[i] = __builtin_bit_cast(uint4, w);
  }
}

// Fragments of NT 32-row (column) blocks from r0 on, for both halves of a step: f[ks][i].
template <typename T, bool COL, int W, int NT> struct StreamReader {
  using S = StreamTile<T, COL, W>;
  uint32_t base;  // block 0, first half
  __device__ __forceinline__ StreamReader(int r0, int lane) {
    if constexpr (!COL) {
      const int row = r0 + (lane & 31);
      base = row * 64 + (((lane >> 5) ^ S::swizzle(row)) << 4);
    } else if constexpr (sizeof(T) == 2) {
      const int i = lane & 15, q = i >> 2, p = i & 3, e = r0 + 16 * ((lane >> 4) & 1) + 4 * p;
      base = (8 * (lane >> 5) + q) * S::RB + (((e >> 3) ^ (q << 2)) << 4) + ((e & 7) << 1);
    } else {
      const int col = r0 + (lane & 31);
      base = 4 * (lane >> 5) * S::RB + ((((col >> 2) ^ ((lane >> 5) << 3)) << 4)) + ((col & 3) << 2);
    }
  }
  __device__ __forceinline__ void read(const char* smem, uint32_t tile, int ks, uint4 (&f)[NT]) const {
    if constexpr (!COL) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const li_u32x4 w = *reinterpret_cast<const li_u32x4*>(smem + (((tile + base) ^ (ks << 5)) + i * 2048));
        f[i] = make_uint4(w.x, w.y, w.z, w.w);
      }
    } else if constexpr (sizeof(T) == 2) {
      const uint32_t at = lin_lds(smem) + tile + ks * 16 * S::RB;  // block i: chunk 4 i, permuted by q << 2
      if constexpr (NT == 4) {
        lin_tr4<S::RB, 0, 0, 0, 0>(at + base, at + (base ^ 64), at + (base ^ 128), at + (base ^ 192), f);
      } else {
        static_assert(NT == 2, "two or four blocks");
        uint4 g[4];  // (the other two are the second half of the step's, read by both())
        lin_tr4<S::RB, 0, 0, 16 * S::RB, 16 * S::RB>(at + base, at + (base ^ 64), at + base, at + (base ^ 64), g);
        f[0] = g[0];
        f[1] = g[1];
      }
    } else {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) w[t] = *reinterpret_cast<const uint32_t*>(smem + (tile + (base ^ (i << 7)) + (ks * 8 + t) * S::RB));  // block i: chunk 8 i, permuted
        f[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  // both halves at once
  __device__ __forceinline__ void both(const char* smem, uint32_t tile, uint4 (&f)[2][NT]) const {
    if constexpr (COL && sizeof(T) == 2 && NT == 2) {
      const uint32_t at = lin_lds(smem) + tile;
      uint4 g[4];
      lin_tr4<S::RB, 0, 0, 16 * S::RB, 16 * S::RB>(at + base, at + (base ^ 64), at + base, at + (base ^ 64), g);
      f[0][0] = g[0];
      f[0][1] = g[1];
      f[1][0] = g[2];
      f[1][1] = g[3];
    } else {
      read(smem, tile, 0, f[0]);
      read(smem, tile, 1, f[1]);
    }
  }
};

template <typename T> __device__ __forceinline__ float frag_sum(const uint4& w, float s) {
  float v[LT<T>::E];
  unpack16<T>(w, v);
#pragma unroll
  for (int i = 0; i < LT<T>::E; ++i) s += v[i];
  return s;
}
#endif  // __HIP_DEVICE_COMPILE__

constexpr int kStreamN = 128;
template <int BM> constexpr int stream_stages() { return BM == 192 ? 4 : 3; }
template <int BM> constexpr int stream_lds() { return stream_stages<BM>() * (BM + kStreamN) * 64; }

// (The activation is a parameter of the kernel: with all of them in it, twelve times over, its code does not fit the instruction cache.)
template <typename T, int BM, bool ACOL, bool BCOL, int MODE, int ACT>
__global__ __launch_bounds__(256, 2) void linear_stream_kernel(LinArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BN = kStreamN, NTM = BM / 64, NTN = 2, STAGE = (BM + BN) * 64, NST = stream_stages<BM>();
  static_assert(BM != 192 || !ACOL, "192-row tiles: row-major A");
  using TA = StreamTile<T, ACOL, BM>;
  using TB = StreamTile<T, BCOL, BN>;
  constexpr int BK = TA::BK;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1, wave_u = __builtin_amdgcn_readfirstlane(wave);
  // Workgroups go round-robin over the 8 XCDs: each of them gets a run of tiles.  A run walks ngroup columns of tiles (their part
  // of B stays in the XCD's L2) row by row of A.
  const int tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN, total = tm * tn * a.nsplit;
  const int per = (total + 7) >> 3;
  const int item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || item >= total) return;
  const int split = item / (tm * tn), tile = item % (tm * tn);
  const int grp = tile / (tm * a.ngroup), in_grp = tile - grp * tm * a.ngroup, width = min(a.ngroup, tn - grp * a.ngroup);
  const int m0 = in_grp / width * BM, n0 = (grp * a.ngroup + in_grp % width) * BN;
  const int k0 = MODE == LIN_PART ? split * a.kspan : 0;
  const int k1 = MODE == LIN_PART ? min(a.K, k0 + a.kspan) : a.K;

  const T* Ap = static_cast<const T*>(a.A) + (ACOL ? (int64_t)k0 * a.lda + m0 : (int64_t)m0 * a.lda + k0);
  const T* Bp = static_cast<const T*>(a.B) + (BCOL ? (int64_t)k0 * a.ldb + n0 : (int64_t)n0 * a.ldb + k0);
  const int64_t sa = ACOL ? (int64_t)BK * a.lda : BK, sb = BCOL ? (int64_t)BK * a.ldb : BK;
  const TA ta(a.lda, a.M - m0, wave, lane);
  const TB tb(a.ldb, a.N - n0, wave, lane);
  const StreamReader<T, ACOL, BM, NTM> ra(wm * (BM / 2), lane);
  const StreamReader<T, BCOL, BN, NTN> rb(wn * (BN / 2), lane);

  li_f32x16 acc[NTM][NTN];
#pragma unroll
  for (int i = 0; i < NTM; ++i)
#pragma unroll
    for (int j = 0; j < NTN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  float colsum[NTM];
#pragma unroll
  for (int i = 0; i < NTM; ++i) colsum[i] = 0.f;
  const bool sums = ACOL && a.part_bias && n0 == 0 && wn == 0;

  const int steps = (k1 - k0 + BK - 1) / BK;
  constexpr int NP = TA::N + TB::N;  // a wave's transfers of a step
  __amdgpu_buffer_rsrc_t rsrc_a, rsrc_b;
  char* into = smem;
  int krem;
  auto fetch_begin = [&](int t) {
    rsrc_a = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(Ap + t * sa), 0, kLinReach, 0x00020000);
    rsrc_b = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(Bp + t * sb), 0, kLinReach, 0x00020000);
    krem = k1 - k0 - t * BK;  // past the last step: zeros, nothing is read
  };
  auto fetch_piece = [&](int i) {
    if (i < TA::N) ta.piece(i, rsrc_a, into, wave_u, krem);
    else tb.piece(i - TA::N, rsrc_b, into + BM * 64, wave_u, krem);
  };
  auto fetch_end = [&]() { into = into == smem + (NST - 1) * STAGE ? smem : into + STAGE; };
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) {
    fetch_begin(i);
#pragma unroll
    for (int j = 0; j < NP; ++j) fetch_piece(j);
    fetch_end();
  }
  uint32_t at = 0;
  for (int t = 0; t < steps; ++t) {
    // this step's transfers have landed (the next ones' may be in flight), and everybody has read what the next fetch overwrites
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * NP) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    fetch_begin(t + NST - 1);
    uint4 fa[2][NTM], fb[2][NTN];
    rb.both(smem, at + BM * 64, fb);
    ra.read(smem, at, 0, fa[0]);
    if constexpr (!ACOL) ra.read(smem, at, 1, fa[1]);
    // The transfers are issued between the matrix instructions: the CU takes one in 16 cycles or more, and a wave that issues them in
    // a row waits there (400 of a step's 1350 cycles) with nothing for the matrix unit to do.
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if constexpr (ACOL)
        if (ks) ra.read(smem, at, 1, fa[1]);
      if (sums) {
#pragma unroll
        for (int i = 0; i < NTM; ++i) colsum[i] = frag_sum<T>(fa[ks][i], colsum[i]);
      }
#pragma unroll
      for (int i = 0; i < NTM; ++i) {
#pragma unroll
        for (int j = 0; j < NTN; ++j) acc[i][j] = lmma(fb[ks][j], fa[ks][i], acc[i][j], T());
        __builtin_amdgcn_sched_barrier(0);
        constexpr int SLOTS = 2 * NTM;
        const int slot = ks * NTM + i;
#pragma unroll
        for (int q = 0; q < NP; ++q)
          if (q * SLOTS / NP == slot) fetch_piece(q);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    fetch_end();
    at = at == (NST - 1) * STAGE ? 0 : at + STAGE;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no transfer may meet the images
  __syncthreads();
  if (sums) {
#pragma unroll
    for (int i = 0; i < NTM; ++i) {
      const float s = colsum[i] + __shfl_xor(colsum[i], 32, 64);
      const int m = m0 + wm * (BM / 2) + 32 * i + (lane & 31);
      if (lane < 32 && m < a.M) a.part_bias[(int64_t)split * a.M + m] = s;
    }
  }
  lin_epilogue<T, BN / 2, NTM, NTN, MODE, ACT, true>(acc, smem, a, split, m0 + wm * (BM / 2), n0 + wn * (BN / 2), wave, lane);
#endif
}

#if defined(__HIP_DEVICE_COMPILE__)
// the epilogue of one element
template <typename T> __device__ __forceinline__ void lin_finish(const LinArgs& a, int m, int n, float v) {
  const int64_t at = (int64_t)m * a.N + n;
  if (a.bias) v += to_f32<T>(static_cast<const T*>(a.bias)[n]);
  if (a.z) static_cast<T*>(a.z)[at] = from_f32<T>(v);
  v = act_of<T>(v, a.act);
  if (a.gamma) v *= to_f32<T>(static_cast<const T*>(a.gamma)[n]);
  if (a.row_scale) v *= to_f32<T>(static_cast<const T*>(a.row_scale)[m / a.rows_per_scale]);
  if (a.residual) v += to_f32<T>(static_cast<const T*>(a.residual)[at]);
  static_cast<T*>(a.C)[at] = from_f32<T>(v);
}
#endif

// A few rows: one wave a column, the weight's row read once for all of them.
template <typename T, int R>
__global__ __launch_bounds__(256) void linear_few_kernel(LinArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int E = LT<T>::E;
  const int lane = lane_id(), n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= a.N) return;
  const T* w = static_cast<const T*>(a.B) + (int64_t)n * a.ldb;
  const T* x = static_cast<const T*>(a.A);
  float acc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = 0.f;
  for (int k = lane * E; k < a.K; k += 64 * E) {
    float wv[E], xv[E];
    unpack16<T>(load_some<T>(w + k, a.K - k), wv);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      unpack16<T>(load_some<T>(x + (int64_t)r * a.lda + k, r < a.M ? a.K - k : 0), xv);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[r] = fmaf(wv[e], xv[e], acc[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = wave_sum(acc[r]);
  float v = acc[0];
#pragma unroll
  for (int r = 1; r < R; ++r) v = lane == r ? acc[r] : v;
  if (lane < R && lane < a.M) {
    lin_finish<T>(a, lane, n, v);
  }
#endif
}

// A long contraction and few tiles: 8 waves of a workgroup share one tile's contraction and add their sums through LDS, in order.
// Tile: R x R with R = 16 NTL.  Fragments come from memory as they are (16 rows by 64 bytes, neighbouring lines in the next steps of
// a wave), one unit of U steps ahead; a row past the end is the last one again, whose results are not kept.
#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ li_f32x4 lmma16(const uint4& a, const uint4& b, li_f32x4 acc, bf16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(li_bf16x8, a), __builtin_bit_cast(li_bf16x8, b), acc, 0, 0, 0);
}
__device__ __forceinline__ li_f32x4 lmma16(const uint4& a, const uint4& b, li_f32x4 acc, float) {
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), acc, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), acc, 0, 0, 0);
}
#endif
template <typename T, int NTL>
__global__ __launch_bounds__(512, 2) void linear_shared_kernel(LinArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int E = LT<T>::E, NW = 8, R = 16 * NTL, U = NTL == 1 ? 4 : 2, UK = U * 4 * E;
  __shared__ __attribute__((aligned(16))) float red[NW][R][R + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, quad = lane >> 4;
  // a run of tiles an XCD, rows fastest: the weight's rows, which are the many, are read into one L2
  const int tm = (a.M + R - 1) / R, total = tm * ((a.N + R - 1) / R), per = (total + 7) >> 3;
  const int item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || item >= total) return;
  const int m0 = item % tm * R, n0 = item / tm * R;
  const T *ap[NTL], *bp[NTL];
  li_f32x4 acc[NTL][NTL];
#pragma unroll
  for (int i = 0; i < NTL; ++i) {
    ap[i] = static_cast<const T*>(a.A) + (int64_t)min(m0 + 16 * i + l16, a.M - 1) * a.lda + quad * E;
    bp[i] = static_cast<const T*>(a.B) + (int64_t)min(n0 + 16 * i + l16, a.N - 1) * a.ldb + quad * E;
#pragma unroll
    for (int j = 0; j < NTL; ++j) acc[i][j] = li_f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int units = (a.K + UK - 1) / UK;
  struct Unit { uint4 a[U][NTL], b[U][NTL]; } one, two;
  auto load = [&](int u, Unit& f) {  // past the last unit: zeros
    const int k = u * UK;
    if (k + UK <= a.K) {
#pragma unroll
      for (int s = 0; s < U; ++s)
#pragma unroll
        for (int i = 0; i < NTL; ++i) {
          __builtin_memcpy(&f.a[s][i], ap[i] + k + s * 4 * E, 16);
          __builtin_memcpy(&f.b[s][i], bp[i] + k + s * 4 * E, 16);
        }
    } else {
#pragma unroll
      for (int s = 0; s < U; ++s)
#pragma unroll
        for (int i = 0; i < NTL; ++i) {
          const int at = k + s * 4 * E;
          f.a[s][i] = load_some<T>(ap[i] + at, a.K - at - quad * E);
          f.b[s][i] = load_some<T>(bp[i] + at, a.K - at - quad * E);
        }
    }
  };
  auto add = [&](const Unit& f) {
#pragma unroll
    for (int s = 0; s < U; ++s)
#pragma unroll
      for (int i = 0; i < NTL; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = lmma16(f.b[s][j], f.a[s][i], acc[i][j], T());
  };
  int u = wave;
  load(u, one);
  for (; u < units; u += 2 * NW) {
    load(u + NW, two);
    add(one);
    load(u + 2 * NW, one);
    add(two);
  }
#pragma unroll
  for (int i = 0; i < NTL; ++i)
#pragma unroll
    for (int j = 0; j < NTL; ++j) *reinterpret_cast<li_f32x4*>(&red[wave][16 * i + l16][16 * j + 4 * quad]) = acc[i][j];
  __syncthreads();
  for (int e = tid; e < R * R; e += NW * 64) {
    const int i = e / R, j = e % R, m = m0 + i, n = n0 + j;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[w][i][j];
    if (m < a.M && n < a.N) lin_finish<T>(a, m, n, v);
  }
#endif
}

// dz and the column sums of its terms (15168 x 768 of bf16 with z: 70 MB in 16.8 us, 4.2 TB/s).  Block: 32 chunks of 8 columns x 8 row lanes, over `rows` rows; the row lanes are added
// in order and each block row leaves one part.
struct DzArgs {
  const void *dy, *z, *gamma, *row_scale;
  void* dz;                 // may be null (dz = dy)
  float *part_b, *part_g;   // [parts][N], either may be null
  void *db, *dg;            // where there is one part: the column sums themselves, either may be null
  int M, N, rows_per_scale, act, rows;  // rows: of a block
};
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(DzArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int E = LT<T>::E;
  __shared__ float red[2][8][256 + 8];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int n = blockIdx.x * 256 + cx * 8, nn = a.N - n;
  float gamma[8], sb[8], sg[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    gamma[i] = a.gamma && i < nn ? to_f32<T>(static_cast<const T*>(a.gamma)[n + i]) : 1.f;
    sb[i] = sg[i] = 0.f;
  }
  const int r0 = blockIdx.y * a.rows, r1 = min(a.M, r0 + a.rows);
  if (nn > 0) {
    for (int m = r0 + ry; m < r1; m += 8) {
      const int64_t at = (int64_t)m * a.N + n;
      const float rs = a.row_scale ? to_f32<T>(static_cast<const T*>(a.row_scale)[m / a.rows_per_scale]) : 1.f;
      float dy[8], z[8];
#pragma unroll
      for (int e = 0; e < 8; e += E) {
        unpack16<T>(load_some<T>(static_cast<const T*>(a.dy) + at + e, nn - e), dy + e);
        if (a.z) unpack16<T>(load_some<T>(static_cast<const T*>(a.z) + at + e, nn - e), z + e);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float du = dy[e] * rs;
        if (a.part_g || a.dg) sg[e] = fmaf(du, act_of<T>(z[e], a.act), sg[e]);
        dy[e] = du * gamma[e];
        if (a.act != EVE_ACT_IDENTITY) dy[e] *= act_slope<T>(z[e], a.act);
        sb[e] += dy[e];
      }
      if (a.dz) {
#pragma unroll
        for (int e = 0; e < 8; e += E) store_some<T>(static_cast<T*>(a.dz) + at + e, pack16<T>(dy + e), nn - e);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    red[0][ry][cx * 8 + i] = sb[i];
    red[1][ry][cx * 8 + i] = sg[i];
  }
  __syncthreads();
  const int c = threadIdx.x, nc = blockIdx.x * 256 + c;
  if (nc < a.N) {
    float b = 0.f, g = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      b += red[0][r][c];
      g += red[1][r][c];
    }
    if (a.part_b) a.part_b[(int64_t)blockIdx.y * a.N + nc] = b;
    if (a.part_g) a.part_g[(int64_t)blockIdx.y * a.N + nc] = g;
    if (a.db) static_cast<T*>(a.db)[nc] = from_f32<T>(b);
    if (a.dg) static_cast<T*>(a.dg)[nc] = from_f32<T>(g);
  }
#endif
}

// The sums that close a backward, one launch: dW as the sum of its splits (blocks from 0 on, 1024 elements each), and the column
// sums dbias and dgamma, many parts of few columns (32 columns a block, 8 runs of parts); each in a fixed order.
struct SumArgs {
  const float *part_w, *part_c[2];
  void *dw, *dc[2];  // null: not asked for
  int64_t n_w;
  int parts_w, n_c, parts_c, blocks_w, blocks_c;
};
template <typename T>
__global__ __launch_bounds__(256) void linear_sum_kernel(SumArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ float red[8][32];
  if ((int)blockIdx.x < a.blocks_w) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (i + 4 <= a.n_w && (a.n_w & 3) == 0) {
#pragma unroll 4
      for (int q = 0; q < a.parts_w; ++q) {
        const float4 x = *reinterpret_cast<const float4*>(a.part_w + q * a.n_w + i);
        s[0] += x.x;
        s[1] += x.y;
        s[2] += x.z;
        s[3] += x.w;
      }
    } else {
      for (int e = 0; e < 4; ++e)
        if (i + e < a.n_w)
          for (int q = 0; q < a.parts_w; ++q) s[e] += a.part_w[q * a.n_w + i + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < a.n_w) static_cast<T*>(a.dw)[i + e] = from_f32<T>(s[e]);
    return;
  }
  const int bid = blockIdx.x - a.blocks_w, which = bid / a.blocks_c;
  const float* p = which ? a.part_c[1] : a.part_c[0];
  T* o = static_cast<T*>(which ? a.dc[1] : a.dc[0]);
  if (!o) return;
  const int c = threadIdx.x & 31, run = threadIdx.x >> 5, n = bid % a.blocks_c * 32 + c, len = (a.parts_c + 7) / 8;
  float s = 0.f;
  if (n < a.n_c) {
#pragma unroll 8
    for (int q = run * len; q < min(a.parts_c, (run + 1) * len); ++q) s += p[(int64_t)q * a.n_c + n];
  }
  red[run][c] = s;
  __syncthreads();
  if (run == 0 && n < a.n_c) {
#pragma unroll
    for (int r = 1; r < 8; ++r) s += red[r][c];
    o[n] = from_f32<T>(s);
  }
#endif
}

// ---------------------------------------------------------------------------------------------------------- host
namespace {

constexpr int kFewRows = 4;

int lin_cus() {
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

int check_dims(int rows, int T, int K, int N, int act, int dtype) {
  EVE_REQUIRE(dtype == EVE_F32 || dtype == EVE_BF16, EVE_ERR_ARG, "eve_linear: dtype %d", dtype);
  EVE_REQUIRE(act >= EVE_ACT_QUICK_GELU && act <= EVE_ACT_IDENTITY, EVE_ERR_ARG, "eve_linear: activation %d", act);
  EVE_REQUIRE(rows >= 0 && K >= 0 && N >= 0 && T >= 1, EVE_ERR_ARG, "eve_linear: negative size");
  EVE_REQUIRE(rows <= 0x7ff00000 && K <= (1 << 24) && N <= (1 << 24), EVE_ERR_UNSUPPORTED, "eve_linear: too large");
  return EVE_OK;
}

// Which kernel a product runs on: the rows of the streaming kernel's tile, or (negative) the edge of the general one's.
// The streaming kernel wants 16-byte rows.  Its tile -- 192 rows (256 of a k-major A) or 128, which has 15 % more LDS traffic a row --
// is the one whose fullest CU has less to do: 15168 x 768 is 474 tiles of 192 rows (64 us for a contraction of 2304), 714 of 128
// (70 us), 360 of 256 (74 us: two on some CUs, one on others).  Problems of fewer tiles go to the general kernel's 64 x 64 tiles;
// in float32, which the matrix unit bounds, wherever the CUs have less to do so (400 rows of 1024 -> 4096: 44 us instead of 71).
bool rows16(const void* p, int ld, int size) { return ((uintptr_t)p & 15) == 0 && (int64_t)ld * size % 16 == 0 && ld < (1 << 20); }
int choose_tile(bool aligned, bool acol, int64_t M, int64_t N, int64_t splits, int size, int cus) {
  const int64_t tn = (N + 127) / 128 * splits;
  if ((M + 127) / 128 * tn < cus / 2) return -64;
  if (size == 4 && !acol) {
    const int64_t n64 = (M + 63) / 64 * ((N + 63) / 64), n128 = (M + 127) / 128 * tn;
    if ((n64 > cus ? n64 : cus) * 29 < (n128 > cus ? n128 : cus) * 67) return -64;
  }
  if (!aligned) return -128;
  const int large = acol ? 256 : 192;
  const int64_t n_large = (M + large - 1) / large * tn, n_small = (M + 127) / 128 * tn;
  return (n_large + cus - 1) / cus * large * 100 <= (n_small + cus - 1) / cus * 128 * 115 ? large : 128;
}
bool product_aligned(const LinArgs& a, bool acol, bool bcol, int size) {
  // (a k-major operand's chunks run along its rows or columns of the result)
  return rows16(a.A, a.lda, size) && rows16(a.B, a.ldb, size) && rows16(a.C, a.N, size) && (int64_t)a.K * size % 16 * (acol && bcol ? 0 : 1) == 0 &&
         (!acol || (int64_t)a.M * size % 16 == 0) && rows16(a.residual, a.N, size) && rows16(a.z, a.N, size) && rows16(a.bias, a.N, size) && rows16(a.gamma, a.N, size);
}

template <typename T, int BT, bool ACOL, bool BCOL, int MODE>
int launch_tile(const LinArgs& a, hipStream_t st) {
  const int64_t total = (int64_t)((a.M + BT - 1) / BT) * ((a.N + BT - 1) / BT) * a.nsplit;
  EVE_REQUIRE(total <= kMaxThreads / tile_threads<BT>() - 8, EVE_ERR_UNSUPPORTED, "eve_linear: too many tiles");
  constexpr int lds = 2 * 2 * BT * 128 > 4 * 32 * (BT / 2 + 4) * 4 ? 2 * 2 * BT * 128 : 4 * 32 * (BT / 2 + 4) * 4;
  linear_tile_kernel<T, BT, ACOL, BCOL, MODE><<<dim3((unsigned)((total + 7) / 8 * 8)), dim3(tile_threads<BT>()), lds, st>>>(a);
  EVE_CHECK_LAUNCH("eve_linear (product)");
  return EVE_OK;
}
template <typename T, int BM, bool ACOL, bool BCOL, int MODE, int ACT = EVE_ACT_IDENTITY>
int launch_stream(LinArgs a, hipStream_t st) {
  const int tn = ceil_div(a.N, kStreamN);
  const int64_t total = (int64_t)ceil_div(a.M, BM) * tn * a.nsplit;
  EVE_REQUIRE(total <= kMaxThreads / 256 - 8, EVE_ERR_UNSUPPORTED, "eve_linear: too many tiles");
  // half an L2 (2 MiB) of B a group, and groups of equal width
  const int64_t panel = (int64_t)kStreamN * (MODE == LIN_PART ? a.kspan : a.K) * (int)sizeof(T);
  int width = (int)((2 << 20) / (panel > 0 ? panel : 1));
  width = width < 1 ? 1 : width > tn ? tn : width;
  a.ngroup = ceil_div(tn, ceil_div(tn, width));
  constexpr int lds = stream_lds<BM>();
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(linear_stream_kernel<T, BM, ACOL, BCOL, MODE, ACT>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    EVE_REQUIRE(e == hipSuccess, EVE_ERR_LAUNCH, "eve_linear: %d bytes of LDS: %s", lds, hipGetErrorString(e));
  }
  linear_stream_kernel<T, BM, ACOL, BCOL, MODE, ACT><<<dim3((unsigned)((total + 7) / 8 * 8)), dim3(256), lds, st>>>(a);
  EVE_CHECK_LAUNCH("eve_linear (product)");
  return EVE_OK;
}
template <typename T, int BM, bool ACOL, bool BCOL, int MODE>
int launch_stream_act(const LinArgs& a, hipStream_t st) {
  if constexpr (MODE == LIN_FWD) {
    switch (a.act) {
      case EVE_ACT_QUICK_GELU: return launch_stream<T, BM, ACOL, BCOL, MODE, EVE_ACT_QUICK_GELU>(a, st);
      case EVE_ACT_GELU: return launch_stream<T, BM, ACOL, BCOL, MODE, EVE_ACT_GELU>(a, st);
      case EVE_ACT_RELU: return launch_stream<T, BM, ACOL, BCOL, MODE, EVE_ACT_RELU>(a, st);
      default: break;
    }
  }
  return launch_stream<T, BM, ACOL, BCOL, MODE>(a, st);
}
template <typename T, bool ACOL, bool BCOL, int MODE>
int product(const LinArgs& a, int tile, hipStream_t st) {
  constexpr int LARGE = ACOL ? 256 : 192;
  switch (tile) {
    case LARGE: return launch_stream_act<T, LARGE, ACOL, BCOL, MODE>(a, st);
    case 128: return launch_stream_act<T, 128, ACOL, BCOL, MODE>(a, st);
    case -128: return launch_tile<T, 128, ACOL, BCOL, MODE>(a, st);
    default: return launch_tile<T, 64, ACOL, BCOL, MODE>(a, st);
  }
}

// Problems of few 64 x 64 tiles leave CUs idle while a long contraction goes by; then tiles of 16 or 32, whose contraction a
// workgroup's waves share, are quicker.  A tile takes a CU 10 (16 x 16), 21 (32 x 32) and 41 or, in float32, 72 (64 x 64); a launch
// takes its tiles over the CUs, one tile at least (32 x 32: whole rounds, as two at a time on a CU gain it nothing): 40 rows of 4096 -> 1024 in bf16 take 9.6, 17 and 29 us, in float32 17, 33 and 101;
// 400 rows 52, 31 and 31 us; 617 rows of 768 -> 2304 in float32 65, 47 and 35.
// -> 1 or 2 (tiles of 16 of a side), 0: the general kernel.  A larger tile is kept unless a tenth is gained.
int shared_tiles(int64_t M, int64_t N, int cost64, int cus) {
  auto cost = [&](int r, int tile) {
    const int64_t n = ((M + r - 1) / r) * ((N + r - 1) / r);
    if (r == 32) return (n + cus - 1) / cus * cus * tile;
    return (n > cus ? n : cus) * tile;
  };
  const int64_t c64 = cost(64, cost64), c32 = cost(32, 21), c16 = cost(16, 10);
  const int ntl = c32 * 11 < c64 * 10 ? 2 : 0;
  return c16 * 11 < (ntl ? c32 : c64) * 10 ? 1 : ntl;
}
template <typename T, int NTL>
int launch_shared(const LinArgs& a, hipStream_t st) {
  constexpr int R = 16 * NTL;
  const int64_t total = (int64_t)((a.M + R - 1) / R) * ((a.N + R - 1) / R);
  EVE_REQUIRE(total <= kMaxThreads / 512 - 8, EVE_ERR_UNSUPPORTED, "eve_linear: too many tiles");
  linear_shared_kernel<T, NTL><<<dim3((unsigned)((total + 7) / 8 * 8)), dim3(512), 0, st>>>(a);
  EVE_CHECK_LAUNCH("eve_linear_fwd (shared contraction)");
  return EVE_OK;
}

template <typename T>
int fwd_typed(const LinArgs& a, hipStream_t st) {
  if (a.M <= kFewRows) {
    const dim3 grid((a.N + 3) / 4), block(256);
    if (a.M == 1) linear_few_kernel<T, 1><<<grid, block, 0, st>>>(a);
    else if (a.M == 2) linear_few_kernel<T, 2><<<grid, block, 0, st>>>(a);
    else linear_few_kernel<T, 4><<<grid, block, 0, st>>>(a);
    EVE_CHECK_LAUNCH("eve_linear_fwd (few rows)");
    return EVE_OK;
  }
  const int tile = choose_tile(product_aligned(a, false, false, sizeof(T)), false, a.M, a.N, 1, sizeof(T), lin_cus());
  if (tile == -64) {
    const int ntl = shared_tiles(a.M, a.N, sizeof(T) == 2 ? 41 : 72, lin_cus());
    if (ntl == 1) return launch_shared<T, 1>(a, st);
    if (ntl == 2) return launch_shared<T, 2>(a, st);
  }
  return product<T, false, false, LIN_FWD>(a, tile, st);
}

struct BwdPlan { int dz_rows, parts, nsplit, kspan; size_t dz, part_b, part_g, part_w, part_s, bytes; };

BwdPlan bwd_plan(int rows, int K, int N, int dtype, int cus) {
  BwdPlan p;
  const size_t size = dtype == EVE_BF16 ? 2 : 4;
  // rows of a dz block: 32 (128: 29 us for 15168 x 768 of bf16, too few workgroups), fewer until there are four workgroups a CU
  // (1899 x 1001 of float32: 32 rows 21.7 us, 8 rows 14.1); up to 64 rows are one part, which needs no launch for sums
  p.dz_rows = 32;
  while (p.dz_rows > 8 && (int64_t)ceil_div(N, 256) * ceil_div(rows, p.dz_rows) < 4 * (int64_t)cus) p.dz_rows /= 2;
  if (rows <= 64) p.dz_rows = 64;
  while (ceil_div(rows, p.dz_rows) > 32768) p.dz_rows *= 2;
  p.parts = ceil_div(rows, p.dz_rows);
  // dW [N, K]: the contraction over the rows is split until there are about two tiles of 256 x 128 a CU, 256 rows each at least; one
  // a CU if that leaves few idle and no more than 1280 rows a split, where the parts cost more than the company on a CU gives.  15168
  // rows, 768 x 768 (18 tiles): 14 splits 35 us with the sums, 28 splits 41; 2304 x 768 (54): 4 splits 105 and 6 us,
  // 9 splits 69 and 11; off 16-byte boundaries, 8000 rows, 2047 x 1023 (64): 4 splits 215 us in all, 8 splits 180.  (The bound of 1280
  // rows is for those: on 16-byte boundaries it changes little, 15168 rows, 2048 x 1024: 4 splits 80 us, 8 splits 81; 10000 rows: 61 and 63.)
  // (Float32 off 16-byte boundaries goes by its tiles of 128 x 128, as the matrix unit bounds it: 1899 rows, 1001 x 750: 5 splits 45 us
  // and 8, 6 splits 55 and 9; 8000 rows, 2047 x 1023: 4 splits 337 us in all, 8 splits 368.)
  const bool large = size == 2 || ((size_t)N * size % 16 == 0 && (size_t)K * size % 16 == 0);
  const int64_t tiles = (int64_t)ceil_div(N, large ? 256 : 128) * ceil_div(K, 128);
  int64_t want = tiles > 0 ? cus / tiles : 1;
  if (want * tiles * 16 < (int64_t)cus * 15 || rows > 1280 * want) want = tiles > 0 ? 2 * (int64_t)cus / tiles : 1;
  if (want > rows / 256) want = rows / 256;
  if (want < 1) want = 1;
  p.kspan = (int)align_up((size_t)((rows + want - 1) / want), 64);
  if (p.kspan < 64) p.kspan = 64;
  p.nsplit = rows > 0 ? ceil_div(rows, p.kspan) : 1;
  p.dz = 0;
  p.part_b = p.dz + align_up((size_t)rows * N * size, 256);
  p.part_g = p.part_b + align_up((size_t)p.parts * N * 4, 256);
  p.part_w = p.part_g + align_up((size_t)p.parts * N * 4, 256);
  p.part_s = p.part_w + (p.nsplit > 1 ? align_up((size_t)p.nsplit * N * K * 4, 256) : 0);
  p.bytes = p.part_s + align_up((size_t)p.nsplit * N * 4, 256);
  return p;
}

template <typename T>
int bwd_typed(const DzArgs& dzin, const void* x, const void* w, void* dx, void* dw, void* dbias, void* dgamma, int K, char* ws,
              const BwdPlan& p, hipStream_t st) {
  DzArgs d = dzin;
  const int rows = d.M, N = d.N;
  d.rows = p.dz_rows;
  const bool plain = d.act == EVE_ACT_IDENTITY && !d.gamma && !d.row_scale;  // dz = dy
  LinArgs w_ = {};
  w_.A = plain ? d.dy : ws + p.dz; w_.B = x; w_.C = dw; w_.M = N; w_.N = K; w_.K = rows; w_.lda = N; w_.ldb = K;
  w_.nsplit = p.nsplit; w_.kspan = p.kspan; w_.part = reinterpret_cast<float*>(ws + p.part_w);
  const int tile_w = choose_tile(product_aligned(w_, true, true, sizeof(T)), true, N, K, p.nsplit, sizeof(T), lin_cus());
  // dz = dy: dbias is summed by the dW product while it has dy in registers, where the streaming kernel runs it
  const bool with_dw = plain && dbias && dw && !dgamma && tile_w > 0 && rows > 0 && N > 0 && K > 0;
  if (with_dw) w_.part_bias = reinterpret_cast<float*>(ws + p.part_s);
  d.dz = plain || !(dx || dw) ? nullptr : ws + p.dz;
  const bool direct = p.parts == 1 && !with_dw;
  d.db = direct ? dbias : nullptr;
  d.dg = direct ? dgamma : nullptr;
  d.part_b = dbias && !with_dw && !direct ? reinterpret_cast<float*>(ws + p.part_b) : nullptr;
  d.part_g = dgamma && !direct ? reinterpret_cast<float*>(ws + p.part_g) : nullptr;
  if (N > 0 && rows > 0 && (d.dz || d.part_b || d.part_g || d.db || d.dg)) {
    linear_dz_kernel<T><<<dim3(ceil_div(N, 256), p.parts), dim3(256), 0, st>>>(d);
    EVE_CHECK_LAUNCH("eve_linear_bwd (dz)");
  }
  const void* dz = plain ? d.dy : d.dz;
  if (dx && rows > 0 && K > 0) {
    LinArgs a = {};
    a.A = dz; a.B = w; a.C = dx; a.M = rows; a.N = K; a.K = N; a.lda = N; a.ldb = K; a.nsplit = 1;
    const int rc = product<T, false, true, LIN_PLAIN>(a, choose_tile(product_aligned(a, false, true, sizeof(T)), false, rows, K, 1, sizeof(T), lin_cus()), st);
    if (rc != EVE_OK) return rc;
  }
  if (dw && N > 0 && K > 0) {
    int rc = p.nsplit == 1 ? product<T, true, true, LIN_PLAIN>(w_, tile_w, st) : product<T, true, true, LIN_PART>(w_, tile_w, st);
    if (rc != EVE_OK) return rc;
  }
  SumArgs s = {};
  if (dw && N > 0 && K > 0 && p.nsplit > 1) {
    s.part_w = w_.part; s.dw = dw; s.n_w = (int64_t)N * K; s.parts_w = p.nsplit;
    s.blocks_w = (int)((s.n_w + 1023) / 1024);
  }
  s.blocks_c = 1;
  if (N > 0 && (dbias || dgamma) && !direct) {
    s.part_c[0] = with_dw ? w_.part_bias : d.part_b; s.part_c[1] = d.part_g; s.dc[0] = dbias; s.dc[1] = dgamma;
    s.n_c = N; s.parts_c = with_dw ? p.nsplit : p.parts; s.blocks_c = ceil_div(N, 32);
  }
  const int64_t blocks = s.blocks_w + (s.n_c ? 2 * (int64_t)s.blocks_c : 0);
  EVE_REQUIRE(blocks <= kMaxThreads / 256, EVE_ERR_UNSUPPORTED, "eve_linear: too many weights");
  if (blocks > 0) {
    linear_sum_kernel<T><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(s);
    EVE_CHECK_LAUNCH("eve_linear_bwd (sums)");
  }
  return EVE_OK;
}

}  // namespace
}  // namespace eve

using namespace eve;

extern "C" int eve_linear_fwd(const void* x, const void* w, const void* bias, const void* gamma, const void* row_scale,
                              const void* residual, void* y, void* z, int rows, int rows_per_scale, int K, int N, int act, int dtype,
                              void* stream) {
  const int rc = check_dims(rows, rows_per_scale, K, N, act, dtype);
  if (rc != EVE_OK) return rc;
  if (rows == 0 || N == 0) return EVE_OK;
  EVE_REQUIRE(y && (K == 0 || (x && w)), EVE_ERR_ARG, "eve_linear_fwd: null pointer");
  LinArgs a = {};
  a.A = x; a.B = w; a.C = y; a.M = rows; a.N = N; a.K = K; a.lda = K; a.ldb = K; a.nsplit = 1;
  a.bias = bias; a.gamma = gamma; a.row_scale = row_scale; a.residual = residual; a.z = z;
  a.rows_per_scale = rows_per_scale; a.act = act;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == EVE_BF16 ? fwd_typed<bf16_t>(a, st) : fwd_typed<float>(a, st);
}

extern "C" size_t eve_linear_bwd_workspace_bytes(int rows, int K, int N, int dtype) {
  if (check_dims(rows, 1, K, N, EVE_ACT_IDENTITY, dtype) != EVE_OK) return 0;
  return bwd_plan(rows, K, N, dtype, lin_cus()).bytes;
}

extern "C" int eve_linear_bwd(const void* dy, const void* x, const void* w, const void* z, const void* gamma,
                              const void* row_scale, void* dx, void* dw, void* dbias, void* dgamma, int rows, int rows_per_scale,
                              int K, int N, int act, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_dims(rows, rows_per_scale, K, N, act, dtype);
  if (rc != EVE_OK) return rc;
  EVE_REQUIRE(rows == 0 || N == 0 || dy, EVE_ERR_ARG, "eve_linear_bwd: null gradient");
  EVE_REQUIRE(rows == 0 || N == 0 || K == 0 || ((!dx || w) && (!dw || x)), EVE_ERR_ARG, "eve_linear_bwd: null operand");
  EVE_REQUIRE(rows == 0 || N == 0 || z || (act == EVE_ACT_IDENTITY && !dgamma), EVE_ERR_ARG,
              "eve_linear_bwd: the activation's and gamma's gradients need z");
  const BwdPlan p = bwd_plan(rows, K, N, dtype, lin_cus());
  EVE_REQUIRE(p.bytes == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= p.bytes), EVE_ERR_WORKSPACE,
              "eve_linear_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, p.bytes);
  DzArgs d = {};
  d.dy = dy; d.z = z; d.gamma = gamma; d.row_scale = row_scale; d.M = rows; d.N = N; d.rows_per_scale = rows_per_scale; d.act = act;
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  return dtype == EVE_BF16 ? bwd_typed<bf16_t>(d, x, w, dx, dw, dbias, dgamma, K, ws, p, st)
                           : bwd_typed<float>(d, x, w, dx, dw, dbias, dgamma, K, ws, p, st);
}
