// The matrix products around the encoder's attention (reference models/multiway_transformer.py:104-106, :129-130, :341), gfx950:
//   z = x W^T + bias,   u = act(z),   y = residual + row_scale[row / T] gamma u
// with everything after the product done on the fp32 accumulator in the epilogue, and the gradient
//   dz = dy row_scale gamma act'(z)   (one pass, with the column sums dbias = sum dz, dgamma = sum dy row_scale u)
//   dx = dz W,   dW = dz^T x.
//
// One tile kernel serves the three products.  An operand is row-major (its contraction index is contiguous in memory: x, W in the
// forward, dz in dx) or k-major (the contraction index is the row: W in dx, dz and x in dW).  Row-major tiles lie in LDS as
// [rows][128 bytes] and are read as 16-byte fragments; k-major tiles lie as in memory, [k][columns], and are transposed on the
// way to the matrix unit (bf16: ds_read_b64_tr_b16).  Chunks of 16 bytes are XOR-swizzled so that either read spreads over the
// banks.  Any size goes: what lies outside an operand arrives as zeros, rows need no alignment.
// dW has few tiles and a long contraction (the rows of the batch): it is split, with fp32 parts added in order.
#include "act.h"
#include "common.h"

namespace eve {

typedef __attribute__((ext_vector_type(8))) __bf16 li_bf16x8;
typedef __attribute__((ext_vector_type(4))) short li_s16x4;
typedef __attribute__((ext_vector_type(8))) short li_s16x8;
typedef __attribute__((ext_vector_type(16))) float li_f32x16;

enum { LIN_FWD = 0, LIN_PLAIN = 1, LIN_PART = 2 };

struct LinArgs {
  const void *A, *B;       // operands; rows of the result come from A, columns from B
  void* C;                 // [M, N] of the type
  float* part;             // LIN_PART: [nsplit][M][N]
  int M, N, K, lda, ldb;
  int nsplit, ksteps;      // LIN_PART: splits of the contraction, tile steps of each
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
template <typename T, bool COL, int W> struct LinTile {
  static constexpr int E = LT<T>::E, BK = LT<T>::BK;
  static constexpr int BYTES = W * 128;
  static constexpr int N = BYTES / 16 / 256;
  uint4 w[N];
  // ext: rows (columns) of the operand from the tile's first on; kext: contraction indices from the step's first on
  __device__ __forceinline__ void load(const T* p, int64_t ld, int ext, int kext, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * 256;
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
      const int idx = tid + i * 256;
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

// BT x BT tile, 4 waves of (BT/2) x (BT/2); two LDS stages, the next step's tiles in registers meanwhile.
template <typename T, int BT, bool ACOL, bool BCOL, int MODE>
__global__ __launch_bounds__(256) void linear_tile_kernel(LinArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BK = LT<T>::BK, E = LT<T>::E, NT = BT / 64, NKS = BK / (2 * E);
  constexpr int STAGE = 2 * BT * 128;
  constexpr int EP = BT / 2 + 4;  // floats of a row of a wave's epilogue image
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  // Workgroups go round-robin over the 8 XCDs: each of them gets a run of tiles, columns fastest, so that the tiles it works on
  // at a time share a few row panels of A through its L2.
  const int tm = (a.M + BT - 1) / BT, tn = (a.N + BT - 1) / BT, total = tm * tn * a.nsplit;
  const int per = (total + 7) >> 3;
  const int item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || item >= total) return;
  const int split = item / (tm * tn), tile = item % (tm * tn);
  const int m0 = (tile / tn) * BT, n0 = (tile % tn) * BT;
  const int k0 = MODE == LIN_PART ? split * a.ksteps * BK : 0;
  const int k1 = MODE == LIN_PART ? min(a.K, k0 + a.ksteps * BK) : a.K;

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

  LinTile<T, ACOL, BT> ta;
  LinTile<T, BCOL, BT> tb;
  const int steps = (k1 - k0 + BK - 1) / BK;
  auto fetch = [&](int t) {
    ta.load(Ap + t * sa, a.lda, a.M - m0, k1 - k0 - t * BK, tid);
    tb.load(Bp + t * sb, a.ldb, a.N - n0, k1 - k0 - t * BK, tid);
  };
  if (steps > 0) fetch(0);
  for (int t = 0; t < steps; ++t) {
    char* as = smem + (t & 1) * STAGE;
    char* bs = as + BT * 128;
    ta.store(as, tid);
    tb.store(bs, tid);
    __syncthreads();
    if (t + 1 < steps) fetch(t + 1);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      uint4 fa[NT], fb[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) fa[i] = lfrag<T, ACOL, BT>(as, wm * (BT / 2) + 32 * i, ks, lane);
#pragma unroll
      for (int j = 0; j < NT; ++j) fb[j] = lfrag<T, BCOL, BT>(bs, wn * (BT / 2) + 32 * j, ks, lane);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = lmma(fa[i], fb[j], acc[i][j], T());
    }
  }
  __syncthreads();  // the stages become the waves' epilogue images

  // 32 rows at a time through the wave's own image, then 8 columns of a row a lane
  constexpr int CH = BT / 2 / 8, RPI = 64 / CH;  // chunks of 8 columns of an image row; rows a pass
  float* img = reinterpret_cast<float*>(smem) + wave * 32 * EP;
  const int ch = lane % CH, n = n0 + wn * (BT / 2) + ch * 8, nn = a.N - n;
  float bias[8], gamma[8];
  if constexpr (MODE == LIN_FWD) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bias[i] = a.bias && i < nn ? to_f32<T>(static_cast<const T*>(a.bias)[n + i]) : 0.f;
      gamma[i] = a.gamma && i < nn ? to_f32<T>(static_cast<const T*>(a.gamma)[n + i]) : 1.f;
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) img[((r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) * EP + 32 * j + (lane & 31)] = acc[i][j][r];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the image is the wave's own: no barrier, but its lanes exchange through it
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int it = 0; it < 32 / RPI; ++it) {
      const int rr = it * RPI + lane / CH, m = m0 + wm * (BT / 2) + 32 * i + rr;
      float v[8];
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(img + rr * EP + ch * 8);
      *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(img + rr * EP + ch * 8 + 4);
      if (m < a.M && nn > 0) {
        const int64_t at = (int64_t)m * a.N + n;
        if constexpr (MODE == LIN_PART) {
          float* p = a.part + (int64_t)split * a.M * a.N + at;
          store_some<float>(p, __builtin_bit_cast(uint4, *reinterpret_cast<float4*>(v)), nn);
          store_some<float>(p + 4, __builtin_bit_cast(uint4, *reinterpret_cast<float4*>(v + 4)), nn - 4);
        } else {
          if constexpr (MODE == LIN_FWD) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += bias[e];
            if (a.z) {
#pragma unroll
              for (int e = 0; e < 8; e += E) store_some<T>(static_cast<T*>(a.z) + at + e, pack16<T>(v + e), nn - e);
            }
            if (a.act != EVE_ACT_IDENTITY) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = act_of<T>(v[e], a.act);
            }
            const float rs = a.row_scale ? to_f32<T>(static_cast<const T*>(a.row_scale)[m / a.rows_per_scale]) : 1.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= gamma[e] * rs;
            if (a.residual) {
#pragma unroll
              for (int e = 0; e < 8; e += E) {
                float r[E];
                unpack16<T>(load_some<T>(static_cast<const T*>(a.residual) + at + e, nn - e), r);
#pragma unroll
                for (int f = 0; f < E; ++f) v[e + f] += r[f];
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 8; e += E) store_some<T>(static_cast<T*>(a.C) + at + e, pack16<T>(v + e), nn - e);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
#endif
}

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
    const int64_t at = (int64_t)lane * a.N + n;
    if (a.bias) v += to_f32<T>(static_cast<const T*>(a.bias)[n]);
    if (a.z) static_cast<T*>(a.z)[at] = from_f32<T>(v);
    v = act_of<T>(v, a.act);
    if (a.gamma) v *= to_f32<T>(static_cast<const T*>(a.gamma)[n]);
    if (a.row_scale) v *= to_f32<T>(static_cast<const T*>(a.row_scale)[lane / a.rows_per_scale]);
    if (a.residual) v += to_f32<T>(static_cast<const T*>(a.residual)[at]);
    static_cast<T*>(a.C)[at] = from_f32<T>(v);
  }
#endif
}

// dz and the column sums of its terms.  Block: 32 chunks of 8 columns x 8 row lanes, over kDzRows rows; the row lanes are added
// in order and each block row leaves one part.
struct DzArgs {
  const void *dy, *z, *gamma, *row_scale;
  void* dz;                 // may be null (dz = dy)
  float *part_b, *part_g;   // [parts][N], either may be null
  int M, N, rows_per_scale, act;
};
constexpr int kDzRows = 128;
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
  const int r0 = blockIdx.y * kDzRows, r1 = min(a.M, r0 + kDzRows);
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
        if (a.part_g) sg[e] = fmaf(du, act_of<T>(z[e], a.act), sg[e]);
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
  }
#endif
}

// out[i] = sum over the parts, in order; blockIdx.y picks one of two problems
struct SumArgs { const float* part[2]; void* out[2]; int64_t n; int parts; };
template <typename T>
__global__ __launch_bounds__(256) void linear_sum_kernel(SumArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const float* p = blockIdx.y ? a.part[1] : a.part[0];
  T* o = static_cast<T*>(blockIdx.y ? a.out[1] : a.out[0]);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (!o || i >= a.n) return;
  float s = 0.f;
#pragma unroll 8
  for (int q = 0; q < a.parts; ++q) s += p[q * a.n + i];
  o[i] = from_f32<T>(s);
#endif
}

// ---------------------------------------------------------------------------------------------------------- host
namespace {

constexpr int kFewRows = 8;

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

int tile_edge(int64_t M, int64_t N, int64_t splits, int cus) {
  return ((M + 127) / 128) * ((N + 127) / 128) * splits >= cus ? 128 : 64;
}

template <typename T, int BT, bool ACOL, bool BCOL, int MODE>
int launch_tile(const LinArgs& a, hipStream_t st) {
  const int64_t total = (int64_t)((a.M + BT - 1) / BT) * ((a.N + BT - 1) / BT) * a.nsplit;
  EVE_REQUIRE(total <= 0x7ffffff0LL, EVE_ERR_UNSUPPORTED, "eve_linear: too many tiles");
  constexpr int lds = 2 * 2 * BT * 128 > 4 * 32 * (BT / 2 + 4) * 4 ? 2 * 2 * BT * 128 : 4 * 32 * (BT / 2 + 4) * 4;
  linear_tile_kernel<T, BT, ACOL, BCOL, MODE><<<dim3((unsigned)((total + 7) / 8 * 8)), dim3(256), lds, st>>>(a);
  EVE_CHECK_LAUNCH("eve_linear (product)");
  return EVE_OK;
}
template <typename T, bool ACOL, bool BCOL, int MODE>
int product(const LinArgs& a, int edge, hipStream_t st) {
  return edge == 128 ? launch_tile<T, 128, ACOL, BCOL, MODE>(a, st) : launch_tile<T, 64, ACOL, BCOL, MODE>(a, st);
}

template <typename T>
int fwd_typed(const LinArgs& a, hipStream_t st) {
  if (a.M <= kFewRows) {
    const dim3 grid((a.N + 3) / 4), block(256);
    if (a.M == 1) linear_few_kernel<T, 1><<<grid, block, 0, st>>>(a);
    else if (a.M == 2) linear_few_kernel<T, 2><<<grid, block, 0, st>>>(a);
    else if (a.M <= 4) linear_few_kernel<T, 4><<<grid, block, 0, st>>>(a);
    else linear_few_kernel<T, 8><<<grid, block, 0, st>>>(a);
    EVE_CHECK_LAUNCH("eve_linear_fwd (few rows)");
    return EVE_OK;
  }
  return product<T, false, false, LIN_FWD>(a, tile_edge(a.M, a.N, 1, lin_cus()), st);
}

struct BwdPlan { int parts, edge_w, nsplit, ksteps; size_t dz, part_b, part_g, part_w, bytes; };

BwdPlan bwd_plan(int rows, int K, int N, int dtype, int cus) {
  BwdPlan p;
  const size_t size = dtype == EVE_BF16 ? 2 : 4;
  const int bk = dtype == EVE_BF16 ? 64 : 32;
  p.parts = ceil_div(rows, kDzRows);
  const int steps = ceil_div(rows, bk);
  // dW [N, K]: the contraction over the rows is split until there are about two tiles a CU, with at least four steps each
  const int64_t t128 = (int64_t)ceil_div(N, 128) * ceil_div(K, 128);
  int64_t want = t128 > 0 ? 2 * (int64_t)cus / t128 : 1;
  if (want > steps / 4) want = steps / 4;
  if (want < 1) want = 1;
  p.edge_w = tile_edge(N, K, want, cus);
  p.ksteps = (int)((steps + want - 1) / want);
  if (p.ksteps < 1) p.ksteps = 1;
  p.nsplit = steps > 0 ? ceil_div(steps, p.ksteps) : 1;
  p.dz = 0;
  p.part_b = p.dz + align_up((size_t)rows * N * size, 256);
  p.part_g = p.part_b + align_up((size_t)p.parts * N * 4, 256);
  p.part_w = p.part_g + align_up((size_t)p.parts * N * 4, 256);
  p.bytes = p.part_w + (p.nsplit > 1 ? align_up((size_t)p.nsplit * N * K * 4, 256) : 0);
  return p;
}

template <typename T>
int bwd_typed(const DzArgs& dzin, const void* x, const void* w, void* dx, void* dw, void* dbias, void* dgamma, int K, char* ws,
              const BwdPlan& p, hipStream_t st) {
  DzArgs d = dzin;
  const int rows = d.M, N = d.N;
  const bool plain = d.act == EVE_ACT_IDENTITY && !d.gamma && !d.row_scale;  // dz = dy
  d.dz = plain || !(dx || dw) ? nullptr : ws + p.dz;
  d.part_b = dbias ? reinterpret_cast<float*>(ws + p.part_b) : nullptr;
  d.part_g = dgamma ? reinterpret_cast<float*>(ws + p.part_g) : nullptr;
  if (N > 0 && rows > 0 && (d.dz || dbias || dgamma)) {
    linear_dz_kernel<T><<<dim3(ceil_div(N, 256), p.parts), dim3(256), 0, st>>>(d);
    EVE_CHECK_LAUNCH("eve_linear_bwd (dz)");
  }
  if (N > 0 && (dbias || dgamma)) {
    SumArgs s = {{d.part_b, d.part_g}, {dbias, dgamma}, N, p.parts};
    linear_sum_kernel<T><<<dim3(ceil_div(N, 256), 2), dim3(256), 0, st>>>(s);
    EVE_CHECK_LAUNCH("eve_linear_bwd (column sums)");
  }
  const void* dz = plain ? d.dy : d.dz;
  if (dx && rows > 0 && K > 0) {
    LinArgs a = {};
    a.A = dz; a.B = w; a.C = dx; a.M = rows; a.N = K; a.K = N; a.lda = N; a.ldb = K; a.nsplit = 1;
    const int rc = product<T, false, true, LIN_PLAIN>(a, tile_edge(rows, K, 1, lin_cus()), st);
    if (rc != EVE_OK) return rc;
  }
  if (dw && N > 0 && K > 0) {
    LinArgs a = {};
    a.A = dz; a.B = x; a.C = dw; a.M = N; a.N = K; a.K = rows; a.lda = N; a.ldb = K;
    a.nsplit = p.nsplit; a.ksteps = p.ksteps; a.part = reinterpret_cast<float*>(ws + p.part_w);
    if (p.nsplit == 1) return product<T, true, true, LIN_PLAIN>(a, p.edge_w, st);
    const int rc = product<T, true, true, LIN_PART>(a, p.edge_w, st);
    if (rc != EVE_OK) return rc;
    SumArgs s = {{a.part, nullptr}, {dw, nullptr}, (int64_t)N * K, p.nsplit};
    linear_sum_kernel<T><<<dim3((unsigned)(((int64_t)N * K + 255) / 256)), dim3(256), 0, st>>>(s);
    EVE_CHECK_LAUNCH("eve_linear_bwd (sum of the splits)");
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
