// vt_scaled.h -- scaled int8 operators: linear layers and gated feed-forward
// products with int8 weights (one scale per output channel) and int8 rows (one
// scale per token), and their input gradients. Part of vt_hip_gemm.hip's
// translation unit, whose int8 products they run.
//
//   quantise     top_i = max_k |x_ik|, t_i = top_i / 127,
//                q_ik = round(x_ik * (127 / top_i)), ties to even
//   linear       y_ij = t_i s_j sum_k q_ik W_kj + b_j
//   gated        g, u like y of two weights, h = act(g) u
//   linear_grad  dx_ik = sum_j dy_ij s_j W_kj
//   gated_grad   dx_ik = sum_j dh_ij (u act'(g) sg_j Wg_kj + act(g) su_j Wu_kj)
//
// Weights are in the packed layout of vt_pack_b_i8 with K and N rounded up
// with zeros (scaled_kp, scaled_np). The gate and up projections of a gated
// product are one packed matrix of alternating blocks of 32 columns, so a wave
// that holds a gate column's sums also holds the up column's.

namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v4b __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

// K and N of the packed weights. K in whole pairs of 64-deep slices, from 1024
// on in the 256-deep groups that the persistent kernels take (at most a fifth
// more to read there; at small K it would be up to four times as much). N in
// whole 64-column blocks: the gradient contracts over N in steps of 64, and a
// gated product's 64 columns are 32 of the gate and 32 of the up weight.
__host__ __device__ constexpr int64_t scaled_kp(int64_t K) {
  return K < 1024 ? (K + 127) / 128 * 128 : (K + 255) / 256 * 256;
}
constexpr int64_t scaled_np(int64_t N, bool pair) {
  return pair ? 2 * ((N + 31) / 32 * 32) : (N + 63) / 64 * 64;
}

// Packed column of projection column j (which: 0 gate, 1 up).
__host__ __device__ constexpr int64_t pair_col(int64_t j, int which) {
  return (j >> 5) * 64 + which * 32 + (j & 31);
}

// Float side of packed weights: np scales, np bias terms, and the bound of a
// gated product's gradient terms (pack_bound_kernel).
constexpr int64_t scaled_meta(int64_t np) { return 2 * np + 16; }

enum ElemType { kF32 = VT_TYPE_F32, kF16 = VT_TYPE_F16, kBF16 = VT_TYPE_BF16 };

int64_t elem_size(int type) {
  return type == VT_TYPE_F32 ? 4 : type == VT_TYPE_F16 || type == VT_TYPE_BF16 ? 2 : 1;
}

// ---------------------------------------------------------------------------
// Rows to int8
// ---------------------------------------------------------------------------

// A row's magnitude as an integer that orders like it, NaN above infinity.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

constexpr uint32_t kInfBits = 0x7f800000u;
// Below this magnitude (2^-120) 127 / top would leave float32's range: such a
// row counts as zeros.
constexpr uint32_t kLeastTop = 0x03800000u;

struct RowScale {
  float scale, inv;
};

// The scale of a row whose largest magnitude has these bits. A row that holds
// NaN or an infinity has the scale NaN (and rounds to zeros): its outputs are
// NaN, never a clipped value.
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  RowScale r = {0.0f, 0.0f};
  if (top >= kInfBits) {
    r.scale = __uint_as_float(0x7fc00000u);
  } else if (top >= kLeastTop) {
    const float t = __uint_as_float(top);
    r.scale = t * (1.0f / 127.0f);
    r.inv = 127.0f / t;
  }
  return r;
}

// round(v * inv), ties to even, as the low byte: adding 1.5 * 2^23 rounds at
// the units place. The product is rounded to 32 bits first (no fma).
__device__ __forceinline__ uint32_t round_byte(float v, float inv) {
#pragma clang fp contract(off)
  const float p = v * inv;
  return __float_as_uint(p + 12582912.0f);
}

__device__ __forceinline__ int pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), cd = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
  return (int)(ab | cd << 16);
}

template <int TYPE>
struct Elem;
template <>
struct Elem<kF32> {
  typedef float T;
};
template <>
struct Elem<kF16> {
  typedef _Float16 T;
};
template <>
struct Elem<kBF16> {
  typedef __bf16 T;
};

// 16 elements of a row from `pos`, zero past `len`. Pieces that lie within the
// row are read as 16-byte vectors at any alignment (the target's global loads
// need none; element loads took rows of odd lengths three times as long).
template <int TYPE>
__device__ __forceinline__ void load16(const typename Elem<TYPE>::T *row, int64_t pos, int64_t len, float (&v)[16]) {
  typedef typename Elem<TYPE>::T T;
  constexpr int PER = 16 / sizeof(T);
  if (pos + 16 <= len) {
    typedef T VT __attribute__((ext_vector_type(PER), aligned(sizeof(T))));
#pragma unroll
    for (int i = 0; i < 16 / PER; ++i) {
      const VT x = *(const VT *)(row + pos + i * PER);
#pragma unroll
      for (int e = 0; e < PER; ++e) v[i * PER + e] = (float)x[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = pos + e < len ? (float)row[pos + e] : 0.0f;
  }
}

struct QuantArgs {
  const void *X;
  int8_t *Q;
  float *T;
  int64_t ldx, ldq, K, Kp;
};

template <int THREADS>
__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t *red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
  if (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) m = max(m, red[i]);
  }
  return m;
}

// One workgroup per row; a thread holds NC pieces of 16 elements in registers
// between the maximum and the rounding (NC = 0: longer rows, read twice). Bound
// by one read and half a write of the row and, at small M, by the chain of
// load, reduction and store: 2000 x 4096 bfloat16 in 6.8 us (3.6 TB/s), 333 x
// 1001 float32 in 3.5.
template <int TYPE, int THREADS, int NC>
__global__ __launch_bounds__(THREADS) void quant_rows_kernel(QuantArgs p) {
  __shared__ uint32_t red[THREADS / 64];
  typedef typename Elem<TYPE>::T T;
  const int64_t row = blockIdx.x;
  const T *x = (const T *)p.X + row * p.ldx;
  int8_t *q = p.Q + row * p.ldq;
  const int tid = threadIdx.x;
  float v[NC ? NC : 1][16];
  uint32_t top = 0;
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int64_t pos = (int64_t)(tid + THREADS * i) * 16;
      load16<TYPE>(x, pos, p.K, v[i]);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = max(top, magnitude(v[i][e]));
    }
  } else {
    for (int64_t pos = tid * 16; pos < p.K; pos += THREADS * 16) {
      load16<TYPE>(x, pos, p.K, v[0]);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = max(top, magnitude(v[0][e]));
    }
  }
  top = block_max<THREADS>(top, red);
  const RowScale r = row_scale(top);
  if (tid == 0) p.T[row] = r.scale;
  auto put = [&](int64_t pos, const float (&w)[16]) {
    if (pos >= p.Kp) return;
    v4i o;
#pragma unroll
    for (int d = 0; d < 4; ++d)
      o[d] = r.inv == 0.0f ? 0
                           : pack_bytes(round_byte(w[4 * d], r.inv), round_byte(w[4 * d + 1], r.inv),
                                        round_byte(w[4 * d + 2], r.inv), round_byte(w[4 * d + 3], r.inv));
    *(v4i *)(q + pos) = o;
  };
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) put((int64_t)(tid + THREADS * i) * 16, v[i]);
  } else {
    for (int64_t pos = tid * 16; pos < p.Kp; pos += THREADS * 16) {
      load16<TYPE>(x, pos, p.K, v[0]);
      put(pos, v[0]);
    }
  }
}

// 16 bytes of an int8 row of any pitch and alignment to a row of Kp bytes,
// zeros past K.
__device__ __forceinline__ void pad_piece(const QuantArgs &p, int64_t row, int64_t pos) {
  const int8_t *x = (const int8_t *)p.X + row * p.ldx;
  v4i o = v4i{0, 0, 0, 0};
  if (pos + 16 <= p.K) {
    o = ld_any(x + pos);
  } else {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      uint32_t b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = pos + d * 4 + e < p.K ? (uint32_t)(uint8_t)x[pos + d * 4 + e] : 0u;
      o[d] = (int)(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24);
    }
  }
  *(v4i *)(p.Q + row * p.ldq + pos) = o;
}

__global__ __launch_bounds__(256) void pad_rows_kernel(QuantArgs p) {
  const int64_t pos = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 16;
  if (pos < p.Kp) pad_piece(p, blockIdx.x, pos);
}

// ---------------------------------------------------------------------------
// Packing
// ---------------------------------------------------------------------------

struct ScaledPackArgs {
  const int8_t *W0, *W1;         // [K][ldw], W1 the up projection or null
  const float *s0, *s1, *bias;   // bias null: zeros
  int8_t *Bp;
  float *meta;
  int64_t ldw0, ldw1;
  int K, N, Kp, Np;
};

// One workgroup packs 64 rows of 64 packed columns (any N, pitch and
// alignment: done once per weight, so element loads do).
__global__ __launch_bounds__(256) void pack_scaled_kernel(ScaledPackArgs p) {
  __shared__ int8_t tile[64 * 68];
  const int kb = blockIdx.x, cb = blockIdx.y, tid = threadIdx.x;
  const int c = tid & 63;
  const int pc = cb * 64 + c;
  const int j = p.W1 ? cb * 32 + (c & 31) : pc;
  const bool up = p.W1 && c >= 32;
  const int8_t *w = up ? p.W1 : p.W0;
  const int64_t ldw = up ? p.ldw1 : p.ldw0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = (tid >> 6) + 4 * i, k = kb * 64 + r;
    tile[r * 68 + c] = k < p.K && j < p.N ? w[(int64_t)k * ldw + j] : (int8_t)0;
  }
  if (kb == 0 && tid < 64) {
    const float *s = up ? p.s1 : p.s0;
    p.meta[pc] = j < p.N ? s[j] : 0.0f;
    p.meta[p.Np + pc] = p.bias && j < p.N ? p.bias[j] : 0.0f;
    if (cb == 0 && tid < 16) p.meta[2 * (int64_t)p.Np + tid] = 0.0f;
  }
  __syncthreads();
  const int t = tid >> 6, l = tid & 63;
  v4i v;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t b = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      b |= (uint32_t)(uint8_t)tile[(16 * (l >> 4) + 4 * q + e) * 68 + t * 16 + (l & 15)] << (8 * e);
    v[q] = (int)b;
  }
  const int64_t kbt = p.Kp / 64;
  if (kb < kbt)   // K = 0 has no tiles
    *(v4i *)(p.Bp + (((int64_t)cb * 4 + t) * kbt + kb) * 1024 + l * 16) = v;
}

// meta[2 Np] = max over j of |s_gate s_up| * sum_k |W| of either projection:
// the largest |u sg| or |g su| that rows of t = 1, q = 1 can give. A workgroup
// adds up 64 columns, its waves every fourth row; the maximum of non-negative
// floats is the maximum of their bits, whatever the order.
__global__ __launch_bounds__(256) void pack_bound_kernel(ScaledPackArgs p) {
  __shared__ int32_t part[4][2][64];   // K <= 131071: at most 2^24 a column
  const int c = threadIdx.x & 63, wave = threadIdx.x >> 6, j = blockIdx.x * 64 + c;
  int32_t a0 = 0, a1 = 0;
  if (j < p.N) {
#pragma unroll 8
    for (int k = wave; k < p.K; k += 4) {
      a0 += abs((int)p.W0[(int64_t)k * p.ldw0 + j]);
      a1 += abs((int)p.W1[(int64_t)k * p.ldw1 + j]);
    }
  }
  part[wave][0][c] = a0;
  part[wave][1][c] = a1;
  __syncthreads();
  if (wave) return;
  uint32_t bits = 0;
  if (j < p.N) {
    const int32_t b0 = part[0][0][c] + part[1][0][c] + part[2][0][c] + part[3][0][c];
    const int32_t b1 = part[0][1][c] + part[1][1][c] + part[2][1][c] + part[3][1][c];
    bits = magnitude((float)max(b0, b1) * fabsf(p.s0[j]) * fabsf(p.s1[j]));
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, o));
  if (c == 0) atomicMax((uint32_t *)(p.meta + 2 * (int64_t)p.Np), bits);
}

// ---------------------------------------------------------------------------
// What follows the int32 sums
// ---------------------------------------------------------------------------

// g / (1 + exp(-z)) as (g y) (y / (1 + y^2)) with y = exp(z / 2) = 2^x: a small value
// stays clear of the smallest float32 exponents (which the exponential and the
// reciprocal drop) until it is multiplied by g, and z keeps all of its bits. (32
// added to the exponent instead took those near z = 0: 4.5 roundings of the
// product instead of 1.5.) From y = 2^13 on, y^2 is all of 1 + y^2 in 24 bits. (fmed3
// clamps in one instruction; a NaN reaches the result by its factor g.)
__device__ __forceinline__ float logistic_of(float g, float x) {
  const float y = __builtin_amdgcn_exp2f(__builtin_amdgcn_fmed3f(x, -200.0f, 13.0f));
  return (g * y) * (y * __builtin_amdgcn_rcpf(fmaf(y, y, 1.0f)));
}

// act(g), and its slope. gelu is the tanh form: (1 + tanh z) / 2 is
// 1 / (1 + exp(-2 z)) with z = c (g + a g^3); past |g| = 16 it is 0 or 1, so g
// is held there inside (its cube would leave float32's range). TERMS: for
// gradient terms, which are rounded to steps of 2^-24 of their row's bound or
// more, nothing has to be kept of a value below 2^-126.
template <int ACT, bool TERMS>
__device__ __forceinline__ float act_of(float g, float &slope) {
  const float c = 0.7978845608028654f, a = 0.044715f;
  const float h = ACT == VT_ACT_GELU ? __builtin_amdgcn_fmed3f(g, -16.0f, 16.0f) : g;
  const float hh = h * h, z = ACT == VT_ACT_GELU ? h * fmaf(a, hh, 1.0f) : g;   // gelu: over 2 c
  const float log2e = (ACT == VT_ACT_GELU ? 2.0f * c : 1.0f) * 1.4426950408889634f;
  if constexpr (!TERMS) return logistic_of(g, z * (0.5f * log2e));
  const float p = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -log2e));
  const float dz = ACT == VT_ACT_GELU ? 2.0f * c * fmaf(3.0f * a, hh, 1.0f) : 1.0f;
  slope = p * fmaf(h * dz, 1.0f - p, 1.0f);
  return g * p;
}

// Row normaliser of 16-bit gradient terms: the power of two that takes a bound
// of the row's terms to 2^14 .. 2^15, so no term overflows float16 and terms
// 2^28 below the bound still keep all of its 11 bits. NaN for a row without a
// bound (its gradients are NaN).
__device__ __forceinline__ float normaliser(float bound) {
  const uint32_t b = magnitude(bound);
  if (b >= kInfBits) return __uint_as_float(0x7fc00000u);
  if (b == 0) return 1.0f;
  const int e = (int)(b >> 23) - 127;   // bound < 2^(e + 1)
  return __uint_as_float((uint32_t)(max(-126, min(126, 14 - e)) + 127) << 23);
}

// f(0), f(1), .. f(N - 1) with compile-time arguments.
template <class F, int... I>
__device__ __forceinline__ void each(F &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}

// What becomes of a product's sums: a linear layer's or gated product's output,
// the 16-bit gradient terms of a gated product, or the gradient itself.
enum ScaledOp { kLinear = 0, kGated = 1, kGradTerms = 2, kGrad = 3 };

struct ScaledOut {
  const float *t;      // row scales
  const float *meta;   // channel scales [Np], bias [Np]
  const void *D;       // kGradTerms: dh [M][ldd] of `type`
  const float *norm;   // kGradTerms, kGrad: row normalisers
  void *Y;             // output [M][ldy] of `type`; kGradTerms: float16 terms [M][Np]
  int64_t ldy, ldd;
  int64_t lo;          // kGradTerms: elements from the high to the low halves, 0 for none
  int M, N, Np;        // N: columns of the output (kGradTerms: of dh)
  int act, type;
};

// Two floats as 16-bit elements, the first in the low half.
__device__ __forceinline__ uint32_t pack16(float a, float b, int type) {
  typedef __bf16 v2b __attribute__((ext_vector_type(2)));
  const uint32_t bf = __builtin_bit_cast(uint32_t, v2b{(__bf16)a, (__bf16)b});
  const uint32_t hf = __builtin_bit_cast(uint32_t, v2h{(_Float16)a, (_Float16)b});
  return type == VT_TYPE_BF16 ? bf : hf;
}

__device__ __forceinline__ float from16(uint32_t bits, int type) {
  return type == VT_TYPE_BF16 ? __uint_as_float(bits << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// E: bytes of the floating type in tile16 (2 or 4), and LOW whether it writes
// the low halves of gradient terms; everything else goes by `type` and `lo`.
template <int OP, int E = 2, bool LOW = E == 4>
struct ScaledTile : ScaledOut {
  static constexpr bool kScaled = true;
  static constexpr int OE = OP == kGradTerms ? 2 : E;   // bytes of what tile16 writes
  static constexpr int P = OP == kGated || OP == kGradTerms ? 2 : 1;   // projections taken together

  // f(the activation, at compile time): one branch around many pairs. A branch
  // for each kept a wave at one pair's chain of dependent instructions (a tile's
  // epilogue 10.4 us, with gradient terms 22).
  template <class F>
  __device__ __forceinline__ void by_act(F &&f) const {
    if constexpr (P == 1) f(std::integral_constant<int, VT_ACT_SILU>());
    else if (act == VT_ACT_SILU) f(std::integral_constant<int, VT_ACT_SILU>());
    else f(std::integral_constant<int, VT_ACT_GELU>());
  }

  // g and u of a pair of sums -> h, or (kGradTerms) the terms of Wg and Wu.
  template <int ACT>
  __device__ __forceinline__ void pair(int32_t ag, int32_t au, float t_row, float sg, float su, float d, float &first,
                                       float &second) const {
    const float g = (float)ag * t_row * sg, u = (float)au * t_row * su;
    float slope;
    const float a = act_of<ACT, OP == kGradTerms>(g, slope);
    if constexpr (OP == kGated) {
      first = a * u;
    } else {
      // Rounded to 32 bits here: a product fused into the conversion to float16
      // rounds once, and the low half that is left of it would be another's.
      first = d * u * slope * sg;
      second = d * a * su;
      asm("" : "+v"(first), "+v"(second));
    }
  }

  __device__ __forceinline__ int to16() const { return OP == kGradTerms ? VT_TYPE_F16 : type; }

  // 8 elements to y[at ..].
  __device__ __forceinline__ void store8(int64_t at, const float (&v)[8], int to) const {
    if (to == VT_TYPE_F32) {
      float *y = (float *)Y + at;
      __builtin_nontemporal_store(v4f{v[0], v[1], v[2], v[3]}, (v4f_any *)y);
      __builtin_nontemporal_store(v4f{v[4], v[5], v[6], v[7]}, (v4f_any *)(y + 4));
    } else {
      v4i w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (int)pack16(v[2 * i], v[2 * i + 1], to);
      __builtin_nontemporal_store(w, (v4i_any *)((uint16_t *)Y + at));
    }
  }
  // `count` (any) of them.
  __device__ __forceinline__ void store8(int64_t at, const float (&v)[8], int count, int to) const {
    if (count >= 8) return store8(at, v, to);
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < count) {
        if (to == VT_TYPE_F32) ((float *)Y)[at + e] = v[e];
        else ((uint16_t *)Y)[at + e] = (uint16_t)pack16(v[e], 0.0f, to);
      }
  }

  // 8 elements of dh from column j, zero past the last.
  struct D8 {
    uint32_t w[8];
  };
  __device__ __forceinline__ D8 load_d8(int64_t row, int j) const {
    D8 d;
#pragma unroll
    for (int e = 0; e < 8; ++e) d.w[e] = 0;
    if (type == VT_TYPE_F32) {
      const float *x = (const float *)D + row * ldd + j;
      if (j + 8 <= N) {
        const v4f a = *(const v4f_any *)x, b = *(const v4f_any *)(x + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d.w[e] = __float_as_uint(a[e]);
          d.w[4 + e] = __float_as_uint(b[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (j + e < N) d.w[e] = __float_as_uint(x[e]);
      }
    } else {
      const uint16_t *x = (const uint16_t *)D + row * ldd + j;
      if (j + 8 <= N) {
        const v4i a = ld_any((const int8_t *)x);
#pragma unroll
        for (int e = 0; e < 4; ++e) d.w[e] = (uint32_t)a[e];
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (j + e < N) d.w[e >> 1] |= (uint32_t)x[e] << (16 * (e & 1));
      }
    }
    return d;
  }
  __device__ __forceinline__ float d_value(const D8 &d, int e) const {
    return type == VT_TYPE_F32 ? __uint_as_float(d.w[e]) : from16(d.w[e >> 1] >> (16 * (e & 1)) & 0xffffu, type);
  }

  // A wave's sums, MI strips of ROWS rows by WP packed columns from (row0,
  // col0): write(mi) puts a strip as it lies in the accumulators into the wave's
  // LDS (rows of 4 WP bytes, 16-byte chunk k of a row at k ^ swz(row)), and the
  // lanes take it from there row by row, 8 output columns each, so scales, dh
  // and outputs are whole 16-byte pieces. The strips are a loop (`write` alone
  // is unrolled): this code runs once per tile, and a short call waits for it
  // to be fetched (unrolled, the gradient's kernel of 18 KB took 11 us for one
  // slice). Every strip's dh is loaded one strip ahead, before the stores that
  // it would otherwise wait for (both count in vmcnt, in order). Rows past
  // row_max and columns past the last are not stored; a wave that has none of
  // those runs without their branches (with them an iteration took 550 cycles,
  // and the epilogue of the gradient's kernel 6.5 us). `early`: the row
  // normalisers of the wave's first and second 64 rows, when they were loaded
  // before.
  template <int MI, int ROWS, int WP, class WRITE, class SWZ>
  __device__ __forceinline__ void strips(WRITE write, SWZ swz, int row0, int col0, int row_max, int lane,
                                         const LDS_AS int8_t *lds, const float *early = nullptr) const {
    constexpr int LPR = WP / P / 8, RPI = 64 / LPR, IT = ROWS / RPI;   // lanes per row, rows at a time, times
    static_assert(IT >= 1 && MI * ROWS <= 128, "whole iterations; two registers hold the rows' scales");
    const int j8 = 8 * (lane % LPR), lr = lane / LPR;
    const int lp = P == 1 ? j8 : (j8 >> 5) * 64 + (j8 & 31);   // the lane's first packed column, less col0
    const int pc = col0 + lp, j = (P == 1 ? col0 : col0 / 2) + j8;
    const int count = OP == kGradTerms ? 8 : N - j;
    const bool cols = pc < Np && count > 0;
    const bool whole = __builtin_amdgcn_readfirstlane(
        row0 + MI * ROWS <= row_max && (P == 1 ? col0 + WP : col0 / 2 + WP / 2) <= N && col0 + WP <= Np);
    float s0[8], s1[P == 2 ? 8 : 1], bias[OP == kLinear ? 8 : 1];
    if constexpr (OP != kGrad) {
      const float *m = meta + min(pc, Np - 8 - (P == 2 ? 32 : 0));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s0[e] = m[e];
        if constexpr (P == 2) s1[e] = m[32 + e];
        if constexpr (OP == kLinear) bias[e] = m[Np + e];
      }
    }
    float tr[2], nr[2];
#pragma unroll
    for (int h = 0; h < (MI * ROWS > 64 ? 2 : 1); ++h) {
      const int row = min(row0 + 64 * h + lane, M - 1);
      if constexpr (OP != kGrad) tr[h] = t[row];
      if constexpr (OP == kGradTerms) nr[h] = norm[row];
      if constexpr (OP == kGrad) nr[h] = early[h];
    }
    D8 d[OP == kGradTerms ? IT : 1], ahead[OP == kGradTerms ? IT : 1];
    auto load_d = [&](int mi) {
      if constexpr (OP == kGradTerms) {
#pragma unroll
        for (int it = 0; it < IT; ++it)
          ahead[it] = load_d8(min(row0 + mi * ROWS + it * RPI + lr, M - 1), min(j, N));
      }
    };
    load_d(0);
#pragma unroll 1
    for (int mi = 0; mi < MI; ++mi) {
      if constexpr (OP == kGradTerms) {
#pragma unroll
        for (int it = 0; it < IT; ++it) d[it] = ahead[it];
        load_d(min(mi + 1, MI - 1));
      }
      each([&](auto i) __attribute__((always_inline)) {
        if (mi == decltype(i)::value) write(i);
      }, std::make_integer_sequence<int, MI>());
      const bool second = MI * ROWS > 64 && mi * ROWS >= 64;
#pragma unroll (IT > 4 ? 4 : IT)
      for (int it = 0; it < IT; ++it) {
        const int r = it * RPI + lr, rel = mi * ROWS + r, row = row0 + rel;
        const LDS_AS int8_t *at = lds + r * (4 * WP);
        auto chunk = [&](int k) { return *(const LDS_AS v4i *)(at + ((k ^ swz(r)) << 4)); };
        const v4i a0 = chunk(lp / 4), a1 = chunk(lp / 4 + 1);
        v4i u0, u1;
        if constexpr (P == 2) {
          u0 = chunk(lp / 4 + 8);
          u1 = chunk(lp / 4 + 9);
        }
        float t_row, n_row;
        if constexpr (OP != kGrad) t_row = __shfl(second ? tr[1] : tr[0], rel & 63);
        if constexpr (OP == kGradTerms || OP == kGrad) n_row = __shfl(second ? nr[1] : nr[0], rel & 63);
        float v[8], v2[P == 2 ? 8 : 1];
        by_act([&](auto kind) __attribute__((always_inline)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int a = e < 4 ? a0[e & 3] : a1[e & 3];
            if constexpr (OP == kLinear) {
              v[e] = (float)a * t_row * s0[e] + bias[e];
            } else if constexpr (OP == kGrad) {
              v[e] = __builtin_bit_cast(float, a) * n_row;
            } else {
              const int u = e < 4 ? u0[e & 3] : u1[e & 3];
              pair<decltype(kind)::value>(a, u, t_row, s0[e], s1[e], OP == kGradTerms ? d_value(d[it], e) * n_row : 0.0f,
                                          v[e], v2[e]);
            }
          }
        });
        if constexpr (OP == kGradTerms) {
          if (!whole && (!cols || row >= row_max)) continue;
          const int64_t to = (int64_t)row * Np + pc;
          store8(to, v, VT_TYPE_F16);
          store8(to + 32, v2, VT_TYPE_F16);
          if (lo) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              v[e] -= (float)(_Float16)v[e];
              v2[e] -= (float)(_Float16)v2[e];
            }
            store8(to + lo, v, VT_TYPE_F16);
            store8(to + lo + 32, v2, VT_TYPE_F16);
          }
        } else if (whole) {
          store8((int64_t)row * ldy + j, v, type);
        } else if (cols && row < row_max) {
          store8((int64_t)row * ldy + j, v, count, type);
        }
      }
    }
  }

  // Blocks of 16 x 16 sums (element e of lane l: row 4 (l / 16) + e, column
  // l % 16) of 16 MI rows and 16 NI packed columns, G block rows to a strip; the
  // strips' swizzle is store_strip16_lds' (distinct banks for an instruction's
  // writes).
  template <int G, int MI, int NI, class ACC>
  __device__ __forceinline__ void blocks16(const ACC (&acc)[MI][NI], int row0, int col0, int lane, LDS_AS int8_t *lds,
                                           const float *early) const {
    const int g = lane >> 4, c = lane & 15;
    strips<MI / G, 16 * G, NI * 16>(
        [&](auto strip) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int ni = 0; ni < NI; ++ni)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *(LDS_AS decltype(acc[0][0][0] + 0) *)(lds + (16 * i + 4 * g + e) * (64 * NI) +
                                                       ((((ni ^ g) << 2) + (c >> 2)) << 4) + (c & 3) * 4) =
                    acc[strip * G + i][ni][e];
        },
        [](int row) { return ((row >> 2) & 3) << 2; }, row0, col0, M, lane, lds, early);
  }

  // Rows [r0, r0 + 16) of `W` output columns from out0 leave the wave's LDS, in
  // 16-byte pieces of whole rows (vector j of a lane: row (64 j + lane) / RC,
  // chunk lane % RC). 16-byte chunk k of a row is at k ^ swz(row). Rows below
  // row_min and columns below out_min are the neighbouring tile's.
  template <int W, class SWZ>
  __device__ __forceinline__ void store_rows(LDS_AS int8_t *lds, SWZ swz, int r0, int out0, int64_t plane, int lane,
                                             int row_min, int out_min) const {
    constexpr int PITCH = W * OE, RC = PITCH / 16, PER = 16 / OE;
    const int out_n = OP == kGradTerms ? Np : N;
    const int64_t ld = OP == kGradTerms ? Np : ldy;
#pragma unroll 4
    for (int j = 0; j < (16 * RC + 63) / 64; ++j) {
      const int idx = 64 * j + lane, row = idx / RC, k = idx % RC;
      LDS_AS int8_t *from = lds + row * PITCH + ((k ^ swz(row)) << 4);
      const int col = out0 + k * PER;
      if (r0 + row < row_min || col < out_min) continue;
      int8_t *y = (int8_t *)Y + ((int64_t)(r0 + row) * ld + plane + col) * OE;
      if (col + PER <= out_n) {
        __builtin_nontemporal_store(*(LDS_AS v4i *)from, (v4i_any *)y);
      } else {
#pragma unroll 1
        for (int e = 0; col + e < out_n; ++e) {
          if constexpr (OE == 4) ((int32_t *)y)[e] = ((LDS_AS int32_t *)from)[e];
          else ((uint16_t *)y)[e] = ((LDS_AS uint16_t *)from)[e];
        }
      }
    }
  }

  // Four elements of consecutive rows of one column into the wave's LDS.
  template <int PITCH>
  __device__ __forceinline__ void put4(LDS_AS int8_t *at, float a, float b, float c, float d) const {
    if constexpr (OE == 4) {
      *(LDS_AS float *)at = a;
      *(LDS_AS float *)(at + PITCH) = b;
      *(LDS_AS float *)(at + 2 * PITCH) = c;
      *(LDS_AS float *)(at + 3 * PITCH) = d;
    } else {
      const uint32_t ab = pack16(a, b, to16()), cd = pack16(c, d, to16());
      *(LDS_AS uint16_t *)at = (uint16_t)ab;
      *(LDS_AS uint16_t *)(at + PITCH) = (uint16_t)(ab >> 16);
      *(LDS_AS uint16_t *)(at + 2 * PITCH) = (uint16_t)cd;
      *(LDS_AS uint16_t *)(at + 3 * PITCH) = (uint16_t)(cd >> 16);
    }
  }

  typedef typename std::conditional<E == 4, float, uint16_t>::type DBits;
  __device__ __forceinline__ float d_value(DBits b) const {
    if constexpr (E == 4) return b;
    else return type == VT_TYPE_BF16 ? __uint_as_float((uint32_t)b << 16) : (float)__builtin_bit_cast(_Float16, b);
  }

  // The persistent kernels' tiles, in the same layout but the other order: the
  // outputs are formed where the sums lie, in registers, and go through the LDS
  // as they are stored. That is half the LDS traffic for 16-bit outputs, and the
  // strips, unrolled, overlap: 8192^3 in 403 us against 409 (`strips` unrolled)
  // and 417 (a loop), gated 2000 x 4096 x 14336 219 against 227 and 232.
  // Blocks of 16 MI rows from row0 and 16 NI packed columns from col0. Each
  // strip of 16 rows goes through the wave's LDS to whole 16-byte pieces of
  // output rows, chunk k of strip row r at k ^ (OE * ((r / 4) % 4)): the writes
  // of one instruction then fall on distinct banks, as in store_strip16_lds.
  // Rows below row_min and packed columns below col_min are the neighbouring
  // tile's. All loads are issued before the stores they would otherwise wait
  // for (both count in vmcnt, in order): the scales first, a strip's dh one
  // strip ahead.
  template <int MI, int NI, bool EDGE>
  __device__ __forceinline__ void tile16(const v4i (&acc)[MI][NI], int row0, int col0, int row_min, int col_min,
                                         int lane, LDS_AS int8_t *lds) const {
    constexpr int NB = OP == kGated ? NI / 2 : NI;   // blocks of output columns
    constexpr int ND = OP == kGradTerms ? NI / 2 : 1;  // and of dh's
    constexpr int W = NB * 16, PITCH = W * OE, RC = PITCH / 16;
    const int g = lane >> 4, c = lane & 15;
    float s[NI], bias[OP == kLinear ? NI : 1];
    v4f tr[OP == kGradTerms ? 1 : MI], nr;
    auto trow = [](int mi) { return OP == kGradTerms ? 0 : mi; };
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      s[ni] = meta[col0 + ni * 16 + c];
      if constexpr (OP == kLinear) bias[ni] = meta[Np + col0 + ni * 16 + c];
    }
    if constexpr (OP != kGradTerms) {
#pragma unroll
      for (int mi = 0; mi < MI; ++mi) tr[mi] = *(const v4f_any *)(t + row0 + mi * 16 + 4 * g);
    }
    DBits d[ND][4];
    auto load_scales = [&](int mi) {
      if constexpr (OP == kGradTerms) {
        tr[0] = *(const v4f_any *)(t + row0 + mi * 16 + 4 * g);
        nr = *(const v4f_any *)(norm + row0 + mi * 16 + 4 * g);
      }
    };
    auto load_block = [&](int mi, int b) {
      const int j = min(col0 / 2 + b * 16 + c, N - 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) d[b][e] = ((const DBits *)D)[(int64_t)(row0 + mi * 16 + 4 * g + e) * ldd + j];
    };
    if constexpr (OP == kGradTerms) {
      load_scales(0);
#pragma unroll
      for (int b = 0; b < ND; ++b) load_block(0, b);
    }
    auto swz = [](int row) { return (((row >> 2) & 3) * OE) & (RC - 1); };
    int wb[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) wb[b] = 4 * g * PITCH + (((b * OE + (c * OE >> 4)) ^ swz(4 * g)) << 4) + (c * OE & 15);
    auto flush = [&](const float (&v)[NB][4], int mi, int64_t plane) {
#pragma unroll
      for (int b = 0; b < NB; ++b) put4<PITCH>(lds + wb[b], v[b][0], v[b][1], v[b][2], v[b][3]);
      store_rows<W>(lds, swz, row0 + mi * 16, OP == kGated ? col0 / 2 : col0, plane, lane, EDGE ? row_min : 0,
                    OP == kGated ? col_min / 2 : col_min);
    };
    each([&](auto strip) __attribute__((always_inline)) {
      constexpr int mi = decltype(strip)::value;
      float v[NB][4];
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (OP == kLinear) {
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[ni][e] = (float)acc[mi][ni][e] * tr[trow(mi)][e] * s[ni] + bias[ni];
      } else {
        by_act([&](auto kind) __attribute__((always_inline)) {
#pragma unroll
          for (int b = 0; b < NI / 2; ++b) {
            const int ng = (b >> 1) * 4 + (b & 1);
            const bool in = OP != kGradTerms || col0 / 2 + b * 16 + c < N;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int32_t ag = acc[mi][ng][e], au = acc[mi][ng + 2][e];
              if constexpr (OP == kGated) {
                float none;
                pair<decltype(kind)::value>(ag, au, tr[trow(mi)][e], s[ng], s[ng + 2], 0.0f, v[b][e], none);
              } else {
                const float de = in ? d_value(d[b][e]) * nr[e] : 0.0f;
                pair<decltype(kind)::value>(ag, au, tr[trow(mi)][e], s[ng], s[ng + 2], de, v[ng][e], v[ng + 2][e]);
              }
            }
            // A block's dh of the next strip takes the registers of this one's, and
            // four pairs' chains run at a time: more spilled registers.
            if constexpr (OP == kGradTerms) {
              __builtin_amdgcn_sched_barrier(0);
              if constexpr (mi + 1 < MI) {
                load_block(mi + 1, b);
                if (b == NI / 2 - 1) load_scales(mi + 1);
              }
            }
          }
        });
      }
      flush(v, mi, 0);
      if constexpr (OP == kGradTerms && LOW) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[b][e] -= (float)(_Float16)v[b][e];
        flush(v, mi, lo);
      }
      __builtin_amdgcn_sched_barrier(0);
    }, std::make_integer_sequence<int, MI>());
  }

  // Blocks of 32 x 32 sums (element e of lane l: row 8 (e / 4) + 4 (l / 32) +
  // e % 4, column l % 32) of 32 MI rows and 64 packed columns; an instruction's
  // two rows are 4 apart, and chunk k of row r is at k ^ (8 ((r / 4) % 2)).
  template <int MI, int NI>
  __device__ __forceinline__ void tile32(const v16i (&acc)[MI][NI], int row0, int col0, int lane,
                                         LDS_AS int8_t *lds) const {
    static_assert(NI == 2, "a gate and an up block");
    const int g = lane >> 5, c = lane & 31;
    strips<MI, 32, 64>(
        [&](auto mi) __attribute__((always_inline)) {
#pragma unroll
          for (int ni = 0; ni < NI; ++ni)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              *(LDS_AS int32_t *)(lds + (8 * (e >> 2) + 4 * g + (e & 3)) * 256 + ((((ni ^ g) << 3) + (c >> 2)) << 4) +
                                  (c & 3) * 4) = acc[mi][ni][e];
        },
        [](int row) { return ((row >> 2) & 1) << 3; }, row0, col0, M, lane, lds);
  }

  // One element: the sums of packed columns pc (and, of a pair, pc + 32) of a
  // row, to output column j.
  __device__ __forceinline__ void element(int32_t a0, int32_t a1, int row, int pc, int j, float t_row) const {
    auto put = [&](int64_t at, float v, int to) {
      if (to == VT_TYPE_F32) ((float *)Y)[at] = v;
      else ((uint16_t *)Y)[at] = (uint16_t)pack16(v, 0.0f, to);
    };
    const float s0 = meta[pc];
    if constexpr (OP == kLinear) {
      if (j < N) put((int64_t)row * ldy + j, (float)a0 * t_row * s0 + meta[Np + pc], type);
    } else {
      float first, second = 0.0f, d = 0.0f;
      if (OP == kGradTerms && j < N) {
        const int64_t at = (int64_t)row * ldd + j;
        d = norm[row] * (type == VT_TYPE_F32 ? ((const float *)D)[at] : from16(((const uint16_t *)D)[at], type));
      }
      by_act([&](auto kind) __attribute__((always_inline)) {
        pair<decltype(kind)::value>(a0, a1, t_row, s0, meta[pc + 32], d, first, second);
      });
      if constexpr (OP == kGated) {
        if (j < N) put((int64_t)row * ldy + j, first, type);
      } else {
        const int64_t at = (int64_t)row * Np + pc;
        put(at, first, VT_TYPE_F16);
        put(at + 32, second, VT_TYPE_F16);
        if (lo) {
          put(at + lo, first - (float)(_Float16)first, VT_TYPE_F16);
          put(at + lo + 32, second - (float)(_Float16)second, VT_TYPE_F16);
        }
      }
    }
  }
};

template <int OP, int E, int BN>
__global__ __launch_bounds__(256, 1) void scaled_dma16_kernel(GemmArgs p, ScaledTile<OP, E> out) {
  dma16_tiles<false, true, true, BN, false>(p, out);
}

// Terms of float16 gradients: 16-bit dh, and low halves. (A branch on `lo` in the
// kernel for both 16-bit types cost the bfloat16 one registers and 1.5 - 3 %.)
template <int BN>
__global__ __launch_bounds__(256, 1) void terms_low_dma16_kernel(GemmArgs p, ScaledTile<kGradTerms, 2, true> out) {
  dma16_tiles<false, true, true, BN, false>(p, out);
}

// The same from int32 sums in memory: `slices` partial sums [M][Np] each.
template <int OP>
__global__ __launch_bounds__(256) void finish_kernel(const int32_t *S, int slices, ScaledTile<OP> out) {
  const int row = blockIdx.x, j = blockIdx.y * 256 + threadIdx.x;
  const int pc = OP == kLinear ? j : (int)pair_col(j, 0);
  if (pc >= out.Np) return;
  const int32_t *s = S + (int64_t)row * out.Np + pc;
  int32_t a0 = 0, a1 = 0;
#pragma unroll 4
  for (int i = 0; i < slices; ++i) {
    a0 = add_wrap(a0, s[0]);
    if (OP != kLinear) a1 = add_wrap(a1, s[32]);
    s += (int64_t)out.M * out.Np;
  }
  out.element(a0, a1, row, pc, j, out.t[row]);
}

// ---------------------------------------------------------------------------
// Up to 64 rows
// ---------------------------------------------------------------------------

struct ScaledSkinnyArgs {
  const void *X;      // int8 rows (XB 0), or the floating rows themselves
  const int8_t *Bp;
  float *t;           // XB > 0 with partial sums: the rows' scales for finish_kernel
  int32_t *ws;        // [k_split][M][Np] partial sums, or null
  uint64_t *fin;      // finishing words, or null
  int64_t ldx;
  int x_type;
  int K, Kp, nbt;     // nbt: 16-column blocks of a projection
  int hpw, groups, k_split, kb_per_split, fin_bits;
};

// Values of floating rows that a workgroup rounds to int8 itself: two pieces
// of 16 for each of its 512 threads.
constexpr int kFusedValues = 16384;

// M <= 16 MB rows over packed weights, bound by reading the weights once: the
// scheme of packed_skinny_kernel (a group of 8-column half blocks per
// workgroup, its 8 waves taking 64-row blocks in turn, S of them in flight in
// registers), for P projections whose column groups it takes together, and
// with what follows the sums in its epilogue. XB > 0: X holds float32 (4) or
// 16-bit (2) rows, at most kFusedValues with their padding; every workgroup
// finds the rows' scales and keeps the rounded rows in LDS. Their loads are
// issued before the first weights' and waited for behind them, so the stream
// of weights starts no later. One row of 4096: 11.6 us for 58.7 MB of weights
// to 14336 columns (5.1 TB/s), 19.5 us for a gated product's 117 MB (6.0); with
// the rounding and the scaling as kernels of their own 14.7 and 23.2.
//
// K slices finish through 64-bit words as in packed_skinny_kernel: the words'
// two sums are two rows of a column (P = 1) or the two projections of one
// element (P = 2).
template <int OP, int NBW, int MB, int XB>
__global__ __launch_bounds__(512) void scaled_skinny_kernel(ScaledSkinnyArgs p, ScaledOut o) {
  constexpr int P = OP == kGated ? 2 : 1, NT = NBW * P, WAVES = 8, S = packed_stages(NT);
  static_assert(XB == 0 || MB == 1, "rows are rounded here for M <= 16");
  __shared__ v4i red[WAVES * NT * 64];
  __shared__ __attribute__((aligned(16))) int8_t arows[XB ? kFusedValues + 16 * 32 : 16];
  __shared__ uint32_t tops[16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = gridDim.x, w = blockIdx.x;
  const int q = G >> 3, r = G & 7, x = w & 7;
  const int wl = x * q + (x < r ? x : r) + (w >> 3);
  const int group = wl % p.groups, split = wl / p.groups;
  const int h0 = group * p.hpw, h1 = min(h0 + p.hpw, 2 * p.nbt);   // half blocks [h0, h1) of a projection
  const int nb0 = h0 >> 1, live = ((h1 - 1) >> 1) - nb0 + 1;
  const int kbt = p.Kp / 64, kb_beg = split * p.kb_per_split, kb_end = min(kb_beg + p.kb_per_split, kbt);
  const int acol = (lane >> 4) * 16, M = o.M;
  auto col_lo = [&](int n) { return (n == 0 && (h0 & 1)) ? 8 : 0; };
  auto col_hi = [&](int n) { return n >= live ? 0 : (n == live - 1 && (h1 & 1)) ? 8 : 16; };
  // 16-column block nb of projection `which` among the packed ones
  auto block = [&](int nb, int which) { return P == 1 ? nb : (nb >> 1) * 4 + (nb & 1) + 2 * which; };

  // This thread's pieces of the floating rows.
  uint32_t raw[XB ? 2 : 1][XB ? XB * 4 : 1];
  const int per_row = p.Kp / 16;
  if constexpr (XB > 0) {
    if (tid < 16) tops[tid] = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int idx = tid + 512 * i, row = idx / per_row, pos = (idx - row * per_row) * 16;
#pragma unroll
      for (int e = 0; e < XB * 4; ++e) raw[i][e] = 0;
      if (row < M) {
        const int8_t *src = (const int8_t *)p.X + ((int64_t)row * p.ldx + pos) * XB;
        if (pos + 16 <= p.K) {
#pragma unroll
          for (int v = 0; v < XB; ++v) {
            const v4i y = ld_any(src + v * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[i][v * 4 + e] = (uint32_t)y[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (pos + e < p.K) {
              if constexpr (XB == 4) raw[i][e] = ((const uint32_t *)src)[e];
              else raw[i][e >> 1] |= (uint32_t)((const uint16_t *)src)[e] << (16 * (e & 1));
            }
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }

  const bool dead_lo = (h0 & 1) && (lane & 15) < 8, dead_hi = (h1 & 1) && (lane & 15) >= 8;
  const int8_t *b_tile[NT];
  uint32_t b_lane[NBW];
#pragma unroll
  for (int n = 0; n < NBW; ++n) {
    const bool dead = ((n == 0 || live == 1) && dead_lo) || (n >= live - 1 && dead_hi);
    b_lane[n] = (uint32_t)(dead ? lane ^ 8 : lane) * 16;
#pragma unroll
    for (int i = 0; i < P; ++i)
      b_tile[i * NBW + n] = p.Bp + (int64_t)block(nb0 + min(n, live - 1), i) * kbt * 1024;
  }
  const int8_t *a_src[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int row = min(mb * 16 + (lane & 15), M - 1);
    a_src[mb] = XB ? arows + row * (p.Kp + 32) + acol : (const int8_t *)p.X + (int64_t)row * p.ldx + acol;
  }
  v4i acc[MB][NT];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[mb][n] = v4i{0, 0, 0, 0};

  const int first = kb_beg + wave;
  const int steps = first < kb_end ? (kb_end - first + WAVES - 1) / WAVES : 0;
  v4i a[S][MB], b[S][NT];
  auto load_b = [&](int s, v4i (&bv)[NT]) {
    const int kb = first + s * WAVES;
#pragma unroll
    for (int n = 0; n < NT; ++n)
      bv[n] = __builtin_nontemporal_load((const v4i *)(b_tile[n] + (int64_t)kb * 1024 + b_lane[n % NBW]));
  };
  auto load_a = [&](int s, v4i (&av)[MB]) {
    const int kb = first + s * WAVES;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      if constexpr (XB > 0) av[mb] = *(const LDS_AS v4i *)((const LDS_AS int8_t *)a_src[mb] + kb * 64);
      else av[mb] = *(const v4i *)(a_src[mb] + kb * 64);
    }
  };
  auto load = [&](int s, v4i (&av)[MB], v4i (&bv)[NT]) {
    load_b(s, bv);
    load_a(s, av);
  };
  auto multiply = [&](const v4i (&av)[MB], const v4i (&bv)[NT]) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int n = 0; n < NT; ++n)
        acc[mb][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[mb], bv[n], acc[mb][n], 0, 0, 0);
  };
  // Rounds the rows, between the first weights' loads and their use.
  auto round_rows = [&]() {
    if constexpr (XB > 0) {
      float v[2][16];
      uint32_t top[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if constexpr (XB == 4) {
            v[i][e] = __uint_as_float(raw[i][e]);
          } else {
            const uint32_t h = raw[i][e >> 1] >> (16 * (e & 1));
            v[i][e] = p.x_type == VT_TYPE_BF16 ? __uint_as_float(h << 16)
                                               : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
          }
          top[i] = max(top[i], magnitude(v[i][e]));
        }
        // the 8 threads of 128 columns share a row (Kp is a multiple of 128)
#pragma unroll
        for (int d = 4; d; d >>= 1) top[i] = max(top[i], (uint32_t)__shfl_xor((int)top[i], d));
      }
      lds_barrier();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = (tid + 512 * i) / per_row;
        if (row < M && (tid & 7) == 0) atomicMax(&tops[row], top[i]);
      }
      lds_barrier();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int idx = tid + 512 * i, row = idx / per_row, pos = (idx - row * per_row) * 16;
        if (row < M) {
          const float inv = row_scale(tops[row]).inv;
          v4i out;
#pragma unroll
          for (int d = 0; d < 4; ++d)
            out[d] = inv == 0.0f ? 0
                                 : pack_bytes(round_byte(v[i][4 * d], inv), round_byte(v[i][4 * d + 1], inv),
                                              round_byte(v[i][4 * d + 2], inv), round_byte(v[i][4 * d + 3], inv));
          st_lds_b128(arows, row * (p.Kp + 32) + pos, out);
        }
      }
      lds_barrier();
      if (p.ws && wl == 0 && tid < M) p.t[tid] = row_scale(tops[tid]).scale;
    }
  };
  if (steps >= S) {
#pragma unroll
    for (int s = 0; s < S; ++s) load_b(s, b[s]);
    if constexpr (XB > 0) __builtin_amdgcn_sched_barrier(0);
    round_rows();
#pragma unroll
    for (int s = 0; s < S; ++s) load_a(s, a[s]);
    int s0 = 0;
    for (; s0 + 2 * S <= steps; s0 += S) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        multiply(a[s], b[s]);
        load(s0 + s + S, a[s], b[s]);
      }
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s0 + s < steps) multiply(a[s], b[s]);
      if (s0 + s + S < steps) load(s0 + s + S, a[s], b[s]);
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (s0 + s + S < steps) multiply(a[s], b[s]);
  } else {
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (s < steps) load_b(s, b[s]);
    if constexpr (XB > 0) __builtin_amdgcn_sched_barrier(0);
    round_rows();
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (s < steps) load_a(s, a[s]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (s < steps) multiply(a[s], b[s]);
  }

  auto row_t = [&](int row) { return XB ? row_scale(tops[row]).scale : o.t[row]; };
  auto finish = [&](int32_t a0, int32_t a1, int row, int col, float t_row) {
    ScaledTile<OP> out;
    (ScaledOut &)out = o;
    out.element(a0, a1, row, P == 1 ? col : (int)pair_col(col, 0), col, t_row);
  };
  // The sum over the waves of element e of source lane `src` of tile n.
  auto sum = [&](int n, int src, int e) {
    int32_t s = 0;
#pragma unroll
    for (int wv = 0; wv < WAVES; ++wv) s = add_wrap(s, ((const int32_t *)&red[(wv * NT + n) * 64 + src])[e]);
    return s;
  };
  if (MB == 1 && p.fin) {
#pragma unroll
    for (int n = 0; n < NT; ++n) red[(wave * NT + n) * 64 + lane] = acc[0][n];
    __syncthreads();
    const int fw = p.fin_bits;
    const uint64_t field = (1ull << fw) - 1;
    const int64_t bias = (int64_t)kFinBiasPerRow * p.kb_per_split * 64;
    constexpr int PER_BLOCK = P == 1 ? 128 : 256;   // words of a column block
    for (int t = tid; t < NBW * PER_BLOCK; t += 512) {
      const int n = t / PER_BLOCK, rw = t % PER_BLOCK >> 4, c = t & 15;
      const int row = P == 1 ? 2 * rw : rw, src = (row >> 2) * 16 + c, e = row & 3;
      const int32_t s0 = sum(n, src, e), s1 = P == 1 ? sum(n, src, e + 1) : sum(n + NBW, src, e);
      if (c < col_lo(n) || c >= col_hi(n) || row >= M) continue;
      const int col = (nb0 + n) * 16 + c;
      const uint64_t lo = (uint64_t)((int64_t)s0 + bias), hi = (uint64_t)((int64_t)s1 + bias);
      uint64_t *word = p.fin + ((int64_t)rw * p.nbt * 16 + col);
      const uint64_t old = __hip_atomic_fetch_add(word, (1ull << (2 * fw)) | (hi << fw) | lo, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT);
      if ((old >> (2 * fw)) != (uint64_t)(p.k_split - 1)) continue;
      const int64_t all_bias = bias * p.k_split;
      const int32_t v0 = (int32_t)((int64_t)((old & field) + lo) - all_bias);
      const int32_t v1 = (int32_t)((int64_t)(((old >> fw) & field) + hi) - all_bias);
      finish(v0, v1, row, col, row_t(row));
      if (P == 1 && row + 1 < M) finish(v1, 0, row + 1, col, row_t(row + 1));
      __hip_atomic_store(word, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    return;
  }
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    if (mb > 0) __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) red[(wave * NT + n) * 64 + lane] = acc[mb][n];
    __syncthreads();
    for (int t = tid; t < NBW * 256; t += 512) {
      const int n = t >> 8, r16 = (t >> 4) & 15, c = t & 15;
      const int src = (r16 >> 2) * 16 + c, e = r16 & 3, row = mb * 16 + r16;
      if (row >= M || c < col_lo(n) || c >= col_hi(n)) continue;
      const int32_t s0 = sum(n, src, e), s1 = P == 1 ? 0 : sum(n + NBW, src, e);
      const int col = (nb0 + n) * 16 + c;
      if (!p.ws) {
        finish(s0, s1, row, col, row_t(row));
      } else {
        int32_t *ws = p.ws + ((int64_t)split * M + row) * o.Np;
        ws[P == 1 ? col : pair_col(col, 0)] = s0;
        if (P == 2) ws[pair_col(col, 1)] = s1;
      }
    }
  }
}

struct TermArgs {
  QuantArgs pad;       // gated: int8 rows to copy to the pitch of the products (Q null: none)
  const void *D;
  const float *t;      // gated: row scales
  const float *meta;
  float *norm;         // out: row normalisers
  _Float16 *Y;         // linear: terms [M][Np]
  int64_t ldd, lo;
  int M, N, Np;
};

// 16 float16 terms of a row, and what float16 leaves of them.
__device__ __forceinline__ void put_terms(_Float16 *y, int64_t lo, const float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v8h h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[e] = (_Float16)v[8 * i + e];
      l[e] = (_Float16)(v[8 * i + e] - (float)h[e]);
    }
    *(v8h *)(y + 8 * i) = h;
    if (lo) *(v8h *)(y + lo + 8 * i) = l;
  }
}

// One workgroup per row of dy. LINEAR: the row's terms dy s, normalised by
// their own largest; NC pieces of 16 stay in each thread's registers between
// the maximum and the rounding (0: longer rows, read twice). Else only the
// normaliser of a gated product's terms, from the row's largest |dh|, its
// scale and the weights' bound: |q| <= 128, |act(g)| <= |g| and |act'| <= 1.13.
// Bound by its pass over dy: 4096 x 4096 bfloat16 in 16 us (4.2 TB/s read and
// written; by single elements 24), normalisers of 2048 x 14336 in 13 (4.5).
template <int TYPE, bool LINEAR, int THREADS, int NC>
__global__ __launch_bounds__(THREADS) void row_terms_kernel(TermArgs p) {
  __shared__ uint32_t red[THREADS / 64];
  typedef typename Elem<TYPE>::T T;
  const int64_t row = blockIdx.x;
  const T *d = (const T *)p.D + row * p.ldd;
  const int tid = threadIdx.x;
  float v[NC ? NC : 1][16];
  uint32_t top = 0;
  if constexpr (!LINEAR) {
    if (p.pad.Q)
      for (int pos = tid * 16; pos < p.pad.Kp; pos += THREADS * 16) pad_piece(p.pad, row, pos);
  }
  auto load = [&](int pos, float (&x)[16]) {
    load16<TYPE>(d, pos, p.N, x);
    if constexpr (LINEAR) {
      if (pos < p.Np) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v4f s = *(const v4f *)(p.meta + pos + 4 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * i + e] *= s[e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, magnitude(x[e]));
  };
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) load((tid + THREADS * i) * 16, v[i]);
  } else {
    for (int pos = tid * 16; pos < p.N; pos += THREADS * 16) load(pos, v[0]);
  }
  top = block_max<THREADS>(top, red);
  float bound = __uint_as_float(top);
  if (!LINEAR && top < kInfBits) bound *= fabsf(p.t[row]) * p.meta[2 * (int64_t)p.Np] * (128.0f * 1.13f);
  float norm = normaliser(bound);
  // dh times it stays in float32's range, whatever the scales
  if (!LINEAR && top < kInfBits) norm = fminf(norm, normaliser(__uint_as_float(top)) * 0x1p80f);
  if (tid == 0) p.norm[row] = norm;
  if constexpr (LINEAR) {
    _Float16 *y = p.Y + row * p.Np;
    auto put = [&](int pos, float (&x)[16]) {
      if (pos >= p.Np) return;
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] *= norm;
      put_terms(y + pos, p.lo, x);
    };
    if constexpr (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) put((tid + THREADS * i) * 16, v[i]);
    } else {
      for (int pos = tid * 16; pos < p.Np; pos += THREADS * 16) {
        load(pos, v[0]);
        put(pos, v[0]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// dx = terms . W^T
// ---------------------------------------------------------------------------

struct GradArgs {
  const _Float16 *T;     // terms [M][Np]; low halves `lo` elements after them
  const int8_t *Bp;
  int64_t lo;
  int M, Kp, Np;
  int tiles_m, tiles_n, group_m;
  int planes;            // 2: terms in two halves
  int splits;            // workgroups along the contraction, each writing its own partial sums
};

// v_mfma_f32_16x16x32_f16 accumulating in place in AGPRs (see mfma16_in_place:
// the same register pressure and the same rules). Its B operand is written by
// VALU instructions, of which two must lie between a write and the MFMA: the
// conversions of a half step's operands end at least two slots before it
// (tests/test_scaled_asm.py checks the compiled code).
__device__ __forceinline__ void mfma16h_in_place(v4f &acc, const v4i &a, const v4i &b) {
  asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

// BM x 256 tiles of dx (BM 256: waves of 128 x 128; 128: of 128 x 64; 64: of
// 64 x 64, two workgroups to a CU), one tile per workgroup. A slice is 64 packed columns deep: the terms' rows (128
// bytes, 16-byte chunk c of row r at c ^ (r % 8)) and 4 x 4 whole packed tiles,
// both by DMA into three LDS stages, two slices ahead. A slice is multiplied in
// two halves of 32; half (s, h) multiplies fragments read in the half before,
// while it reads the next half's and turns its int8 values into float16:
//   (s, 0)  reads half (s, 1) from stage s; DMAs of slice s + 2 begin. At its
//           end slice s + 1 has landed (vmcnt: only slice s + 2's first DMAs
//           remain), and the barrier publishes it.
//   (s, 1)  reads half (s + 1, 0) from stage s + 1; the other DMAs of slice
//           s + 2. Its MFMAs consume the last fragments of stage s, so after
//           the barrier at its end stage s may be refilled (by slice s + 3).
// `planes` 2: the terms' low halves are multiplied by the same weights in a
// second pass over the slices. With `splits`, a workgroup takes its share of the
// slices and writes float32 partial sums.
//
// Bound by the float16 MFMA rate: 4096^3 on 256 x 256 tiles in 102 - 107 us (1290
// - 1350 TFLOP/s; register-staged 128 x 128 tiles took 168), 2048 x 4096 x 28672
// on 128 x 256 tiles in 381 - 417 (1150 - 1260). The conversions, 10 vector
// operations per B operand of 32 x 16 weights, issue between the MFMAs: 1.35
// vector instructions to one. A call of few slices is bound by what surrounds
// them, which 64-row tiles halve: 100 x 333 over 2432 packed columns in 13.4 us
// with its terms and sums, on 128-row tiles 16.5.
template <int BM>
__global__ __launch_bounds__(256, 1) void grad_dma_kernel(GradArgs p, ScaledTile<kGrad> out) {
  static_assert(BM == 256 || BM == 128 || BM == 64, "256x256, 128x256 or 64x256 tiles");
  constexpr int WCOLS = BM == 256 ? 2 : 4, WTN = 256 / WCOLS, MI = BM == 64 ? 4 : 8, NI = WTN / 16;
  constexpr int A_BYTES = BM * 128, B_BYTES = 64 * 256, NSTAGE = 3, B_REGION = NSTAGE * A_BYTES;
  constexpr int DA = A_BYTES / 4096, DB = 4, DMAS = DA + DB, FIRST = DMAS / 2;
  __shared__ __attribute__((aligned(1024))) int8_t smem[NSTAGE * (A_BYTES + B_BYTES)];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WCOLS, wn = wave % WCOLS;
  const int g = lane >> 4, j = lane & 15;

  const int total = gridDim.x, w = blockIdx.x;
  const int q = total >> 3, r = total & 7, x = w & 7;
  const int wl = x * q + (x < r ? x : r) + (w >> 3);
  const int tiles = p.tiles_m * p.tiles_n, split = wl / tiles, tile = wl - split * tiles;
  const int group = p.group_m * p.tiles_n, gid = tile / group, first_m = gid * p.group_m;
  const int gm = min(p.tiles_m - first_m, p.group_m), within = tile - gid * group;
  const int m0 = (first_m + within % gm) * BM, n0 = (within / gm) * 256;

  // The normalisers of the wave's rows, loaded ahead of everything.
  float norms[2] = {1.0f, 1.0f};
  if (out.norm) {
#pragma unroll
    for (int h = 0; h < 2; ++h) norms[h] = out.norm[min(m0 + wm * 128 + 64 * h + lane, p.M - 1)];
  }
  const int kbt = p.Kp / 64;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(LDS_AS int8_t *)smem;
  uint32_t a_lane[DA], b_lane[DB];
#pragma unroll
  for (int i = 0; i < DA; ++i) {
    const int row = min(m0 + (wave * DA + i) * 8 + (lane >> 3), p.M - 1) - m0;
    a_lane[i] = (uint32_t)(row * p.Np * 2 + ((lane & 7) ^ (lane >> 3)) * 16);
  }
#pragma unroll
  for (int i = 0; i < DB; ++i)
    b_lane[i] = (uint32_t)((wave * kbt + min(n0 / 64 + i, kbt - 1)) * 1024 + lane * 16);
  const int8_t *const a_tile = (const int8_t *)(p.T + (int64_t)m0 * p.Np);
  // This workgroup's slices, of all planes' in turn.
  const int per_plane = p.Np / 64, all = per_plane * p.planes;
  const int s_beg = all * split / p.splits, slices = all * (split + 1) / p.splits - s_beg;   // all * splits < 2^23
  const int64_t b_step = (int64_t)4 * kbt * 1024;
  const int plane = s_beg / per_plane, s_in = s_beg - plane * per_plane;
  const int8_t *a_next = a_tile + (int64_t)s_in * 128 + plane * p.lo * 2, *b_next = p.Bp + s_in * b_step;
  int left = per_plane - s_in, d_left = slices;   // slices left of the plane, and to fetch after the next one
  // The next slice's bases; past the last one it is fetched again (and not read).
  auto next_slice = [&](const int8_t *&ab, const int8_t *&bb) {
    ab = a_next;
    bb = b_next;
    if (--d_left > 0) {
      if (--left == 0) {
        left = per_plane;
        a_next = a_tile + p.lo * 2;
        b_next = p.Bp;
      } else {
        a_next += 128;
        b_next += b_step;
      }
    }
  };
  auto dma = [&](int d, int stage, const int8_t *ab, const int8_t *bb) {
    if (d < DA) dma_b128(ab, a_lane[d], lds0 + stage * A_BYTES + (wave * DA + d) * 1024);
    else dma_b128(bb, b_lane[d - DA], lds0 + B_REGION + stage * B_BYTES + (wave * DB + d - DA) * 1024);
  };

  // Fragment addresses within a stage, less the blocks' constant parts.
  const int a_row = (wm * 128 + j) * 128;
  const int a_frag[2] = {a_row + ((g ^ (j & 7)) << 4), a_row + (((4 + g) ^ (j & 7)) << 4)};
  const int b_frag = B_REGION + (g >> 1) * 4096 + wn * (WTN / 64) * 1024 + (8 * (g & 1) + (j >> 1)) * 16 + (j & 1) * 8;
  v4f acc[MI][NI];
  auto fence_acc = [&]() {
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) asm volatile("" : "+a"(acc[mi][ni]));
  };
#pragma unroll
  for (int mi = 0; mi < MI; ++mi)
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = v4f{0, 0, 0, 0};
  fence_acc();
  asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");

  v4i fa[MI], fb0[NI], fb1[NI];
  v2i raw[NI];
  auto read_a = [&](int at, int mi) { fa[mi] = ld_lds_b128(smem, at + mi * 2048); };
  auto read_b = [&](int at, int ni) { raw[ni] = ld_lds_tr8(smem, at + (ni >> 2) * 1024 + (ni & 3) * 256); };
  const v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};
  // Operation o of a half step's 10 NI that turn its raw bytes into float16,
  // exactly: a byte b = w + 128 below the exponent byte 0x64 is 1024 + b.
  uint32_t biased = 0, pair = 0;
  auto convert = [&](auto op, v4i *gb) __attribute__((always_inline)) {
    constexpr int o = decltype(op)::value, ni = o / 10, d = o / 5 & 1;
    if constexpr (o % 5 == 0) biased = (uint32_t)raw[ni][d] ^ 0x80808080u;
    else if constexpr (o % 5 == 1) pair = __builtin_amdgcn_perm(0x64646464u, biased, 0x04010400u);
    else if constexpr (o % 5 == 3) pair = __builtin_amdgcn_perm(0x64646464u, biased, 0x04030402u);
    else gb[ni][2 * d + (o % 5 == 4)] = __builtin_bit_cast(int, __builtin_bit_cast(v2h, pair) - off);
  };
  constexpr int SLOTS = MI * NI, CONV0 = SLOTS / 4, DSTEP = SLOTS / (DMAS / 2 + 1);
  constexpr int OPS = BM == 64 ? 4 : 2, CONV1 = CONV0 + 10 * NI / OPS;   // conversions' operations in a slot
  static_assert(CONV1 <= SLOTS - 2, "conversions end two slots before the half step does");
  // One half step: MFMAs from fa and fb (odd rows right to left, so a row's
  // first reuses the last B operand); the next half's fragments from at_a and
  // at_b, B's converted into gb; DMAs d0 .. d1 - 1 of a slice into `stage`.
  auto half = [&](v4i *fb, v4i *gb, int at_a, int at_b, auto first, auto last, int stage, const int8_t *ab,
                  const int8_t *bb) __attribute__((always_inline)) {
    constexpr int d0 = decltype(first)::value, d1 = decltype(last)::value;
    each([&](auto at) __attribute__((always_inline)) {
      constexpr int slot = decltype(at)::value, mi = slot / NI, pos = slot % NI, ni = (mi & 1) ? NI - 1 - pos : pos;
      mfma16h_in_place(acc[mi][ni], fa[mi], fb[ni]);
      if constexpr (slot < NI) read_b(at_b, slot);
      if constexpr (pos == NI - 1) read_a(at_a, mi);
      if constexpr (slot >= CONV0 && slot < CONV1)
        each([&](auto o) __attribute__((always_inline)) {
          convert(std::integral_constant<int, OPS * (slot - CONV0) + decltype(o)::value>(), gb);
        }, std::make_integer_sequence<int, OPS>());
      if constexpr (slot % DSTEP == 2 && d0 + slot / DSTEP < d1) dma(d0 + slot / DSTEP, stage, ab, bb);
      __builtin_amdgcn_sched_barrier(0);
    }, std::make_integer_sequence<int, SLOTS>());
  };
  using Zero = std::integral_constant<int, 0>;
  using First = std::integral_constant<int, FIRST>;
  using All = std::integral_constant<int, DMAS>;

  const int8_t *ab, *bb;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    next_slice(ab, bb);
#pragma unroll
    for (int d = 0; d < DMAS; ++d) dma(d, i, ab, bb);
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(DMAS) : "memory");   // slice 0 landed
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) read_a(a_frag[0], mi);
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) read_b(b_frag, ni);
  each([&](auto o) __attribute__((always_inline)) { convert(o, fb0); }, std::make_integer_sequence<int, 10 * NI>());
  __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): no scalar load completes inside the loop
  int st = 0;
  for (int s = 0; s < slices; ++s) {
    const int st1 = st == 2 ? 0 : st + 1, st2 = st == 0 ? 2 : st - 1;   // stages of slices s + 1, s + 2
    next_slice(ab, bb);
    half(fb0, fb1, a_frag[1] + st * A_BYTES, b_frag + 8192 + st * B_BYTES, Zero(), First(), st2, ab, bb);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(FIRST) : "memory");
    half(fb1, fb0, a_frag[0] + st1 * A_BYTES, b_frag + st1 * B_BYTES, First(), All(), st2, ab, bb);
    asm volatile("s_barrier" ::: "memory");
    st = st1;
  }
  // No DMA may write the LDS that the stores go through, and the last MFMAs'
  // results must be there.
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier\n\ts_nop 7\n\ts_nop 7" ::: "memory");
  fence_acc();
  if (p.splits > 1) out.Y = (float *)out.Y + (int64_t)split * p.M * p.Kp;
  constexpr int STRIP = 64 * WTN * 4;   // 64 of a wave's rows
  static_assert(4 * STRIP <= (int)sizeof(smem), "the stages hold every wave's strip");
  float unit[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) unit[h] = out.norm ? 1.0f / norms[h] : 1.0f;
  out.blocks16<4>(acc, m0 + wm * 128, n0 + wn * WTN, lane, (LDS_AS int8_t *)smem + wave * STRIP, unit);
}

// dx from the partial sums [slices][M][Kp] of a split contraction, over the
// rows' normalisers: 4 columns of a row per thread. Latency-bound where splits
// are chosen (300 x 999 in 4.1 us), and cheaper than adding in memory, whose
// order would change results from call to call.
struct GradSumArgs {
  const float *ws;
  const float *norm;
  void *X;
  int64_t ldx;
  int M, K, Kp, slices, type;
};

__global__ __launch_bounds__(256) void grad_sum_kernel(GradSumArgs p) {
  const int64_t row = blockIdx.x;
  const int col = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (col >= p.K) return;
  const float *w = p.ws + row * p.Kp + col;
  const int64_t step = (int64_t)p.M * p.Kp;
  v4f v = {0, 0, 0, 0};
  for (int i = 0; i < p.slices; i += 8) {   // 8 loads in flight; the order of the sums does not depend on them
    v4f part[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) part[u] = *(const v4f *)(w + min(i + u, p.slices - 1) * step);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u < p.slices) v += part[u];
  }
  v *= 1.0f / p.norm[row];
  const int64_t at = row * p.ldx + col;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < p.K) {
      if (p.type == VT_TYPE_F32) ((float *)p.X)[at + e] = v[e];
      else ((uint16_t *)p.X)[at + e] = (uint16_t)pack16(v[e], 0.0f, p.type);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

bool float_type(int type) { return type == VT_TYPE_F32 || type == VT_TYPE_F16 || type == VT_TYPE_BF16; }

constexpr int64_t kScaledMax = (int64_t)1 << 30;
// The longest sums: 131071 products of -128 and -128 stay below 2^31.
constexpr int64_t kScaledMaxK = 131071;
// Rows: kernels that take one per workgroup stay below 2^32 threads.
constexpr int64_t kScaledMaxM = ((int64_t)1 << 24) - 1;
// Packed columns: a tile's 256 rows of float16 terms stay within 32-bit offsets.
constexpr int64_t kScaledMaxN = 65535 * 64;
// Bytes of int8 rows, of gradient terms or of partial sums that a call keeps at
// once: calls of more take their rows in parts, and split contractions less. (A
// part is 1 ms of work and more: 8192 x 4096 over 2 x 14336 float32 gradients in
// two parts of 470 MB.)
constexpr int64_t kScaledBytes = (int64_t)512 << 20;
// Pitch of int8 rows from which on they are copied before the products.
constexpr int64_t kFarRows = (int64_t)1 << 23;

// Threads of a row. Few long rows are spread over 1024 (48 x 14336 bfloat16:
// 4.4 -> 3.7 us); many are no faster so, nor on a wave each (700 x 4096: 1 us
// slower).
template <int TYPE>
void launch_quant_typed(const QuantArgs &a, int64_t M, hipStream_t s) {
  const dim3 grid((unsigned)M);
  if (a.Kp <= 1024) hipLaunchKernelGGL((quant_rows_kernel<TYPE, 64, 1>), grid, dim3(64), 0, s, a);
  else if (a.Kp <= 4096) hipLaunchKernelGGL((quant_rows_kernel<TYPE, 256, 1>), grid, dim3(256), 0, s, a);
  else if (a.Kp <= 16384 && M < 512) hipLaunchKernelGGL((quant_rows_kernel<TYPE, 1024, 1>), grid, dim3(1024), 0, s, a);
  else if (a.Kp <= 8192) hipLaunchKernelGGL((quant_rows_kernel<TYPE, 256, 2>), grid, dim3(256), 0, s, a);
  else if (a.Kp <= 16384) hipLaunchKernelGGL((quant_rows_kernel<TYPE, 256, 4>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((quant_rows_kernel<TYPE, 256, 0>), grid, dim3(256), 0, s, a);
}

int launch_quant(const QuantArgs &a, int type, int64_t M, hipStream_t s) {
  switch (type) {
    case VT_TYPE_F32: launch_quant_typed<kF32>(a, M, s); break;
    case VT_TYPE_F16: launch_quant_typed<kF16>(a, M, s); break;
    default: launch_quant_typed<kBF16>(a, M, s); break;
  }
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

// int8 rows and their scales, as the products read them.
struct Rows {
  const int8_t *q;
  const float *t;
  int64_t ld;
};

// Whether int8 rows can be read where they are: in whole 16-byte aligned
// pieces, no further apart than the tile kernels' 32-bit offsets reach.
bool rows_in_place(const void *X, int type, int64_t ldx, int64_t K) {
  return ldx <= kFarRows &&
         (type == VT_TYPE_I8_PADDED || (type == VT_TYPE_I8 && K == scaled_kp(K) && ldx % 16 == 0 && aligned16(X)));
}

// X (any type) -> rows of Kp int8 values: in place, or copied (int8) or rounded
// to a workspace. `pad`: a copy is left to the caller, who gets its arguments.
int take_rows(const void *X, int type, int64_t ldx, const float *T, int64_t M, int64_t K, Scratch &scr, Rows *out,
              QuantArgs *pad = nullptr) {
  const int64_t Kp = scaled_kp(K);
  if (rows_in_place(X, type, ldx, K) || (Kp == 0 && !float_type(type))) {   // no values: nothing to copy
    *out = Rows{(const int8_t *)X, T, ldx};
    return VT_OK;
  }
  void *w = nullptr;
  const size_t q_bytes = (size_t)M * Kp;
  if (int rc = scr.take(kRows, q_bytes + (size_t)M * sizeof(float), &w)) return rc;
  QuantArgs a = {X, (int8_t *)w, (float *)((int8_t *)w + q_bytes), ldx, Kp, K, Kp};
  *out = Rows{a.Q, float_type(type) ? a.T : T, Kp};
  if (float_type(type)) return launch_quant(a, type, M, (hipStream_t)scr.stream);
  if (pad) {
    *pad = a;
    return VT_OK;
  }
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)M, (unsigned)((Kp + 4095) / 4096)), dim3(256), 0,
                     (hipStream_t)scr.stream, a);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

GemmArgs scaled_args(const Rows &rows, const int8_t *Bp, int64_t M, int64_t Kp, int64_t Np, int bm, int bn) {
  GemmArgs a = {};
  a.A = rows.q;
  a.B = Bp;
  a.lda = rows.ld;
  a.ldb = Kp / 64;
  a.M = (int)M; a.N = (int)Np; a.K = (int)Kp;
  a.tiles_m = (int)((M + bm - 1) / bm);
  a.tiles_n = (int)((Np + bn - 1) / bn);
  a.group_m = 4;
  a.batch_count = 1;
  a.k_last = a.K;
  return a;
}

template <int OP>
int launch_finish(const int32_t *sums, int slices, const ScaledTile<OP> &out, hipStream_t s) {
  const int cols = OP == kLinear ? out.Np : out.Np / 2;
  const dim3 grid((unsigned)out.M, (unsigned)((cols + 255) / 256));
  hipLaunchKernelGGL((finish_kernel<OP>), grid, dim3(256), 0, s, sums, slices, out);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

// Tiles of the forward products and gradient terms: the kernel with the least
// estimated time. Fitted to calls over 100 .. 5295 rows, 704 .. 28672 packed
// columns and K 256 .. 14336 (us, r rounds of tiles over the CUs, s 64-deep
// slices), each kernel on each of them; the choice is within 5 % of the fastest
// where that is over 15 us:
//   persistent 256x256  r (14 + 0.64 s)       whole rounds; 700 x 4096 x 14336
//                                              52.1 (128x128 tiles 61.5)
//   persistent 256x128  r (8 + 0.42 s)        5295 x 4864 x 4096 119.5 (256x256
//                                              127.9, 128x128 135.5)
//   128x128             5.2 + r (1.6 + 0.287 s), r fractional above 1 (several
//                                              workgroups share a CU)
//                                              2566 x 10240 x 1536 56.2 (256x128
//                                              69.8); 590 x 6912 x 24064 131 (154)
//   64x128              4.3 + r (0.5 + 0.195 s), r at least 1.2
//                                              4096 x 256 x 4096 14.5 (128x128
//                                              16.6, 256x256 18.0)
//   128x128, K in ks slices: the partial sums' kernel, 3.5 and their traffic
//                                              1092 x 9728 x 704 22.9 (44.8)
// Gradient terms take longer after the sums (3 us per round of 128x128 tiles,
// by the same per element for the others).
struct TilePlan {
  int bm, bn, ks;
  bool persistent;
  int64_t tiles;
};

TilePlan tile_plan(bool terms, int64_t M, int64_t Np, int64_t Kp, int cus) {
  const double slices = Kp / 64.0, more = terms ? 3.0 : 0.0;
  TilePlan best = {};
  double least = 0;
  auto offer = [&](int bm, int bn, int ks, bool persistent) {
    const int64_t tiles = (M + bm - 1) / bm * ((Np + bn - 1) / bn);
    const double share = (double)(tiles * ks) / cus;
    double us;
    if (persistent) {
      const double rounds = (double)((tiles + cus - 1) / cus);
      us = bn == 256 ? rounds * (14 + 0.64 * slices + 3 * more) : rounds * (8 + 0.42 * slices + 1.6 * more);
    } else if (bm == 64) {
      us = 4.3 + std::max(share, 1.2) * (0.5 + 0.195 * slices + 0.5 * more);
    } else {
      us = 5.2 + std::max(share, 1.0) * (1.6 + 0.287 * slices / ks + (ks > 1 ? 0 : more));
      if (ks > 1) us += 3.5 + 8.0 * ks * M * Np / 8.0e6;
    }
    if (least == 0 || us < least) {
      least = us;
      best = {bm, bn, ks, persistent, tiles};
    }
  };
  if (M >= 256 && Np >= 256 && Kp % 256 == 0) {
    offer(256, 256, 1, true);
    offer(256, 128, 1, true);
  }
  if (Kp > 128) offer(128, 128, 1, false);   // their kernel is built for more than one pair of slices
  offer(64, 128, 1, false);
  for (int ks = 2; ks <= 16; ++ks)
    if (Kp % (128 * ks) == 0 && Kp / ks >= 512) offer(128, 128, ks, false);
  return best;
}

template <int OP, int BN>
void launch_dma16(const GemmArgs &a, const ScaledOut &o, int64_t wgs, hipStream_t s) {
  if (o.type == VT_TYPE_F32) {
    ScaledTile<OP, 4> out;
    (ScaledOut &)out = o;
    hipLaunchKernelGGL((scaled_dma16_kernel<OP, 4, BN>), dim3((unsigned)wgs), dim3(256), 0, s, a, out);
  } else if (OP == kGradTerms && o.lo) {
    ScaledTile<kGradTerms, 2, true> out;
    (ScaledOut &)out = o;
    hipLaunchKernelGGL((terms_low_dma16_kernel<BN>), dim3((unsigned)wgs), dim3(256), 0, s, a, out);
  } else {
    ScaledTile<OP, 2> out;
    (ScaledOut &)out = o;
    hipLaunchKernelGGL((scaled_dma16_kernel<OP, 2, BN>), dim3((unsigned)wgs), dim3(256), 0, s, a, out);
  }
}

// The int8 product of rows and packed weights, and what follows it, on tiles.
template <int OP>
int launch_scaled(const Rows &rows, const int8_t *Bp, int64_t Kp, const ScaledOut &o, Scratch &scr) {
  ScaledTile<OP> out;
  (ScaledOut &)out = o;
  hipStream_t s = (hipStream_t)scr.stream;
  const int cus = scr.st->num_cus;
  const int64_t M = out.M, Np = out.Np;
  const Problem q = {rows.q, Bp, nullptr, nullptr, M, Np, Kp, rows.ld, Kp / 64, 0, Np, 1, 0, 0, 0, 0};
  void *w = nullptr;
  if (Kp == 0) return launch_finish(nullptr, 0, out, s);
  const TilePlan plan = tile_plan(OP == kGradTerms, M, Np, Kp, cus);
  if (plan.tiles > 0x7fffffff) return fail(VT_EUNSUPPORTED, "grid of %lld tiles too large", (long long)plan.tiles);
  if (plan.ks > 1) {
    if (int rc = scr.take(kPartials, (size_t)plan.ks * M * Np * sizeof(int32_t), &w)) return rc;
    const int64_t kc = Kp / plan.ks;
    Problem sl = q;
    sl.K = kc;
    sl.batch = plan.ks;
    sl.sa = kc;
    sl.sb = kc / 64 * 1024;
    sl.C = (int32_t *)w;
    sl.ldc = Np;
    sl.sc = M * Np;
    if (int rc = launch_mfma_tiles<128, 128, true>(sl, s, cus)) return rc;
    return launch_finish((const int32_t *)w, plan.ks, out, s);
  }
  const GemmArgs a = scaled_args(rows, Bp, M, Kp, Np, plan.bm, plan.bn);
  if (plan.persistent) {
    const int64_t wgs = std::min<int64_t>(plan.tiles, cus);
    if (plan.bn == 256) launch_dma16<OP, 256>(a, o, wgs, s);
    else launch_dma16<OP, 128>(a, o, wgs, s);
  } else {
    const dim3 grid((unsigned)plan.tiles);
    if (plan.bm == 64) {
      if (Kp <= 128) hipLaunchKernelGGL((gemm_mfma_kernel<64, 128, 1, false, true, false, true, ScaledTile<OP>>), grid, dim3(256), 0, s, a, out);
      else hipLaunchKernelGGL((gemm_mfma_kernel<64, 128, 1, false, false, false, true, ScaledTile<OP>>), grid, dim3(256), 0, s, a, out);
    } else {
      hipLaunchKernelGGL((gemm_mfma_kernel<128, 128, 1, false, false, false, true, ScaledTile<OP>>), grid, dim3(256), 0, s, a, out);
    }
  }
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

// Column groups and K slices for up to 64 rows: packed_geometry's rules, for
// groups that hold both projections' columns.
struct ScaledGeom {
  int hpw, groups, ks;
};

template <int P>
ScaledGeom skinny_geom(int64_t M, int64_t nbt, int64_t Kp, int cus) {
  const int64_t units = 2 * nbt, most = 2 * kPackedNBW / P, kbt = Kp / 64;
  auto halves = [&](int64_t ks) {
    if ((units + most - 1) / most * ks >= 192) return most;
    return std::max<int64_t>(1, std::min(most, (units * ks + cus - 1) / cus));
  };
  int64_t hpw = halves(1), ks = 1;
  const int64_t groups = (units + hpw - 1) / hpw;
  if (groups < 192) {
    ks = std::max<int64_t>(1, std::min({(224 + groups - 1) / groups, (kbt + kPackedWaves - 1) / kPackedWaves, (int64_t)64}));
  } else if (hpw < most) {
    // narrow groups read A for longer than a split takes to sum (packed_a_split)
    int64_t least = 0;
    for (int64_t k = 1; k <= 4 && (k == 1 || kbt >= k * kPackedWaves); k *= 2) {
      const int64_t chunk = (kbt + k - 1) / k * 64, h = halves(k), wgs = (units + h - 1) / h * k;
      int64_t ns = (wgs + cus - 1) / cus * chunk * (315 * h * P + 32 * M) / 1000;
      if (k > 1) ns += M <= kSkinnyFinMaxM && skinny_fin_bits((int)k, chunk) > 0 ? 2000 : 3500 + 8 * M * nbt * 16 * P * k / 1500;
      if (k == 1 || ns < least) {
        least = ns;
        ks = k;
      }
    }
    hpw = halves(ks);
  }
  return {(int)hpw, (int)((units + hpw - 1) / hpw), (int)ks};
}

template <int OP, int NBW, int XB>
void launch_skinny_blocks(const ScaledSkinnyArgs &a, const ScaledOut &o, dim3 grid, hipStream_t s) {
  if constexpr (XB > 0) {
    hipLaunchKernelGGL((scaled_skinny_kernel<OP, NBW, 1, XB>), grid, dim3(512), 0, s, a, o);
  } else {
    switch ((o.M + 15) / 16) {
      case 1: hipLaunchKernelGGL((scaled_skinny_kernel<OP, NBW, 1, 0>), grid, dim3(512), 0, s, a, o); break;
      case 2: hipLaunchKernelGGL((scaled_skinny_kernel<OP, NBW, 2, 0>), grid, dim3(512), 0, s, a, o); break;
      case 3: hipLaunchKernelGGL((scaled_skinny_kernel<OP, NBW, 3, 0>), grid, dim3(512), 0, s, a, o); break;
      default: hipLaunchKernelGGL((scaled_skinny_kernel<OP, NBW, 4, 0>), grid, dim3(512), 0, s, a, o); break;
    }
  }
}

template <int OP, int XB>
void launch_skinny_rows(const ScaledSkinnyArgs &a, const ScaledOut &o, dim3 grid, hipStream_t s) {
  const int blocks = (a.hpw + 1) / 2;
  if constexpr (OP == kGated) {
    if (blocks == 1) launch_skinny_blocks<OP, 1, XB>(a, o, grid, s);
    else launch_skinny_blocks<OP, 2, XB>(a, o, grid, s);
  } else {
    switch (blocks) {
      case 1: launch_skinny_blocks<OP, 1, XB>(a, o, grid, s); break;
      case 2: launch_skinny_blocks<OP, 2, XB>(a, o, grid, s); break;
      case 3: launch_skinny_blocks<OP, 3, XB>(a, o, grid, s); break;
      default: launch_skinny_blocks<OP, 4, XB>(a, o, grid, s); break;
    }
  }
}

// Up to 64 rows of a forward call: X of any type (rows already int8 in `rows`
// when it is null).
template <int OP>
int launch_skinny(const void *X, int type, int64_t ldx, int64_t K, const Rows &rows, const int8_t *Bp, ScaledOut o, Scratch &scr) {
  constexpr int P = OP == kGated ? 2 : 1;
  hipStream_t s = (hipStream_t)scr.stream;
  const int64_t Kp = scaled_kp(K), nbt = (o.N + 15) / 16;
  const ScaledGeom g = skinny_geom<P>(o.M, nbt, Kp, scr.st->num_cus);
  ScaledSkinnyArgs a = {};
  a.X = X ? X : rows.q;
  a.Bp = Bp;
  a.ldx = X ? ldx : rows.ld;
  a.x_type = type;
  a.K = (int)K; a.Kp = (int)Kp; a.nbt = (int)nbt;
  a.hpw = g.hpw;
  a.groups = g.groups;
  a.kb_per_split = (int)((Kp / 64 + g.ks - 1) / g.ks);
  a.k_split = (int)((Kp / 64 + a.kb_per_split - 1) / a.kb_per_split);
  void *w = nullptr;
  if (a.k_split > 1) {
    const int bits = o.M <= kSkinnyFinMaxM ? skinny_fin_bits(a.k_split, (int64_t)a.kb_per_split * 64) : 0;
    if (bits > 0) {
      const int64_t words = (P == 1 ? (o.M + 1) / 2 : o.M) * nbt * 16;
      if (int rc = scr.take(kFinWords, (size_t)words * sizeof(uint64_t), &w)) return rc;
      a.fin = (uint64_t *)w;
      a.fin_bits = bits;
    } else {
      if (int rc = scr.take(kPartials, (size_t)a.k_split * o.M * o.Np * sizeof(int32_t), &w)) return rc;
      a.ws = (int32_t *)w;
      if (X) {
        if (int rc = scr.take(kRows, (size_t)o.M * sizeof(float), &w)) return rc;
        a.t = (float *)w;
        o.t = a.t;
      }
    }
  }
  const dim3 grid((unsigned)(a.groups * a.k_split));
  if (!X) launch_skinny_rows<OP, 0>(a, o, grid, s);
  else if (type == VT_TYPE_F32) launch_skinny_rows<OP, 4>(a, o, grid, s);
  else launch_skinny_rows<OP, 2>(a, o, grid, s);
  VT_HIP_CHECK(hipGetLastError());
  if (!a.ws) return VT_OK;
  ScaledTile<OP> out;
  (ScaledOut &)out = o;
  return launch_finish(a.ws, a.k_split, out, s);
}

template <int TYPE, bool LINEAR>
void launch_row_terms_typed(const TermArgs &a, hipStream_t s) {
  const dim3 grid((unsigned)a.M);
  if constexpr (LINEAR) {
    if (a.Np <= 1024) hipLaunchKernelGGL((row_terms_kernel<TYPE, true, 64, 1>), grid, dim3(64), 0, s, a);
    else if (a.Np <= 4096) hipLaunchKernelGGL((row_terms_kernel<TYPE, true, 256, 1>), grid, dim3(256), 0, s, a);
    else if (a.Np <= 8192) hipLaunchKernelGGL((row_terms_kernel<TYPE, true, 256, 2>), grid, dim3(256), 0, s, a);
    else if (a.Np <= 16384) hipLaunchKernelGGL((row_terms_kernel<TYPE, true, 256, 4>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((row_terms_kernel<TYPE, true, 256, 0>), grid, dim3(256), 0, s, a);
  } else if (a.N <= 1024) {
    hipLaunchKernelGGL((row_terms_kernel<TYPE, false, 64, 0>), grid, dim3(64), 0, s, a);
  } else {
    hipLaunchKernelGGL((row_terms_kernel<TYPE, false, 256, 0>), grid, dim3(256), 0, s, a);
  }
}

template <bool LINEAR>
int launch_row_terms(const TermArgs &a, int type, hipStream_t s) {
  switch (type) {
    case VT_TYPE_F32: launch_row_terms_typed<kF32, LINEAR>(a, s); break;
    case VT_TYPE_F16: launch_row_terms_typed<kF16, LINEAR>(a, s); break;
    default: launch_row_terms_typed<kBF16, LINEAR>(a, s); break;
  }
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

// Tiles and splits of a gradient product by the least estimated time (us). A
// slice takes a workgroup, on an idle card and on a busy one (the clock falls),
//   64 x 256     0.48 .. 0.53, as if two workgroups on a CU ran one behind the
//                other; 3.7 around the slices, half of it under the other workgroup
//   128 x 256    0.66 .. 0.87; 6.3
//   256 x 256    1.17 .. 1.55; 10
// and partial sums are written and read at 4 TB/s and take a second launch. On 37
// shapes, every tile timed at 1, 2, 4, .. 32 splits, the choice among those is
// within 5 % of the fastest: 100 x 333 over 2432 columns 13.4 on 64-row tiles (128: 16.5), 1024 x 4096 over
// 4096 45.8 (53.5; 256: 66.8), 1088 rows of that 56.2 on 128-row tiles (64: 63.2),
// 4096^3 124 on 256-row tiles (128: 137, 64: 151).
struct GradGeom {
  int bm, splits;
};

GradGeom grad_geom(int64_t M, int64_t Kp, int64_t slices, int cus) {
  static const struct { int bm; double idle, busy, around, next; } kTiles[] = {
      {256, 1.17, 1.55, 10.0, 10.0}, {128, 0.66, 0.87, 6.3, 6.3}, {64, 0.48, 0.53, 3.7, 1.85}};
  GradGeom best = {128, 1};
  double least = 0;
  for (const auto &t : kTiles)
    for (int splits = 1; splits <= 32 && splits <= slices; splits += splits < 8 ? 1 : splits / 4) {
      if (splits > 1 && splits * M * Kp * 4 > kScaledBytes) break;
      const int64_t wgs = (M + t.bm - 1) / t.bm * ((Kp + 255) / 256) * splits, rounds = (wgs + cus - 1) / cus;
      const double slice = t.idle + (t.busy - t.idle) * std::min(1.0, (double)wgs / cus);
      double us = (double)rounds * (double)((slices + splits - 1) / splits) * slice + t.around + (double)(rounds - 1) * t.next;
      if (splits > 1) us += 2.5 + 8.0 * splits * M * Kp / 4e6;
      if (least == 0 || us < least) {
        least = us;
        best = {t.bm, splits};
      }
    }
  return best;
}

int launch_grad_tiles(const GradArgs &a, int bm, const ScaledOut &o, hipStream_t s) {
  ScaledTile<kGrad> out;
  (ScaledOut &)out = o;
  const int64_t wgs = (int64_t)a.tiles_m * a.tiles_n * a.splits;
  if (wgs > 0x7fffffff) return fail(VT_EUNSUPPORTED, "gradient grid too large");
  if (bm == 256) hipLaunchKernelGGL(grad_dma_kernel<256>, dim3((unsigned)wgs), dim3(256), 0, s, a, out);
  else if (bm == 128) hipLaunchKernelGGL(grad_dma_kernel<128>, dim3((unsigned)wgs), dim3(256), 0, s, a, out);
  else hipLaunchKernelGGL(grad_dma_kernel<64>, dim3((unsigned)wgs), dim3(256), 0, s, a, out);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

// An empty contraction: zeros (a kernel, which a captured graph may hold).
__global__ __launch_bounds__(256) void zero_rows_kernel(ScaledOut o) {
  const int64_t at = blockIdx.x * o.ldy;
  for (int j = threadIdx.x; j < o.N; j += 256) {
    if (o.type == VT_TYPE_F32) ((float *)o.Y)[at + j] = 0.0f;
    else ((uint16_t *)o.Y)[at + j] = 0;
  }
}

int launch_zero(const ScaledOut &o, hipStream_t s) {
  hipLaunchKernelGGL(zero_rows_kernel, dim3((unsigned)o.M), dim3(256), 0, s, o);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

// dx = terms . W^T. o: the gradient, its rows' normalisers and type.
int launch_grad(GradArgs a, const ScaledOut &o, Scratch &scr) {
  hipStream_t s = (hipStream_t)scr.stream;
  const GradGeom g = grad_geom(a.M, a.Kp, (int64_t)a.Np / 64 * a.planes, scr.st->num_cus);
  a.group_m = 4;
  a.tiles_m = (a.M + g.bm - 1) / g.bm;
  a.tiles_n = (a.Kp + 255) / 256;
  a.splits = g.splits;
  if (g.splits == 1)
    return launch_grad_tiles(a, g.bm, o, s);
  void *w = nullptr;
  if (int rc = scr.take(kPartials, (size_t)g.splits * a.M * a.Kp * sizeof(float), &w)) return rc;
  ScaledOut part = o;
  part.Y = w;
  part.ldy = part.N = part.Np = a.Kp;
  part.norm = nullptr;
  part.type = VT_TYPE_F32;
  if (int rc = launch_grad_tiles(a, g.bm, part, s)) return rc;
  const GradSumArgs r = {(const float *)w, o.norm, o.Y, o.ldy, a.M, o.N, a.Kp, g.splits, o.type};
  hipLaunchKernelGGL(grad_sum_kernel, dim3((unsigned)a.M, (unsigned)((o.N + 1023) / 1024)), dim3(256), 0, s, r);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

// A call's checks that need no device. x_ld / y_ld: row pitches of the row
// operand [M][xc] and the output [M][yc].
struct ScaledCall {
  const char *who;
  const void *X;
  int x_type;
  int64_t ldx, xc;
  const float *T;
  const int8_t *Bp;
  const float *meta;
  void *Y;
  int y_type;
  int64_t ldy, yc;
  int64_t M, K, N;
  bool pair;
};

int check_scaled(const ScaledCall &c, bool *empty) {
  *empty = false;
  if (c.M < 0 || c.K < 0 || c.N < 0)
    return fail(VT_EINVAL, "%s: negative size (M=%lld K=%lld N=%lld)", c.who, (long long)c.M, (long long)c.K, (long long)c.N);
  if (c.M > kScaledMaxM) return fail(VT_EINVAL, "%s: more than %lld rows (M=%lld)", c.who, (long long)kScaledMaxM, (long long)c.M);
  if (c.N > kScaledMaxN / (c.pair ? 2 : 1))
    return fail(VT_EINVAL, "%s: packed columns beyond %lld (N=%lld)", c.who, (long long)kScaledMaxN, (long long)c.N);
  if (c.K > kScaledMaxK)
    return fail(VT_EINVAL, "%s: int32 sums hold K <= %lld (K=%lld)", c.who, (long long)kScaledMaxK, (long long)c.K);
  const bool i8 = c.x_type == VT_TYPE_I8 || c.x_type == VT_TYPE_I8_PADDED;
  if (!float_type(c.x_type) && !i8) return fail(VT_EINVAL, "%s: unknown input type %d", c.who, c.x_type);
  if (!float_type(c.y_type)) return fail(VT_EINVAL, "%s: unknown output type %d", c.who, c.y_type);
  if (c.M == 0 || c.yc == 0) {
    *empty = true;
    return VT_OK;
  }
  if (!c.Y) return fail(VT_EINVAL, "%s: output is null", c.who);
  const int64_t Kp = scaled_kp(c.K), Np = scaled_np(c.N, c.pair);
  if (!c.meta || (c.K > 0 && c.N > 0 && !c.Bp)) return fail(VT_EINVAL, "%s: weights are null", c.who);
  if (c.xc > 0 && !c.X) return fail(VT_EINVAL, "%s: input is null", c.who);
  if (i8 && !c.T) return fail(VT_EINVAL, "%s: int8 rows without scales", c.who);
  const int64_t need = c.x_type == VT_TYPE_I8_PADDED ? Kp : c.xc;
  if (c.ldx < need) return fail(VT_EINVAL, "%s: input pitch %lld < %lld", c.who, (long long)c.ldx, (long long)need);
  if (c.ldy < c.yc) return fail(VT_EINVAL, "%s: output pitch %lld < %lld", c.who, (long long)c.ldy, (long long)c.yc);
  if (c.ldx > ((int64_t)1 << 40) || c.ldy > ((int64_t)1 << 40)) return fail(VT_EINVAL, "%s: pitch beyond 2^40", c.who);
  if (c.x_type == VT_TYPE_I8_PADDED && Kp > 0 && (c.ldx % 16 || !aligned16(c.X)))
    return fail(VT_EINVAL, "%s: padded int8 rows need a pitch of whole 16 bytes and a 16-byte aligned base", c.who);
  if ((uintptr_t)c.X % elem_size(c.x_type) || (uintptr_t)c.Y % elem_size(c.y_type) || !aligned16(c.Bp) || !aligned16(c.meta))
    return fail(VT_EINVAL, "%s: operands are not aligned to their elements, or packed weights not to 16 bytes", c.who);
  Extent ex, ey, eb, em, et;
  if (!operand_extent(c.X, 1, 0, c.M, c.ldx, need, elem_size(c.x_type), &ex) ||
      !operand_extent(c.Y, 1, 0, c.M, c.ldy, c.yc, elem_size(c.y_type), &ey) ||
      !operand_extent(c.Bp, 1, 0, 1, 0, Kp * Np, 1, &eb) ||
      !operand_extent(c.meta, 1, 0, 1, 0, scaled_meta(Np), 4, &em))
    return fail(VT_EINVAL, "%s: extent beyond 2^56 bytes", c.who);
  if ((c.X && overlaps(ey, ex)) || (c.Bp && overlaps(ey, eb)) || overlaps(ey, em))
    return fail(VT_EINVAL, "%s: the output overlaps an input in memory", c.who);
  if (c.T) {
    if ((uintptr_t)c.T % 4) return fail(VT_EINVAL, "%s: scales are not aligned to their elements", c.who);
    if (!operand_extent(c.T, 1, 0, 1, 0, c.M, 4, &et)) return fail(VT_EINVAL, "%s: extent beyond 2^56 bytes", c.who);
    if (overlaps(ey, et)) return fail(VT_EINVAL, "%s: the output overlaps an input in memory", c.who);
  }
  return VT_OK;
}

int open_scratch(void *stream, Scratch *scr) {
  int dev = 0;
  DeviceState *st = nullptr;
  if (int rc = current_device(&dev, &st)) return rc;
  scr->st = st;
  scr->stream = stream;
  return VT_OK;
}

// Rows that a call of M takes at a time, whose workspaces hold row_bytes each:
// parts of equal numbers of whole tiles, 64 rows at least.
int64_t rows_at_once(int64_t M, int64_t row_bytes) {
  const int64_t tile = 256 * row_bytes <= kScaledBytes ? 256 : 64;
  const int64_t most = std::max(kScaledBytes / row_bytes / tile * tile, tile);
  if (M <= most) return M;
  const int64_t parts = (M + most - 1) / most;
  return ((M + parts - 1) / parts + tile - 1) / tile * tile;
}

// Rows [r, r + rows) of a call.
ScaledCall part_of(ScaledCall c, int64_t r, int64_t rows) {
  if (c.X) c.X = (const int8_t *)c.X + r * c.ldx * elem_size(c.x_type);
  if (c.T) c.T += r;
  c.Y = (int8_t *)c.Y + r * c.ldy * elem_size(c.y_type);
  c.M = rows;
  return c;
}

int forward_rows(const ScaledCall &c, int act, void *stream) {
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const int64_t Kp = scaled_kp(c.K), Np = scaled_np(c.N, c.pair);
  ScaledOut o = {};
  o.meta = c.meta; o.Y = c.Y; o.ldy = c.ldy;
  o.M = (int)c.M; o.N = (int)c.N; o.Np = (int)Np;
  o.act = act; o.type = c.y_type;
  Rows rows = {};
  const bool skinny = c.M <= kSkinnyMaxM && Kp > 0;
  if (skinny && float_type(c.x_type) && c.M <= 16 && c.M * Kp <= kFusedValues)
    return c.pair ? launch_skinny<kGated>(c.X, c.x_type, c.ldx, c.K, rows, c.Bp, o, scr)
                  : launch_skinny<kLinear>(c.X, c.x_type, c.ldx, c.K, rows, c.Bp, o, scr);
  if (int rc = take_rows(c.X, c.x_type, c.ldx, c.T, c.M, c.K, scr, &rows)) return rc;
  o.t = rows.t;
  if (skinny)
    return c.pair ? launch_skinny<kGated>(nullptr, 0, 0, c.K, rows, c.Bp, o, scr)
                  : launch_skinny<kLinear>(nullptr, 0, 0, c.K, rows, c.Bp, o, scr);
  return c.pair ? launch_scaled<kGated>(rows, c.Bp, Kp, o, scr) : launch_scaled<kLinear>(rows, c.Bp, Kp, o, scr);
}

int forward(const ScaledCall &c, int act, void *stream) {
  bool empty = false;
  if (int rc = check_scaled(c, &empty)) return rc;
  if (act != VT_ACT_SILU && act != VT_ACT_GELU) return fail(VT_EINVAL, "%s: unknown activation %d", c.who, act);
  if (empty) return VT_OK;
  const bool copied = !rows_in_place(c.X, c.x_type, c.ldx, c.K);
  const int64_t step = copied ? rows_at_once(c.M, scaled_kp(c.K) + 4) : c.M;
  for (int64_t r = 0; r < c.M; r += step)
    if (int rc = forward_rows(part_of(c, r, std::min(step, c.M - r)), act, stream)) return rc;
  return VT_OK;
}

// Terms in float16, normalised by row, and in a second half what float16
// leaves of each: two products, 22 bits. Only bfloat16 gradients do without:
// their own rounding to 8 bits is 8 times that of an 11-bit term, so the error
// grows by 1 / 128 (1.7e-3 of the result's norm either way, 4096^3), and the
// second product would double the largest part of the call. Float16 gradients
// have as many bits as such a term: one half alone gave 1.4 times their error.
bool two_halves(int type) { return type != VT_TYPE_BF16; }

int backward_rows(const ScaledCall &c, const int8_t *Q, int q_type, int64_t ldq, const float *t, int act, void *stream) {
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  hipStream_t s = (hipStream_t)stream;
  const int64_t Kp = scaled_kp(c.K), Np = scaled_np(c.N, c.pair);
  ScaledOut o = {};
  o.Y = c.Y; o.ldy = c.ldy;
  o.M = (int)c.M; o.N = (int)c.K; o.Np = (int)Kp;
  o.type = c.y_type;
  if (Np == 0) return launch_zero(o, s);
  const bool split = two_halves(c.x_type);
  const int64_t lo = split ? c.M * Np : 0;
  void *w = nullptr;
  const size_t t_bytes = ((size_t)c.M * Np * 2 * (split ? 2 : 1) + 255) / 256 * 256;
  if (int rc = scr.take(kTerms, t_bytes + (size_t)c.M * sizeof(float), &w)) return rc;
  _Float16 *terms = (_Float16 *)w;
  float *norm = (float *)((int8_t *)w + t_bytes);
  TermArgs ta = {{}, c.X, t, c.meta, norm, terms, c.ldx, lo, (int)c.M, (int)c.N, (int)Np};
  if (!c.pair) {
    if (int rc = launch_row_terms<true>(ta, c.x_type, s)) return rc;
  } else {
    Rows rows;
    if (int rc = take_rows(Q, q_type, ldq, t, c.M, c.K, scr, &rows, &ta.pad)) return rc;
    if (int rc = launch_row_terms<false>(ta, c.x_type, s)) return rc;
    ScaledOut f = {};
    f.t = rows.t; f.meta = c.meta; f.D = c.X; f.norm = norm; f.Y = terms;
    f.ldd = c.ldx; f.lo = lo;
    f.M = (int)c.M; f.N = (int)c.N; f.Np = (int)Np;
    f.act = act; f.type = c.x_type;
    if (int rc = launch_scaled<kGradTerms>(rows, c.Bp, Kp, f, scr)) return rc;
  }
  o.norm = norm;
  const GradArgs g = {terms, c.Bp, lo, (int)c.M, (int)Kp, (int)Np, 0, 0, 0, split ? 2 : 1, 1};
  return launch_grad(g, o, scr);
}

// The gradient in x^: D [M][ldd] of N columns, X the output [M][ldx] of K.
int backward(const ScaledCall &c, const int8_t *Q, int q_type, int64_t ldq, const float *t, int act, void *stream) {
  bool empty = false;
  if (int rc = check_scaled(c, &empty)) return rc;
  if (act != VT_ACT_SILU && act != VT_ACT_GELU) return fail(VT_EINVAL, "%s: unknown activation %d", c.who, act);
  if (!float_type(c.x_type) || c.x_type != c.y_type)
    return fail(VT_EINVAL, "%s: the gradients have one floating type", c.who);
  if (c.pair) {
    if (q_type != VT_TYPE_I8 && q_type != VT_TYPE_I8_PADDED)
      return fail(VT_EINVAL, "%s: the rows are int8 with scales", c.who);
    if (!empty) {
      ScaledCall r = c;   // the same checks of the int8 rows against the output
      r.X = Q; r.x_type = q_type; r.ldx = ldq; r.xc = c.K; r.T = t;
      if (int rc = check_scaled(r, &empty)) return rc;
    }
  }
  if (empty) return VT_OK;
  int64_t row_bytes = scaled_np(c.N, c.pair) * (two_halves(c.x_type) ? 4 : 2) + 4;
  if (c.pair && !rows_in_place(Q, q_type, ldq, c.K)) row_bytes = std::max(row_bytes, scaled_kp(c.K) + 4);
  const int64_t step = rows_at_once(c.M, row_bytes);
  for (int64_t r = 0; r < c.M; r += step)
    if (int rc = backward_rows(part_of(c, r, std::min(step, c.M - r)), c.pair ? Q + r * ldq : nullptr, q_type, ldq,
                               c.pair ? t + r : nullptr, act, stream))
      return rc;
  return VT_OK;
}

}  // namespace

extern "C" {

int64_t vt_quant_pitch(int64_t K) {
  if (K < 0 || K >= kScaledMax) return fail(VT_EINVAL, "vt_quant_pitch: needs 0 <= K < 2^30");
  return scaled_kp(K);
}

int vt_quant_rows(const void *X, int32_t x_type, int64_t ldx, int8_t *Q, int64_t ldq, float *T, int64_t M, int64_t K,
                  void *stream) {
  g_err.clear();
  if (M < 0 || K < 0 || M > kScaledMaxM || K >= kScaledMax)
    return fail(VT_EINVAL, "vt_quant_rows: needs 0 <= M <= %lld, 0 <= K < 2^30 (M=%lld K=%lld)", (long long)kScaledMaxM,
                (long long)M, (long long)K);
  if (!float_type(x_type)) return fail(VT_EINVAL, "vt_quant_rows: unknown input type %d", (int)x_type);
  if (M == 0) return VT_OK;
  const int64_t Kp = scaled_kp(K);
  if (!T || (K > 0 && (!X || !Q))) return fail(VT_EINVAL, "vt_quant_rows: X, Q or T is null");
  if (ldx < K || ldq < Kp || ldx > ((int64_t)1 << 40) || ldq > ((int64_t)1 << 40))
    return fail(VT_EINVAL, "vt_quant_rows: ldx=%lld must be %lld .. 2^40, ldq=%lld %lld .. 2^40", (long long)ldx,
                (long long)K, (long long)ldq, (long long)Kp);
  if (ldq % 16 || !aligned16(Q) || (uintptr_t)X % elem_size(x_type) || (uintptr_t)T % 4)
    return fail(VT_EINVAL, "vt_quant_rows: Q needs 16-byte aligned rows, X and T their elements' alignment");
  Extent ex, eq, et;
  if (!operand_extent(X, 1, 0, M, ldx, K, elem_size(x_type), &ex) || !operand_extent(Q, 1, 0, M, ldq, Kp, 1, &eq) ||
      !operand_extent(T, 1, 0, 1, 0, M, 4, &et))
    return fail(VT_EINVAL, "vt_quant_rows: extent beyond 2^56 bytes");
  if (overlaps(ex, eq) || overlaps(ex, et) || overlaps(eq, et))
    return fail(VT_EINVAL, "vt_quant_rows: operands overlap in memory");
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const QuantArgs a = {X, Q, T, ldx, ldq, K, Kp};
  return launch_quant(a, x_type, M, (hipStream_t)stream);
}

int64_t vt_scaled_size(int64_t K, int64_t N, int32_t pair, int64_t *meta_floats) {
  if (K < 0 || N < 0 || K > kScaledMaxK || N > kScaledMaxN / (pair ? 2 : 1))
    return fail(VT_EINVAL, "vt_scaled_size: needs 0 <= K <= %lld and 0 <= N <= %lld (K=%lld N=%lld)", (long long)kScaledMaxK,
                (long long)(kScaledMaxN / (pair ? 2 : 1)), (long long)K, (long long)N);
  const int64_t Np = scaled_np(N, pair != 0);
  if (meta_floats) *meta_floats = scaled_meta(Np);
  return scaled_kp(K) * Np;
}

int vt_scaled_pack(const int8_t *W0, const int8_t *W1, int64_t ldw0, int64_t ldw1, const float *s0, const float *s1,
                   const float *bias, int64_t K, int64_t N, int8_t *Bp, float *meta, void *stream) {
  g_err.clear();
  const bool pair = s1 != nullptr;
  const int64_t size = vt_scaled_size(K, N, pair, nullptr);
  if (size < 0) return (int)size;
  if (N == 0) return VT_OK;
  if (!meta || !s0 || (K > 0 && (!W0 || !Bp || (pair && !W1))))
    return fail(VT_EINVAL, "vt_scaled_pack: weights, scales or outputs are null");
  if ((pair && bias) || (!pair && W1)) return fail(VT_EINVAL, "vt_scaled_pack: a pair has two weights and scales and no bias");
  if (ldw0 < N || (pair && ldw1 < N)) return fail(VT_EINVAL, "vt_scaled_pack: weight pitch below N=%lld", (long long)N);
  if (ldw0 > ((int64_t)1 << 40) || ldw1 > ((int64_t)1 << 40)) return fail(VT_EINVAL, "vt_scaled_pack: pitch beyond 2^40");
  if (!aligned16(Bp) || !aligned16(meta)) return fail(VT_EINVAL, "vt_scaled_pack: outputs need 16-byte aligned bases");
  const int64_t Kp = scaled_kp(K), Np = scaled_np(N, pair);
  Extent e0, e1, eb;
  if (!operand_extent(W0, 1, 0, K, ldw0, N, 1, &e0) || !operand_extent(Bp, 1, 0, 1, 0, size, 1, &eb) ||
      (pair && !operand_extent(W1, 1, 0, K, ldw1, N, 1, &e1)))
    return fail(VT_EINVAL, "vt_scaled_pack: extent beyond 2^56 bytes");
  if ((uintptr_t)s0 % 4 || (uintptr_t)s1 % 4 || (uintptr_t)bias % 4)
    return fail(VT_EINVAL, "vt_scaled_pack: scales and bias need their elements' alignment");
  if (K > 0 && (overlaps(e0, eb) || (pair && overlaps(e1, eb))))
    return fail(VT_EINVAL, "vt_scaled_pack: Bp overlaps the weights in memory");
  Extent em, ev;
  bool shared = !operand_extent(meta, 1, 0, 1, 0, scaled_meta(Np), 4, &em) ||
                (K > 0 && (overlaps(em, eb) || overlaps(em, e0) || (pair && overlaps(em, e1))));
  for (const float *v : {s0, s1, bias})
    if (v) shared |= !operand_extent(v, 1, 0, 1, 0, N, 4, &ev) || overlaps(ev, em) || (K > 0 && overlaps(ev, eb));
  if (shared) return fail(VT_EINVAL, "vt_scaled_pack: meta shares memory with another operand, or scales with Bp");
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const ScaledPackArgs a = {W0, W1, s0, s1, bias, Bp, meta, ldw0, ldw1, (int)K, (int)N, (int)Kp, (int)Np};
  hipLaunchKernelGGL(pack_scaled_kernel, dim3((unsigned)std::max<int64_t>(Kp / 64, 1), (unsigned)(Np / 64)), dim3(256), 0,
                     (hipStream_t)stream, a);
  VT_HIP_CHECK(hipGetLastError());
  if (pair) {
    hipLaunchKernelGGL(pack_bound_kernel, dim3((unsigned)((N + 63) / 64)), dim3(256), 0, (hipStream_t)stream, a);
    VT_HIP_CHECK(hipGetLastError());
  }
  return VT_OK;
}

int vt_scaled_linear(const void *X, int32_t x_type, int64_t ldx, const float *T, int64_t M, int64_t K, const int8_t *Bp,
                     const float *meta, int64_t N, void *Y, int32_t y_type, int64_t ldy, void *stream) {
  g_err.clear();
  const ScaledCall c = {"vt_scaled_linear", X, x_type, ldx, K, T, Bp, meta, Y, y_type, ldy, N, M, K, N, false};
  return forward(c, VT_ACT_SILU, stream);
}

int vt_scaled_gated(const void *X, int32_t x_type, int64_t ldx, const float *T, int64_t M, int64_t K, const int8_t *Bp,
                    const float *meta, int64_t N, int32_t act, void *Y, int32_t y_type, int64_t ldy, void *stream) {
  g_err.clear();
  const ScaledCall c = {"vt_scaled_gated", X, x_type, ldx, K, T, Bp, meta, Y, y_type, ldy, N, M, K, N, true};
  return forward(c, act, stream);
}

int vt_scaled_linear_grad(const void *dY, int32_t type, int64_t ldd, int64_t M, int64_t K, const int8_t *Bp,
                          const float *meta, int64_t N, void *dX, int64_t ldx, void *stream) {
  g_err.clear();
  const ScaledCall c = {"vt_scaled_linear_grad", dY, type, ldd, N, nullptr, Bp, meta, dX, type, ldx, K, M, K, N, false};
  return backward(c, nullptr, 0, 0, nullptr, VT_ACT_SILU, stream);
}

int vt_scaled_gated_grad(const void *dH, int32_t type, int64_t ldd, const int8_t *Q, int32_t q_type, int64_t ldq,
                         const float *T, int64_t M, int64_t K, const int8_t *Bp, const float *meta, int64_t N, int32_t act,
                         void *dX, int64_t ldx, void *stream) {
  g_err.clear();
  const ScaledCall c = {"vt_scaled_gated_grad", dH, type, ldd, N, nullptr, Bp, meta, dX, type, ldx, K, M, K, N, true};
  return backward(c, Q, q_type, ldq, T, act, stream);
}

}  // extern "C"
