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

// K and N of the packed weights. K in whole 64-deep slices, from 1024 on in
// the 256-deep groups that the 16x16x64 persistent kernels take (at most a
// fifth more to read there; at small K it would be up to four times as much).
// N in whole 64-column blocks: the gradient contracts over N in steps of 64,
// and a gated product's 64 columns are 32 of the gate and 32 of the up weight.
__host__ __device__ constexpr int64_t scaled_kp(int64_t K) {
  return K < 1024 ? (K + 63) / 64 * 64 : (K + 255) / 256 * 256;
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

// 16 elements of a row from `pos`, zero past `len`. ALIGNED: the row starts on
// 16 bytes, so pieces that lie within the row are read as vectors.
template <int TYPE, bool ALIGNED>
__device__ __forceinline__ void load16(const typename Elem<TYPE>::T *row, int64_t pos, int64_t len, float (&v)[16]) {
  typedef typename Elem<TYPE>::T T;
  constexpr int PER = 16 / sizeof(T);
  if (ALIGNED && pos + 16 <= len) {
    typedef T VT __attribute__((ext_vector_type(PER)));
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
// between the maximum and the rounding (NC = 0: longer rows, read twice).
template <int TYPE, bool ALIGNED, int THREADS, int NC>
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
      load16<TYPE, ALIGNED>(x, pos, p.K, v[i]);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = max(top, magnitude(v[i][e]));
    }
  } else {
    for (int64_t pos = tid * 16; pos < p.K; pos += THREADS * 16) {
      load16<TYPE, ALIGNED>(x, pos, p.K, v[0]);
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
      load16<TYPE, ALIGNED>(x, pos, p.K, v[0]);
      put(pos, v[0]);
    }
  }
}

// int8 rows of any pitch and alignment -> rows of Kp bytes, zeros past K.
__global__ __launch_bounds__(256) void pad_rows_kernel(QuantArgs p) {
  const int64_t row = blockIdx.y, pos = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 16;
  if (pos >= p.Kp) return;
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
// the largest |u sg| or |g su| that rows of t = 1, q = 1 can give. One
// workgroup per packed pair of column blocks; the maximum of non-negative
// floats is the maximum of their bits, whatever the order.
__global__ __launch_bounds__(256) void pack_bound_kernel(ScaledPackArgs p) {
  __shared__ uint32_t red[4];
  const int j = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  uint32_t bits = 0;
  if (j < p.N) {
    int64_t a0 = 0, a1 = 0;
    for (int k = lane; k < p.K; k += 64) {
      a0 += abs((int)p.W0[(int64_t)k * p.ldw0 + j]);
      a1 += abs((int)p.W1[(int64_t)k * p.ldw1 + j]);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
      a0 += __shfl_xor((long long)a0, o);
      a1 += __shfl_xor((long long)a1, o);
    }
    bits = magnitude((float)max(a0, a1) * fabsf(p.s0[j]) * fabsf(p.s1[j]));
  }
  bits = block_max<256>(bits, red);
  if (threadIdx.x == 0) atomicMax((uint32_t *)(p.meta + 2 * (int64_t)p.Np), bits);
}

// ---------------------------------------------------------------------------
// What follows the int32 sums
// ---------------------------------------------------------------------------

// 2^32 / (1 + exp(-z)): the factor keeps a small value clear of the smallest
// float32 exponents (which the exponential and the reciprocal drop) until it
// is multiplied by g. From 2^60 on, exp(z) is all of 1 + exp(z).
constexpr float kLogisticUnit = 0x1p-32f;
__device__ __forceinline__ float logistic32(float z) {
  const float e = __builtin_amdgcn_exp2f(fminf(z * 1.4426950408889634f, 60.0f) + 32.0f);
  return e * __builtin_amdgcn_rcpf(1.0f + e * kLogisticUnit);
}

// act(g), and its slope. gelu is the tanh form: (1 + tanh z) / 2 is
// 1 / (1 + exp(-2 z)) with z = c (g + a g^3); past |g| = 16 it is 0 or 1, so g
// is held there inside (its cube would leave float32's range).
template <int ACT>
__device__ __forceinline__ float act_of(float g, float &slope) {
  if (ACT == VT_ACT_SILU) {
    const float p32 = logistic32(g), p = p32 * kLogisticUnit;
    slope = p * (1.0f + g * (1.0f - p));
    return g * p32 * kLogisticUnit;
  }
  const float c = 0.7978845608028654f, a = 0.044715f;
  const float h = fminf(fmaxf(g, -16.0f), 16.0f);
  const float p32 = logistic32(2.0f * c * (h + a * h * h * h)), p = p32 * kLogisticUnit;
  slope = p + h * 2.0f * p * (1.0f - p) * c * (1.0f + 3.0f * a * h * h);
  return g * p32 * kLogisticUnit;
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

struct FinishArgs {
  const int32_t *S;      // int32 sums [M][Np]
  const float *t;        // row scales
  const float *meta;     // channel scales and bias, packed order
  const void *D;         // dh (terms)
  const float *norm;     // row normalisers (terms)
  void *Y;               // output [M][ldy], or terms [M][Np] (float16; low halves after them)
  int64_t ldd, ldy;
  int64_t lo;            // terms: elements from the high to the low half, 0 for none
  int M, N, Np;
};

// OP 0 linear, 1 gated, 2 gradient terms of gated.
template <int TYPE, int OP, int ACT>
__global__ __launch_bounds__(256) void finish_kernel(FinishArgs p) {
  typedef typename Elem<TYPE>::T T;
  const int64_t row = blockIdx.y;
  const int j = blockIdx.x * 256 + threadIdx.x;
  const int64_t pg = OP ? pair_col(j, 0) : j, pu = pair_col(j, 1);
  if (OP == 2 ? pu >= p.Np : j >= p.N) return;
  const float t = p.t[row];
  const int32_t *s = p.S + row * p.Np;
  const float g = (float)s[pg] * t * p.meta[pg];
  if constexpr (OP == 0) {
    ((T *)p.Y)[row * p.ldy + j] = (T)(g + p.meta[p.Np + j]);
  } else {
    const float u = (float)s[pu] * t * p.meta[pu];
    float slope;
    const float a = act_of<ACT>(g, slope);
    if constexpr (OP == 1) {
      ((T *)p.Y)[row * p.ldy + j] = (T)(a * u);
    } else {
      const float d = j < p.N ? (float)((const T *)p.D)[row * p.ldd + j] * p.norm[row] : 0.0f;
      const float tg = d * u * slope * p.meta[pg], tu = d * a * p.meta[pu];
      _Float16 *y = (_Float16 *)p.Y + row * p.Np;
      const _Float16 hg = (_Float16)tg, hu = (_Float16)tu;
      y[pg] = hg;
      y[pu] = hu;
      if (p.lo) {
        y[p.lo + pg] = (_Float16)(tg - (float)hg);
        y[p.lo + pu] = (_Float16)(tu - (float)hu);
      }
    }
  }
}

struct TermArgs {
  const void *D;
  const float *t;      // gated: row scales
  const float *meta;
  float *norm;         // out: row normalisers
  _Float16 *Y;         // linear: terms [M][Np]
  int64_t ldd, lo;
  int M, N, Np;
};

// One workgroup per row of dy. LINEAR: the row's terms dy s, normalised by
// their own largest; else only the normaliser of a gated product's terms,
// from the row's largest |dh|, its scale and the weights' bound: |q| <= 128,
// |act(g)| <= |g| and |act'| <= 1.13.
template <int TYPE, bool LINEAR>
__global__ __launch_bounds__(256) void row_terms_kernel(TermArgs p) {
  __shared__ uint32_t red[4];
  typedef typename Elem<TYPE>::T T;
  const int64_t row = blockIdx.x;
  const T *d = (const T *)p.D + row * p.ldd;
  uint32_t top = 0;
  for (int j = threadIdx.x; j < p.N; j += 256)
    top = max(top, magnitude(LINEAR ? (float)d[j] * p.meta[j] : (float)d[j]));
  top = block_max<256>(top, red);
  float bound = __uint_as_float(top);
  if (!LINEAR && top < kInfBits) bound *= fabsf(p.t[row]) * p.meta[2 * (int64_t)p.Np] * (128.0f * 1.13f);
  float norm = normaliser(bound);
  // dh times it stays in float32's range, whatever the scales
  if (!LINEAR && top < kInfBits) norm = fminf(norm, normaliser(__uint_as_float(top)) * 0x1p80f);
  if (threadIdx.x == 0) p.norm[row] = norm;
  if constexpr (LINEAR) {
    _Float16 *y = p.Y + row * p.Np;
    for (int j = threadIdx.x; j < p.Np; j += 256) {
      const float v = j < p.N ? (float)d[j] * p.meta[j] * norm : 0.0f;
      const _Float16 h = (_Float16)v;
      y[j] = h;
      if (p.lo) y[p.lo + j] = (_Float16)(v - (float)h);
    }
  }
}

// ---------------------------------------------------------------------------
// dx = terms . W^T
// ---------------------------------------------------------------------------

struct GradArgs {
  const _Float16 *T;     // terms [M][Np]; low halves `lo` elements after them
  const int8_t *Bp;
  const float *norm;
  void *X;               // dx [M][ldx]
  int64_t ldx, lo;
  int M, K, Kp, Np;
  int tiles_m, tiles_n;
};

// 8 int8 values as float16, exactly: a byte b = w + 128 below the exponent byte
// 0x64 is the float16 1024 + b.
__device__ __forceinline__ v8h bytes_to_half(v2i w) {
  v8h r;
  const v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const uint32_t b = (uint32_t)w[d] ^ 0x80808080u;
    const v2h lo = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - off;
    const v2h hi = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - off;
    r[4 * d] = lo[0];
    r[4 * d + 1] = lo[1];
    r[4 * d + 2] = hi[0];
    r[4 * d + 3] = hi[1];
  }
  return r;
}

// 128 x 128 tiles of dx, 4 waves of 64 x 64. The contraction runs over packed
// columns in steps of 64: the forward pass's packed weights serve as they are,
// since ds_read_b64_tr_b8 of 8 columns' 16 consecutive k gives a lane 8
// consecutive columns of one k, the operand of v_mfma_f32_16x16x32_f16.
template <int TYPE, bool SPLIT>
__global__ __launch_bounds__(256) void grad_kernel(GradArgs p) {
  constexpr int BM = 128, BN = 128;
  constexpr int A_BYTES = BM * 128, B_BYTES = 64 * BN;
  __shared__ __attribute__((aligned(16))) int8_t smem[2 * A_BYTES * (SPLIT ? 2 : 1) + 2 * B_BYTES];
  constexpr int A_STAGE = A_BYTES * (SPLIT ? 2 : 1);
  int8_t *const Bs0 = smem + 2 * A_STAGE;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  const int total = gridDim.x, w = blockIdx.x;
  const int q = total >> 3, r = total & 7, x = w & 7;
  const int wl = x * q + (x < r ? x : r) + (w >> 3);
  const int m0 = wl / p.tiles_n * BM, n0 = wl % p.tiles_n * BN;
  const int kbt = p.Kp / 64;
  v4i ra[SPLIT ? 8 : 4], rb[2];
  auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = min(m0 + (tid >> 3) + 32 * i, p.M - 1);
      const _Float16 *src = p.T + (int64_t)row * p.Np + c0 + (tid & 7) * 8;
      ra[i] = *(const v4i *)src;
      if constexpr (SPLIT) ra[4 + i] = *(const v4i *)(src + p.lo);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int ch = tid + 256 * i, t = ch >> 6;          // tile t: column block t / 2, k block t % 2
      const int kb = min(n0 / 64 + (t & 1), kbt - 1);
      rb[i] = *(const v4i *)(p.Bp + ((int64_t)(c0 / 16 + (t >> 1)) * kbt + kb) * 1024 + (ch & 63) * 16);
    }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = (tid >> 3) + 32 * i, off = row * 128 + (((tid & 7) ^ (row & 7)) << 4);
      st_lds_b128(smem + buf * A_STAGE, off, ra[i]);
      if constexpr (SPLIT) st_lds_b128(smem + buf * A_STAGE + A_BYTES, off, ra[4 + i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) st_lds_b128(Bs0 + buf * B_BYTES, (tid + 256 * i) * 16, rb[i]);
  };
  v4f acc[4][4];
#pragma unroll
  for (int mi = 0; mi < 4; ++mi)
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = v4f{0, 0, 0, 0};
  const int steps = p.Np / 64;
  if (steps > 0) {
    load(0);
    store(0);
  }
  __syncthreads();
  for (int s = 0; s < steps; ++s) {
    const int buf = s & 1;
    if (s + 1 < steps) load((s + 1) * 64);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v8h fb[4];
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) {
        // lane group g takes columns 8 (g % 2) .. of block 2 h + g / 2; output
        // block ni of the wave is k block wn, its 16 k's number ni
        const int g = lane >> 4, j = lane & 15;
        const int t = (2 * h + (g >> 1)) * 2 + wn;
        fb[ni] = bytes_to_half(ld_lds_tr8(Bs0 + buf * B_BYTES,
                                          t * 1024 + (16 * ni + 8 * (g & 1) + (j >> 1)) * 16 + (j & 1) * 8));
      }
#pragma unroll
      for (int mi = 0; mi < 4; ++mi) {
        const int row = wm * 64 + mi * 16 + (lane & 15);
        const int off = row * 128 + (((h * 4 + (lane >> 4)) ^ (row & 7)) << 4);
        const v8h fa = __builtin_bit_cast(v8h, ld_lds_b128(smem + buf * A_STAGE, off));
#pragma unroll
        for (int ni = 0; ni < 4; ++ni)
          acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa, fb[ni], acc[mi][ni], 0, 0, 0);
        if constexpr (SPLIT) {
          const v8h fl = __builtin_bit_cast(v8h, ld_lds_b128(smem + buf * A_STAGE + A_BYTES, off));
#pragma unroll
          for (int ni = 0; ni < 4; ++ni)
            acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl, fb[ni], acc[mi][ni], 0, 0, 0);
        }
      }
    }
    if (s + 1 < steps) store(buf ^ 1);
    __syncthreads();
  }
  typedef typename Elem<TYPE>::T T;
#pragma unroll
  for (int mi = 0; mi < 4; ++mi)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = m0 + wm * 64 + mi * 16 + 4 * (lane >> 4) + e;
      if (row >= p.M) continue;
      const float un = 1.0f / p.norm[row];   // a power of two: exact
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) {
        const int col = n0 + wn * 64 + ni * 16 + (lane & 15);
        if (col < p.K) ((T *)p.X)[(int64_t)row * p.ldx + col] = (T)(acc[mi][ni][e] * un);
      }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

bool float_type(int type) { return type == VT_TYPE_F32 || type == VT_TYPE_F16 || type == VT_TYPE_BF16; }

constexpr int64_t kScaledMax = (int64_t)1 << 30;

template <int TYPE, bool ALIGNED>
void launch_quant_typed(const QuantArgs &a, int64_t M, hipStream_t s) {
  const dim3 grid((unsigned)M);
  if (a.Kp <= 1024) hipLaunchKernelGGL((quant_rows_kernel<TYPE, ALIGNED, 64, 1>), grid, dim3(64), 0, s, a);
  else if (a.Kp <= 4096) hipLaunchKernelGGL((quant_rows_kernel<TYPE, ALIGNED, 256, 1>), grid, dim3(256), 0, s, a);
  else if (a.Kp <= 8192) hipLaunchKernelGGL((quant_rows_kernel<TYPE, ALIGNED, 256, 2>), grid, dim3(256), 0, s, a);
  else if (a.Kp <= 16384) hipLaunchKernelGGL((quant_rows_kernel<TYPE, ALIGNED, 256, 4>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((quant_rows_kernel<TYPE, ALIGNED, 256, 0>), grid, dim3(256), 0, s, a);
}

int launch_quant(const QuantArgs &a, int type, int64_t M, hipStream_t s) {
  const int64_t e = elem_size(type);
  const bool al = aligned16(a.X) && a.ldx * e % 16 == 0;
  switch (type) {
    case VT_TYPE_F32: al ? launch_quant_typed<kF32, true>(a, M, s) : launch_quant_typed<kF32, false>(a, M, s); break;
    case VT_TYPE_F16: al ? launch_quant_typed<kF16, true>(a, M, s) : launch_quant_typed<kF16, false>(a, M, s); break;
    default: al ? launch_quant_typed<kBF16, true>(a, M, s) : launch_quant_typed<kBF16, false>(a, M, s); break;
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

// X (any type) -> rows of Kp int8 values: int8 rows that are already so are
// used where they are, others are copied (int8) or rounded to a workspace.
int take_rows(const void *X, int type, int64_t ldx, const float *T, int64_t M, int64_t K, Scratch &scr, Rows *out) {
  const int64_t Kp = scaled_kp(K);
  if ((type == VT_TYPE_I8 && K == Kp && ldx % 16 == 0 && aligned16(X)) || type == VT_TYPE_I8_PADDED) {
    *out = Rows{(const int8_t *)X, T, ldx};
    return VT_OK;
  }
  void *w = nullptr;
  const size_t q_bytes = (size_t)M * Kp;
  if (int rc = scr.take(kRows, q_bytes + (size_t)M * sizeof(float), &w)) return rc;
  QuantArgs a = {X, (int8_t *)w, (float *)((int8_t *)w + q_bytes), ldx, Kp, K, Kp};
  *out = Rows{a.Q, type == VT_TYPE_I8 ? T : a.T, Kp};
  if (type == VT_TYPE_I8) {
    for (int64_t r0 = 0; r0 < M; r0 += 65535) {
      QuantArgs b = a;
      b.X = (const int8_t *)X + r0 * ldx;
      b.Q = a.Q + r0 * Kp;
      const unsigned rows = (unsigned)std::min<int64_t>(M - r0, 65535);
      hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)((Kp + 4095) / 4096), rows), dim3(256), 0,
                         (hipStream_t)scr.stream, b);
    }
    VT_HIP_CHECK(hipGetLastError());
    return VT_OK;
  }
  return launch_quant(a, type, M, (hipStream_t)scr.stream);
}

template <int OP, int ACT>
int launch_finish_typed(const FinishArgs &a, int type, hipStream_t s) {
  const int cols = OP == 2 ? a.Np / 2 : a.N;
  for (int r0 = 0; r0 < a.M; r0 += 65535) {
    FinishArgs b = a;
    b.S = a.S + (int64_t)r0 * a.Np;
    b.t = a.t + r0;
    b.D = a.D ? (const int8_t *)a.D + (int64_t)r0 * a.ldd * elem_size(type) : nullptr;
    b.norm = a.norm ? a.norm + r0 : nullptr;
    b.Y = (int8_t *)a.Y + (OP == 2 ? (int64_t)r0 * a.Np * 2 : (int64_t)r0 * a.ldy * elem_size(type));
    const dim3 grid((unsigned)((cols + 255) / 256), (unsigned)std::min(a.M - r0, 65535));
    switch (type) {
      case VT_TYPE_F32: hipLaunchKernelGGL((finish_kernel<kF32, OP, ACT>), grid, dim3(256), 0, s, b); break;
      case VT_TYPE_F16: hipLaunchKernelGGL((finish_kernel<kF16, OP, ACT>), grid, dim3(256), 0, s, b); break;
      default: hipLaunchKernelGGL((finish_kernel<kBF16, OP, ACT>), grid, dim3(256), 0, s, b); break;
    }
  }
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

template <int OP>
int launch_finish(const FinishArgs &a, int type, int act, hipStream_t s) {
  if (OP == 0 || act == VT_ACT_SILU) return launch_finish_typed<OP, VT_ACT_SILU>(a, type, s);
  return launch_finish_typed<OP, VT_ACT_GELU>(a, type, s);
}

// int32 sums [M][Np] of rows and packed weights into a workspace.
int take_sums(const Rows &rows, const int8_t *Bp, int64_t M, int64_t Kp, int64_t Np, Scratch &scr, int32_t **out) {
  void *w = nullptr;
  if (int rc = scr.take(kSums, (size_t)M * Np * sizeof(int32_t), &w)) return rc;
  *out = (int32_t *)w;
  const Problem q = {rows.q, Bp, nullptr, *out, M, Np, Kp, rows.ld, 0, 0, Np, 1, 0, 0, 0, 0};
  return run_packed(q, 0, scr);
}

template <bool LINEAR>
int launch_row_terms(const TermArgs &a, int type, hipStream_t s) {
  const dim3 grid((unsigned)a.M);
  switch (type) {
    case VT_TYPE_F32: hipLaunchKernelGGL((row_terms_kernel<kF32, LINEAR>), grid, dim3(256), 0, s, a); break;
    case VT_TYPE_F16: hipLaunchKernelGGL((row_terms_kernel<kF16, LINEAR>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((row_terms_kernel<kBF16, LINEAR>), grid, dim3(256), 0, s, a); break;
  }
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

int launch_grad(GradArgs a, int type, hipStream_t s) {
  a.tiles_m = (a.M + 127) / 128;
  a.tiles_n = (a.Kp + 127) / 128;
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
  if (tiles > 0x7fffffff) return fail(VT_EUNSUPPORTED, "gradient grid too large");
  const dim3 grid((unsigned)tiles);
  switch (type) {
    case VT_TYPE_F32: hipLaunchKernelGGL((grad_kernel<kF32, true>), grid, dim3(256), 0, s, a); break;
    case VT_TYPE_F16: hipLaunchKernelGGL((grad_kernel<kF16, false>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((grad_kernel<kBF16, false>), grid, dim3(256), 0, s, a); break;
  }
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
  if (c.M >= kScaledMax || c.K >= kScaledMax || c.N >= kScaledMax / 2)
    return fail(VT_EINVAL, "%s: size beyond 2^30", c.who);
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
  if (c.x_type == VT_TYPE_I8_PADDED && (c.ldx % 16 || !aligned16(c.X)))
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

// K == 0: the sums are zero. Cleared by a kernel (a captured memset is none of
// the library's).
__global__ __launch_bounds__(256) void zero_sums_kernel(int32_t *S, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) S[i] = 0;
}

int forward(const ScaledCall &c, int act, void *stream) {
  bool empty = false;
  if (int rc = check_scaled(c, &empty)) return rc;
  if (act != VT_ACT_SILU && act != VT_ACT_GELU) return fail(VT_EINVAL, "%s: unknown activation %d", c.who, act);
  if (empty) return VT_OK;
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  hipStream_t s = (hipStream_t)stream;
  const int64_t Kp = scaled_kp(c.K), Np = scaled_np(c.N, c.pair);
  Rows rows;
  if (int rc = take_rows(c.X, c.x_type, c.ldx, c.T, c.M, c.K, scr, &rows)) return rc;
  int32_t *sums = nullptr;
  if (c.K > 0) {
    if (int rc = take_sums(rows, c.Bp, c.M, Kp, Np, scr, &sums)) return rc;
  } else {
    void *w = nullptr;
    if (int rc = scr.take(kSums, (size_t)c.M * Np * sizeof(int32_t), &w)) return rc;
    sums = (int32_t *)w;
    const int64_t n = c.M * Np;
    if (n > ((int64_t)1 << 38)) return fail(VT_EUNSUPPORTED, "%s: output too large", c.who);
    hipLaunchKernelGGL(zero_sums_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, sums, n);
  }
  const FinishArgs f = {sums, rows.t, c.meta, nullptr, nullptr, c.Y, 0, c.ldy, 0, (int)c.M, (int)c.N, (int)Np};
  return c.pair ? launch_finish<1>(f, c.y_type, act, s) : launch_finish<0>(f, c.y_type, act, s);
}

// The gradient in x^: D [M][ldd] of N columns, X the output [M][ldx] of K.
int backward(const ScaledCall &c, const int8_t *Q, int q_type, int64_t ldq, const float *t, int act, void *stream) {
  bool empty = false;
  if (int rc = check_scaled(c, &empty)) return rc;
  if (act != VT_ACT_SILU && act != VT_ACT_GELU) return fail(VT_EINVAL, "%s: unknown activation %d", c.who, act);
  if (!float_type(c.x_type) || c.x_type != c.y_type)
    return fail(VT_EINVAL, "%s: the gradients have one floating type", c.who);
  const int64_t Kp = scaled_kp(c.K), Np = scaled_np(c.N, c.pair);
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
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  hipStream_t s = (hipStream_t)stream;
  // Terms in float16, normalised by row; of float32 gradients also what
  // float16 leaves of each (two products).
  const bool split = c.x_type == VT_TYPE_F32;
  const int64_t lo = split ? c.M * Np : 0;
  void *w = nullptr;
  const size_t t_bytes = ((size_t)c.M * Np * 2 * (split ? 2 : 1) + 255) / 256 * 256;
  if (int rc = scr.take(kTerms, t_bytes + (size_t)c.M * sizeof(float), &w)) return rc;
  _Float16 *terms = (_Float16 *)w;
  float *norm = (float *)((int8_t *)w + t_bytes);
  const TermArgs ta = {c.X, t, c.meta, norm, terms, c.ldx, lo, (int)c.M, (int)c.N, (int)Np};
  if (!c.pair || c.N == 0) {
    if (int rc = launch_row_terms<true>(ta, c.x_type, s)) return rc;
  } else {
    if (int rc = launch_row_terms<false>(ta, c.x_type, s)) return rc;
    Rows rows;
    if (int rc = take_rows(Q, q_type, ldq, t, c.M, c.K, scr, &rows)) return rc;
    int32_t *sums = nullptr;
    if (int rc = take_sums(rows, c.Bp, c.M, Kp, Np, scr, &sums)) return rc;
    const FinishArgs f = {sums, rows.t, c.meta, c.X, norm, terms, c.ldx, 0, lo, (int)c.M, (int)c.N, (int)Np};
    if (int rc = launch_finish<2>(f, c.x_type, act, s)) return rc;
  }
  const GradArgs g = {terms, c.Bp, norm, c.Y, c.ldy, lo, (int)c.M, (int)c.K, (int)Kp, (int)Np, 0, 0};
  return launch_grad(g, c.y_type, s);
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
  if (M < 0 || K < 0 || M >= kScaledMax || K >= kScaledMax)
    return fail(VT_EINVAL, "vt_quant_rows: needs 0 <= M, K < 2^30 (M=%lld K=%lld)", (long long)M, (long long)K);
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
  if (K < 0 || N < 0 || K >= kScaledMax || N >= kScaledMax / 2)
    return fail(VT_EINVAL, "vt_scaled_size: needs 0 <= K < 2^30, 0 <= N < 2^29 (K=%lld N=%lld)", (long long)K, (long long)N);
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
  if (Np / 64 > 65535) return fail(VT_EUNSUPPORTED, "vt_scaled_pack: N=%lld too large", (long long)N);
  Extent e0, e1, eb;
  if (!operand_extent(W0, 1, 0, K, ldw0, N, 1, &e0) || !operand_extent(Bp, 1, 0, 1, 0, size, 1, &eb) ||
      (pair && !operand_extent(W1, 1, 0, K, ldw1, N, 1, &e1)))
    return fail(VT_EINVAL, "vt_scaled_pack: extent beyond 2^56 bytes");
  if (K > 0 && (overlaps(e0, eb) || (pair && overlaps(e1, eb))))
    return fail(VT_EINVAL, "vt_scaled_pack: Bp overlaps the weights in memory");
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const ScaledPackArgs a = {W0, W1, s0, s1, bias, Bp, meta, ldw0, ldw1, (int)K, (int)N, (int)Kp, (int)Np};
  hipLaunchKernelGGL(pack_scaled_kernel, dim3((unsigned)std::max<int64_t>(Kp / 64, 1), (unsigned)(Np / 64)), dim3(256), 0,
                     (hipStream_t)stream, a);
  VT_HIP_CHECK(hipGetLastError());
  if (pair) {
    hipLaunchKernelGGL(pack_bound_kernel, dim3((unsigned)((N + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
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
