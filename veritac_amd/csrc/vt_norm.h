// vt_norm.h -- root-mean-square norm of rows, with the residual's addition in
// front and int8 rows with scales, or rows of x's type, behind, and its
// gradients. Part of vt_hip_gemm.hip's translation unit, after vt_scaled.h.
//
//   h_ij = x_ij + r_ij, rounded to x's type (x itself without r)
//   y_ij = h_ij g_j / sqrt(mean_j h_ij^2 + eps)
//   rows: z = h g, top_i = max_j |z_ij|, q = round(z (127 / top)), t = top / 127 / sqrt(..)
//   dx_ij = (z_ij - n_ij mean_j(z_ij n_ij)) / sqrt(..) + dh_ij, z = dy g, n = h / sqrt(..)
//   dg_j = sum_i dy_ij n_ij
//
// A row's int8 values do not depend on its norm, which is a factor of its scale
// only, so one reduction (of the squares' sum and the largest |z|) serves both.
// Everything is float32 between the loads and the one rounding at the store.

namespace {

// 8 elements of a row as they lie in memory, and their values. Apart, since a
// value's conversion in a branch around its load waits for that load there. `late`:
// by how many elements they begin before the piece, whose end is past the row's:
// a row's last piece is read as the row's last 8 elements and moved, without a
// branch (element loads of it, each waited for, took 3 us of an odd row's 8).
template <int TYPE>
struct Raw8 {
  v4i w[TYPE == kF32 ? 2 : 1];
  int late;

  __device__ __forceinline__ void settle() {
    if (!__any(late)) return;
    if constexpr (TYPE == kF32) {
#pragma unroll
      for (int b = 4; b; b >>= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int from = e + b < 8 ? w[(e + b) >> 2 & 1][(e + b) & 3] : 0, is = w[e >> 2][e & 3];
          w[e >> 2][e & 3] = (late & b) ? from : is;
        }
      if (late >= 8) w[0] = w[1] = v4i{0, 0, 0, 0};
    } else {
      uint64_t lo = (uint32_t)w[0][0] | (uint64_t)(uint32_t)w[0][1] << 32, hi = (uint32_t)w[0][2] | (uint64_t)(uint32_t)w[0][3] << 32;
      if (late & 4) {
        lo = hi;
        hi = 0;
      }
      const int s = 16 * (late & 3);
      lo = s ? lo >> s | hi << (64 - s) : lo;
      hi >>= s;
      if (late >= 8) lo = hi = 0;
      w[0] = v4i{(int)(uint32_t)lo, (int)(lo >> 32), (int)(uint32_t)hi, (int)(hi >> 32)};
    }
    late = 0;
  }
};

// From `pos`, zero past `len`, as 16-byte vectors at any alignment; rows of fewer
// than 8 by elements.
template <int TYPE>
__device__ __forceinline__ Raw8<TYPE> raw8(const typename Elem<TYPE>::T *row, int64_t pos, int64_t len) {
  constexpr int N = TYPE == kF32 ? 2 : 1;
  Raw8<TYPE> r;
  if (len >= 8) {
    const int64_t at = min(pos, len - 8);
    r.late = (int)min(pos - at, (int64_t)8);
#pragma unroll
    for (int i = 0; i < N; ++i) r.w[i] = *(const v4i_any *)(row + at + i * (8 / N));
  } else {
    r.late = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) r.w[i] = v4i{0, 0, 0, 0};
    typedef typename std::conditional<TYPE == kF32, uint32_t, uint16_t>::type Bits;
    const Bits *b = (const Bits *)row;
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (pos + e < len) {
        if constexpr (TYPE == kF32) r.w[e >> 2][e & 3] = (int)b[pos + e];
        else r.w[0][e >> 1] |= (int)((uint32_t)b[pos + e] << (16 * (e & 1)));
      }
  }
  return r;
}

// Of a settled piece.
template <int TYPE>
__device__ __forceinline__ float raw_value(const Raw8<TYPE> &r, int e) {
  if constexpr (TYPE == kF32) {
    const int b = r.w[e >> 2][e & 3];
    return __int_as_float(b);
  } else {
    const uint32_t b = (uint32_t)r.w[0][e >> 1] >> (16 * (e & 1)) & 0xffffu;
    return from16(b, TYPE);
  }
}

template <int TYPE>
__device__ __forceinline__ void raw_values(Raw8<TYPE> r, float (&v)[8]) {
  r.settle();
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = raw_value<TYPE>(r, e);
}

template <int TYPE>
__device__ __forceinline__ void load8(const typename Elem<TYPE>::T *row, int64_t pos, int64_t len, float (&v)[8]) {
  raw_values<TYPE>(raw8<TYPE>(row, pos, len), v);
}

template <int TYPE>
__device__ __forceinline__ void store8(typename Elem<TYPE>::T *row, int64_t pos, int64_t len, const float (&v)[8]) {
  typedef typename Elem<TYPE>::T T;
  constexpr int PER = 16 / sizeof(T);
  if (pos + 8 <= len) {
    typedef T VT __attribute__((ext_vector_type(PER), aligned(sizeof(T))));
#pragma unroll
    for (int i = 0; i < 8 / PER; ++i) {
      VT x;
#pragma unroll
      for (int e = 0; e < PER; ++e) x[e] = (T)v[i * PER + e];
      *(VT *)(row + pos + i * PER) = x;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (pos + e < len) row[pos + e] = (T)v[e];
  }
}

// The norm's weights, float32 or of the rows' type.
template <int TYPE>
__device__ __forceinline__ void load_gain(const void *g, bool wide, int64_t pos, int64_t len, float (&v)[8]) {
  if (wide || TYPE == kF32) load8<kF32>((const float *)g, pos, len, v);
  else load8<TYPE>((const typename Elem<TYPE>::T *)g, pos, len, v);
}

// Sum and maximum over a workgroup, of two values at once.
template <int THREADS, class A, class B, class FA, class FB>
__device__ __forceinline__ void block_two(A &a, B &b, FA fa, FB fb, uint64_t *red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    a = fa(a, __builtin_bit_cast(A, __shfl_xor(__builtin_bit_cast(int, a), o)));
    b = fb(b, __builtin_bit_cast(B, __shfl_xor(__builtin_bit_cast(int, b), o)));
  }
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0)
      red[threadIdx.x >> 6] = (uint64_t)__builtin_bit_cast(uint32_t, a) << 32 | __builtin_bit_cast(uint32_t, b);
    __syncthreads();
    uint64_t w = red[0];
    a = __builtin_bit_cast(A, (uint32_t)(w >> 32));
    b = __builtin_bit_cast(B, (uint32_t)w);
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) {
      w = red[i];
      a = fa(a, __builtin_bit_cast(A, (uint32_t)(w >> 32)));
      b = fb(b, __builtin_bit_cast(B, (uint32_t)w));
    }
    __syncthreads();   // red is the next row's after this
  }
}

__device__ __forceinline__ float add_f(float a, float b) { return a + b; }
__device__ __forceinline__ uint32_t max_u(uint32_t a, uint32_t b) { return max(a, b); }

// The power of two that a row is scaled by: 1, unless the squares' sum has left
// float32's range at the top, or is so small beside an eps of next to nothing
// that squares were lost at the bottom. 2^100 keeps the mean of one least value's
// square (2^-149) over the longest row a normal number, and eps f^2 below 2^120;
// a larger eps leaves room for 2^80.
__device__ __forceinline__ float row_factor(float squares, float eps) {
  if (magnitude(squares) >= kInfBits) return 0x1p-80f;
  if (squares >= 0x1p-80f || eps >= 0x1p-60f) return 1.0f;
  return eps < 0x1p-80f ? 0x1p100f : 0x1p80f;
}

// 1 / sqrt(mean + eps) of a row scaled by f, over f: n = (h f) * this.
__device__ __forceinline__ float inverse_rms(float squares, float f, float k, float eps) {
  return 1.0f / sqrtf(squares / k + eps * f * f);
}

// What dx needs of a row scaled by f besides it: dx = ((z - h f c) a b) + dh.
struct RowUse {
  float c, a, b;
};
// c = dot / k inv^2 and inv f = a b. A row that was too small (f > 1) has a dot
// product that would vanish in the division, and float32 may have no normal number
// for inv f: two factors then, of which b is 1 in any other row.
__device__ __forceinline__ RowUse row_use(float dot, float k, float inv, float f) {
  RowUse r = {dot / k * inv * inv, inv * f, 1.0f};
  if (f != 1.0f) {
    if (f > 1.0f) r.c = dot * inv / k * inv;
    if (!(r.a >= 0x1p-126f && magnitude(r.a) < kInfBits)) {
      r.a = inv;
      r.b = f;
    }
  }
  return r;
}

struct NormArgs {
  const void *X, *R, *G;   // R null: no residual
  void *H, *Y;             // H: h, null without a residual; Y: [M][ldy] of the type, or int8 rows
  float *T;                // scales of int8 rows, null: Y is floating
  int64_t ldx, ldr, ldh, ldy, M, K, Kp;
  float eps;
  int gain32;
};

// A workgroup takes rows w, w + grid, ..; a thread holds NC pieces of 8 elements
// of the row and of the gain in registers (NC = 0: longer rows, read again after
// the reduction, and the gain with them). Bound by one read of x and r and one
// write of h and y: 8192 x 4096 bfloat16 with a residual into int8 rows in 44.5 us
// (235 MB, 5.3 TB/s; a large copy reaches 5.2). One row in 2.9: its chain of load,
// reduction and store.
template <int TYPE, int THREADS, int NC, bool ROWS>
__global__ __launch_bounds__(THREADS) void norm_kernel(NormArgs p) {
  __shared__ uint64_t red[THREADS / 64];
  typedef typename Elem<TYPE>::T T;
  constexpr int N = NC ? NC : 1;
  const int tid = threadIdx.x;
  float g[N][8];
  auto pos_of = [&](int i) { return (int64_t)(tid + THREADS * i) * 8; };
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) load_gain<TYPE>(p.G, p.gain32, pos_of(i), p.K, g[i]);
  }
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    const T *x = (const T *)p.X + row * p.ldx, *r = (const T *)p.R + row * p.ldr;
    // h of a piece, in x's precision; again: as the thread has stored it (over r, maybe)
    auto load_h = [&](int64_t pos, float (&v)[8], bool again) {
      if (again && p.H) {
        load8<TYPE>((const T *)p.H + row * p.ldh, pos, p.K, v);
        return;
      }
      load8<TYPE>(x, pos, p.K, v);
      if (p.R) {
        float w[8];
        load8<TYPE>(r, pos, p.K, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)(T)(v[e] + w[e]);
      }
    };
    float v[N][8];
    float squares = 0.0f;
    uint32_t top = 0;
    auto gather = [&](const float (&h)[8], const float (&w)[8], float f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = h[e] * f;
        squares = fmaf(a, a, squares);
        if constexpr (ROWS) top = max(top, magnitude(a * w[e]));
      }
    };
    auto all = [&](float f, bool first) {
      squares = 0.0f;
      top = 0;
      if constexpr (NC > 0) {
#pragma unroll
        for (int i = 0; i < NC; ++i) gather(v[i], g[i], f);
      } else {
        for (int64_t pos = tid * 8; pos < p.K; pos += THREADS * 8) {
          load_h(pos, v[0], !first);
          if (first && p.H) store8<TYPE>((T *)p.H + row * p.ldh, pos, p.K, v[0]);
          load_gain<TYPE>(p.G, p.gain32, pos, p.K, g[0]);
          gather(v[0], g[0], f);
        }
      }
      block_two<THREADS>(squares, top, add_f, max_u, red);
    };
    if constexpr (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) load_h(pos_of(i), v[i], false);
      if (p.H) {
#pragma unroll
        for (int i = 0; i < NC; ++i) store8<TYPE>((T *)p.H + row * p.ldh, pos_of(i), p.K, v[i]);
      }
    }
    all(1.0f, true);
    const float f = row_factor(squares, p.eps);
    if (f != 1.0f) all(f, false);
    const float inv = inverse_rms(squares, f, (float)p.K, p.eps);
    const RowScale s = row_scale(top);
    if (ROWS && tid == 0) p.T[row] = p.K ? s.scale * inv : 0.0f;
    auto put = [&](int64_t pos, const float (&h)[8], const float (&w)[8]) {
      if constexpr (ROWS) {
        if (pos >= p.Kp) return;
        uint32_t b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = round_byte(h[e] * f * w[e], s.inv);
        v2i o = {pack_bytes(b[0], b[1], b[2], b[3]), pack_bytes(b[4], b[5], b[6], b[7])};
        if (s.inv == 0.0f) o = v2i{0, 0};
        *(v2i *)((int8_t *)p.Y + row * p.ldy + pos) = o;
      } else {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = h[e] * f * w[e] * inv;
        store8<TYPE>((T *)p.Y + row * p.ldy, pos, p.K, y);
      }
    };
    if constexpr (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) put(pos_of(i), v[i], g[i]);
    } else {
      for (int64_t pos = tid * 8; pos < (ROWS ? p.Kp : p.K); pos += THREADS * 8) {
        load_h(pos, v[0], true);
        load_gain<TYPE>(p.G, p.gain32, pos, p.K, g[0]);
        put(pos, v[0], g[0]);
      }
    }
  }
}

struct NormGradArgs {
  const void *D, *H, *G, *E;   // dy, h, the gain and the residual's own gradient (or null)
  void *X;                     // dx
  float *part;                 // [groups][K] partial sums of the gain's gradient, null: not wanted
  float *stats;                // rows longer than kNormGradRow: four floats a row: f, inv, and c and b of RowUse
  int64_t ldd, ldh, lde, ldx, M, K;
  float eps;
  int gain32;
};

// A workgroup takes rows w, w + grid, .. whole, and keeps its part of the gain's
// gradient in registers over them: dy, h and dh are read once. 4096 x 4096 bfloat16
// in 25 - 29 us (134 MB, 4.6 - 5.4 TB/s; 31 with each load's conversion in the branch
// around it), 333 x 1001 float32 in 5.8.
template <int TYPE, int THREADS, int NC>
__global__ __launch_bounds__(THREADS) void norm_grad_kernel(NormGradArgs p) {
  __shared__ uint64_t red[THREADS / 64];
  typedef typename Elem<TYPE>::T T;
  const int tid = threadIdx.x;
  float g[NC][8], sum[NC][8];
  auto pos_of = [&](int i) { return (int64_t)(tid + THREADS * i) * 8; };
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    load_gain<TYPE>(p.G, p.gain32, pos_of(i), p.K, g[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[i][e] = 0.0f;
  }
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    float d[NC][8], h[NC][8], x[NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      load8<TYPE>((const T *)p.D + row * p.ldd, pos_of(i), p.K, d[i]);
      load8<TYPE>((const T *)p.H + row * p.ldh, pos_of(i), p.K, h[i]);
      if (p.E) load8<TYPE>((const T *)p.E + row * p.lde, pos_of(i), p.K, x[i]);
    }
    float squares, dot;
    auto all = [&](float f) {
      squares = dot = 0.0f;
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = h[i][e] * f;
          squares = fmaf(a, a, squares);
          dot = fmaf(d[i][e] * g[i][e], a, dot);
        }
      block_two<THREADS>(squares, dot, add_f, add_f, red);
    };
    all(1.0f);
    const float f = row_factor(squares, p.eps);
    if (f != 1.0f) all(f);
    const float inv = inverse_rms(squares, f, (float)p.K, p.eps);
    const RowUse use = row_use(dot, (float)p.K, inv, f);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = h[i][e] * f;
        sum[i][e] = fmaf(d[i][e], a * inv, sum[i][e]);
        y[e] = (d[i][e] * g[i][e] - a * use.c) * use.a;
      }
      if (use.b != 1.0f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= use.b;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = p.E ? x[i][e] + y[e] : y[e];
      store8<TYPE>((T *)p.X + row * p.ldx, pos_of(i), p.K, x[i]);
    }
  }
  if (p.part) {
#pragma unroll
    for (int i = 0; i < NC; ++i) store8<kF32>(p.part + blockIdx.x * p.K, pos_of(i), p.K, sum[i]);
  }
}

// Rows too long for a workgroup's registers: first what dx needs of each row, a
// workgroup each up to 2^20 (as many as CUs hold, which take rows in turn, are 2 %
// slower over 4096 x 16384; a launch has less than 2^22),
template <int TYPE>
__global__ __launch_bounds__(1024) void norm_stats_kernel(NormGradArgs p) {
  __shared__ uint64_t red[16];
  typedef typename Elem<TYPE>::T T;
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    float squares, dot;
    auto all = [&](float f) {
      squares = dot = 0.0f;
      for (int64_t pos = threadIdx.x * 8; pos < p.K; pos += 8192) {
        float d[8], h[8], g[8];
        load8<TYPE>((const T *)p.D + row * p.ldd, pos, p.K, d);
        load8<TYPE>((const T *)p.H + row * p.ldh, pos, p.K, h);
        load_gain<TYPE>(p.G, p.gain32, pos, p.K, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = h[e] * f;
          squares = fmaf(a, a, squares);
          dot = fmaf(d[e] * g[e], a, dot);
        }
      }
      block_two<1024>(squares, dot, add_f, add_f, red);
    };
    all(1.0f);
    const float f = row_factor(squares, p.eps);
    if (f != 1.0f) all(f);
    if (threadIdx.x == 0) {
      const float inv = inverse_rms(squares, f, (float)p.K, p.eps);
      float *s = p.stats + row * 4;
      const RowUse use = row_use(dot, (float)p.K, inv, f);
      s[0] = f;
      s[1] = inv;
      s[2] = use.c;
      s[3] = use.b;
    }
  }
}

// then dx and the gain's gradient, 2048 columns of rows w, w + gridDim.x, .. each.
template <int TYPE>
__global__ __launch_bounds__(256) void norm_apply_kernel(NormGradArgs p) {
  typedef typename Elem<TYPE>::T T;
  const int64_t pos = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
  float g[8], sum[8];
  load_gain<TYPE>(p.G, p.gain32, pos, p.K, g);
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.0f;
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    const v4f s = *(const v4f *)(p.stats + row * 4);
    const float f = s[0], inv = s[1], c = s[2], b = s[3], a1 = b == 1.0f ? inv * f : inv;
    float d[8], h[8], x[8];
    load8<TYPE>((const T *)p.D + row * p.ldd, pos, p.K, d);
    load8<TYPE>((const T *)p.H + row * p.ldh, pos, p.K, h);
    if (p.E) load8<TYPE>((const T *)p.E + row * p.lde, pos, p.K, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = h[e] * f;
      sum[e] = fmaf(d[e], a * inv, sum[e]);
      d[e] = (d[e] * g[e] - a * c) * a1;
    }
    if (b != 1.0f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] *= b;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p.E ? x[e] + d[e] : d[e];
    store8<TYPE>((T *)p.X + row * p.ldx, pos, p.K, x);
  }
  if (p.part) store8<kF32>(p.part + blockIdx.x * p.K, pos, p.K, sum);
}

// The sums of `groups` rows of K partial sums, in one order: 64 columns a
// workgroup, its 16 waves every 16th row, 8 loads in flight (512 x 4096 in 4.2 us;
// on four waves 9.4).
struct GainSumArgs {
  const float *part;
  void *out;
  int64_t K;
  int groups, type;
};

__global__ __launch_bounds__(1024) void gain_sum_kernel(GainSumArgs p) {
  __shared__ float red[16][64];
  const int c = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + c;
  float s = 0.0f;
  if (col < p.K) {
    for (int i = wave; i < p.groups; i += 128) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = i + 16 * u < p.groups ? p.part[(int64_t)(i + 16 * u) * p.K + col] : 0.0f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
  }
  red[wave][c] = s;
  __syncthreads();
  if (wave || col >= p.K) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += red[i][c];
  if (p.type == VT_TYPE_F32) ((float *)p.out)[col] = s;
  else ((uint16_t *)p.out)[col] = (uint16_t)pack16(s, 0.0f, p.type);
}

// int8 rows as the values they stand for (8192 x 4096 to bfloat16 in 16 us: 101 MB).
struct DequantArgs {
  const int8_t *Q;
  const float *T;
  void *Y;
  int64_t ldq, ldy, M, K;
};

template <int TYPE>
__global__ __launch_bounds__(256) void dequant_kernel(DequantArgs p) {
  typedef typename Elem<TYPE>::T T;
  const int64_t pieces = (p.K + 7) / 8;
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    const float t = p.T[row];
    const int8_t *q = p.Q + row * p.ldq;
    for (int64_t i = threadIdx.x; i < pieces; i += 256) {
      const int64_t pos = i * 8;
      typedef int8_t V8 __attribute__((ext_vector_type(8), aligned(1)));
      float v[8];
      if (pos + 8 <= p.K) {
        const V8 b = *(const V8 *)(q + pos);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)b[e] * t;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = pos + e < p.K ? (float)q[pos + e] * t : 0.0f;
      }
      store8<TYPE>((T *)p.Y + row * p.ldy, pos, p.K, v);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// Workgroups for rows of `threads` threads each: as many as are resident at once.
int64_t resident(int64_t rows, int threads, int cus) { return std::min<int64_t>(rows, (int64_t)cus * (2048 / threads)); }

template <int TYPE, bool ROWS>
void launch_norm_typed(const NormArgs &a, int cus, hipStream_t s) {
  const int64_t k = ROWS ? a.Kp : a.K;
  auto grid = [&](int threads) { return dim3((unsigned)resident(a.M, threads, cus)); };
  if (k <= 512) hipLaunchKernelGGL((norm_kernel<TYPE, 64, 1, ROWS>), grid(64), dim3(64), 0, s, a);
  else if (k <= 2048) hipLaunchKernelGGL((norm_kernel<TYPE, 256, 1, ROWS>), grid(256), dim3(256), 0, s, a);
  else if (k <= 4096) hipLaunchKernelGGL((norm_kernel<TYPE, 512, 1, ROWS>), grid(512), dim3(512), 0, s, a);
  else if (k <= 8192) hipLaunchKernelGGL((norm_kernel<TYPE, 1024, 1, ROWS>), grid(1024), dim3(1024), 0, s, a);
  else if (k <= 16384) hipLaunchKernelGGL((norm_kernel<TYPE, 1024, 2, ROWS>), grid(1024), dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((norm_kernel<TYPE, 1024, 0, ROWS>), grid(1024), dim3(1024), 0, s, a);
}

template <int TYPE>
int launch_norm(const NormArgs &a, int cus, hipStream_t s) {
  if (a.T) launch_norm_typed<TYPE, true>(a, cus, s);
  else launch_norm_typed<TYPE, false>(a, cus, s);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

// Longest rows whose gradients a workgroup holds in registers.
constexpr int64_t kNormGradRow = 8192;

template <int TYPE>
int launch_norm_grad(NormGradArgs a, void *dgain, int gain_type, Scratch &scr) {
  hipStream_t s = (hipStream_t)scr.stream;
  const int cus = scr.st->num_cus;
  const int threads = a.K <= 512 ? 64 : a.K <= 2048 ? 256 : a.K <= 4096 ? 512 : a.K <= kNormGradRow ? 1024 : 256;
  // One workgroup more of a row's size costs the gain's sums a row more to read.
  const int64_t groups = a.K <= kNormGradRow ? std::min<int64_t>(a.M, (int64_t)cus * (1024 / threads))
                                             : std::min<int64_t>(a.M, std::max<int64_t>(1, cus * 8 / ((a.K + 2047) / 2048)));
  void *w = nullptr;
  if (dgain || a.K > kNormGradRow) {
    const size_t part = dgain ? ((size_t)groups * a.K * sizeof(float) + 255) / 256 * 256 : 0;
    const size_t stats = a.K > kNormGradRow ? (size_t)a.M * 4 * sizeof(float) : 0;
    if (int rc = scr.take(kPartials, part + stats, &w)) return rc;
    a.part = dgain ? (float *)w : nullptr;
    a.stats = (float *)((int8_t *)w + part);
  }
  const dim3 grid((unsigned)groups);
  if (a.M == 0) ;   // dgain = 0
  else if (threads == 64) hipLaunchKernelGGL((norm_grad_kernel<TYPE, 64, 1>), grid, dim3(64), 0, s, a);
  else if (a.K <= 2048) hipLaunchKernelGGL((norm_grad_kernel<TYPE, 256, 1>), grid, dim3(256), 0, s, a);
  else if (threads == 512) hipLaunchKernelGGL((norm_grad_kernel<TYPE, 512, 1>), grid, dim3(512), 0, s, a);
  else if (threads == 1024) hipLaunchKernelGGL((norm_grad_kernel<TYPE, 1024, 1>), grid, dim3(1024), 0, s, a);
  else {
    hipLaunchKernelGGL((norm_stats_kernel<TYPE>), dim3((unsigned)std::min<int64_t>(a.M, 1 << 20)), dim3(1024), 0, s, a);
    VT_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL((norm_apply_kernel<TYPE>), dim3((unsigned)groups, (unsigned)((a.K + 2047) / 2048)), dim3(256), 0, s, a);
  }
  VT_HIP_CHECK(hipGetLastError());
  if (!dgain) return VT_OK;
  const GainSumArgs g = {a.part, dgain, a.K, (int)groups, gain_type};
  hipLaunchKernelGGL(gain_sum_kernel, dim3((unsigned)((a.K + 63) / 64)), dim3(1024), 0, s, g);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

// An operand of a call: [rows][ld] of `cols` elements of `elem` bytes, from a
// base and rows aligned to `align` of them. Null and empty ones are left out.
struct Operand {
  const char *name;
  const void *p;
  int64_t rows, ld, cols, elem;
  bool out;
  int64_t align = 1;
};

// Pitches, alignment and extents of up to 16 operands, and that no output
// shares memory with another operand.
int check_operands(const char *who, const Operand *o, int count) {
  Extent e[16];
  for (int i = 0; i < count; ++i) {
    if (!o[i].p || o[i].rows == 0 || o[i].cols == 0) continue;
    if (o[i].rows > 1 && (o[i].ld < o[i].cols || o[i].ld > ((int64_t)1 << 40)))
      return fail(VT_EINVAL, "%s: pitch of %s (%lld) must be %lld .. 2^40", who, o[i].name, (long long)o[i].ld, (long long)o[i].cols);
    if ((uintptr_t)o[i].p % (o[i].elem * o[i].align) || (o[i].rows > 1 && o[i].ld % o[i].align))
      return fail(VT_EINVAL, "%s: %s is not aligned to %lld bytes", who, o[i].name, (long long)(o[i].elem * o[i].align));
    if (!operand_extent(o[i].p, 1, 0, o[i].rows, o[i].ld, o[i].cols, o[i].elem, &e[i]))
      return fail(VT_EINVAL, "%s: extent of %s beyond 2^56 bytes", who, o[i].name);
    for (int j = 0; j < i; ++j)
      if (o[j].p && o[j].rows && o[j].cols && (o[i].out || o[j].out) && overlaps(e[i], e[j]))
        return fail(VT_EINVAL, "%s: %s and %s share memory", who, o[j].name, o[i].name);
  }
  return VT_OK;
}

int check_norm_sizes(const char *who, int64_t M, int64_t K, int32_t type, int32_t gain_type, float eps) {
  if (M < 0 || K < 0 || M > kScaledMaxM || K >= kScaledMax)
    return fail(VT_EINVAL, "%s: needs 0 <= M <= %lld, 0 <= K < 2^30 (M=%lld K=%lld)", who, (long long)kScaledMaxM, (long long)M,
                (long long)K);
  if (!float_type(type)) return fail(VT_EINVAL, "%s: unknown type %d", who, (int)type);
  if (gain_type != VT_TYPE_F32 && gain_type != type)
    return fail(VT_EINVAL, "%s: the gain is float32 or of the rows' type (got %d)", who, (int)gain_type);
  if (!(eps >= 0.0f) || eps > 3.0e38f) return fail(VT_EINVAL, "%s: eps must be a number of at least 0", who);
  return VT_OK;
}

// f(the element type, at compile time).
template <class F>
int by_type(int type, F &&f) {
  switch (type) {
    case VT_TYPE_F32: return f(std::integral_constant<int, kF32>());
    case VT_TYPE_F16: return f(std::integral_constant<int, kF16>());
    default: return f(std::integral_constant<int, kBF16>());
  }
}

}  // namespace

extern "C" {

int vt_norm(const void *X, int64_t ldx, const void *R, int64_t ldr, int32_t type, const void *gain, int32_t gain_type,
            float eps, void *H, int64_t ldh, void *Y, int64_t ldy, float *T, int64_t M, int64_t K, void *stream) {
  g_err.clear();
  const char *who = "vt_norm";
  if (int rc = check_norm_sizes(who, M, K, type, gain_type, eps)) return rc;
  if (M == 0 || (K == 0 && !T)) return VT_OK;
  if (K > 0 && (!X || !gain || !Y || !R != !H)) return fail(VT_EINVAL, "%s: an operand is null, or only one of R and H given", who);
  const int64_t e = elem_size(type), Kp = scaled_kp(K);
  const bool in_place = H == R && ldh == ldr;
  const Operand o[] = {{"X", X, M, ldx, K, e, false}, {"R", in_place ? nullptr : R, M, ldr, K, e, false},
                       {"gain", gain, 1, K, K, elem_size(gain_type), false}, {"H", H, M, ldh, K, e, true},
                       {"Y", Y, M, ldy, T ? Kp : K, T ? 1 : e, true, T ? 16 : 1}, {"T", T, 1, M, M, 4, true}};
  if (int rc = check_operands(who, o, 6)) return rc;
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const NormArgs a = {X, R, gain, H, Y, T, ldx, ldr, ldh, ldy, M, K, Kp, eps, gain_type == VT_TYPE_F32};
  return by_type(type, [&](auto t) { return launch_norm<decltype(t)::value>(a, scr.st->num_cus, (hipStream_t)stream); });
}

int vt_norm_grad(const void *dY, int64_t ldd, const void *H, int64_t ldh, const void *dH, int64_t lde, int32_t type,
                 const void *gain, int32_t gain_type, float eps, void *dX, int64_t ldx, void *dgain, int64_t M, int64_t K,
                 void *stream) {
  g_err.clear();
  const char *who = "vt_norm_grad";
  if (int rc = check_norm_sizes(who, M, K, type, gain_type, eps)) return rc;
  if (K > (int64_t)65535 * 2048) return fail(VT_EUNSUPPORTED, "%s: rows of more than 65535 times 2048 (K=%lld)", who, (long long)K);
  if (K == 0 || (M == 0 && !dgain)) return VT_OK;
  if (!gain || (M > 0 && (!dY || !H || !dX))) return fail(VT_EINVAL, "%s: an operand is null", who);
  const int64_t e = elem_size(type), ge = elem_size(gain_type);
  const Operand o[] = {{"dY", dY, M, ldd, K, e, false}, {"H", H, M, ldh, K, e, false}, {"dH", dH, M, lde, K, e, false},
                       {"gain", gain, 1, K, K, ge, false}, {"dX", dX, M, ldx, K, e, true}, {"dgain", dgain, 1, K, K, ge, true}};
  if (int rc = check_operands(who, o, 6)) return rc;
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const NormGradArgs a = {dY, H, gain, dH, dX, nullptr, nullptr, ldd, ldh, lde, ldx, M, K, eps, gain_type == VT_TYPE_F32};
  return by_type(type, [&](auto t) { return launch_norm_grad<decltype(t)::value>(a, dgain, gain_type, scr); });
}

int vt_dequant_rows(const int8_t *Q, int64_t ldq, const float *T, void *Y, int32_t y_type, int64_t ldy, int64_t M, int64_t K,
                    void *stream) {
  g_err.clear();
  const char *who = "vt_dequant_rows";
  if (M < 0 || K < 0 || M > kScaledMaxM || K >= kScaledMax)
    return fail(VT_EINVAL, "%s: needs 0 <= M <= %lld, 0 <= K < 2^30 (M=%lld K=%lld)", who, (long long)kScaledMaxM, (long long)M,
                (long long)K);
  if (!float_type(y_type)) return fail(VT_EINVAL, "%s: unknown output type %d", who, (int)y_type);
  if (M == 0 || K == 0) return VT_OK;
  if (!Q || !T || !Y) return fail(VT_EINVAL, "%s: an operand is null", who);
  const Operand o[] = {{"Q", Q, M, ldq, K, 1, false}, {"T", T, 1, M, M, 4, false}, {"Y", Y, M, ldy, K, elem_size(y_type), true}};
  if (int rc = check_operands(who, o, 3)) return rc;
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const DequantArgs a = {Q, T, Y, ldq, ldy, M, K};
  const dim3 grid((unsigned)resident(M, 256, scr.st->num_cus));
  return by_type(y_type, [&](auto t) {
    hipLaunchKernelGGL((dequant_kernel<decltype(t)::value>), grid, dim3(256), 0, (hipStream_t)stream, a);
    VT_HIP_CHECK(hipGetLastError());
    return VT_OK;
  });
}

}  // extern "C"
