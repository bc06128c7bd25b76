// vt_adapter.h -- low-rank adapters of many requests beside an int8 linear layer,
// and their gradients. Part of vt_hip_gemm.hip's translation unit, after
// vt_norm.h.
//
//   u_ir = c sum_k x_ik A_ark, a the row's adapter    (A [L][R][K]: down)
//   y_ij = t_i s_j sum_k q_ik W_kj + b_j + sum_r u_ir B_ajr    (B [L][N][R]: up)
//   h_ir = c sum_j dy_ij B_ajr
//   dx_ik = sum_j dy_ij s_j W_kj + sum_r h_ir A_ark
//   dA_ark = sum_i h_ir x_ik, dB_ajr = sum_i u_ir dy_ij, over the adapter's rows
//
// u and h are float32 [M][Rp] and come from a kernel of their own; the second
// product is added where the int8 product's (or the gradient's) sums lie in
// registers, so y and dx are rounded and written once. Adapters are laid out
// with the rank padded to Rp (whole 16s) and the long side to that of the packed
// weights, zeros in between, once with the contraction's index innermost for each
// product that reads them.

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int kMaxRank = 128, kMaxAdapters = 65535;   // adapters: a side of a grid
constexpr int64_t rank_pad(int64_t R) { return (R + 15) / 16 * 16; }

// One pair of an adapter's layouts: [L][Rp][Kp] for x . A^T and [L][Np][Rp] for
// u . B^T forward, [L][Rp][Np] for dy . B and [L][Kp][Rp] for h . A backward.
struct AdapterLayout {
  int64_t Kp, Np, Rp, L;
  int64_t first(bool back) const { return L * Rp * (back ? Np : Kp); }
  int64_t second(bool back) const { return L * Rp * (back ? Kp : Np); }
};

AdapterLayout adapter_layout(int64_t K, int64_t N, int64_t R, int64_t L) {
  return {scaled_kp(K), scaled_np(N, false), rank_pad(R), L};
}

struct AdapterPackArgs {
  const uint8_t *A, *B;   // down [L][R][K], up [L][N][R]
  uint8_t *first, *second;
  int K, N, R, Kp, Np, Rp;
  int back, elem;
};

// A workgroup lays out 64 of an adapter's long side by all of its rank, through
// LDS, reading and writing along whichever side is innermost. blockIdx.z: down or
// up.
template <class T>
__global__ __launch_bounds__(256) void adapter_pack_kernel(AdapterPackArgs p) {
  __shared__ T tile[64][kMaxRank + 2];
  const bool up = blockIdx.z;
  const int len = up ? p.N : p.K, lenp = up ? p.Np : p.Kp, a = blockIdx.y, j0 = blockIdx.x * 64;
  if (j0 >= lenp) return;
  const T *src = (const T *)(up ? p.B : p.A) + (int64_t)a * p.R * len;
  for (int i = threadIdx.x; i < 64 * p.Rp; i += 256) {
    // down is [R][K], up [N][R]
    const int j = up ? i / p.Rp : i & 63, r = up ? i % p.Rp : i >> 6;
    T v = T(0);
    if (j0 + j < len && r < p.R) v = up ? src[(int64_t)(j0 + j) * p.R + r] : src[(int64_t)r * len + j0 + j];
    tile[j][r] = v;
  }
  __syncthreads();
  // forward, down keeps its order and up too; backward both turn
  const bool rank_inner = up != (p.back != 0);
  T *dst = (T *)(up != (p.back != 0) ? p.second : p.first) + (int64_t)a * p.Rp * lenp;
  for (int i = threadIdx.x; i < 64 * p.Rp; i += 256) {
    if (rank_inner) dst[(int64_t)(j0 + i / p.Rp) * p.Rp + i % p.Rp] = tile[i / p.Rp][i % p.Rp];
    else dst[(int64_t)(i >> 6) * lenp + j0 + (i & 63)] = tile[i & 63][i >> 6];
  }
}

// ---------------------------------------------------------------------------
// u = c x . A^T
// ---------------------------------------------------------------------------

struct ShrinkArgs {
  const void *X;        // rows [M][ldx] of the adapters' type, or int8
  const float *t;       // int8 rows' scales
  const void *P;        // [L][Rp][lenp]
  const int32_t *which; // [M], or null: all rows have adapter 0
  float *U;             // [M][Rp]
  int64_t ldx;
  float scale;
  int M, len, lenp, L, Rp;
};

// 8 elements of a row from `pos` as floats, zero past `len`; int8 rows too.
template <int TYPE, bool I8>
__device__ __forceinline__ void load_row8(const void *row, int pos, int len, float (&v)[8]) {
  if constexpr (I8) {
    const int8_t *q = (const int8_t *)row;
    typedef int8_t V8 __attribute__((ext_vector_type(8), aligned(1)));
    if (pos + 8 <= len) {
      const V8 b = *(const V8 *)(q + pos);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)b[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = pos + e < len ? (float)q[pos + e] : 0.0f;
    }
  } else {
    load8<TYPE>((const typename Elem<TYPE>::T *)row, pos, len, v);
  }
}

// What a row's sums are multiplied by: a NaN for an adapter that is not there.
template <bool I8>
__device__ __forceinline__ float shrink_factor(const ShrinkArgs &p, int row, int a) {
  if (a >= p.L) return __uint_as_float(0x7fc00000u);
  return I8 ? p.scale * p.t[row] : p.scale;
}

// Up to 64 rows, each with an adapter of its own maybe: 16 ranks of a row to a
// workgroup, a wave for each, 8 columns a lane. Bound by the latency of its few
// loads and, with many adapters, by reading them.
template <int TYPE, bool I8>
__global__ __launch_bounds__(1024) void shrink_rows_kernel(ShrinkArgs p) {
  typedef typename Elem<TYPE>::T T;
  const int row = blockIdx.x, rank = blockIdx.y * 16 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int a = p.which ? p.which[row] : 0;
  float s = 0.0f;
  if (a >= 0 && a < p.L) {
    const void *x = I8 ? (const void *)((const int8_t *)p.X + row * p.ldx) : (const void *)((const T *)p.X + row * p.ldx);
    const T *w = (const T *)p.P + ((int64_t)a * p.Rp + rank) * p.lenp;
#pragma unroll 4
    for (int pos = lane * 8; pos < p.lenp; pos += 512) {
      float v[8], b[8];
      load_row8<TYPE, I8>(x, pos, p.len, v);
      load8<TYPE>(w, pos, p.lenp, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(v[e], b[e], s);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  }
  if (lane == 0) p.U[(int64_t)row * p.Rp + rank] = a < 0 ? 0.0f : s * shrink_factor<I8>(p, row, a);
}

// A 16 x 32 by 32 x 16 product (16 x 16 x 16 steps of 4 in float32) of fragments
// of 8 values a lane: row or column lane % 16, k 8 (lane / 16) + e. In float32 the
// order of k within the 32 is another, the same on both sides.
template <int TYPE>
struct Frag;
template <>
struct Frag<kF32> {
  float v[8];
};
template <>
struct Frag<kF16> {
  v8h v;
};
template <>
struct Frag<kBF16> {
  v8bf v;
};

template <int TYPE>
__device__ __forceinline__ Frag<TYPE> to_frag(const float (&f)[8]) {
  Frag<TYPE> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = (typename Elem<TYPE>::T)f[e];
  return r;
}
// 8 stored values, 16-byte aligned.
template <int TYPE>
__device__ __forceinline__ Frag<TYPE> load_frag(const typename Elem<TYPE>::T *p) {
  Frag<TYPE> r;
  if constexpr (TYPE == kF32) {
    const v4f a = *(const v4f *)p, b = *(const v4f *)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r.v[e] = a[e];
      r.v[4 + e] = b[e];
    }
  } else {
    r.v = *(const decltype(r.v) *)p;
  }
  return r;
}
template <int TYPE>
__device__ __forceinline__ v4f mfma16(const Frag<TYPE> &a, const Frag<TYPE> &b, v4f c) {
  if constexpr (TYPE == kF16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0);
  else if constexpr (TYPE == kBF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
  else {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], c, 0, 0, 0);
    return c;
  }
}
// The adapters of 16 rows, one after another: f(adapter, its rows as bits). a: that
// of row lane % 16, negative for none. All rows are multiplied by each and only its
// own are taken: a row is never touched by what another's adapter holds.
template <class F>
__device__ __forceinline__ void each_adapter(int a, F &&f) {
  uint32_t todo = (uint32_t)__ballot(a >= 0) & 0xffff;
  while (todo) {
    const int cur = __builtin_amdgcn_readlane(a, __builtin_ctz(todo));
    const uint32_t rows = (uint32_t)__ballot(a == cur) & 0xffff;
    todo &= ~rows;
    f(cur, rows);
  }
}

// More rows: 16 rows by 16 ranks to a workgroup, whose 8 waves take 32-deep
// slices in turn (4 of them in flight) and join through LDS.
template <int TYPE, bool I8>
__global__ __launch_bounds__(512) void shrink_tiles_kernel(ShrinkArgs p) {
  typedef typename Elem<TYPE>::T T;
  constexpr int WAVES = 8, U = 4;
  __shared__ float red[WAVES][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int row0 = blockIdx.x * 16, rank0 = blockIdx.y * 16;
  const int row = min(row0 + c, p.M - 1);
  int a = p.which ? p.which[row] : 0;
  if (a >= p.L) a = -1;
  const void *x = I8 ? (const void *)((const int8_t *)p.X + row * p.ldx) : (const void *)((const T *)p.X + row * p.ldx);
  const T *w = (const T *)p.P + (int64_t)(rank0 + c) * p.lenp + 8 * g;
  const int64_t step = (int64_t)p.Rp * p.lenp;
  v4f acc = {0, 0, 0, 0};
  for (int k0 = wave * 32; k0 < p.lenp; k0 += WAVES * U * 32) {
    Frag<TYPE> xa[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[8];
      load_row8<TYPE, I8>(x, k0 + u * WAVES * 32 + 8 * g, p.len, v);
      xa[u] = to_frag<TYPE>(v);
    }
    each_adapter(a, [&](int cur, uint32_t rows) {
      Frag<TYPE> b[U];
      v4f part = {0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < U; ++u) b[u] = load_frag<TYPE>(w + cur * step + min(k0 + u * WAVES * 32, p.lenp - 32));
#pragma unroll
      for (int u = 0; u < U; ++u) part = mfma16<TYPE>(xa[u], b[u], part);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (rows >> (4 * g + e) & 1) acc[e] += part[e];
    });
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) red[wave][4 * g + e][c] = acc[e];
  __syncthreads();
  if (threadIdx.x < 256) {
    const int r = threadIdx.x >> 4, rank = threadIdx.x & 15, i = row0 + r;
    if (i < p.M) {
      float s = 0.0f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) s += red[v][r][rank];
      const int ad = p.which ? p.which[i] : 0;
      p.U[(int64_t)i * p.Rp + rank0 + rank] = ad < 0 ? 0.0f : s * shrink_factor<I8>(p, i, ad);
    }
  }
}

// ---------------------------------------------------------------------------
// u . B^T, where the int8 product's sums lie
// ---------------------------------------------------------------------------

// u and the adapters' second layout: row i adds sum_r U[i][r] V[which_i][col][r].
struct LowRank {
  const float *U;
  const void *V;          // [L][colsp][Rp]
  const int32_t *which;
  int64_t colsp;
  int L, Rp, rows;
};

// The adapter of a row for the second product: that of no adapter is below 0,
// and that of one which is not there (its u is NaN) is any.
__device__ __forceinline__ int adapter_of(const LowRank &l, int row) {
  return l.which ? min(l.which[row], l.L - 1) : 0;
}

// One element of it, 8 ranks at a time.
template <int TYPE>
__device__ __forceinline__ float low_rank_element(const LowRank &l, int row, int64_t col) {
  const int a = adapter_of(l, row);
  if (a < 0) return 0.0f;
  const float *u = l.U + (int64_t)row * l.Rp;
  const typename Elem<TYPE>::T *v = (const typename Elem<TYPE>::T *)l.V + (a * l.colsp + col) * l.Rp;
  float s = 0.0f;
  for (int r = 0; r < l.Rp; r += 8) {
    const Frag<TYPE> b = load_frag<TYPE>(v + r);
    const v4f x = *(const v4f *)(u + r), y = *(const v4f *)(u + r + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(x[e], (float)b.v[e], s);
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(y[e], (float)b.v[4 + e], s);
  }
  return s;
}

__device__ __forceinline__ float low_rank_element(const LowRank &l, int type, int row, int64_t col) {
  if (type == VT_TYPE_F32) return low_rank_element<kF32>(l, row, col);
  return type == VT_TYPE_F16 ? low_rank_element<kF16>(l, row, col) : low_rank_element<kBF16>(l, row, col);
}

// Blocks of 16 x 16 in the accumulators' layout: d[ni] element e is row row0 +
// 4 (lane / 16) + e, column col0 + 16 ni + lane % 16. Columns below colsp, any rows.
// 16-bit adapters: 16 ranks are one 32-deep product, of u in two halves (16 bits
// of it in bfloat16, 22 in float16; u is then as exact as the 16-bit y that it is
// added to needs, 2^-8 of a step) against the same 16 values. float16 halves are of
// u times a power of two for each row, so that none overflows or is lost.
template <int TYPE, int NI>
__device__ __forceinline__ void low_rank16(const LowRank &l, int row0, int col0, int lane, v4f (&d)[NI]) {
  typedef typename Elem<TYPE>::T T;
  const int g = lane >> 4, c = lane & 15, row = min(row0 + c, l.rows - 1);
  const float *u = l.U + (int64_t)row * l.Rp;
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) d[ni] = v4f{0, 0, 0, 0};
  each_adapter(adapter_of(l, row), [&](int cur, uint32_t rows) {
    const T *v = (const T *)l.V + (cur * l.colsp + col0 + c) * l.Rp;
    v4f t[NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) t[ni] = v4f{0, 0, 0, 0};
    if constexpr (TYPE == kF32) {
      for (int r = 0; r < l.Rp; r += 16) {
        const v4f a = *(const v4f *)(u + r + 4 * g);
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) {
          const v4f b = *(const v4f *)(v + (int64_t)ni * 16 * l.Rp + r + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) t[ni] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], t[ni], 0, 0, 0);
        }
      }
    } else {
      for (int r = 0; r < l.Rp; r += 16) {
        const int at = r + 8 * (g & 1);
        const v4f a0 = *(const v4f *)(u + at), a1 = *(const v4f *)(u + at + 4);
        float f[8];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f[e] = e < 4 ? a0[e & 3] : a1[e & 3];
          top = max(top, magnitude(f[e]));
        }
        float back = 1.0f;
        if constexpr (TYPE == kF16) {
          top = max(top, (uint32_t)__shfl_xor((int)top, 16));
          const float norm = normaliser(__uint_as_float(top));
          back = 1.0f / norm;
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= norm;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float hi = (float)(T)f[e];
          // (inf - inf of an infinite u would make a NaN of its low half)
          f[e] = g < 2 ? hi : magnitude(hi) < kInfBits ? f[e] - hi : 0.0f;
        }
        const Frag<TYPE> a = to_frag<TYPE>(f);
        if constexpr (TYPE == kF16) {
          v4f un;
#pragma unroll
          for (int e = 0; e < 4; ++e) un[e] = __shfl(back, 4 * g + e);
#pragma unroll
          for (int ni = 0; ni < NI; ++ni) {
            const v4f p = mfma16<TYPE>(a, load_frag<TYPE>(v + (int64_t)ni * 16 * l.Rp + at), v4f{0, 0, 0, 0});
#pragma unroll
            for (int e = 0; e < 4; ++e) t[ni][e] = fmaf(p[e], un[e], t[ni][e]);
          }
        } else {
#pragma unroll
          for (int ni = 0; ni < NI; ++ni) t[ni] = mfma16<TYPE>(a, load_frag<TYPE>(v + (int64_t)ni * 16 * l.Rp + at), t[ni]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool mine = rows >> (4 * g + e) & 1;
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) d[ni][e] = mine ? t[ni][e] : d[ni][e];
    }
  });
}

// A linear layer's outputs with adapters. TYPE: of adapters and outputs.
template <int TYPE>
struct AdaptedTile : ScaledTile<kLinear, TYPE == kF32 ? 4 : 2> {
  LowRank low;
  static constexpr int OE = TYPE == kF32 ? 4 : 2;

  template <int MI, int NI, bool EDGE>
  __device__ __forceinline__ void tile16(const v4i (&acc)[MI][NI], int row0, int col0, int row_min, int col_min, int lane,
                                         LDS_AS int8_t *lds) const {
    constexpr int W = NI * 16, PITCH = W * OE, RC = PITCH / 16;
    const int g = lane >> 4, c = lane & 15;
    float s[NI], b[NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      s[ni] = this->meta[col0 + ni * 16 + c];
      b[ni] = this->meta[this->Np + col0 + ni * 16 + c];
    }
    auto swz = [](int row) { return (((row >> 2) & 3) * OE) & (RC - 1); };
    int wb[NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) wb[ni] = 4 * g * PITCH + (((ni * OE + (c * OE >> 4)) ^ swz(4 * g)) << 4) + (c * OE & 15);
    each([&](auto strip) __attribute__((always_inline)) {
      constexpr int mi = decltype(strip)::value;
      const v4f tr = *(const v4f_any *)(this->t + row0 + mi * 16 + 4 * g);
      v4f d[NI];
      low_rank16<TYPE, NI>(low, row0 + mi * 16, col0, lane, d);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ((float)acc[mi][ni][e] * tr[e] * s[ni] + b[ni]) + d[ni][e];
        this->template put4<PITCH>(lds + wb[ni], v[0], v[1], v[2], v[3]);
      }
      this->template store_rows<W>(lds, swz, row0 + mi * 16, col0, 0, lane, EDGE ? row_min : 0, col_min);
      __builtin_amdgcn_sched_barrier(0);
    }, std::make_integer_sequence<int, MI>());
  }

  // 32 x 32 blocks (element e of lane l: row 8 (e / 4) + 4 (l / 32) + e % 4, column
  // l % 32), two of them beside each other, as the sums of four 16 x 16 products
  // each: those go through the wave's LDS, 16 rows by 64 columns of float32 at a
  // time, to where the int32 sums lie, which then leave the same way.
  template <int MI, int NI>
  __device__ __forceinline__ void tile32(const v16i (&acc)[MI][NI], int row0, int col0, int lane, LDS_AS int8_t *lds) const {
    static_assert(NI == 2, "strips of 64 columns");
    if (col0 >= this->Np) return;   // the same for the whole wave, behind the last barrier
    const int g = lane >> 5, c = lane & 31;
    LDS_AS float *f = (LDS_AS float *)lds;   // [32][64]
    each([&](auto strip) __attribute__((always_inline)) {
      constexpr int mi = decltype(strip)::value;
      const int first = row0 + mi * 32;
      if (first >= this->M) return;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v4f d[4];
        low_rank16<TYPE, 4>(low, first + 16 * h, col0, lane, d);
#pragma unroll
        for (int ni = 0; ni < 4; ++ni)
#pragma unroll
          for (int e = 0; e < 4; ++e) f[(16 * h + 4 * (lane >> 4) + e) * 64 + ni * 16 + (lane & 15)] = d[ni][e];
      }
#pragma unroll
      for (int ni = 0; ni < 2; ++ni) {
        const int j = col0 + ni * 32 + c;
        const float s = this->meta[j], b = this->meta[this->Np + j];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int r = 8 * (e >> 2) + 4 * g + (e & 3);
          LDS_AS float *at = f + r * 64 + ni * 32 + c;
          *at = ((float)acc[mi][ni][e] * this->t[min(first + r, this->M - 1)] * s + b) + *at;
        }
      }
      // 8 columns of a row to a lane
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 3), k = (lane & 7) * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = f[r * 64 + k + e];
        if (first + r < this->M && col0 + k < this->N)
          this->store8((int64_t)(first + r) * this->ldy + col0 + k, v, this->N - (col0 + k), this->type);
      }
    }, std::make_integer_sequence<int, MI>());
  }

  __device__ __forceinline__ void element(int32_t a0, int32_t, int row, int pc, int j, float t_row) const {
    if (j >= this->N) return;
    const float v = ((float)a0 * t_row * this->meta[pc] + this->meta[this->Np + pc]) + low_rank_element(low, this->type, row, j);
    const int64_t at = (int64_t)row * this->ldy + j;
    if (this->type == VT_TYPE_F32) ((float *)this->Y)[at] = v;
    else ((uint16_t *)this->Y)[at] = (uint16_t)pack16(v, 0.0f, this->type);
  }
};

// dx with the adapters' part.
template <int TYPE>
struct AdaptedGrad : ScaledTile<kGrad> {
  LowRank low;

  template <int G, int MI, int NI, class ACC>
  __device__ __forceinline__ void blocks16(const ACC (&acc)[MI][NI], int row0, int col0, int lane, LDS_AS int8_t *lds,
                                           const float *early) const {
    const int g = lane >> 4, c = lane & 15;
    const float one[2] = {1.0f, 1.0f};
    this->template strips<MI / G, 16 * G, NI * 16>(
        [&](auto strip) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < G; ++i) {
            constexpr int first = decltype(strip)::value * G;
            const int rel = (first + i) * 16;
            v4f d[NI];
            // columns past the last are not stored, and read from before it
            low_rank16<TYPE, NI>(low, row0 + rel, min(col0, (int)low.colsp - NI * 16), lane, d);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float unit = __shfl(rel >= 64 ? early[1] : early[0], (rel + 4 * g + e) & 63);
#pragma unroll
              for (int ni = 0; ni < NI; ++ni)
                *(LDS_AS float *)(lds + (16 * i + 4 * g + e) * (64 * NI) + ((((ni ^ g) << 2) + (c >> 2)) << 4) + (c & 3) * 4) =
                    acc[first + i][ni][e] * unit + d[ni][e];
            }
          }
        },
        [](int row) { return ((row >> 2) & 3) << 2; }, row0, col0, M, lane, lds, one);
  }
};

template <int TYPE, int BM>
__global__ __launch_bounds__(256, 1) void adapted_dx_kernel(GradArgs p, AdaptedGrad<TYPE> out) {
  grad_tiles<BM>(p, out);
}

// Up to 64 rows: by elements, whose type is the outputs'.
template <int NBW, int MB, int XB>
__global__ __launch_bounds__(512) void adapted_skinny_kernel(ScaledSkinnyArgs p, AdaptedTile<kBF16> o) {
  skinny_rows<kLinear, NBW, MB, XB>(p, o);
}

__global__ __launch_bounds__(256) void adapted_finish_kernel(const int32_t *S, int slices, AdaptedTile<kBF16> out) {
  finish_rows<kLinear>(S, slices, out);
}

// dx from partial sums, with the adapters' part.
__global__ __launch_bounds__(256) void adapted_dx_sum_kernel(GradSumArgs p, LowRank low) {
  sum_grad_slices(p, [&](int row, int col) { return low_rank_element(low, p.type, row, col); });
}

// ---------------------------------------------------------------------------
// dA = h^T x, dB = u^T dy
// ---------------------------------------------------------------------------

struct OuterArgs {
  const float *H;          // [M][Rp]
  const void *Z;           // [M][ldz] of the type
  const int32_t *which;
  float *part;             // [splits][L][Rp][colsp], null: one split, straight to Out
  void *Out;               // [L][R][cols], or (turned) [L][cols][R]
  int64_t ldz;
  int M, cols, colsp, L, R, Rp, splits, turned;
};

// 16 ranks by 128 columns of one adapter over one range of rows to a workgroup.
// Its waves take 4 rows at a time in turn, as 4-deep float32 products (nothing is
// rounded on the way, whatever the type): lane l holds 8 columns of row l / 16,
// and product j takes column j of every lane's. The rows of other adapters are
// left out by a list of this one's rows, made in order 1024 rows at a time.
template <int TYPE>
__global__ __launch_bounds__(256) void outer_kernel(OuterArgs p) {
  typedef typename Elem<TYPE>::T T;
  constexpr int ROWS = 1024;
  __shared__ int list[ROWS];
  __shared__ int counts[4][4];
  __shared__ float red[4][16][132];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const int ranks = p.Rp / 16, tiles = (p.cols + 127) / 128;
  const int tile = blockIdx.x % tiles, rank0 = blockIdx.x / tiles % ranks * 16;
  const int a = blockIdx.y, split = blockIdx.z;
  const int col = tile * 128 + 8 * c;
  const int beg = (int)((int64_t)p.M * split / p.splits), end = (int)((int64_t)p.M * (split + 1) / p.splits);
  v4f acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = v4f{0, 0, 0, 0};
  for (int r0 = beg; r0 < end; r0 += ROWS) {
    int n = min(ROWS, end - r0);
    if (p.which) {
      // thread t looks at rows t, t + 256, ..: a wave's 64 rows are consecutive
      bool has[4];
      uint64_t mask[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = r0 + i * 256 + tid;
        has[i] = row < r0 + n && p.which[row] == a;
        mask[i] = __ballot(has[i]);
        if (lane == 0) counts[i][wave] = __popcll(mask[i]);
      }
      __syncthreads();
      int total = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if (w == wave && has[i]) list[total + __popcll(mask[i] & ((1ull << lane) - 1))] = r0 + i * 256 + tid;
          total += counts[i][w];
        }
      }
      n = total;
      __syncthreads();
    }
    constexpr int U = 4;
    for (int i0 = wave * 4 * U; i0 < n; i0 += 16 * U) {
      float h[U], z[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + 4 * u + g;
        h[u] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) z[u][e] = 0.0f;
        if (i < n) {
          const int row = p.which ? list[i] : r0 + i;
          h[u] = p.H[(int64_t)row * p.Rp + rank0 + c];
          load8<TYPE>((const T *)p.Z + row * p.ldz, col, p.cols, z[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(h[u], z[u][j], acc[j], 0, 0, 0);
    }
    if (p.which) __syncthreads();   // the list is the next rows'
  }
  // element e of product j: rank rank0 + 4 g + e, column tile * 128 + 8 c + j
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[wave][4 * g + e][8 * c + j] = acc[j][e];
  __syncthreads();
  for (int i = tid; i < 16 * 128; i += 256) {
    // along the innermost side of what is written
    const bool turn = !p.part && p.turned;
    const int r = turn ? i & 15 : i >> 7, k = turn ? i >> 4 : i & 127, at = tile * 128 + k;
    const float s = (red[0][r][k] + red[1][r][k]) + (red[2][r][k] + red[3][r][k]);
    if (p.part) {
      if (at < p.colsp) p.part[(((int64_t)split * p.L + a) * p.Rp + rank0 + r) * p.colsp + at] = s;
    } else if (at < p.cols && rank0 + r < p.R) {
      const int64_t to = p.turned ? ((int64_t)a * p.cols + at) * p.R + rank0 + r : ((int64_t)a * p.R + rank0 + r) * p.cols + at;
      ((T *)p.Out)[to] = (T)s;
    }
  }
}

// The splits' sums, in one order.
template <int TYPE>
__global__ __launch_bounds__(256) void outer_sum_kernel(OuterArgs p) {
  typedef typename Elem<TYPE>::T T;
  const int64_t count = (int64_t)p.R * p.cols, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  const int a = blockIdx.y;
  const int r = (int)(p.turned ? i % p.R : i / p.cols), k = (int)(p.turned ? i / p.R : i % p.cols);
  const float *w = p.part + ((int64_t)a * p.Rp + r) * p.colsp + k;
  const int64_t step = (int64_t)p.L * p.Rp * p.colsp;
  float s = 0.0f;
  for (int n = 0; n < p.splits; n += 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = n + u < p.splits ? w[(n + u) * step] : 0.0f;
#pragma unroll
    for (int u = 0; u < 8; ++u) s += v[u];
  }
  ((T *)p.Out)[a * count + i] = (T)s;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

template <int TYPE, bool I8>
int launch_shrink(const ShrinkArgs &a, hipStream_t s) {
  if (a.M <= kSkinnyMaxM)
    hipLaunchKernelGGL((shrink_rows_kernel<TYPE, I8>), dim3((unsigned)a.M, (unsigned)(a.Rp / 16)), dim3(1024), 0, s, a);
  else
    hipLaunchKernelGGL((shrink_tiles_kernel<TYPE, I8>), dim3((unsigned)((a.M + 15) / 16), (unsigned)(a.Rp / 16)), dim3(512), 0, s, a);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

int shrink(const ShrinkArgs &a, int type, bool i8, hipStream_t s) {
  return by_type(type, [&](auto t) {
    constexpr int TYPE = decltype(t)::value;
    return i8 ? launch_shrink<TYPE, true>(a, s) : launch_shrink<TYPE, false>(a, s);
  });
}

template <int TYPE>
int launch_outer(OuterArgs a, Scratch &scr) {
  hipStream_t s = (hipStream_t)scr.stream;
  const int64_t per = (int64_t)((a.cols + 127) / 128) * (a.Rp / 16), wgs = per * a.L;
  // Rows are split until there are two workgroups for each CU, of 64 rows at
  // least, as far as the partial sums stay within their bound.
  const int64_t bytes = (int64_t)a.L * a.Rp * a.colsp * sizeof(float);
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>({(2 * scr.st->num_cus + wgs - 1) / wgs, (a.M + 63) / 64, kScaledBytes / bytes}));
  a.splits = (int)splits;
  if (splits > 1) {
    void *w = nullptr;
    if (int rc = scr.take(kPartials, (size_t)(splits * bytes), &w)) return rc;
    a.part = (float *)w;
  }
  if (per > 0x7fffffff) return fail(VT_EUNSUPPORTED, "gradient grid too large");
  hipLaunchKernelGGL((outer_kernel<TYPE>), dim3((unsigned)per, (unsigned)a.L, (unsigned)splits), dim3(256), 0, s, a);
  VT_HIP_CHECK(hipGetLastError());
  if (splits > 1) {
    hipLaunchKernelGGL((outer_sum_kernel<TYPE>), dim3((unsigned)(((int64_t)a.R * a.cols + 255) / 256), (unsigned)a.L), dim3(256), 0, s, a);
    VT_HIP_CHECK(hipGetLastError());
  }
  return VT_OK;
}

// What launch_skinny, launch_tiles and launch_grad need of outputs with adapters.
struct AdaptedSkinny : AdaptedTile<kBF16> {
  template <int NBW, int MB, int XB>
  static void skinny(const ScaledSkinnyArgs &a, const AdaptedSkinny &o, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((adapted_skinny_kernel<NBW, MB, XB>), grid, dim3(512), 0, s, a, (const AdaptedTile<kBF16> &)o);
  }
  static int finish(const int32_t *sums, int slices, const AdaptedSkinny &o, hipStream_t s) {
    hipLaunchKernelGGL(adapted_finish_kernel, dim3((unsigned)o.M, (unsigned)((o.Np + 255) / 256)), dim3(256), 0, s, sums, slices,
                       (const AdaptedTile<kBF16> &)o);
    VT_HIP_CHECK(hipGetLastError());
    return VT_OK;
  }
};

template <int TYPE>
struct AdaptedDx : AdaptedGrad<TYPE> {
  static void tiles(const GradArgs &a, int bm, const AdaptedDx &o, dim3 wgs, hipStream_t s) {
    const AdaptedGrad<TYPE> &out = o;
    if (bm == 256) hipLaunchKernelGGL((adapted_dx_kernel<TYPE, 256>), wgs, dim3(256), 0, s, a, out);
    else if (bm == 128) hipLaunchKernelGGL((adapted_dx_kernel<TYPE, 128>), wgs, dim3(256), 0, s, a, out);
    else hipLaunchKernelGGL((adapted_dx_kernel<TYPE, 64>), wgs, dim3(256), 0, s, a, out);
  }
  static void sums(const GradSumArgs &r, const AdaptedDx &o, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL(adapted_dx_sum_kernel, grid, dim3(256), 0, s, r, o.low);
  }
};

// Rows of a forward call, whose u is there.
int adapted_rows(const ScaledCall &c, const LowRank &low, Scratch &scr) {
  const int64_t Kp = scaled_kp(c.K), Np = scaled_np(c.N, false);
  AdaptedSkinny o = {};
  o.meta = c.meta; o.Y = c.Y; o.ldy = c.ldy;
  o.M = (int)c.M; o.N = (int)c.N; o.Np = (int)Np;
  o.type = c.y_type;
  o.low = low;
  Rows rows = {};
  const bool skinny = c.M <= kSkinnyMaxM && Kp > 0;
  if (skinny && float_type(c.x_type) && c.M <= 16 && c.M * Kp <= kFusedValues)
    return launch_skinny<kLinear>(c.X, c.x_type, c.ldx, c.K, rows, c.Bp, o, scr);
  if (int rc = take_rows(c.X, c.x_type, c.ldx, c.T, c.M, c.K, scr, &rows)) return rc;
  o.t = rows.t;
  if (skinny) return launch_skinny<kLinear>(nullptr, 0, 0, c.K, rows, c.Bp, o, scr);
  hipStream_t s = (hipStream_t)scr.stream;
  if (Kp == 0) return AdaptedSkinny::finish(nullptr, 0, o, s);
  const TilePlan plan = tile_plan(false, c.M, Np, Kp, scr.st->num_cus);
  if (plan.ks > 1) {
    const int32_t *sums = nullptr;
    if (int rc = sliced_sums(plan, rows, c.Bp, c.M, Np, Kp, scr, &sums)) return rc;
    return AdaptedSkinny::finish(sums, plan.ks, o, s);
  }
  return by_type(c.y_type, [&](auto t) {
    AdaptedTile<decltype(t)::value> out = {};
    (ScaledOut &)out = o;
    out.low = low;
    return launch_tiles(plan, rows, c.Bp, Kp, out, scr);
  });
}

// Rows of a gradient in x, whose h is there.
int adapted_dx_rows(const ScaledCall &c, const LowRank &low, void *stream) {
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const int64_t Kp = scaled_kp(c.K), Np = scaled_np(c.N, false);
  const bool split = two_halves(c.x_type);
  const int64_t lo = split ? c.M * Np : 0;
  void *w = nullptr;
  const size_t t_bytes = ((size_t)c.M * Np * 2 * (split ? 2 : 1) + 255) / 256 * 256;
  if (int rc = scr.take(kTerms, t_bytes + (size_t)c.M * sizeof(float), &w)) return rc;
  _Float16 *terms = (_Float16 *)w;
  float *norm = (float *)((int8_t *)w + t_bytes);
  const TermArgs ta = {{}, c.X, nullptr, c.meta, norm, terms, c.ldx, lo, (int)c.M, (int)c.N, (int)Np};
  if (int rc = launch_row_terms<true>(ta, c.x_type, (hipStream_t)stream)) return rc;
  const GradArgs g = {terms, c.Bp, lo, (int)c.M, (int)Kp, (int)Np, 0, 0, 0, split ? 2 : 1, 1};
  return by_type(c.x_type, [&](auto t) {
    AdaptedDx<decltype(t)::value> o = {};
    o.Y = c.Y; o.ldy = c.ldy;
    o.M = (int)c.M; o.N = (int)c.K; o.Np = (int)Kp;
    o.type = c.y_type; o.norm = norm;
    o.low = low;
    return launch_grad(g, o, scr);
  });
}

LowRank low_at(LowRank l, int64_t r, int64_t rows) {
  l.U += r * l.Rp;
  if (l.which) l.which += r;
  l.rows = (int)rows;
  return l;
}

struct AdapterCall {
  const char *who;
  int type;
  const void *P;
  int64_t L, R, K, N, M;
  bool back;
  float scale;
  const int32_t *which;
  float *U;
};

int check_adapters(const AdapterCall &c) {
  if (!float_type(c.type)) return fail(VT_EINVAL, "%s: adapters are float32, float16 or bfloat16 (type %d)", c.who, c.type);
  if (c.L < 1 || c.L > kMaxAdapters) return fail(VT_EINVAL, "%s: needs 1 to %d adapters (got %lld)", c.who, kMaxAdapters, (long long)c.L);
  if (c.R < 1 || c.R > kMaxRank) return fail(VT_EINVAL, "%s: needs a rank of 1 to %d (got %lld)", c.who, kMaxRank, (long long)c.R);
  if (c.K < 0 || c.N < 0 || c.K > kScaledMaxK || c.N > kScaledMaxN)
    return fail(VT_EINVAL, "%s: needs 0 <= K <= %lld and 0 <= N <= %lld (K=%lld N=%lld)", c.who, (long long)kScaledMaxK,
                (long long)kScaledMaxN, (long long)c.K, (long long)c.N);
  return VT_OK;
}

}  // namespace

extern "C" {

int64_t vt_adapter_size(int64_t K, int64_t N, int64_t R, int64_t L, int32_t type) {
  const AdapterCall c = {"vt_adapter_size", type, nullptr, L, R, K, N, 0, false, 0.0f, nullptr, nullptr};
  if (int rc = check_adapters(c)) return rc;
  const AdapterLayout l = adapter_layout(K, N, R, L);
  return (l.first(false) + l.second(false)) * elem_size(type);
}

int vt_adapter_pack(const void *down, const void *up, int32_t type, int64_t K, int64_t N, int64_t R, int64_t L, int32_t back,
                    void *P, void *stream) {
  g_err.clear();
  const char *who = "vt_adapter_pack";
  const AdapterCall c = {who, type, P, L, R, K, N, 0, back != 0, 0.0f, nullptr, nullptr};
  if (int rc = check_adapters(c)) return rc;
  const AdapterLayout l = adapter_layout(K, N, R, L);
  const int64_t e = elem_size(type), size = l.first(false) + l.second(false);
  if (size == 0) return VT_OK;
  if (!P || (K > 0 && !down) || (N > 0 && !up)) return fail(VT_EINVAL, "%s: an operand is null", who);
  const Operand o[] = {{"down", down, 1, L * R * K, L * R * K, e, false}, {"up", up, 1, L * R * N, L * R * N, e, false},
                       {"P", P, 1, size, size, e, true, 16 / e}};
  if (int rc = check_operands(who, o, 3)) return rc;
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const AdapterPackArgs a = {(const uint8_t *)down, (const uint8_t *)up, (uint8_t *)P, (uint8_t *)P + l.first(back != 0) * e,
                             (int)K, (int)N, (int)R, (int)l.Kp, (int)l.Np, (int)l.Rp, back != 0, (int)e};
  const dim3 grid((unsigned)(std::max(l.Kp, l.Np) / 64), (unsigned)L, 2);
  if (e == 4) hipLaunchKernelGGL(adapter_pack_kernel<uint32_t>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(adapter_pack_kernel<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, a);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

int vt_adapted_linear(const void *X, int32_t x_type, int64_t ldx, const float *T, int64_t M, int64_t K, const int8_t *Bp,
                      const float *meta, int64_t N, const void *P, int64_t R, int64_t L, float scale, const int32_t *which,
                      float *U, void *Y, int32_t type, int64_t ldy, void *stream) {
  g_err.clear();
  const char *who = "vt_adapted_linear";
  const ScaledCall c = {who, X, x_type, ldx, K, T, Bp, meta, Y, type, ldy, N, M, K, N, false};
  const AdapterCall ad = {who, type, P, L, R, K, N, M, false, scale, which, U};
  if (int rc = check_adapters(ad)) return rc;
  const int64_t Rp = rank_pad(R);
  ScaledCall checked = c;
  if (!Y) {   // u alone
    checked.Y = U;
    checked.y_type = VT_TYPE_F32;
    checked.ldy = checked.yc = Rp;
  }
  bool empty = false;
  if (int rc = check_scaled(checked, &empty)) return rc;
  const bool i8 = !float_type(x_type);
  if (!i8 && x_type != type) return fail(VT_EINVAL, "%s: floating rows have the adapters' type", who);
  if (M == 0) return VT_OK;
  const AdapterLayout l = adapter_layout(K, N, R, L);
  const int64_t e = elem_size(type), size = l.first(false) + l.second(false);
  if (!U || (size > 0 && !P)) return fail(VT_EINVAL, "%s: adapters or U are null", who);
  const Operand o[] = {{"X", X, M, ldx, x_type == VT_TYPE_I8_PADDED ? l.Kp : K, elem_size(x_type), false},
                       {"T", T, 1, M, M, 4, false}, {"weights", Bp, 1, 0, l.Kp * l.Np, 1, false},
                       {"scales", meta, 1, 0, scaled_meta(l.Np), 4, false}, {"adapters", P, 1, size, size, e, false, 16 / e},
                       {"which", which, 1, M, M, 4, false}, {"U", U, 1, M * Rp, M * Rp, 4, true, 4}, {"Y", Y, M, ldy, N, e, true}};
  if (int rc = check_operands(who, o, 8)) return rc;
  const bool copied = !rows_in_place(X, x_type, ldx, K);
  const int64_t step = copied ? rows_at_once(M, l.Kp + 4) : M;
  const LowRank low = {U, (const int8_t *)P + l.first(false) * e, which, l.Np, (int)L, (int)Rp, (int)M};
  {
    Scratch scr;
    if (int rc = open_scratch(stream, &scr)) return rc;
    const ShrinkArgs a = {X, T, P, which, U, ldx, scale, (int)M, (int)K, (int)l.Kp, (int)L, (int)Rp};
    if (int rc = shrink(a, type, i8, (hipStream_t)stream)) return rc;
  }
  if (empty || !Y) return VT_OK;
  for (int64_t r = 0; r < M; r += step) {
    Scratch scr;
    if (int rc = open_scratch(stream, &scr)) return rc;
    const int64_t rows = std::min(step, M - r);
    if (int rc = adapted_rows(part_of(c, r, rows), low_at(low, r, rows), scr)) return rc;
  }
  return VT_OK;
}

int vt_adapted_grad(const void *dY, int32_t type, int64_t ldd, const void *X, int64_t ldx, int64_t M, int64_t K, const int8_t *Bp,
                    const float *meta, int64_t N, const void *P, int64_t R, int64_t L, float scale, const int32_t *which,
                    const float *U, float *H, void *dX, int64_t lddx, void *dDown, void *dUp, void *stream) {
  g_err.clear();
  const char *who = "vt_adapted_grad";
  const int64_t Rp = rank_pad(R);
  const ScaledCall c = {who, dY, type, ldd, N, nullptr, Bp, meta, dX ? dX : H, dX ? type : VT_TYPE_F32, dX ? lddx : Rp, dX ? K : Rp, M, K, N, false};
  const AdapterCall ad = {who, type, P, L, R, K, N, M, true, scale, which, H};
  if (int rc = check_adapters(ad)) return rc;
  bool empty = false;
  if (int rc = check_scaled(c, &empty)) return rc;
  const AdapterLayout l = adapter_layout(K, N, R, L);
  const int64_t e = elem_size(type), size = l.first(true) + l.second(true);
  if (M > 0 && (!H || (size > 0 && !P) || (dUp && !U) || (dDown && K > 0 && !X)))
    return fail(VT_EINVAL, "%s: adapters, X, U or H are null", who);
  const Operand o[] = {{"dY", dY, M, ldd, N, e, false}, {"X", X, M, ldx, K, e, false}, {"weights", Bp, 1, 0, l.Kp * l.Np, 1, false},
                       {"scales", meta, 1, 0, scaled_meta(l.Np), 4, false}, {"adapters", P, 1, size, size, e, false, 16 / e},
                       {"which", which, 1, M, M, 4, false}, {"U", U, 1, M * Rp, M * Rp, 4, false, 4},
                       {"H", H, 1, M * Rp, M * Rp, 4, true, 4}, {"dX", dX, M, lddx, K, e, true},
                       {"dDown", dDown, 1, L * R * K, L * R * K, e, true}, {"dUp", dUp, 1, L * R * N, L * R * N, e, true}};
  if (int rc = check_operands(who, o, 11)) return rc;
  if (M > 0) {
    Scratch scr;
    if (int rc = open_scratch(stream, &scr)) return rc;
    const ShrinkArgs a = {dY, nullptr, P, which, H, ldd, scale, (int)M, (int)N, (int)l.Np, (int)L, (int)Rp};
    if (int rc = shrink(a, type, false, (hipStream_t)stream)) return rc;
  }
  if (dX && M > 0 && K > 0) {
    const LowRank low = {H, (const int8_t *)P + l.first(true) * e, which, l.Kp, (int)L, (int)Rp, (int)M};
    const int64_t step = rows_at_once(M, l.Np * (two_halves(type) ? 4 : 2) + 4);
    for (int64_t r = 0; r < M; r += step) {
      const int64_t rows = std::min(step, M - r);
      if (l.Np == 0) {
        ScaledOut z = {};
        const ScaledCall p = part_of(c, r, rows);
        z.Y = p.Y; z.ldy = p.ldy; z.M = (int)rows; z.N = (int)K; z.type = type;
        if (int rc = launch_zero(z, (hipStream_t)stream)) return rc;
      } else if (int rc = adapted_dx_rows(part_of(c, r, rows), low_at(low, r, rows), stream)) {
        return rc;
      }
    }
  }
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  auto outer = [&](const float *h, const void *z, int64_t ldz, int64_t cols, int64_t colsp, void *out, bool turned) {
    if (!out || cols == 0) return (int)VT_OK;
    const OuterArgs a = {h, z, which, nullptr, out, ldz, (int)M, (int)cols, (int)colsp, (int)L, (int)R, (int)Rp, 1, turned};
    return by_type(type, [&](auto t) { return launch_outer<decltype(t)::value>(a, scr); });
  };
  if (int rc = outer(H, X, ldx, K, l.Kp, dDown, false)) return rc;
  return outer(U, dY, ldd, N, l.Np, dUp, true);
}

}  // extern "C"
