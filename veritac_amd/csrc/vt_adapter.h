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
// with the rank padded to Rp and the long side to that of the packed weights, zeros
// in between, once for each product that reads them, as that product's fragments:
// a wave's load of one is contiguous.

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int kMaxRank = 128, kMaxAdapters = 65535;   // adapters: a side of a grid
// 16 ranks, or whole 32s: the depth of a 16-bit matrix instruction, half of it for
// the second half of u where the rank is small.
constexpr int64_t rank_pad(int64_t R) { return R <= 16 ? 16 : (R + 31) / 32 * 32; }

// One pair of an adapter's layouts, for x . A^T and u . B^T forward, dy . B and h . A
// backward.
//   first   [L][Rp / 16][len / 32] fragments of 16 ranks by 32 columns: 8 columns of
//           rank r % 16 at ((column / 8 % 4) * 16 + r % 16) * 8
//   second  [L][columns / 16][Rp / G] fragments of 16 columns by G ranks (G = 32, or 16
//           where Rp is, or in float32): E ranks (8, in float32 4) of column c % 16 at
//           ((rank / E % (G / E)) * 16 + c % 16) * E
struct AdapterLayout {
  int64_t Kp, Np, Rp, L;
  int64_t first(bool back) const { return L * Rp * (back ? Np : Kp); }
  int64_t second(bool back) const { return L * Rp * (back ? Kp : Np); }
};

AdapterLayout adapter_layout(int64_t K, int64_t N, int64_t R, int64_t L) {
  return {scaled_kp(K), scaled_np(N, false), rank_pad(R), L};
}

struct AdapterPackArgs {
  const uint8_t *A, *B;       // down [L][R][K], up [L][N][R]
  uint8_t *first[2], *second[2];   // forward and backward, null: not wanted
  int K, N, R, Kp, Np, Rp;
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
  const int tid = threadIdx.x;
  for (int r0 = 0; r0 < p.Rp; r0 += 16) {
    // down is [R][K], up [N][R]; 4 elements a thread under way together
    T v[4];
    int j[4], r[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      j[q] = up ? (tid >> 4) + 16 * q : tid & 63;
      r[q] = r0 + (up ? tid & 15 : (tid >> 6) + 4 * q);
      v[q] = T(0);
      if (j0 + j[q] < len && r[q] < p.R) v[q] = up ? src[(int64_t)(j0 + j[q]) * p.R + r[q]] : src[(int64_t)r[q] * len + j0 + j[q]];
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) tile[j[q]][r[q]] = v[q];
  }
  __syncthreads();
  constexpr int E = sizeof(T) == 4 ? 4 : 8;
  const int G = sizeof(T) == 4 || p.Rp == 16 ? 16 : 32;
#pragma unroll
  for (int back = 0; back < 2; ++back) {
    // forward, down is first and up second; backward the other way
    const bool second = up != (back != 0);
    uint8_t *to = second ? p.second[back] : p.first[back];
    if (!to) continue;
    T *dst = (T *)to + (int64_t)a * p.Rp * lenp;
    if (second) {
      // 4 blocks of 16 columns, contiguous
      const int shift = G == 16 ? 4 : 5;
#pragma unroll 1
      for (int nb = 0; nb < 4; ++nb)
        for (int w = tid; w < 16 * p.Rp; w += 256) {
          const int f = w & ((16 << shift) - 1), c = f / E % 16, r = (w >> (4 + shift) << shift) + f / (16 * E) * E + f % E;
          dst[(int64_t)(j0 + nb * 16) * p.Rp + w] = tile[nb * 16 + c][r];
        }
    } else {
      // 2 fragments of 32 columns for each 16 ranks
      for (int i = tid; i < 64 * p.Rp; i += 256) {
        const int rb = i / 1024, w = i % 1024, f = w % 512;
        const int r = rb * 16 + f / 8 % 16, j = w / 512 * 32 + f / 128 * 8 + f % 8;
        dst[((int64_t)rb * (lenp / 32) + j0 / 32) * 512 + w] = tile[j][r];
      }
    }
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
  int8_t *Q;            // few rows: also rounds floating rows to int8 rows of lenp (null: not)
  float *T;             // and their scales
};

// One or two of them over the same rows, by blockIdx.z.
struct ShrinkPair {
  ShrinkArgs of[2];
};

// A 16 x 32 by 32 x 16 product of fragments of 8 values a lane: row or column lane %
// 16, k 8 (lane / 16) + e (in float32 eight products of depth 4).
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
// 8 elements of a row from `pos`, zero past `len`; int8 rows too.
template <int TYPE, bool I8>
struct RowPiece {
  typename std::conditional<I8, v2i, Raw8<TYPE>>::type w;
  __device__ __forceinline__ void load(const void *row, int pos, int len) {
    if constexpr (I8) {
      typedef v2i V __attribute__((aligned(1)));
      const uint8_t *q = (const uint8_t *)row;
      if (pos + 8 <= len) {
        w = *(const V *)(q + pos);
      } else {
        w = v2i{0, 0};
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (pos + e < len) w[e >> 2] |= (int)((uint32_t)q[pos + e] << (8 * (e & 3)));
      }
    } else {
      w = raw8<TYPE>((const typename Elem<TYPE>::T *)row, pos, len);
    }
  }
  __device__ __forceinline__ void settle() {
    if constexpr (!I8) w.settle();
  }
  __device__ __forceinline__ float value(int e) const {
    if constexpr (I8) return (float)(int8_t)((uint32_t)w[e >> 2] >> (8 * (e & 3)));
    else return raw_value<TYPE>(w, e);
  }
  __device__ __forceinline__ Frag<TYPE> frag() const {
    Frag<TYPE> f;
    if constexpr (!I8 && TYPE != kF32) {
      f.v = __builtin_bit_cast(decltype(f.v), w.w);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f.v[e] = (typename Elem<TYPE>::T)value(e);
    }
    return f;
  }
};

// What a row's sums are multiplied by: a NaN for an adapter that is not there.
template <bool I8>
__device__ __forceinline__ float shrink_factor(const ShrinkArgs &p, int row, int a) {
  if (a >= p.L) return __uint_as_float(0x7fc00000u);
  return I8 ? p.scale * p.t[row] : p.scale;
}

// Up to 64 rows, each with an adapter of its own maybe: 16 ranks of a row to a
// workgroup, whose 16 waves take 32 columns in turn (a fragment, 8 columns of a
// rank a lane) and join through LDS. The first of a row's workgroups rounds it too,
// where the int8 product needs that done: the row is in its cache, and a launch
// less. Bound by the latency of its few loads and, with many adapters, by reading
// them: 48 rows of 4096 with 32 adapters of rank 16, rounded too, in 5.8 us (a wave
// to a rank, row by row in memory, 12.9; and 3 more for the rounding).
template <int TYPE, bool I8>
__global__ __launch_bounds__(1024) void shrink_rows_kernel(ShrinkPair pair) {
  __shared__ uint32_t tops[16];
  __shared__ float red[16][16];
  const ShrinkArgs &p = pair.of[blockIdx.z];
  typedef typename Elem<TYPE>::T T;
  constexpr int U = TYPE == kF32 ? 4 : 8;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
  const int a = p.which ? p.which[row] : 0;
  const void *x = I8 ? (const void *)((const int8_t *)p.X + row * p.ldx) : (const void *)((const T *)p.X + row * p.ldx);
  float s = 0.0f;
  if (a >= 0 && a < p.L) {
    const T *w = (const T *)p.P + ((int64_t)a * (p.Rp / 16) + blockIdx.y) * 16 * p.lenp + lane * 8;
    for (int k0 = wave * 32; k0 < p.lenp; k0 += U * 512) {
      RowPiece<TYPE, I8> v[U];
      Frag<TYPE> b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * 512;
        b[u] = load_frag<TYPE>(w + (int64_t)min(k, p.lenp - 32) * 16);
        v[u].load(x, k + 8 * g, p.len);   // zero past the row's end
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u].settle();
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(v[u].value(e), (float)b[u].v[e], s);
      }
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
  }
  if (lane < 16) red[wave][lane] = s;
  __syncthreads();
  if (tid < 16) {
    s = 0.0f;
#pragma unroll
    for (int v = 0; v < 16; ++v) s += red[v][tid];
    p.U[(int64_t)row * p.Rp + blockIdx.y * 16 + tid] = a < 0 ? 0.0f : s * shrink_factor<I8>(p, row, a);
  }
  if constexpr (!I8) {
    if (!p.Q || blockIdx.y) return;
    uint32_t top = 0;
    for (int pos = tid * 8; pos < p.len; pos += 8192) {
      float v[8];
      load8<TYPE>((const T *)x, pos, p.len, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[e]));
    }
    top = block_max<1024>(top, tops);
    const RowScale r = row_scale(top);
    if (tid == 0) p.T[row] = r.scale;
    for (int pos = tid * 8; pos < p.lenp; pos += 8192) {
      float v[8];
      uint32_t b[8];
      load8<TYPE>((const T *)x, pos, p.len, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = round_byte(v[e], r.inv);
      v2i o = {pack_bytes(b[0], b[1], b[2], b[3]), pack_bytes(b[4], b[5], b[6], b[7])};
      if (r.inv == 0.0f) o = v2i{0, 0};
      *(v2i *)(p.Q + (int64_t)row * p.lenp + pos) = o;
    }
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

// More rows: 16 rows by 16 NR ranks to a workgroup, whose 16 waves take
// neighbouring runs of U 32-deep slices (whole lines of the rows) and join through
// LDS. Bound by what it reads of the rows (once for every 16 NR ranks) and of
// their adapters (once for every 16 rows, from L2), and by the chain of loads in
// front of its one or two steps: 2000 x 4096 with rank 64 in 12.9 us, two of 4096 x
// 4096 with rank 16 at once in 18 (3.7 TB/s; 8 slices instead of 4 in flight are no
// faster). U is what 128 registers hold: with 4 slices the widest form spills, and
// 8192 x 8192 x 8192 adapted with rank 128 takes 942 us in place of 736.
template <int TYPE, bool I8, int NR>
__global__ __launch_bounds__(1024) void shrink_tiles_kernel(ShrinkPair pair) {
  typedef typename Elem<TYPE>::T T;
  constexpr int WAVES = 16, U = TYPE == kF32 || NR > 2 ? 2 : 4;
  __shared__ float red[WAVES][16][16 * NR + 1];
  const ShrinkArgs &p = pair.of[blockIdx.z];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int row0 = blockIdx.x * 16, rank0 = blockIdx.y * 16 * NR;
  const int row = min(row0 + c, p.M - 1);
  int a = p.which ? p.which[row] : 0;
  if (a >= p.L) a = -1;
  const void *x = I8 ? (const void *)((const int8_t *)p.X + row * p.ldx) : (const void *)((const T *)p.X + row * p.ldx);
  const T *w = (const T *)p.P + (int64_t)rank0 * p.lenp + lane * 8;
  const int64_t step = (int64_t)p.Rp * p.lenp;
  v4f acc[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) acc[n] = v4f{0, 0, 0, 0};
  for (int k0 = wave * U * 32; k0 < p.lenp; k0 += WAVES * U * 32) {
    RowPiece<TYPE, I8> xa[U];
#pragma unroll
    for (int u = 0; u < U; ++u) xa[u].load(x, k0 + u * 32 + 8 * g, p.len);
    bool settled = false;
    each_adapter(a, [&](int cur, uint32_t rows) {
      Frag<TYPE> b[NR][U];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int u = 0; u < U; ++u)
          b[n][u] = load_frag<TYPE>(w + cur * step + ((int64_t)n * p.lenp + min(k0 + u * 32, p.lenp - 32)) * 16);
      if (!settled) {   // behind the adapter's loads
#pragma unroll
        for (int u = 0; u < U; ++u) xa[u].settle();
        settled = true;
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        v4f part = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < U; ++u) part = mfma16<TYPE>(xa[u].frag(), b[n][u], part);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (rows >> (4 * g + e) & 1) acc[n][e] += part[e];
      }
    });
  }
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[wave][4 * g + e][16 * n + c] = acc[n][e];
  __syncthreads();
  for (int t = threadIdx.x; t < 256 * NR; t += 1024) {
    const int r = t / (16 * NR), rank = t % (16 * NR), i = row0 + r;
    if (i >= p.M) continue;
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) s += red[v][r][rank];
    const int ad = p.which ? p.which[i] : 0;
    p.U[(int64_t)i * p.Rp + rank0 + rank] = ad < 0 ? 0.0f : s * shrink_factor<I8>(p, i, ad);
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

// Where ranks r .. r + 7 of a column lie (8 of them, or in float32 two fours), in
// elements.
__device__ __forceinline__ int64_t rank_at(const LowRank &l, bool wide, int a, int64_t col, int r) {
  return (a * l.colsp + (col & ~(int64_t)15)) * l.Rp + (wide ? 4 : 8) * (col & 15) +
         (wide ? (r >> 4) * 256 + (r >> 2 & 3) * 64 : (r >> 5) * 512 + (r >> 3 & 3) * 128);
}

// E elements of it at once, 8 ranks at a time, so that their loads are under way
// together; those with a row below 0 are left out. U: LowRank's u, or a copy of it
// in LDS. WIDE: float32 adapters, else `type`.
template <bool WIDE, int E, class FLOATS>
__device__ __forceinline__ void low_rank_elements(const LowRank &l, int type, FLOATS U, const int (&row)[E], const int (&col)[E],
                                                  float (&s)[E]) {
  typedef const v4f *Global;
  typedef const LDS_AS v4f *Local;
  typedef typename std::conditional<std::is_same<FLOATS, const float *>::value, Global, Local>::type Four;
  FLOATS u[E];
  int at[E];
  bool in[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int a = row[i] < 0 ? -1 : adapter_of(l, row[i]);
    in[i] = a >= 0;
    u[i] = U + (int64_t)max(row[i], 0) * l.Rp;
    at[i] = max(a, 0);
    s[i] = 0.0f;
  }
  for (int r = 0; r < l.Rp; r += 8) {
    v4i b[E][WIDE ? 2 : 1];
    v4f x[E], y[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int64_t w = rank_at(l, WIDE, at[i], row[i] < 0 ? 0 : col[i], r);
      if constexpr (WIDE) {
        b[i][0] = *(const v4i *)((const float *)l.V + w);
        b[i][1] = *(const v4i *)((const float *)l.V + w + 64);
      } else {
        b[i][0] = *(const v4i *)((const uint16_t *)l.V + w);
      }
      x[i] = *(Four)(u[i] + r);
      y[i] = *(Four)(u[i] + r + 4);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v;
        if constexpr (WIDE) {
          const int bits = b[i][e >> 2][e & 3];
          v = __int_as_float(bits);
        } else {
          v = from16((uint32_t)b[i][0][e >> 1] >> (16 * (e & 1)) & 0xffffu, type);
        }
        s[i] = fmaf(e < 4 ? x[i][e & 3] : y[i][e & 3], v, s[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) s[i] = in[i] ? s[i] : 0.0f;
}

template <int E, class FLOATS>
__device__ __forceinline__ void low_rank_any(const LowRank &l, int type, FLOATS U, const int (&row)[E], const int (&col)[E],
                                                  float (&s)[E]) {
  if (type == VT_TYPE_F32) low_rank_elements<true>(l, type, U, row, col, s);
  else low_rank_elements<false>(l, type, U, row, col, s);
}

// t[i] += a . b[i] + lo . b[i] for four blocks beside each other. In
// inline assembly with the sums in VGPRs: the kernels that do this keep all of
// their accumulators in AGPRs, where the compiler puts a builtin's too, and
// would spill. Its operands may have been written by the instruction before (two
// wait states), and its results are read by the instruction behind: an 8-pass
// product's by 11 wait states, a 16-pass one's by 19.
template <int TYPE>
__device__ __forceinline__ void four_products(v4f (&t)[4], const Frag<TYPE> &a, const Frag<TYPE> &lo, const Frag<TYPE> (&b)[4]) {
#define VT_FOUR(op, A)                                                                            \
  op " %0, %" A ", %6, %0\n\t" op " %1, %" A ", %7, %1\n\t" op " %2, %" A ", %8, %2\n\t" op " %3, %" A ", %9, %3\n\t"
#define VT_ASM(op) \
  asm volatile("s_nop 1\n\t" VT_FOUR(op, "4") VT_FOUR(op, "5") "s_nop 15\n\ts_nop 7" \
               : "+v"(t[0]), "+v"(t[1]), "+v"(t[2]), "+v"(t[3]) \
               : "v"(a.v), "v"(lo.v), "v"(b[0].v), "v"(b[1].v), "v"(b[2].v), "v"(b[3].v))
  if constexpr (TYPE == kF16) VT_ASM("v_mfma_f32_16x16x32_f16");
  else VT_ASM("v_mfma_f32_16x16x32_bf16");
#undef VT_ASM
#undef VT_FOUR
}
// The same in float32, of depth 4.
__device__ __forceinline__ void four_products(v4f (&t)[4], float a, float b0, float b1, float b2, float b3) {
  asm volatile("s_nop 1\n\t"
               "v_mfma_f32_16x16x4_f32 %0, %4, %5, %0\n\tv_mfma_f32_16x16x4_f32 %1, %4, %6, %1\n\t"
               "v_mfma_f32_16x16x4_f32 %2, %4, %7, %2\n\tv_mfma_f32_16x16x4_f32 %3, %4, %8, %3\n\ts_nop 15\n\ts_nop 7"
               : "+v"(t[0]), "+v"(t[1]), "+v"(t[2]), "+v"(t[3])
               : "v"(a), "v"(b0), "v"(b1), "v"(b2), "v"(b3));
}

// Blocks of 16 x 16 in the accumulators' layout: d[ni] element e is row row0 +
// 4 (lane / 16) + e, column col0 + 16 ni + lane % 16 (below colsp), for one strip of 16
// rows after another.
// 16-bit adapters: u enters in two halves (16 bits of it in bfloat16, 22 in
// float16; it is then as exact as the 16-bit y that it is added to needs, 2^-8 of
// a step), 32 ranks at a time, or 16 with both halves in one product. float16
// halves are of u times a power of two for each row and 32 ranks, so that none
// overflows or is lost.
// One wave to a SIMD runs this, so nothing hides its loads, and they would wait for
// the strip's stores (all count in vmcnt, in order): a strip's u is loaded a strip
// ahead, and the adapter's first groups of ranks (two, or one of wide tiles) stay in registers from strip to
// strip (2000 x 4096 -> 4096, rank 64: 75 us with every load at its use, 56 with
// those of a strip together, 35 without adapters).
template <int TYPE, int NI>
struct LowRankStrips {
  static_assert(NI % 4 == 0, "four blocks at a time");
  typedef typename Elem<TYPE>::T T;
  static constexpr int G = TYPE == kF32 ? 16 : 32, HELD = NI <= 4 ? 2 : 1, UV = TYPE == kF32 ? 1 : 2;
  struct Part {   // an adapter's 16 columns by G ranks
    typename std::conditional<TYPE == kF32, v4f, Frag<TYPE>>::type v;
  };
  struct Ahead {
    int a;
    v4f u[HELD][UV];
  };
  const LowRank &l;
  const int col0, lane, g, c, groups;
  const bool small;   // 16 ranks in all
  int held = -1;
  Part b[HELD][NI];

  __device__ __forceinline__ LowRankStrips(const LowRank &low, int col, int ln)
      : l(low), col0(col), lane(ln), g(ln >> 4), c(ln & 15), groups(max(low.Rp / G, 1)), small(TYPE != kF32 && low.Rp == 16) {}

  __device__ __forceinline__ void load_u(int row0, int group, v4f (&u)[UV]) const {
    const float *at = l.U + (int64_t)min(row0 + c, l.rows - 1) * l.Rp + group * G + (TYPE == kF32 ? 4 : 8) * (small ? g & 1 : g);
#pragma unroll
    for (int i = 0; i < UV; ++i) u[i] = *(const v4f *)(at + 4 * i);
  }
  __device__ __forceinline__ void load_b(int a, int group, Part (&p)[NI]) const {
    const T *v = (const T *)l.V + (a * l.colsp + col0) * l.Rp + group * G * 16 + (TYPE == kF32 ? lane * 4 : (small ? lane & 31 : lane) * 8);
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      if constexpr (TYPE == kF32) p[ni].v = *(const v4f *)(v + ni * 16 * l.Rp);
      else p[ni].v = load_frag<TYPE>(v + ni * 16 * l.Rp);
    }
  }
  // a: adapter_of row row0 + lane % 16
  __device__ __forceinline__ Ahead ahead(int a, int row0) const {
    Ahead r;
    r.a = a;
#pragma unroll
    for (int i = 0; i < HELD; ++i) load_u(row0, min(i, groups - 1), r.u[i]);
    return r;
  }
  // One group of ranks of the rows in `rows`.
  __device__ __forceinline__ void group_products(const v4f (&u)[UV], const Part (&p)[NI], uint32_t rows, v4f (&d)[NI]) const {
    v4f un = {1, 1, 1, 1};
    Frag<TYPE> hi, lo;
    if constexpr (TYPE != kF32) {
      float f[8], h[8];
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = u[e >> 2][e & 3];
        top = max(top, magnitude(f[e]));
      }
      if constexpr (TYPE == kF16) {
        top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        const float norm = normaliser(__uint_as_float(top)), back = 1.0f / norm;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= norm;
#pragma unroll
        for (int e = 0; e < 4; ++e) un[e] = __shfl(back, 4 * g + e);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[e] = (float)(T)f[e];
        // (inf - inf of an infinite u would make a NaN of its low half)
        f[e] = magnitude(h[e]) < kInfBits ? f[e] - h[e] : 0.0f;
        // 16 ranks: the product's other 16 are the low halves
        h[e] = small && g >= 2 ? f[e] : h[e];
        f[e] = small ? 0.0f : f[e];
      }
      hi = to_frag<TYPE>(h);
      lo = to_frag<TYPE>(f);
    }
#pragma unroll
    for (int q = 0; q < NI / 4; ++q) {
      v4f t[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
      if constexpr (TYPE == kF32) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          four_products(t, u[0][e], p[4 * q].v[e], p[4 * q + 1].v[e], p[4 * q + 2].v[e], p[4 * q + 3].v[e]);
      } else {
        const Frag<TYPE> four[4] = {p[4 * q].v, p[4 * q + 1].v, p[4 * q + 2].v, p[4 * q + 3].v};
        four_products<TYPE>(t, hi, lo, four);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool mine = rows >> (4 * g + e) & 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = TYPE == kF16 ? fmaf(t[i][e], un[e], d[4 * q + i][e]) : d[4 * q + i][e] + t[i][e];
          d[4 * q + i][e] = mine ? x : d[4 * q + i][e];
        }
      }
    }
  }
  __device__ __forceinline__ void run(const Ahead &w, int row0, v4f (&d)[NI]) {
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) d[ni] = v4f{0, 0, 0, 0};
    each_adapter(w.a, [&](int cur, uint32_t rows) {
      if (cur != held) {
        load_b(cur, 0, b[0]);
        if constexpr (HELD > 1) {
          if (groups > 1) load_b(cur, 1, b[1]);
        }
        held = cur;
      }
      group_products(w.u[0], b[0], rows, d);
      if constexpr (HELD > 1) {
        if (groups > 1) group_products(w.u[1], b[1], rows, d);
      }
#pragma unroll 1
      for (int i = HELD; i < groups; ++i) {
        v4f u[UV];
        Part p[NI];
        load_u(row0, i, u);
        load_b(cur, i, p);
        group_products(u, p, rows, d);
      }
    });
  }
};

// The adapters of a wave's 128 rows from row0: lane l holds rows l and 64 + l.
struct RowAdapters {
  int a[2];
};
__device__ __forceinline__ RowAdapters row_adapters(const LowRank &l, int row0, int lane) {
  RowAdapters r;
#pragma unroll
  for (int h = 0; h < 2; ++h) r.a[h] = adapter_of(l, min(row0 + 64 * h + lane, l.rows - 1));
  return r;
}
// That of row rel + lane % 16 (rel a multiple of 16).
__device__ __forceinline__ int adapter_at(const RowAdapters &r, int rel, int lane) {
  return __shfl(rel >= 64 ? r.a[1] : r.a[0], (rel & 63) + (lane & 15));
}

// A linear layer's outputs with adapters. TYPE: of adapters and outputs.
template <int TYPE>
struct AdaptedTile : ScaledTile<kLinear, TYPE == kF32 ? 4 : 2> {
  // A wave's 128 x 128 sums and its next fragments leave too few registers for the
  // low-rank products, and what they spill waits for the stores. Whole calls with
  // rank 16 / 64 / 128, u's kernel in both as it was then (its widest form spilled):
  // 4096 x 4096 -> 14336 took 346 / 391 / 465 us on 256 x 256 tiles and 292 / 321 / 414
  // on 256 x 128 (219 without adapters); at 8192^3, whose longer K carries that
  // epilogue, 614 / 711 / 887 and 661 / 738 / 946 (484). One rule for any K: the 4 -
  // 7 % that 256 x 256 tiles had there are given up for the 11 - 18 % elsewhere. With
  // today's u the kept form takes 288 / 301 / 377 and 662 / 635 / 736.
  static constexpr bool kWide = false;
  LowRank low;
  static constexpr int OE = TYPE == kF32 ? 4 : 2;

  // A strip of 16 rows at a time in a loop, of which only the reading of the sums
  // is unrolled: as straight code the low-rank products (3 times, for ranks in
  // fours, ones and several adapters) leave the instruction cache with every strip.
  // Rows and columns that a moved-back tile shares with its neighbour come out the
  // same in both.
  template <int MI, int NI, bool EDGE>
  __device__ __forceinline__ void tile16(const v4i (&acc)[MI][NI], int row0, int col0, int, int, int lane, LDS_AS int8_t *lds) const {
    static_assert(NI == 4, "64 columns");
    constexpr int W = NI * 16, LPR = W / 8, RPI = 64 / LPR, IT = 16 / RPI;
    const int g = lane >> 4, c = lane & 15, j8 = 8 * (lane % LPR), lr = lane / LPR;
    float s[NI], b[NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      s[ni] = this->meta[col0 + ni * 16 + c];
      b[ni] = this->meta[this->Np + col0 + ni * 16 + c];
    }
    const RowAdapters ra = row_adapters(low, row0, lane);
    LowRankStrips<TYPE, NI> strips(low, col0, lane);
    auto next = strips.ahead(adapter_at(ra, 0, lane), row0);
    v4f next_t = *(const v4f_any *)(this->t + row0 + 4 * g);
#pragma unroll 1
    for (int mi = 0; mi < MI; ++mi) {
      const auto now = next;
      const v4f tr = next_t;
      const int after = min(mi + 1, MI - 1) * 16;
      next = strips.ahead(adapter_at(ra, after, lane), row0 + after);
      next_t = *(const v4f_any *)(this->t + row0 + after + 4 * g);
      v4f d[NI];
      strips.run(now, row0 + mi * 16, d);
      // chunk k of strip row r at k ^ (4 (r / 4 % 4)): an instruction's writes fall on distinct banks
      each([&](auto strip) __attribute__((always_inline)) {
        constexpr int i = decltype(strip)::value;
        if (mi != i) return;
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *(LDS_AS float *)(lds + (4 * g + e) * (W * 4) + ((((ni ^ g) << 2) + (c >> 2)) << 4) + (c & 3) * 4) =
                ((float)acc[i][ni][e] * tr[e] * s[ni] + b[ni]) + d[ni][e];
      }, std::make_integer_sequence<int, MI>());
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int r = it * RPI + lr;
        const LDS_AS int8_t *at = lds + r * (W * 4);
        const int swz = ((r >> 2) & 3) << 2;
        const v4f x = *(const LDS_AS v4f *)(at + (((j8 >> 2) ^ swz) << 4)), y = *(const LDS_AS v4f *)(at + ((((j8 >> 2) + 1) ^ swz) << 4));
        const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        if (col0 + j8 < this->N)
          this->store8((int64_t)(row0 + mi * 16 + r) * this->ldy + col0 + j8, v, this->N - (col0 + j8), this->type);
      }
    }
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
    const RowAdapters ra = row_adapters(low, row0, lane);
    LowRankStrips<TYPE, 4> strips(low, col0, lane);
    auto next = strips.ahead(adapter_at(ra, 0, lane), row0);
    each([&](auto strip) __attribute__((always_inline)) {
      constexpr int mi = decltype(strip)::value;
      const int first = row0 + mi * 32;
      if (first >= this->M) return;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        v4f d[4];
        const auto now = next;
        const int after = min(mi * 32 + 16 * h + 16, MI * 32 - 16);
        next = strips.ahead(adapter_at(ra, after, lane), row0 + after);
        strips.run(now, first + 16 * h, d);
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

  // u of all rows (64 at the most) into LDS: its 16 columns' lanes read it again and
  // again.
  template <int THREADS>
  __device__ __forceinline__ void stage(float *lds, int tid) const {
    for (int i = tid * 4; i < this->M * low.Rp; i += THREADS * 4) *(LDS_AS v4f *)((LDS_AS float *)lds + i) = *(const v4f *)(low.U + i);
    lds_barrier();
  }
  // The adapters' part of E elements, before the sums are there.
  template <int E>
  __device__ __forceinline__ void ahead(const int (&row)[E], const int (&col)[E], float (&d)[E], float *lds) const {
    low_rank_any(low, this->type, (const LDS_AS float *)lds, row, col, d);
  }
  __device__ __forceinline__ void element(int32_t a0, int32_t, int row, int pc, int j, float t_row) const {
    if (j >= this->N) return;
    const int rows[1] = {row}, cols[1] = {j};
    float d[1];
    low_rank_any(low, this->type, low.U, rows, cols, d);
    element_with(a0, row, pc, j, t_row, d[0]);
  }
  __device__ __forceinline__ void element_with(int32_t a0, int row, int pc, int j, float t_row, float d) const {
    if (j >= this->N) return;
    const float v = ((float)a0 * t_row * this->meta[pc] + this->meta[this->Np + pc]) + d;
    const int64_t at = (int64_t)row * this->ldy + j;
    if (this->type == VT_TYPE_F32) ((float *)this->Y)[at] = v;
    else ((uint16_t *)this->Y)[at] = (uint16_t)pack16(v, 0.0f, this->type);
  }
};

// dx with the adapters' part: 4096^3 with rank 16 in 112 us, without 102 - 107.
template <int TYPE>
struct AdaptedGrad : ScaledTile<kGrad> {
  LowRank low;

  template <int G, int MI, int NI, class ACC>
  __device__ __forceinline__ void blocks16(const ACC (&acc)[MI][NI], int row0, int col0, int lane, LDS_AS int8_t *lds,
                                           const float *early) const {
    const int g = lane >> 4, c = lane & 15;
    const float one[2] = {1.0f, 1.0f};
    const RowAdapters ra = row_adapters(low, row0, lane);
    // columns past the last are not stored, and read from before it
    LowRankStrips<TYPE, NI> low_strips(low, min(col0, (int)low.colsp - NI * 16), lane);
    auto next = low_strips.ahead(adapter_at(ra, 0, lane), row0);
    this->template strips<MI / G, 16 * G, NI * 16>(
        [&](auto strip) __attribute__((always_inline)) {
          constexpr int first = decltype(strip)::value * G;
#pragma unroll 1
          for (int i = 0; i < G; ++i) {
            const int rel = (first + i) * 16, after = min(rel + 16, MI * 16 - 16);
            const auto now = next;
            next = low_strips.ahead(adapter_at(ra, after, lane), row0 + after);
            v4f d[NI];
            low_strips.run(now, row0 + rel, d);
            v4f unit;
#pragma unroll
            for (int e = 0; e < 4; ++e) unit[e] = __shfl(rel >= 64 ? early[1] : early[0], (rel + 4 * g + e) & 63);
            each([&](auto block) __attribute__((always_inline)) {
              constexpr int k = decltype(block)::value;
              if (i != k) return;
#pragma unroll
              for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni)
                  *(LDS_AS float *)(lds + (16 * k + 4 * g + e) * (64 * NI) + ((((ni ^ g) << 2) + (c >> 2)) << 4) + (c & 3) * 4) =
                      acc[first + k][ni][e] * unit[e] + d[ni][e];
            }, std::make_integer_sequence<int, G>());
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

__global__ __launch_bounds__(256) void adapted_join_kernel(const int32_t *S, int slices, AdaptedTile<kBF16> out) {
  finish_rows<kLinear>(S, slices, out);
}

// dx from partial sums, with the adapters' part.
__global__ __launch_bounds__(256) void adapted_dx_sum_kernel(GradSumArgs p, LowRank low) {
  sum_grad_slices(p, [&](int row, int col, float (&x)[4]) {
    const int rows[4] = {row, row, row, row}, cols[4] = {col, col + 1, col + 2, col + 3};   // below colsp, whole fours
    low_rank_any(low, p.type, low.U, rows, cols, x);
  });
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

// One or two of them over the same rows: the first `x0` of blockIdx.x are the first's.
struct OuterPair {
  OuterArgs of[2];
  int x0;
};

// 16 ranks by 128 columns of one adapter over one range of rows to a workgroup:
// 4096 rows of 2 x 4096 columns with rank 16 in 22 us (67 MB, 3.0 TB/s; the products
// alone are 7; 2 or 8 row groups in flight instead of 4 take 22 and 30).
// Its waves take 4 rows at a time in turn, as 4-deep float32 products (nothing is
// rounded on the way, whatever the type): lane l holds 8 columns of row l / 16,
// and product j takes column j of every lane's. The rows of other adapters are
// left out by a list of this one's rows, made in order 1024 rows at a time; without
// an index all rows are the first adapter's, and the others' sums are empty.
template <int TYPE>
__global__ __launch_bounds__(256, 4) void outer_kernel(OuterPair pair) {
  typedef typename Elem<TYPE>::T T;
  constexpr int ROWS = 1024;
  const int which_of = (int)blockIdx.x >= pair.x0, block = blockIdx.x - (which_of ? pair.x0 : 0);
  const OuterArgs &p = pair.of[which_of];
  __shared__ int list[ROWS];
  __shared__ int counts[4][4];
  __shared__ float red[4][16][132];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const int ranks = p.Rp / 16, tiles = (p.cols + 127) / 128;
  const int tile = block % tiles, rank0 = block / tiles % ranks * 16;
  const int a = blockIdx.y, split = blockIdx.z;
  const int col = tile * 128 + 8 * c;
  const int beg = (int)((int64_t)p.M * split / p.splits), end = p.which || !a ? (int)((int64_t)p.M * (split + 1) / p.splits) : beg;
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
      // all loads under way: rows past the last are the last again, times zero and of zeros
      float h[U];
      Raw8<TYPE> z[U];
      bool in[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + 4 * u + g;
        in[u] = i < n;
        const int at = min(i, n - 1), row = p.which ? list[at] : r0 + at;
        h[u] = p.H[(int64_t)row * p.Rp + rank0 + c];
        z[u] = raw8<TYPE>((const T *)p.Z + row * p.ldz, col, p.cols);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + 4 * u >= n) break;
        z[u].settle();
        const float hu = in[u] ? h[u] : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = raw_value<TYPE>(z[u], j);
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(hu, in[u] ? x : 0.0f, acc[j], 0, 0, 0);
        }
      }
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
__global__ __launch_bounds__(256) void outer_sum_kernel(OuterPair pair) {
  typedef typename Elem<TYPE>::T T;
  const int which_of = (int)blockIdx.x >= pair.x0;
  const OuterArgs &p = pair.of[which_of];
  const int64_t count = (int64_t)p.R * p.cols, i = (int64_t)(blockIdx.x - (which_of ? pair.x0 : 0)) * 256 + threadIdx.x;
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

// `count` (1 or 2) of them over the same rows.
template <int TYPE, bool I8>
int launch_shrink(const ShrinkPair &a, int count, int cus, hipStream_t s) {
  const int64_t M = a.of[0].M, blocks = (M + 15) / 16, ranks = a.of[0].Rp / 16;
  if (M <= kSkinnyMaxM) {
    hipLaunchKernelGGL((shrink_rows_kernel<TYPE, I8>), dim3((unsigned)M, (unsigned)ranks, (unsigned)count), dim3(1024), 0, s, a);
  } else {
    // as many ranks to a workgroup as leave most CUs one
    const bool two = ranks % 2 == 0 && blocks * (ranks / 2) * count >= cus * 3 / 4;
    if (two && TYPE != kF32 && ranks % 4 == 0 && blocks * (ranks / 4) * count >= cus * 3 / 4)
      hipLaunchKernelGGL((shrink_tiles_kernel<TYPE, I8, TYPE == kF32 ? 2 : 4>), dim3((unsigned)blocks, (unsigned)(ranks / 4), (unsigned)count), dim3(1024), 0, s, a);
    else if (two)
      hipLaunchKernelGGL((shrink_tiles_kernel<TYPE, I8, 2>), dim3((unsigned)blocks, (unsigned)(ranks / 2), (unsigned)count), dim3(1024), 0, s, a);
    else
      hipLaunchKernelGGL((shrink_tiles_kernel<TYPE, I8, 1>), dim3((unsigned)blocks, (unsigned)ranks, (unsigned)count), dim3(1024), 0, s, a);
  }
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

int shrink(const ShrinkPair &a, int count, int type, bool i8, const Scratch &scr) {
  return by_type(type, [&](auto t) {
    constexpr int TYPE = decltype(t)::value;
    hipStream_t s = (hipStream_t)scr.stream;
    return i8 ? launch_shrink<TYPE, true>(a, count, scr.st->num_cus, s) : launch_shrink<TYPE, false>(a, count, scr.st->num_cus, s);
  });
}

// `count` (1 or 2) of them over the same rows and adapters.
template <int TYPE>
int launch_outer(OuterPair a, int count, Scratch &scr) {
  hipStream_t s = (hipStream_t)scr.stream;
  const OuterArgs &f = a.of[0];
  int64_t wgs = 0, bytes[2] = {0, 0}, blocks[2] = {0, 0}, sums = 0;
  for (int i = 0; i < count; ++i) {
    const OuterArgs &o = a.of[i];
    blocks[i] = (int64_t)((o.cols + 127) / 128) * (o.Rp / 16);
    bytes[i] = (int64_t)o.L * o.Rp * o.colsp * sizeof(float);
    wgs += blocks[i];
  }
  // Rows are split until there are four workgroups for each CU, of 64 rows at
  // least, as far as the partial sums stay within their bound.
  const int64_t all = wgs * f.L, cus = scr.st->num_cus;
  const int64_t splits = std::max<int64_t>(1, std::min<int64_t>({(4 * cus + all - 1) / all, (f.M + 63) / 64, kScaledBytes / (bytes[0] + bytes[1])}));
  if (wgs > 0x7fffffff) return fail(VT_EUNSUPPORTED, "gradient grid too large");
  void *w = nullptr;
  if (splits > 1)
    if (int rc = scr.take(kPartials, (size_t)(splits * (bytes[0] + bytes[1])), &w)) return rc;
  for (int i = 0; i < count; ++i) {
    a.of[i].splits = (int)splits;
    if (splits > 1) a.of[i].part = (float *)((int8_t *)w + (i ? splits * bytes[0] : 0));
  }
  a.x0 = (int)blocks[0];
  hipLaunchKernelGGL((outer_kernel<TYPE>), dim3((unsigned)wgs, (unsigned)f.L, (unsigned)splits), dim3(256), 0, s, a);
  VT_HIP_CHECK(hipGetLastError());
  if (splits == 1) return VT_OK;
  for (int i = 0; i < count; ++i) {
    blocks[i] = ((int64_t)a.of[i].R * a.of[i].cols + 255) / 256;
    sums += blocks[i];
  }
  a.x0 = (int)blocks[0];
  hipLaunchKernelGGL((outer_sum_kernel<TYPE>), dim3((unsigned)sums, (unsigned)f.L), dim3(256), 0, s, a);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

// What launch_skinny, launch_tiles and launch_grad need of outputs with adapters.
struct AdaptedSkinny : AdaptedTile<kBF16> {
  template <int NBW, int MB, int XB>
  static void skinny(const ScaledSkinnyArgs &a, const AdaptedSkinny &o, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((adapted_skinny_kernel<NBW, MB, XB>), grid, dim3(512), 0, s, a, (const AdaptedTile<kBF16> &)o);
  }
  static int finish(const int32_t *sums, int slices, const AdaptedSkinny &o, hipStream_t s) {
    hipLaunchKernelGGL(adapted_join_kernel, dim3((unsigned)o.M, (unsigned)((o.Np + 255) / 256)), dim3(256), 0, s, sums, slices,
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

// Whether u's kernel rounds a call's rows too: those that the weights' stream does
// not round itself.
bool shrink_rounds(const ScaledCall &c) {
  const int64_t Kp = scaled_kp(c.K);
  return float_type(c.x_type) && c.M <= kSkinnyMaxM && Kp > 0 && !(c.M <= 16 && c.M * Kp <= kFusedValues);
}

// Rows of a forward call, whose u is there (and `ready`: the rows rounded).
int adapted_rows(const ScaledCall &c, const LowRank &low, const Rows *ready, Scratch &scr) {
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
  if (ready) rows = *ready;
  else if (int rc = take_rows(c.X, c.x_type, c.ldx, c.T, c.M, c.K, scr, &rows)) return rc;
  o.t = rows.t;
  if (skinny) return launch_skinny<kLinear>(nullptr, 0, 0, c.K, rows, c.Bp, o, scr);
  hipStream_t s = (hipStream_t)scr.stream;
  if (Kp == 0) return AdaptedSkinny::finish(nullptr, 0, o, s);
  const TilePlan plan = tile_plan(false, c.M, Np, Kp, scr.st->num_cus, true, AdaptedTile<kF32>::kWide);
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
  int64_t L, R, K, N;
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
  const AdapterCall c = {"vt_adapter_size", type, L, R, K, N};
  if (int rc = check_adapters(c)) return rc;
  const AdapterLayout l = adapter_layout(K, N, R, L);
  return (l.first(false) + l.second(false)) * elem_size(type);
}

int vt_adapter_pack(const void *down, const void *up, int32_t type, int64_t K, int64_t N, int64_t R, int64_t L, void *P,
                    void *back, void *stream) {
  g_err.clear();
  const char *who = "vt_adapter_pack";
  const AdapterCall c = {who, type, L, R, K, N};
  if (int rc = check_adapters(c)) return rc;
  const AdapterLayout l = adapter_layout(K, N, R, L);
  const int64_t e = elem_size(type), size = l.first(false) + l.second(false);
  if (size == 0 || (!P && !back)) return VT_OK;
  if ((K > 0 && !down) || (N > 0 && !up)) return fail(VT_EINVAL, "%s: an operand is null", who);
  const Operand o[] = {{"down", down, 1, L * R * K, L * R * K, e, false}, {"up", up, 1, L * R * N, L * R * N, e, false},
                       {"P", P, 1, size, size, e, true, 16 / e}, {"back", back, 1, size, size, e, true, 16 / e}};
  if (int rc = check_operands(who, o, 4)) return rc;
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  AdapterPackArgs a = {(const uint8_t *)down, (const uint8_t *)up, {(uint8_t *)P, (uint8_t *)back}, {nullptr, nullptr},
                       (int)K, (int)N, (int)R, (int)l.Kp, (int)l.Np, (int)l.Rp};
  for (int i = 0; i < 2; ++i)
    if (a.first[i]) a.second[i] = a.first[i] + l.first(i != 0) * e;
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
  const AdapterCall ad = {who, type, L, R, K, N};
  if (int rc = check_adapters(ad)) return rc;
  const int64_t Rp = rank_pad(R);
  bool empty = false;
  if (int rc = check_scaled(c, &empty)) return rc;
  const bool i8 = !float_type(x_type);
  if (!i8 && x_type != type) return fail(VT_EINVAL, "%s: floating rows have the adapters' type", who);
  if (M == 0) return VT_OK;
  const AdapterLayout l = adapter_layout(K, N, R, L);
  const int64_t e = elem_size(type), size = l.first(false) + l.second(false);
  if (!U || (size > 0 && !P)) return fail(VT_EINVAL, "%s: adapters or U are null", who);
  // u is made without outputs too
  if ((K > 0 && !X) || (i8 && !T)) return fail(VT_EINVAL, "%s: input is null, or int8 rows without scales", who);
  const Operand o[] = {{"X", X, M, ldx, x_type == VT_TYPE_I8_PADDED ? l.Kp : K, elem_size(x_type), false},
                       {"T", T, 1, M, M, 4, false}, {"weights", Bp, 1, 0, l.Kp * l.Np, 1, false},
                       {"scales", meta, 1, 0, scaled_meta(l.Np), 4, false}, {"adapters", P, 1, size, size, e, false, 16 / e},
                       {"which", which, 1, M, M, 4, false}, {"U", U, 1, M * Rp, M * Rp, 4, true, 4}, {"Y", Y, M, ldy, N, e, true}};
  if (int rc = check_operands(who, o, 8)) return rc;
  const LowRank low = {U, (const int8_t *)P + l.first(false) * e, which, l.Np, (int)L, (int)Rp, (int)M};
  ShrinkPair pair = {};
  pair.of[0] = ShrinkArgs{X, T, P, which, U, ldx, scale, (int)M, (int)K, (int)l.Kp, (int)L, (int)Rp, nullptr, nullptr};
  const bool out = !empty;
  // few rows are one part
  const int64_t step = rows_in_place(X, x_type, ldx, K) ? M : rows_at_once(M, l.Kp + 4);
  for (int64_t r = 0; r < M && (out || r == 0); r += step) {
    Scratch scr;
    if (int rc = open_scratch(stream, &scr)) return rc;
    Rows rows = {};
    const bool rounds = out && shrink_rounds(c);
    if (rounds) {
      void *w = nullptr;
      if (int rc = scr.take(kRows, (size_t)M * (l.Kp + sizeof(float)), &w)) return rc;
      pair.of[0].Q = (int8_t *)w;
      pair.of[0].T = (float *)((int8_t *)w + M * l.Kp);
      rows = Rows{pair.of[0].Q, pair.of[0].T, l.Kp};
    }
    if (r == 0)
      if (int rc = shrink(pair, 1, type, i8, scr)) return rc;
    if (!out) break;
    const int64_t count = std::min(step, M - r);
    if (int rc = adapted_rows(part_of(c, r, count), low_at(low, r, count), rounds ? &rows : nullptr, scr)) return rc;
  }
  return VT_OK;
}

int vt_adapted_grad(const void *dY, int32_t type, int64_t ldd, const void *X, int64_t ldx, int64_t M, int64_t K, const int8_t *Bp,
                    const float *meta, int64_t N, const void *P, const void *back, int64_t R, int64_t L, float scale,
                    const int32_t *which, float *U, float *H, void *dX, int64_t lddx, void *dDown, void *dUp, void *stream) {
  g_err.clear();
  const char *who = "vt_adapted_grad";
  const int64_t Rp = rank_pad(R);
  const ScaledCall c = {who, dY, type, ldd, N, nullptr, Bp, meta, dX ? dX : H, dX ? type : VT_TYPE_F32, dX ? lddx : Rp, dX ? K : Rp, M, K, N, false};
  const AdapterCall ad = {who, type, L, R, K, N};
  if (int rc = check_adapters(ad)) return rc;
  bool empty = false;
  if (int rc = check_scaled(c, &empty)) return rc;
  const AdapterLayout l = adapter_layout(K, N, R, L);
  const int64_t e = elem_size(type), size = l.first(true) + l.second(true);
  const bool again = P && dUp;   // u has to be made again
  if (M > 0 && (!H || (N > 0 && !dY) || (size > 0 && !back) || (dUp && !U) || ((dDown || again) && K > 0 && !X)))
    return fail(VT_EINVAL, "%s: adapters, dY, X, U or H are null", who);
  const Operand o[] = {{"dY", dY, M, ldd, N, e, false}, {"X", X, M, ldx, K, e, false}, {"weights", Bp, 1, 0, l.Kp * l.Np, 1, false},
                       {"scales", meta, 1, 0, scaled_meta(l.Np), 4, false}, {"adapters", P, 1, size, size, e, false, 16 / e},
                       {"adapters", back, 1, size, size, e, false, 16 / e}, {"which", which, 1, M, M, 4, false},
                       {"U", dUp ? U : nullptr, 1, M * Rp, M * Rp, 4, again, 4},
                       {"H", H, 1, M * Rp, M * Rp, 4, true, 4}, {"dX", dX, M, lddx, K, e, true},
                       {"dDown", dDown, 1, L * R * K, L * R * K, e, true}, {"dUp", dUp, 1, L * R * N, L * R * N, e, true}};
  if (int rc = check_operands(who, o, 12)) return rc;
  if (M > 0) {
    Scratch scr;
    if (int rc = open_scratch(stream, &scr)) return rc;
    ShrinkPair a = {};
    a.of[0] = ShrinkArgs{dY, nullptr, back, which, H, ldd, scale, (int)M, (int)N, (int)l.Np, (int)L, (int)Rp, nullptr, nullptr};
    a.of[1] = ShrinkArgs{X, nullptr, P, which, U, ldx, scale, (int)M, (int)K, (int)l.Kp, (int)L, (int)Rp, nullptr, nullptr};
    if (int rc = shrink(a, again ? 2 : 1, type, false, scr)) return rc;
  }
  if (dX && M > 0 && K > 0) {
    const LowRank low = {H, (const int8_t *)back + l.first(true) * e, which, l.Kp, (int)L, (int)Rp, (int)M};
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
  OuterPair a = {};
  int count = 0;
  if (dDown && K > 0)
    a.of[count++] = OuterArgs{H, X, which, nullptr, dDown, ldx, (int)M, (int)K, (int)l.Kp, (int)L, (int)R, (int)Rp, 1, 0};
  if (dUp && N > 0)
    a.of[count++] = OuterArgs{U, dY, which, nullptr, dUp, ldd, (int)M, (int)N, (int)l.Np, (int)L, (int)R, (int)Rp, 1, 1};
  if (count == 0) return VT_OK;
  return by_type(type, [&](auto t) { return launch_outer<decltype(t)::value>(a, count, scr); });
}

}  // extern "C"
