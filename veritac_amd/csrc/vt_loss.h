// vt_loss.h -- softmax cross entropy over the logits of an int8 linear layer,
// without keeping the logits, and its gradient in the layer's rows. Part of
// vt_hip_gemm.hip's translation unit, after vt_norm.h.
//
//   l_ij = t_i s_j sum_k q_ik W_kj + b_j
//   loss_i = m_i + log(sum_j exp(l_ij - m_i)) - l_i,target_i, m_i = max_j l_ij
//   dx_ik = g_i sum_j (p_ij - [j = target_i]) s_j W_kj, p_ij = exp((l_ij - m_i) - log(sum))
//
// Forward, the product's epilogue reduces each wave's columns of a row to their
// maximum and the sum of exponentials over it, and a second kernel joins a row's
// parts. Backward, the product runs again and its epilogue writes the gradient's
// terms as 16-bit values, which the gradient product of vt_scaled.h multiplies by
// the weights. m and log(sum) are kept apart: together they would lose the sum
// where the logits are large.

namespace {

typedef float v2f __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kIgnored = -1, kInvalid = -2;   // a row's target in its state

// What the backward pass keeps of a row: m, log(sum), the normaliser of its
// gradient terms, and its target.
struct RowState {
  float top, log_sum, norm;
  int target;
};

struct Targets {
  const void *p;
  int64_t ignored;
  int wide;   // int64, else int32
};

__device__ __forceinline__ int64_t target_value(const Targets &t, int64_t row) {
  return t.wide ? ((const int64_t *)t.p)[row] : (int64_t)((const int32_t *)t.p)[row];
}

// max(a, a of the lane that DPP gives), and the sum likewise, within 16 lanes.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
constexpr int kQuadXor1 = 0xb1, kQuadXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;

// Over LANES (16 or 32) neighbouring lanes, in all of them.
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
  v = fmaxf(v, dpp<kQuadXor1>(v));
  v = fmaxf(v, dpp<kQuadXor2>(v));
  v = fmaxf(v, dpp<kHalfMirror>(v));
  v = fmaxf(v, dpp<kMirror>(v));
  if constexpr (LANES == 32) v = fmaxf(v, __shfl_xor(v, 16));
  return v;
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp<kQuadXor1>(v);
  v += dpp<kQuadXor2>(v);
  v += dpp<kHalfMirror>(v);
  v += dpp<kMirror>(v);
  if constexpr (LANES == 32) v += __shfl_xor(v, 16);
  return v;
}

// A class' logit: the same operations in both passes, and in a linear layer's outputs.
__device__ __forceinline__ float logit_of(int32_t sum, float t, float s, float b) { return fmaf((float)sum * t, s, b); }

// exp(v), where v is a logit less its row's maximum (or -inf). The argument's
// rounding, 2^-24 of |v|, is the result's relative error; in log(sum) that is |v|'s mean
// over the classes' shares, ln N at the most, times 2^-24 of either sign: losses over
// 131072 classes are 7.4e-8 off 64 bits, torch's operations in 32 bits 7.3e-8.
__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(v * kLog2e); }

// A maximum that logits are taken from: finite, so that columns masked by -inf
// give 0 and not NaN. (A NaN logit is in no maximum and in every sum.)
__device__ __forceinline__ float base_of(float top) { return fmaxf(top, -3.40282347e38f); }

// (maximum, sum) of NV values of LANES lanes.
template <int LANES, int NV>
__device__ __forceinline__ v2f part_of_row(const float (&v)[NV]) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < NV; ++i) m = fmaxf(m, v[i]);
  m = base_of(lanes_max<LANES>(m));
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) s += exp_of(v[i] - m);
  return v2f{m, lanes_sum<LANES>(s)};
}

__device__ __forceinline__ v2f join_parts(v2f a, v2f b) {
  const float m = fmaxf(a[0], b[0]);
  return v2f{m, a[1] * exp_of(a[0] - m) + b[1] * exp_of(b[0] - m)};
}

// Forward: a tile's logits -> one (maximum, sum) for each of its rows and each
// wave's columns, and the logits of targets among them. All in registers: 16 (or
// 32) lanes hold a row, whose maximum and sum take four (five) DPP steps each, and
// 8 bytes for 128 logits leave the CU. Bound by the int8 product in front: 2048 x
// 4096 x 131072 in 891 us (2.47 POPS), 2048 x 4096 x 65536 in 447.
struct LseTile : ScaledOut {
  static constexpr bool kScaled = true, kWide = true;
  v2f *part;        // [parts][M]
  float *mine;      // [M]
  Targets targets;

  // Element e (of E) of a wave's rows: row0 + row_of(e), values v[e][NI] of columns
  // col + step * ni, W columns from col0 in all.
  template <int LANES, int E, int NI, class ROW>
  __device__ __forceinline__ void rows(const float (&v)[E][NI], int row0, ROW row_of, int row_min, int col0, int col,
                                       int step, int slot, int lane) const {
    v2f mine_part = {0.0f, 0.0f};
    int my_row = -1;
    const int c = lane % LANES;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const v2f ms = part_of_row<LANES, NI>(v[e]);
      if (c == e) {
        mine_part = ms;
        my_row = row0 + row_of(e);
      }
    }
    int rel = -1;   // the row's target, less col0
    if (my_row >= row_min && my_row < M && c < E) {
      part[(int64_t)slot * M + my_row] = mine_part;
      const int64_t at = target_value(targets, my_row);
      if (at != targets.ignored && at >= col0 && at < col0 + step * NI && at < N) rel = (int)(at - col0);
    }
    // A row's target is among a wave's columns once in a vocabulary.
    if (__ballot(rel >= 0)) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int row = row0 + row_of(e), to = __shfl(rel, (lane / LANES) * LANES + e);
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
          if (to >= 0 && col + step * ni == col0 + to) mine[row] = v[e][ni];
      }
    }
  }

  template <int MI, int NI, bool EDGE>
  __device__ __forceinline__ void tile16(const v4i (&acc)[MI][NI], int row0, int col0, int row_min, int col_min, int lane,
                                         LDS_AS int8_t *) const {
    constexpr int W = NI * 16;
    const int g = lane >> 4, c = lane & 15;
    const int slot = col_min / W + (col0 - min(col_min, Np - 2 * W)) / W;
    float s[NI], b[NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      const int j = col0 + ni * 16 + c;
      const bool in = j < N && j >= col_min;
      s[ni] = meta[j];
      b[ni] = meta[Np + j];
      if (!in) {
        s[ni] = 0.0f;
        b[ni] = -__builtin_inff();
      }
    }
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
      const v4f tr = *(const v4f_any *)(t + row0 + mi * 16 + 4 * g);
      float v[4][NI];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) v[e][ni] = logit_of(acc[mi][ni][e], tr[e], s[ni], b[ni]);
      rows<16, 4, NI>(v, row0 + mi * 16 + 4 * g, [](int e) { return e; }, row_min, max(col0, col_min), col0 + c, 16, slot,
                      lane);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  template <int MI, int NI>
  __device__ __forceinline__ void tile32(const v16i (&acc)[MI][NI], int row0, int col0, int lane, LDS_AS int8_t *) const {
    const int g = lane >> 5, c = lane & 31, slot = col0 / (32 * NI);
    float s[NI], b[NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      const int j = col0 + ni * 32 + c;
      s[ni] = j < N ? meta[j] : 0.0f;
      b[ni] = j < N ? meta[Np + j] : -__builtin_inff();
    }
    each([&](auto strip) __attribute__((always_inline)) {
      constexpr int mi = decltype(strip)::value;
      float v[16][NI];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float tr = t[min(row0 + mi * 32 + 8 * (e >> 2) + 4 * g + (e & 3), M - 1)];
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) v[e][ni] = logit_of(acc[mi][ni][e], tr, s[ni], b[ni]);
      }
      rows<32, 16, NI>(v, row0 + mi * 32 + 4 * g, [](int e) { return 8 * (e >> 2) + (e & 3); }, 0, col0, col0 + c, 32, slot,
                       lane);
    }, std::make_integer_sequence<int, MI>());
  }
};

// Backward: a tile's logits -> 16-bit gradient terms (p - [target]) s of its rows,
// times the rows' normalisers, and with LOW what float16 leaves of them (22 bits).
// Without it, for bfloat16 rows, a term has 11 bits, 8 times finer than the gradient's
// own rounding (two_halves): 2048 x 4096 -> 65536 is 1.0e-3 from the 32-bit form, and
// as far from 64 bits as that, 1.7e-3.
template <bool LOW>
struct LossTermsTile : ScaledTile<kGradTerms, 2, LOW> {
  static constexpr bool kWide = true;
  const RowState *state;
  const float *dloss, *count;   // count null: not a mean
  float *norm_out;
  int64_t step;                 // of dloss: 1 for one a row, 0 for one in all

  struct Row {
    float t, top, log_sum, norm;
    int target;
  };
  __device__ __forceinline__ Row row_at(int row) const {
    const v4i w = *(const v4i *)(state + row);
    return Row{this->t[row], __int_as_float(w[0]), __int_as_float(w[1]), __int_as_float(w[2]), w[3]};
  }
  // log p of a class
  __device__ __forceinline__ float log_p(int32_t sum, const Row &r, float s, float b) const {
    return (logit_of(sum, r.t, s, b) - r.top) - r.log_sum;
  }
  __device__ __forceinline__ float term(int32_t sum, const Row &r, float s, float b) const {
    float v = exp_of(log_p(sum, r, s, b)) * s * r.norm;
    if (r.target == kIgnored) v = 0.0f;
    // rounded to 32 bits before its conversion, as its low half assumes
    asm("" : "+v"(v));
    return v;
  }
  // The target's: p - 1 by itself, since p may be next to 1. Once in a row, so
  // behind one branch of the wave.
  __device__ __forceinline__ float target_term(int32_t sum, const Row &r, float s, float b) const {
    float v = expm1f(log_p(sum, r, s, b)) * s * r.norm;
    asm("" : "+v"(v));
    return v;
  }

  // What the gradient product divides a row by: its normaliser over the gradient
  // that reaches its loss.
  __device__ __forceinline__ void put_norm(int row, const Row &r) const {
    float g = dloss[row * step];
    if (count) g /= *count;
    norm_out[row] = r.target == kIgnored ? __builtin_inff() : r.norm / g;
  }

  // A strip of 16 rows at a time in a loop: its sums go through the wave's LDS to 8
  // columns of a row a lane, which then needs one row's state, and the code stays
  // in the instruction cache (2048 x 4096 x 65536 in 540 us, 268 MB of terms written;
  // unrolled, and with a branch for the target in each of its parts, 606).
  template <int MI, int NI, bool EDGE>
  __device__ __forceinline__ void tile16(const v4i (&acc)[MI][NI], int row0, int col0, int row_min, int col_min, int lane,
                                         LDS_AS int8_t *lds) const {
    constexpr int W = NI * 16, LPR = W / 8, RPI = 64 / LPR, IT = 16 / RPI;
    const int g = lane >> 4, c = lane & 15, j8 = 8 * (lane % LPR), lr = lane / LPR, col = col0 + j8;
    float s[8], b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s[e] = this->meta[col + e];
      b[e] = col + e < this->N ? this->meta[this->Np + col + e] : -__builtin_inff();   // no class: p = 0
    }
    Row next[IT];
#pragma unroll
    for (int it = 0; it < IT; ++it) next[it] = row_at(row0 + it * RPI + lr);
#pragma unroll 1
    for (int mi = 0; mi < MI; ++mi) {
      Row now[IT];
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        now[it] = next[it];
        next[it] = row_at(row0 + min(mi + 1, MI - 1) * 16 + it * RPI + lr);
      }
      // chunk k of strip row r at k ^ (4 (r / 4 % 4)): an instruction's writes fall on distinct banks
      each([&](auto strip) __attribute__((always_inline)) {
        constexpr int i = decltype(strip)::value;
        if (mi != i) return;
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *(LDS_AS int32_t *)(lds + (4 * g + e) * (W * 4) + ((((ni ^ g) << 2) + (c >> 2)) << 4) + (c & 3) * 4) = acc[i][ni][e];
      }, std::make_integer_sequence<int, MI>());
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int r = it * RPI + lr, row = row0 + mi * 16 + r, swz = ((r >> 2) & 3) << 2;
        const LDS_AS int8_t *at = lds + r * (W * 4);
        const v4i x = *(const LDS_AS v4i *)(at + (((j8 >> 2) ^ swz) << 4)), y = *(const LDS_AS v4i *)(at + ((((j8 >> 2) + 1) ^ swz) << 4));
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = term(e < 4 ? x[e & 3] : y[e & 3], now[it], s[e], b[e]);
        const int rel = now[it].target - col;
        if (__ballot((unsigned)rel < 8u)) {
#pragma unroll 1
          for (int e = 0; e < 8; ++e) {
            int32_t sum = 0;
            float se = 0.0f, be = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (k == e) {
                sum = k < 4 ? x[k & 3] : y[k & 3];
                se = s[k];
                be = b[k];
              }
            const float w = target_term(sum, now[it], se, be);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (k == e && rel == e) v[k] = w;
          }
        }
        if (EDGE && (row < row_min || col < col_min)) continue;
        const int64_t to = (int64_t)row * this->Np + col;
        this->store8(to, v, VT_TYPE_F16);
        if constexpr (LOW) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] -= (float)(_Float16)v[e];
          this->store8(to + this->lo, v, VT_TYPE_F16);
        }
        if (col == 0) put_norm(row, now[it]);
      }
    }
  }

  template <int MI, int NI>
  __device__ __forceinline__ void tile32(const v16i (&acc)[MI][NI], int row0, int col0, int lane, LDS_AS int8_t *lds) const {
    static_assert(NI == 2, "strips of 64 columns");
    const int g = lane >> 5, c = lane & 31, Np = this->Np, M = this->M;
    if (col0 >= Np) return;   // the same for the whole wave, behind the last barrier
    float s[NI], b[NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      const int j = col0 + ni * 32 + c;
      s[ni] = this->meta[j];
      b[ni] = j < this->N ? this->meta[Np + j] : -__builtin_inff();   // no class: p = 0
    }
    each([&](auto strip) __attribute__((always_inline)) {
      constexpr int mi = decltype(strip)::value;
      const int first = row0 + mi * 32;
      float v[NI][16];
      bool some = false;
      auto row_of = [&](int e) { return row_at(min(first + 8 * (e >> 2) + 4 * g + (e & 3), M - 1)); };
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const Row r = row_of(e);
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) v[ni][e] = term(acc[mi][ni][e], r, s[ni], b[ni]);
        some |= (unsigned)(r.target - col0) < 64u;
      }
      if (col0 == 0 && lane < 32 && first + lane < M) put_norm(first + lane, row_at(first + lane));
      if (__ballot(some)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const Row r = row_of(e);
#pragma unroll
          for (int ni = 0; ni < NI; ++ni)
            if (r.target == col0 + ni * 32 + c) v[ni][e] = target_term(acc[mi][ni][e], r, s[ni], b[ni]);
        }
      }
      auto flush = [&](int64_t plane) {
        // rows of 128 bytes, chunk k of row r at k ^ (r / 4 % 2)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            *(LDS_AS _Float16 *)(lds + (8 * (e >> 2) + 4 * g + (e & 3)) * 128 + (((ni * 4 + (c >> 3)) ^ g) << 4) + (c & 7) * 2) =
                (_Float16)v[ni][e];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int idx = i * 64 + lane, r = idx >> 3, k = idx & 7;
          if (first + r < M)
            __builtin_nontemporal_store(*(const LDS_AS v4i *)(lds + r * 128 + ((k ^ ((r >> 2) & 1)) << 4)),
                                        (v4i_any *)((uint16_t *)this->Y + (int64_t)(first + r) * Np + col0 + k * 8 + plane));
        }
      };
      flush(0);
      if constexpr (LOW) {
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
#pragma unroll
          for (int e = 0; e < 16; ++e) v[ni][e] -= (float)(_Float16)v[ni][e];
        flush(this->lo);
      }
    }, std::make_integer_sequence<int, MI>());
  }
};

// Logits of a few rows (float32 [M][N] of a workspace) -> their parts: one
// workgroup for 4096 columns of a row.
constexpr int kLogitChunk = 4096;

struct LogitArgs {
  const float *L;
  v2f *part;
  float *mine;
  Targets targets;
  int M, N;
};

__global__ __launch_bounds__(256) void logit_parts_kernel(LogitArgs p) {
  __shared__ v2f red[4];
  const int row = blockIdx.y, c0 = blockIdx.x * kLogitChunk;
  const float *l = p.L + (int64_t)row * p.N + c0;
  const int count = min(p.N - c0, kLogitChunk);
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int j = i * 256 + threadIdx.x;
    v[i] = j < count ? l[j] : -__builtin_inff();
  }
  const int64_t at = target_value(p.targets, row);
  if (threadIdx.x == 0 && at != p.targets.ignored && at >= c0 && at < c0 + count) p.mine[row] = l[at - c0];
  v2f ms = part_of_row<32, 16>(v);
  const v2f other = {__shfl_xor(ms[0], 32), __shfl_xor(ms[1], 32)};
  // in one order on both sides: results repeat whichever lane writes
  ms = (threadIdx.x & 32) ? join_parts(other, ms) : join_parts(ms, other);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ms;
  __syncthreads();
  if (threadIdx.x == 0)
    p.part[(int64_t)blockIdx.x * p.M + row] = join_parts(join_parts(red[0], red[1]), join_parts(red[2], red[3]));
}

// A row's parts -> its loss and state. ROWS rows to a workgroup of 1024, whose
// other threads share a row's parts out: 16 rows, so a read is whole 128-byte
// lines (2048 rows of 1024 parts in 13 us), or 1 where the rows are few.
struct LossRowsArgs {
  const v2f *part;
  const float *mine;
  const float *top_scale;   // the weights' largest |s|, in kTopParts parts
  Targets targets;
  float *loss;
  RowState *state;
  int parts, M, N;
};

template <int ROWS>
__global__ __launch_bounds__(1024) void loss_rows_kernel(LossRowsArgs p) {
  constexpr int GROUPS = 1024 / ROWS;
  __shared__ v2f red[GROUPS][ROWS];
  const int r = threadIdx.x % ROWS, g = threadIdx.x / ROWS, row = blockIdx.x * ROWS + r;
  v2f ms = {-3.40282347e38f, 0.0f};
  if (row < p.M)
    for (int i = g; i < p.parts; i += GROUPS) ms = join_parts(ms, p.part[(int64_t)i * p.M + row]);
  red[g][r] = ms;
  __syncthreads();
#pragma unroll
  for (int n = GROUPS / 2; n; n /= 2) {
    if (g < n) red[g][r] = join_parts(red[g][r], red[g + n][r]);
    __syncthreads();
  }
  if (g || row >= p.M) return;
  ms = red[0][r];
  RowState st = {ms[0], logf(ms[1]), 0.0f, kIgnored};
  float loss = 0.0f;
  const int64_t at = target_value(p.targets, row);
  if (at != p.targets.ignored) {
    const bool valid = at >= 0 && at < p.N;
    st.target = valid ? (int)at : kInvalid;
    loss = valid ? (ms[0] - p.mine[row]) + st.log_sum : __uint_as_float(0x7fc00000u);
    // |p - [target]| is at most 1 - p of the target, of which the logits' own rounding
    // leaves no bits below 2^-22 of their size
    const float least = 0x1p-22f * fminf(fmaxf(fabsf(ms[0]), 1.0f), 0x1p20f);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kTopParts; ++i) top = max(top, magnitude(p.top_scale[i]));
    st.norm = loss == loss ? normaliser(fmaxf(-expm1f(-loss), least) * __uint_as_float(top)) : loss;
  }
  p.loss[row] = loss;
  p.state[row] = st;
}

// The rows' losses -> their sum or mean, and how many rows have a target. In 64 bits: one workgroup adds them up.
struct LossSumArgs {
  const float *loss;
  const RowState *state;
  float *out, *count;   // their sum or mean; how many have a target
  int M, mean;
};

__global__ __launch_bounds__(1024) void loss_sum_kernel(LossSumArgs p) {
  __shared__ double sums[16];
  __shared__ int counts[16];
  double s = 0.0;
  int n = 0;
  for (int i = threadIdx.x; i < p.M; i += 1024) {
    s += (double)p.loss[i];
    n += p.state[i].target != kIgnored;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    s += __shfl_xor(s, o);
    n += __shfl_xor(n, o);
  }
  if ((threadIdx.x & 63) == 0) {
    sums[threadIdx.x >> 6] = s;
    counts[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 16; ++i) {
    s += sums[i];
    n += counts[i];
  }
  *p.out = (float)(p.mean ? s / n : s);
  *p.count = (float)n;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

struct LossCall {
  ScaledCall c;
  Targets targets;
  float *loss;
  RowState *state;
};

// Whether the logits of a call go through a workspace: up to 64 rows, whose
// product is bound by reading the weights (their logits are 4 M / K of that), and
// sums over nothing.
bool through_logits(int64_t M, int64_t Kp) { return M <= kSkinnyMaxM || Kp == 0; }

int loss_rows(const LossCall &l, bool logits, void *stream) {
  const ScaledCall &c = l.c;
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  hipStream_t s = (hipStream_t)stream;
  const int64_t Kp = scaled_kp(c.K), Np = scaled_np(c.N, false);
  const int M = (int)c.M, N = (int)c.N;
  LossRowsArgs r = {nullptr, nullptr, c.meta + 2 * Np, l.targets, l.loss, l.state, 0, M, N};
  void *w = nullptr;
  if (logits) {
    r.parts = (N + kLogitChunk - 1) / kLogitChunk;
    const size_t bytes = ((size_t)M * N * sizeof(float) + 255) / 256 * 256;
    if (int rc = scr.take(kTerms, bytes + (size_t)M * r.parts * sizeof(v2f) + (size_t)M * sizeof(float), &w)) return rc;
    r.part = (v2f *)((int8_t *)w + bytes);
    r.mine = (float *)(r.part + (int64_t)M * r.parts);
    ScaledCall f = c;
    f.Y = w;
    f.y_type = VT_TYPE_F32;
    f.ldy = f.yc = c.N;
    if (int rc = forward_rows(f, VT_ACT_SILU, scr)) return rc;
    const LogitArgs a = {(const float *)w, (v2f *)r.part, (float *)r.mine, l.targets, M, N};
    hipLaunchKernelGGL(logit_parts_kernel, dim3((unsigned)r.parts, (unsigned)M), dim3(256), 0, s, a);
    VT_HIP_CHECK(hipGetLastError());
  } else {
    const TilePlan plan = tile_plan(false, c.M, Np, Kp, scr.st->num_cus, false);
    r.parts = (int)((Np + plan.bn - 1) / plan.bn * 2);
    Rows rows;
    if (int rc = scr.take(kPartials, (size_t)M * (r.parts * sizeof(v2f) + sizeof(float)), &w)) return rc;
    r.part = (v2f *)w;
    r.mine = (float *)(r.part + (int64_t)M * r.parts);
    if (int rc = take_rows(c.X, c.x_type, c.ldx, c.T, c.M, c.K, scr, &rows)) return rc;
    LseTile out = {};
    out.t = rows.t; out.meta = c.meta;
    out.M = M; out.N = N; out.Np = (int)Np;
    out.part = (v2f *)r.part;
    out.mine = (float *)r.mine;
    out.targets = l.targets;
    if (int rc = launch_tiles(plan, rows, c.Bp, Kp, out, scr)) return rc;
  }
  if (M >= 512) hipLaunchKernelGGL(loss_rows_kernel<16>, dim3((unsigned)((M + 15) / 16)), dim3(1024), 0, s, r);
  else hipLaunchKernelGGL(loss_rows_kernel<1>, dim3((unsigned)M), dim3(1024), 0, s, r);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

int loss_grad_rows(const ScaledCall &c, const RowState *state, const float *dloss, int64_t step, const float *count, void *stream) {
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const int64_t Kp = scaled_kp(c.K), Np = scaled_np(c.N, false);
  const bool split = two_halves(c.y_type);
  const int64_t lo = split ? c.M * Np : 0;
  void *w = nullptr;
  const size_t t_bytes = ((size_t)c.M * Np * 2 * (split ? 2 : 1) + 255) / 256 * 256;
  if (int rc = scr.take(kTerms, t_bytes + (size_t)c.M * sizeof(float), &w)) return rc;
  float *norm = (float *)((int8_t *)w + t_bytes);
  Rows rows;
  if (int rc = take_rows(c.X, c.x_type, c.ldx, c.T, c.M, c.K, scr, &rows)) return rc;
  ScaledOut f = {};
  f.t = rows.t; f.meta = c.meta; f.Y = w;
  f.lo = lo;
  f.M = (int)c.M; f.N = (int)c.N; f.Np = (int)Np;
  const TilePlan plan = tile_plan(true, c.M, Np, Kp, scr.st->num_cus, false);
  auto terms = [&](auto out) {
    (ScaledOut &)out = f;
    out.state = state;
    out.dloss = dloss;
    out.count = count;
    out.step = step;
    out.norm_out = norm;
    return launch_tiles(plan, rows, c.Bp, Kp, out, scr);
  };
  if (int rc = split ? terms(LossTermsTile<true>()) : terms(LossTermsTile<false>())) return rc;
  ScaledTile<kGrad> o = {};
  o.Y = c.Y; o.ldy = c.ldy;
  o.M = (int)c.M; o.N = (int)c.K; o.Np = (int)Kp;
  o.type = c.y_type; o.norm = norm;
  const GradArgs g = {(const _Float16 *)w, c.Bp, lo, (int)c.M, (int)Kp, (int)Np, 0, 0, 0, split ? 2 : 1, 1};
  return launch_grad(g, o, scr);
}

int check_targets(const char *who, const void *target, int32_t type, int64_t M) {
  if (type != VT_TARGET_I32 && type != VT_TARGET_I64) return fail(VT_EINVAL, "%s: unknown target type %d", who, (int)type);
  if (!target) return fail(VT_EINVAL, "%s: targets are null", who);
  if ((uintptr_t)target % (type == VT_TARGET_I64 ? 8 : 4)) return fail(VT_EINVAL, "%s: targets are not aligned to their elements", who);
  return VT_OK;
}

}  // namespace

extern "C" {

int vt_cross_entropy(const void *X, int32_t x_type, int64_t ldx, const float *T, int64_t M, int64_t K, const int8_t *Bp,
                     const float *meta, int64_t N, const void *target, int32_t target_type, int64_t ignored, float *loss,
                     float *state, int32_t reduction, float *reduced, float *count, void *stream) {
  g_err.clear();
  const char *who = "vt_cross_entropy";
  if (reduction != VT_REDUCE_NONE && reduction != VT_REDUCE_MEAN && reduction != VT_REDUCE_SUM)
    return fail(VT_EINVAL, "%s: unknown reduction %d", who, (int)reduction);
  if (N < 1) return fail(VT_EINVAL, "%s: needs at least one class (N=%lld)", who, (long long)N);
  LossCall l = {};
  l.c = ScaledCall{who, X, x_type, ldx, K, T, Bp, meta, loss, VT_TYPE_F32, 1, 1, M, K, N, false};
  bool empty = false;
  if (int rc = check_scaled(l.c, &empty)) return rc;
  if (reduction == VT_REDUCE_NONE) reduced = count = nullptr;
  else if (!reduced || !count) return fail(VT_EINVAL, "%s: no place for the reduced loss", who);
  if (!empty) {
    if (int rc = check_targets(who, target, target_type, M)) return rc;
    if (!state) return fail(VT_EINVAL, "%s: state is null", who);
    const int64_t Kp = scaled_kp(K), Np = scaled_np(N, false), elem = elem_size(x_type);
    const Operand o[] = {{"X", X, M, ldx, K, elem, false}, {"T", T, 1, M, M, 4, false}, {"weights", Bp, 1, 0, Kp * Np, 1, false},
                         {"scales", meta, 1, 0, scaled_meta(Np), 4, false},
                         {"targets", target, 1, M, M, target_type == VT_TARGET_I64 ? 8 : 4, false},
                         {"loss", loss, 1, M, M, 4, true}, {"state", state, 1, 4 * M, 4 * M, 4, true, 4},
                         {"reduced", reduced, 1, 1, 1, 4, true}, {"count", count, 1, 1, 1, 4, true}};
    if (int rc = check_operands(who, o, 9)) return rc;
    l.targets = Targets{target, ignored, target_type == VT_TARGET_I64};
    l.loss = loss;
    l.state = (RowState *)state;
    int64_t step;
    const bool logits = through_logits(M, Kp);
    if (logits) {
      // rows are logit_parts_kernel's second side
      const int64_t most = std::min<int64_t>(M, 65535);
      step = std::max<int64_t>(1, std::min(most, kScaledBytes / (N * 4 + (N / kLogitChunk + 1) * 8 + 8)));
    } else {
      // parts of 64 columns at the least
      int64_t row_bytes = (Np + 127) / 128 * 2 * 8 + 4;
      if (!rows_in_place(X, x_type, ldx, K)) row_bytes = std::max(row_bytes, Kp + 4);
      step = rows_at_once(M, row_bytes);
    }
    for (int64_t r = 0; r < M; r += step) {
      LossCall p = l;
      p.c = part_of(l.c, r, std::min(step, M - r));
      p.targets.p = (const int8_t *)target + r * (target_type == VT_TARGET_I64 ? 8 : 4);
      p.loss += r;
      p.state += r;
      if (int rc = loss_rows(p, logits, stream)) return rc;
    }
  }
  if (reduction == VT_REDUCE_NONE) return VT_OK;
  Scratch scr;
  if (int rc = open_scratch(stream, &scr)) return rc;
  const LossSumArgs a = {loss, (const RowState *)state, reduced, count, (int)M, reduction == VT_REDUCE_MEAN};
  hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a);
  VT_HIP_CHECK(hipGetLastError());
  return VT_OK;
}

int vt_cross_entropy_grad(const int8_t *Q, int32_t q_type, int64_t ldq, const float *T, int64_t M, int64_t K, const int8_t *Bp,
                          const float *meta, int64_t N, const float *state, const float *dloss, int64_t dloss_step,
                          const float *count, void *dX, int32_t type, int64_t ldx, void *stream) {
  g_err.clear();
  const char *who = "vt_cross_entropy_grad";
  if (N < 1) return fail(VT_EINVAL, "%s: needs at least one class (N=%lld)", who, (long long)N);
  if (q_type != VT_TYPE_I8 && q_type != VT_TYPE_I8_PADDED) return fail(VT_EINVAL, "%s: the rows are int8 with scales", who);
  const ScaledCall c = {who, Q, q_type, ldq, K, T, Bp, meta, dX, type, ldx, K, M, K, N, false};
  bool empty = false;
  if (int rc = check_scaled(c, &empty)) return rc;
  if (dloss_step != 0 && dloss_step != 1) return fail(VT_EINVAL, "%s: one gradient for each row, or one in all", who);
  if (empty) return VT_OK;
  if (!state || !dloss) return fail(VT_EINVAL, "%s: state or dloss is null", who);
  const Operand o[] = {{"state", state, 1, 4 * M, 4 * M, 4, false, 4}, {"dloss", dloss, 1, M, dloss_step ? M : 1, 4, false},
                       {"count", count, 1, 1, 1, 4, false}, {"dX", dX, M, ldx, K, elem_size(type), true}};
  if (int rc = check_operands(who, o, 4)) return rc;
  int64_t row_bytes = scaled_np(N, false) * (two_halves(type) ? 4 : 2) + 4;
  if (!rows_in_place(Q, q_type, ldq, K)) row_bytes = std::max(row_bytes, scaled_kp(K) + 4);
  const int64_t step = rows_at_once(M, row_bytes);
  for (int64_t r = 0; r < M; r += step)
    if (int rc = loss_grad_rows(part_of(c, r, std::min(step, M - r)), (const RowState *)state + r, dloss + r * dloss_step,
                                dloss_step, count, stream))
      return rc;
  return VT_OK;
}

}  // extern "C"
