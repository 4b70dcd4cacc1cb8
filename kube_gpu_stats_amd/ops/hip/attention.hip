// Softmax attention over a padded batch, forward and backward, for gfx950.
//
//   s_ij = c q_i.k_j  for j < n_b (j <= i if causal),  i < n_b
//   o_i = sum_j softmax_j(s_i) v_j,   lse_i = log2 sum_j 2^(s_ij log2 e)
//   delta_i = do_i.o_i,  p_ij = 2^(s_ij log2 e - lse_i),  ds_ij = p_ij (do_i.v_j - delta_i)
//   dq_i = c sum_j ds_ij k_j,  dk_j = c sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// All three kernels hold one side of the score matrix in registers, 32 rows a wave, and
// walk the other side through LDS.  The product is taken the way round that leaves the
// wave's own rows in the lanes (column = lane % 32): softmax statistics are then one
// value a lane, a row's sum one exchange with lane ^ 32, and the probabilities lie in
// the registers as the next product's second operand wants them, up to an order of the
// summed index that Tile::columns reads the first operand in as well.  So the scores
// and probabilities never leave the registers.
//
// Scores, statistics, sums and accumulators are 32 bits.  Rounded to the tensors' type:
// p and ds, as operands of a matrix instruction (half a step each, independent from
// term to term; out, dq, dk and dv are 1.1 to 1.4 times as far from a 64-bit result as with
// p and ds in 32 bits), and the outputs.  The rounding of out would reach dq and dk through
// delta (a third more error than theirs); so the forward pass that a backward follows
// also keeps 8 bits of what it rounded off.
//
// Bound by the matrix units at the clock the power limit leaves where rows are long: 1 x
// 16384, 8 heads of 128 on 2, bf16, causal: forward 538 us (1020 TFLOP/s, matrix units busy
// 61 % of the time), dq 740 to 770 us (1070, 68 %), dk and dv 930 to 980 us (1110, 67 %).
// Start, end and diagonal of a walk take more of 4 x 2048, 32 heads: 155 us (890, 45 %),
// and dq with dk and dv 510 us (940, 44 and 57 %).  For D = 64 by the softmax's arithmetic,
// which issues for longer than the products: 8 x 1536, 12 heads, fp16, no mask: 76 us (765;
// vector instructions 66 %, matrix units 40 %).
#include "decoder.h"
#include "decoder_common.h"

namespace kgs {
namespace {

// A workgroup holds 128 rows in four waves, and two share a CU.  One of 256 rows with four
// or five steps under way instead of two was within 10 % either way (for forward and dq
// best on few key heads, worse on many or short rows; for dk and dv always worse).
constexpr int NW = 4, kThreads = NW * kWave, kRows = NW * 32;
constexpr int kStep = 64;   // keys a step of forward and dq
constexpr int kQStep = 32;  // rows a step of dk, dv

// Matrix products and LDS reads stay on their side of this; arithmetic may cross.  The
// compiler would place each read right before its product, with a wait between them.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0x406); }

__device__ __forceinline__ int length_of(const KgsAttention& a, int b) {
  if (!a.lengths) return a.S;
  const int n = __builtin_amdgcn_readfirstlane(a.lengths[b]);
  return n < 0 ? 0 : n > a.S ? a.S : n;
}

template <class T> __device__ __forceinline__ const char* at(const void* p, const int64_t* st, int b, int s, int h) {
  return reinterpret_cast<const char*>(static_cast<const T*>(p) + b * st[0] + s * st[1] + h * st[2]);
}

// Bytes from row s to the end of row n - 1.
template <class T, int D> __device__ __forceinline__ int64_t span(int n, int s, int64_t stride) {
  return n > s ? ((n - 1 - s) * stride + D) * static_cast<int64_t>(sizeof(T)) : 0;
}

// Stores a wave's accumulator (lane % 32 = row, registers = elements) times f to rows of
// memory, the rows up to `rows` only, by way of the wave's own 32 rows of LDS: as it lies
// in the registers a store would write 8 bytes of each of 32 rows, from LDS it writes
// whole rows.
template <class T, int D>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[D / 32], float f, char* lds, char* p, int64_t stride,
                                           int rows, int lane) {
  using x4 = typename El<T>::x4;
  using Tl = Tile<D>;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = static_cast<T>(acc[t][g * 4 + j] * f);
      *reinterpret_cast<x4*>(lds + Tl::at(lane & 31, t * 4 + g) + (lane >> 5) * 8) = v;
    }
  wave_order();
  constexpr int kPer = 64 / (D / 8);  // rows a store
  const i32x4 to = buffer(p, rows > 0 ? ((rows - 1) * stride + D) * 2 : 0);
#pragma unroll
  for (int i = 0; i < 32 / kPer; ++i) {
    const int row = i * kPer + lane / (D / 8), chunk = lane % (D / 8);
    const i32x4 v = *reinterpret_cast<const i32x4*>(lds + Tl::at(row, chunk));
    store16(v, to, static_cast<int>(row * stride * 2) + chunk * 16);
  }
  wave_order();
}

// What the rounding of acc f took, beside store_rows.
template <class T, int D>
__device__ __forceinline__ void store_low(const f32x16 (&acc)[D / 32], float f, char* lds, uint8_t* p, int64_t stride,
                                          int rows, int lane) {
  constexpr int kPer = 64 / (D / 16);
  const i32x4 to = buffer(p, rows > 0 ? (rows - 1) * stride + D : 0);
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = low_of<T>(acc[t][g * 4 + j] * f);
      const uint32_t lo = __builtin_amdgcn_perm(q[1], q[0], 0x0C0C0501), hi = __builtin_amdgcn_perm(q[3], q[2], 0x0C0C0501);
      const int row = lane & 31, e = t * 32 + g * 8 + (lane >> 5) * 4;
      *reinterpret_cast<uint32_t*>(lds + row * D + ((((e >> 4) ^ (row >> 1)) & (D / 16 - 1)) << 4) + (e & 15)) = lo | (hi << 16);
    }
  wave_order();
#pragma unroll
  for (int i = 0; i < 32 / kPer; ++i) {
    const int row = i * kPer + lane / (D / 16), chunk = lane % (D / 16);
    const i32x4 v = *reinterpret_cast<const i32x4*>(lds + row * D + (((chunk ^ (row >> 1)) & (D / 16 - 1)) << 4));
    store16(v, to, static_cast<int>(row * stride) + chunk * 16);
  }
}

// Registers 8 h .. 8 h + 7 of an accumulator, rounded: the second operand of the product
// that sums over the accumulator's rows.
template <class T> __device__ __forceinline__ typename El<T>::x8 operand(const f32x16& x, int h) {
  typename El<T>::x8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = static_cast<T>(x[h * 8 + j]);
  return r;
}

// The row index that register r of a 32x32 accumulator holds in this lane.
__device__ __forceinline__ int acc_row(int r, int lane) { return (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3); }

// fp16 has the precision for ds, not the range: ds is a probability, one of thousands, times
// products of do, which may be as small as a mean over tokens makes them.  So it is rounded
// times a power of two, which is taken out of the sum at the end; nothing is rounded but ds
// itself.  The power comes from a bound that holds without a look at the products: out is a
// mean of v's rows, so |do_i.v_j - do_i.out_i| <= 2 |do_i| max |v_j|.  dq takes it of each
// row, dk and dv of all rows of the key head.  The norms of v's rows are a launch of their
// own; those of do come with dq.  bf16 has the range and takes none of this.  (Backward of
// 4 x 2048, 32 heads: 571 us, 543 us without; 8 x 1536, 12 heads of 64: 252 us, 238 us; with
// the largest of the products themselves, looked for at every step, 615 us and 297 us.)
template <class T> constexpr bool kRanged = __is_same(T, f16);
constexpr float kNorm = 0x1p20f;  // over any norm of finite fp16; of others nothing is asked
// The largest norms: of v's rows [B, Hk, tiles], of do's by 32 rows [B, H, groups].
__device__ __forceinline__ float* v_norms(const KgsAttention& a) {
  return a.delta + static_cast<int64_t>(a.B) * a.H * ((a.S + 31) / 32) * 64;
}
__device__ __forceinline__ float* do_norms(const KgsAttention& a) {
  return v_norms(a) + static_cast<int64_t>(a.B) * a.Hk * ((a.S + kRows - 1) / kRows);
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x = fmaxf(x, __shfl_xor(x, m, 64));
  return x;
}
// The largest of n floats and 0, in every lane; eight loads a lane under way.
__device__ __forceinline__ float largest(const float* p, int64_t n, int lane) {
  float x = 0.f;
  for (int64_t i = lane; i < n + lane; i += 64 * 8) {
    float y[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) y[u] = p[min(i + u * 64, n - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u) x = fmaxf(x, y[u]);
  }
  return wave_max(x);
}
// The power of two that brings the bound to between 2^14 and 2^15 (1 % for rounding).
__device__ __forceinline__ float power(float norm_do, float norm_v) {
  return ldexpf(1.f, 15 - __builtin_amdgcn_frexp_expf(2.02f * norm_do * norm_v));
}

// Probabilities of fp16 too are rounded times a power of two, a constant: forward the largest
// of a row may have 2^8 times the subtracted maximum's (a lag that is explained there) and
// is 2^14 then; backward a probability is at most 1, and 16 where scores of 2^26 leave their
// difference from lse no better.  Below 2^-14 rounding is coarser than 11 bits: that is 2^-20
// of a row's largest forward, 2^-26 backward.
template <class T> constexpr float kUpForward = kRanged<T> ? 6.f : 0.f;
template <class T> constexpr float kUpBackward = kRanged<T> ? 12.f : 0.f;

// Of 128 rows of v the largest norm.
template <class T, int D> __global__ __launch_bounds__(kThreads) void attention_norms_kernel(KgsAttention a) {
  constexpr int kLanes = D / 8, kAtOnce = kThreads / kLanes;
  __shared__ float most[NW];
  const int tiles = (a.S + kRows - 1) / kRows, tile = blockIdx.x % tiles, bh = blockIdx.x / tiles;
  const int hk = bh % a.Hk, b = bh / a.Hk, n = length_of(a, b), lane = threadIdx.x & 63;
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < kRows / kAtOnce; ++i) {
    const int row = tile * kRows + i * kAtOnce + threadIdx.x / kLanes;
    float sq = 0.f;
    if (row < n) {
      const typename El<T>::x8 x = *reinterpret_cast<const typename El<T>::x8*>(
          at<T>(a.v, a.v_st, b, row, hk) + threadIdx.x % kLanes * 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(static_cast<float>(x[j]), static_cast<float>(x[j]), sq);
    }
#pragma unroll
    for (int s = 1; s < kLanes; s <<= 1) sq += __shfl_xor(sq, s, 64);
    m = fmaxf(m, sq);
  }
  m = wave_max(m);
  if (lane == 0) most[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < NW; ++i) m = fmaxf(m, most[i]);
    v_norms(a)[blockIdx.x] = fminf(sqrtf(m), kNorm);
  }
}

template <class T, int D, bool CAUSAL>
__global__ __launch_bounds__(kThreads, 2) void attention_fwd_kernel(KgsAttention a) {
  using E = El<T>;
  using Tl = Tile<D>;
  constexpr int kTile = kStep * Tl::kRow;
  __shared__ __attribute__((aligned(1024))) char smem[2 * 2 * kTile];  // a step in work, one under way
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (a.S + kRows - 1) / kRows;
  int bh, rank;
  if (!head_item(blockIdx.x, a.B * a.H, tiles, CAUSAL ? 16 : 1, a.lengths != nullptr, bh, rank)) return;
  const int tile = tiles - 1 - rank;  // causal: the long rows first
  const int h = bh % a.H, b = bh / a.H, hk = h / (a.H / a.Hk);
  const int n = length_of(a, b);
  const int q0 = tile * kRows, qw = q0 + wave * 32, row = qw + (lane & 31);

  typename E::x8 q[D / 16];
  const i32x4 dq = buffer(at<T>(a.q, a.q_st, b, qw, h), span<T, D>(n, qw, a.q_st[1]));
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    q[kk] = load16<typename E::x8>(dq, static_cast<int>((lane & 31) * a.q_st[1] * 2) + (kk * 2 + (lane >> 5)) * 16);

  const int end = CAUSAL ? min(n, q0 + kRows) : n;          // keys any row of the workgroup sees
  const int limit = CAUSAL ? min(row + 1, n) : n;           // keys this lane's row sees
  const int open = CAUSAL ? min(qw + 1, n) : n;             // keys that all rows of the wave see
  const int last = CAUSAL ? min(qw + 32, n) : n;            // keys that any row of the wave sees
  const int steps = q0 < n ? (end + kStep - 1) / kStep : 0;

  // The step after the one in work is under way.  Past the last key the descriptors are
  // empty: the copies leave zeros.
  using Cp = typename Tl::template Copy<kStep, NW>;
  Cp ck, cv;
  ck.init(wave, lane, a.k_st[1] * 2);
  cv.init(wave, lane, a.v_st[1] * 2);
  const uint32_t lds = lds_address(smem);
  Walk wk(at<T>(a.k, a.k_st, b, 0, hk), span<T, D>(n, 0, a.k_st[1]));
  Walk wv(at<T>(a.v, a.v_st, b, 0, hk), span<T, D>(n, 0, a.v_st[1]));
  auto fetch = [&](int slot) {  // the next step
    ck.go(wk.descriptor(), lds + slot * 2 * kTile, wave);
    cv.go(wv.descriptor(), lds + slot * 2 * kTile + kTile, wave);
    wk.go(kStep * 2 * a.k_st[1]);
    wv.go(kStep * 2 * a.v_st[1]);
  };

  f32x16 o[D / 32] = {};
  float top = -0x1.fffffep127f, sum = 0.f;  // finite: a power of a difference of infinities is none
  const float c = a.scale * kLog2e;
  if (steps > 0) fetch(0);
  loads_done();
  int slot = 0;
  for (int j = 0; j < steps; ++j) {
    copies_done();
    barrier();  // step j has landed for every wave, and nobody reads the slot before it any more
    fetch(slot ^ 1);
    const int s0 = j * kStep;
    const char* kt = smem + slot * 2 * kTile;
    const char* vt = kt + kTile;
    slot ^= 1;
    if (s0 >= last) continue;
    f32x16 s[2] = {};
    {
      typename E::x8 f[2][2];  // read one step ahead of the products
      auto read = [&](int kk) {
#pragma unroll
        for (int t = 0; t < 2; ++t) f[kk & 1][t] = Tl::template rows<T>(kt, t * 32, kk, lane);
      };
      read(0);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        if (kk + 1 < D / 16) read(kk + 1);
        in_order();
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = E::mfma(f[kk & 1][t], q[kk], s[t]);
        in_order();
      }
    }
    if (s0 + kStep > open) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (s0 + t * 32 + acc_row(r, lane) >= limit) s[t][r] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[t][r]);
    mx *= c;
    // The subtracted maximum may lag by a factor of 2^8: the quotient is the same, and
    // the accumulators are rescaled a few times a row instead of at every step.  Until then
    // each half of the lanes looks at its own keys only (1 x 16384, 8 heads: 560 us to 538 us).
    if (__any(mx > top + 8.f)) {
      const float now = fmaxf(top, fmaxf(mx, other_half(mx))), f = __builtin_amdgcn_exp2f(top - now);
      top = now;
      sum *= f;
#pragma unroll
      for (int t = 0; t < D / 32; ++t) o[t] *= f;
    }
    const float base = top - kUpForward<T>;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[t][r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], c, -base));
        sum += s[t][r];
      }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const typename E::x8 p = operand<T>(s[t], hh);
#pragma unroll
        for (int e = 0; e < D / 32; ++e)
          o[e] = E::mfma(Tl::template columns<T>(vt, t * 32 + hh * 16, e * 32, lane), p, o[e]);
      }
  }
  copies_done();
  barrier();  // the tiles are read; their place is used for the results' way out
  char* const own = smem + wave * 32 * Tl::kRow;
  sum += other_half(sum);
  if (row >= n) sum = 0.f;
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // a NaN stays one
  if (row >= n)
#pragma unroll
    for (int t = 0; t < D / 32; ++t) o[t] = f32x16{};
  store_rows<T, D>(o, inv, own, const_cast<char*>(at<T>(a.out, a.o_st, b, qw, h)), a.o_st[1], a.S - qw, lane);
  if (a.low)
    store_low<T, D>(o, inv, own, a.low + ((static_cast<int64_t>(b) * a.S + qw) * a.H + h) * D, static_cast<int64_t>(a.H) * D,
                    a.S - qw, lane);
  if (a.lse && lane < 32 && row < a.S)
    a.lse[(static_cast<int64_t>(b) * a.H + h) * a.S + row] = row < n ? top - kUpForward<T> + __builtin_amdgcn_logf(sum) : -INFINITY;
}

// dq of 128 rows a workgroup, and delta of those rows for the kernel that follows.
template <class T, int D, bool CAUSAL>
__global__ __launch_bounds__(kThreads, 2) void attention_dq_kernel(KgsAttention a) {
  using E = El<T>;
  using Tl = Tile<D>;
  constexpr int kTile = kStep * Tl::kRow;
  __shared__ __attribute__((aligned(1024))) char smem[2 * 2 * kTile];  // a step in work, one under way
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (a.S + kRows - 1) / kRows;
  int bh, rank;
  if (!head_item(blockIdx.x, a.B * a.H, tiles, CAUSAL ? 16 : 1, a.lengths != nullptr, bh, rank)) return;
  const int tile = tiles - 1 - rank;
  const int h = bh % a.H, b = bh / a.H, hk = h / (a.H / a.Hk);
  const int n = length_of(a, b);
  const int q0 = tile * kRows, qw = q0 + wave * 32, row = qw + (lane & 31);

  typename E::x8 q[D / 16], g[D / 16];
  float delta = 0.f, norm = 0.f;
  {
    const i32x4 dq = buffer(at<T>(a.q, a.q_st, b, qw, h), span<T, D>(n, qw, a.q_st[1]));
    const i32x4 dg = buffer(at<T>(a.dout, a.g_st, b, qw, h), span<T, D>(n, qw, a.g_st[1]));
    const i32x4 dO = buffer(at<T>(a.out, a.o_st, b, qw, h), span<T, D>(n, qw, a.o_st[1]));
    const int r = lane & 31, cb = (lane >> 5) * 16;
    const i32x4 dl = buffer(a.low + ((static_cast<int64_t>(b) * a.S + qw) * a.H + h) * D,
                            n > qw ? (static_cast<int64_t>(n - 1 - qw) * a.H + 1) * D : 0);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      q[kk] = load16<typename E::x8>(dq, static_cast<int>(r * a.q_st[1] * 2) + kk * 32 + cb);
      g[kk] = load16<typename E::x8>(dg, static_cast<int>(r * a.g_st[1] * 2) + kk * 32 + cb);
      const typename E::x8 o = load16<typename E::x8>(dO, static_cast<int>(r * a.o_st[1] * 2) + kk * 32 + cb);
      const u32x2 low = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_raw_buffer_load_b64(rsrc(dl), r * a.H * D + kk * 16 + (lane >> 5) * 8, 0, 0));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int rest = static_cast<int8_t>(low[j >> 2] >> (8 * (j & 3)));
        delta = fmaf(static_cast<float>(g[kk][j]), with_low<T>(o[j], rest), delta);
        if constexpr (kRanged<T>) norm = fmaf(static_cast<float>(g[kk][j]), static_cast<float>(g[kk][j]), norm);
      }
    }
    delta += other_half(delta);
    norm += other_half(norm);
  }
  const float lse = row < n ? a.lse[(static_cast<int64_t>(b) * a.H + h) * a.S + row] : 0.f;

  const int end = CAUSAL ? min(n, q0 + kRows) : n;
  const int limit = CAUSAL ? min(row + 1, n) : n;
  const int open = CAUSAL ? min(qw + 1, n) : n;
  const int last = CAUSAL ? min(qw + 32, n) : n;
  const int steps = q0 < n ? (end + kStep - 1) / kStep : 0;

  // The step after the one in work is under way.  Past the last key the descriptors are
  // empty: the copies leave zeros.
  using Cp = typename Tl::template Copy<kStep, NW>;
  Cp ck, cv;
  ck.init(wave, lane, a.k_st[1] * 2);
  cv.init(wave, lane, a.v_st[1] * 2);
  const uint32_t lds = lds_address(smem);
  Walk wk(at<T>(a.k, a.k_st, b, 0, hk), span<T, D>(n, 0, a.k_st[1]));
  Walk wv(at<T>(a.v, a.v_st, b, 0, hk), span<T, D>(n, 0, a.v_st[1]));
  auto fetch = [&](int slot) {  // the next step
    ck.go(wk.descriptor(), lds + slot * 2 * kTile, wave);
    cv.go(wv.descriptor(), lds + slot * 2 * kTile + kTile, wave);
    wk.go(kStep * 2 * a.k_st[1]);
    wv.go(kStep * 2 * a.v_st[1]);
  };

  f32x16 acc[D / 32] = {};
  const float c = a.scale * kLog2e;
  if (steps > 0) fetch(0);
  float f = 1.f;
  const int groups = (a.S + 31) / 32, group = qw / 32;
  if constexpr (kRanged<T>) {
    norm = fminf(sqrtf(norm), kNorm);
    f = power(norm, largest(v_norms(a) + (static_cast<int64_t>(b) * a.Hk + hk) * tiles, tiles, lane));
    const float most = wave_max(norm);
    if (lane == 0 && group < groups) do_norms(a)[(static_cast<int64_t>(b) * a.H + h) * groups + group] = most;
  }
  loads_done();
  int slot = 0;
  for (int j = 0; j < steps; ++j) {
    copies_done();
    barrier();
    fetch(slot ^ 1);
    const int s0 = j * kStep;
    const char* kt = smem + slot * 2 * kTile;
    const char* vt = kt + kTile;
    slot ^= 1;
    if (s0 >= last) continue;
    // s and do.v of 32 keys
    const auto scores = [&](int t, f32x16& s, f32x16& dp) {
      s = dp = f32x16{};
      typename E::x8 f[2][2];
      auto read = [&](int kk) {
        f[kk & 1][0] = Tl::template rows<T>(kt, t * 32, kk, lane);
        f[kk & 1][1] = Tl::template rows<T>(vt, t * 32, kk, lane);
      };
      read(0);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        if (kk + 1 < D / 16) read(kk + 1);
        in_order();
        s = E::mfma(f[kk & 1][0], q[kk], s);
        dp = E::mfma(f[kk & 1][1], g[kk], dp);
        in_order();
      }
    };
    if (last <= kStep) {
      // The only step of these rows: delta as sum p (do.v).  Few keys have large p, whose
      // rounding in the forward pass would show in delta = do.o.
      delta = 0.f;
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        f32x16 s, dp;
        scores(t, s, dp);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          delta += s0 + t * 32 + acc_row(r, lane) < limit ? __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) * dp[r] : 0.f;
      }
      delta += other_half(delta);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (t && s0 + 32 >= last) break;  // no row sees the second half (16 x 500: 59 us to 58.3 us)
      f32x16 s, dp;
      scores(t, s, dp);
      const bool edge = s0 + t * 32 + 32 > open;
      const float d = delta * f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse));
        s[r] = p * (kRanged<T> ? fmaf(dp[r], f, -d) : dp[r] - delta);
      }
      if (edge) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (s0 + t * 32 + acc_row(r, lane) >= limit) s[r] = 0.f;
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const typename E::x8 ds = operand<T>(s, hh);
#pragma unroll
        for (int e = 0; e < D / 32; ++e)
          acc[e] = E::mfma(Tl::template columns<T>(kt, t * 32 + hh * 16, e * 32, lane), ds, acc[e]);
      }
    }
  }
  copies_done();
  barrier();
  // For dk, dv: the 32 rows' lse (less the power that probabilities are rounded with), then
  // their delta, side by side.  Rows past the end get zeros: with zeros for q and do they are
  // p = 1 times zero there.
  if (group < groups)
    a.delta[(static_cast<int64_t>(b * a.H + h) * groups + group) * 64 + lane] =
        row >= n ? 0.f : lane < 32 ? lse - kUpBackward<T> : delta;
  if constexpr (kRanged<T>) {
#pragma unroll
    for (int t = 0; t < D / 32; ++t) acc[t] *= 1.f / f;
  }
  if (row >= n)
#pragma unroll
    for (int t = 0; t < D / 32; ++t) acc[t] = f32x16{};
  store_rows<T, D>(acc, a.scale, smem + wave * 32 * Tl::kRow, const_cast<char*>(at<T>(a.dq, a.dq_st, b, qw, h)), a.dq_st[1], a.S - qw, lane);
}

// dk and dv of 128 keys a workgroup: walks the query heads that share the key head, and
// of each the rows that see the keys, 32 at a time.  No atomics: the order of the sums
// is fixed.  v's fragments are read from LDS again at every step: with k's, both
// accumulators and v's in registers a SIMD would hold one wave instead of two.
// With splits > 1 a workgroup takes one part of the walk and leaves its sums, 32 bits,
// in the workspace.
template <class T, int D, bool CAUSAL>
__global__ __launch_bounds__(kThreads, 2) void attention_dkv_kernel(KgsAttention a) {
  using E = El<T>;
  using Tl = Tile<D>;
  // a step: q, do, and lse and delta of its rows
  constexpr int kQ = kQStep, kTile = kQ * Tl::kRow, kV = kRows * Tl::kRow, kStage = 2 * kTile + 256;
  __shared__ __attribute__((aligned(1024))) char smem[kV + 2 * kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (a.S + kRows - 1) / kRows;
  int bh, rank;
  if (!head_item(blockIdx.x, a.B * a.Hk, tiles * a.splits, CAUSAL ? 16 : 1, a.lengths != nullptr, bh, rank)) return;
  const int split = rank % a.splits, tile = rank / a.splits;  // causal: the first keys have the most rows
  const int hk = bh % a.Hk, b = bh / a.Hk, G = a.H / a.Hk;
  const int n = length_of(a, b);
  const int k0 = tile * kRows, kw = k0 + wave * 32, key = kw + (lane & 31);

  // v's tile; rows past the end are zero
  const uint32_t lds = lds_address(smem);
  {
    typename Tl::template Copy<kRows, NW> cv;
    cv.init(wave, lane, a.v_st[1] * 2);
    cv.go(buffer(at<T>(a.v, a.v_st, b, k0, hk), span<T, D>(n, k0, a.v_st[1])), lds, wave);
  }
  typename E::x8 k[D / 16];
  const i32x4 dk = buffer(at<T>(a.k, a.k_st, b, kw, hk), span<T, D>(n, kw, a.k_st[1]));
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    k[kk] = load16<typename E::x8>(dk, static_cast<int>((lane & 31) * a.k_st[1] * 2) + (kk * 2 + (lane >> 5)) * 16);

  float f = 1.f;
  if constexpr (kRanged<T>) {
    // (a quarter a wave: where 64 heads share one they are 32768 for 16384 positions)
    __shared__ float most[NW];
    const int64_t all_rows = static_cast<int64_t>(G) * ((a.S + 31) / 32), quarter = (all_rows + NW - 1) / NW;
    const float m = largest(do_norms(a) + (static_cast<int64_t>(b) * a.Hk + hk) * all_rows + wave * quarter,
                            min(quarter, all_rows - wave * quarter), lane);
    if (lane == 0) most[wave] = m;
    barrier();
    f = power(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])),
              largest(v_norms(a) + (static_cast<int64_t>(b) * a.Hk + hk) * tiles, tiles, lane));
    f = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, f)));  // a scalar register
  }
  const int first = CAUSAL ? k0 / kQ : 0;                                 // first step of rows
  const int each = k0 < n ? (n + kQ - 1) / kQ - first : 0;                // steps a head
  const int all = each * G;                                               // the whole walk
  const int lo = static_cast<int>(static_cast<int64_t>(all) * split / a.splits);
  const int hi = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / a.splits);

  using Cp = typename Tl::template Copy<kQ, NW>;
  Cp cq, cg;
  cq.init(wave, lane, a.q_st[1] * 2);
  cg.init(wave, lane, a.g_st[1] * 2);
  // The walk's step that is fetched next: head of the group, step of that head.  Past the
  // end of the walk the descriptors are empty, as in the forward pass.
  int fh = hi > lo ? lo / each : 0, fs = hi > lo ? lo % each : 0, fi = lo;
  const int groups = (a.S + 31) / 32;
  Walk wq, wg, ws;  // q, do, and lse and delta of the rows
  auto head = [&] {
    const int h = hk * G + fh, s = (first + fs) * kQ;
    wq = Walk(at<T>(a.q, a.q_st, b, s, h), span<T, D>(n, s, a.q_st[1]));
    wg = Walk(at<T>(a.dout, a.g_st, b, s, h), span<T, D>(n, s, a.g_st[1]));
    ws = Walk(a.delta + (static_cast<int64_t>(b * a.H + h) * groups + first + fs) * 64, (groups - first - fs) * 256ll);
  };
  if (lo < hi) head();
  auto fetch = [&](int slot) {
    if (fi++ >= hi) wq.left = wg.left = ws.left = 0;
    const uint32_t to = lds + kV + slot * kStage;
    cq.go(wq.descriptor(), to, wave);
    cg.go(wg.descriptor(), to + kTile, wave);
    if (wave == 0) copy4(ws.descriptor(), lane * 4, to + 2 * kTile);
    wq.go(kQ * 2 * a.q_st[1]);
    wg.go(kQ * 2 * a.g_st[1]);
    ws.go(256);
    if (++fs == each) {
      fs = 0;
      if (++fh < G) head();
    }
  };

  f32x16 dka[D / 32] = {}, dva[D / 32] = {};
  const float c = a.scale * kLog2e;
  const float rest = f * 0x1p-12f;  // the probabilities have 2^12 of it
  if (lo < hi) fetch(0);
  loads_done();
  int slot = 0, ss = hi > lo ? lo % each : 0;
  for (int i = lo; i < hi; ++i) {
    copies_done();
    barrier();
    fetch(slot ^ 1);
    const int s0 = (first + ss) * kQ;
    const char* qt = smem + kV + slot * kStage;
    const char* gt = qt + kTile;
    const float* lse = reinterpret_cast<const float*>(gt + kTile);
    slot ^= 1;
    if (++ss == each) ss = 0;
    if (CAUSAL && s0 + kQ <= kw) continue;  // no row of the step sees the wave's keys
    f32x16 s = {}, dp = {};
    {
      typename E::x8 f[2][3];
      auto read = [&](int kk) {
        f[kk & 1][0] = Tl::template rows<T>(qt, 0, kk, lane);
        f[kk & 1][1] = Tl::template rows<T>(gt, 0, kk, lane);
        f[kk & 1][2] = Tl::template rows<T>(smem, wave * 32, kk, lane);
      };
      read(0);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        if (kk + 1 < D / 16) read(kk + 1);
        in_order();
        s = E::mfma(f[kk & 1][0], k[kk], s);
        dp = E::mfma(f[kk & 1][1], f[kk & 1][2], dp);
        in_order();
      }
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const f32x4 l = *reinterpret_cast<const f32x4*>(lse + m * 8 + (lane >> 5) * 4);
      const f32x4 d = *reinterpret_cast<const f32x4*>(lse + 32 + m * 8 + (lane >> 5) * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = m * 4 + j;
        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -l[j]));
        dp[r] = s[r] * (kRanged<T> ? (dp[r] - d[j]) * rest : dp[r] - d[j]);
      }
    }
    if (CAUSAL && s0 < kw + 31) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (s0 + acc_row(r, lane) < key) s[r] = dp[r] = 0.f;
    }
    {
      const typename E::x8 p[2] = {operand<T>(s, 0), operand<T>(s, 1)}, ds[2] = {operand<T>(dp, 0), operand<T>(dp, 1)};
      typename E::x8 f[2][2];
      auto read = [&](int i) {
        f[i & 1][0] = Tl::template columns<T>(gt, i / (D / 32) * 16, i % (D / 32) * 32, lane);
        f[i & 1][1] = Tl::template columns<T>(qt, i / (D / 32) * 16, i % (D / 32) * 32, lane);
      };
      read(0);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const int hh = i / (D / 32), e = i % (D / 32);
        if (i + 1 < D / 16) read(i + 1);
        in_order();
        dva[e] = E::mfma(f[i & 1][0], p[hh], dva[e]);
        dka[e] = E::mfma(f[i & 1][1], ds[hh], dka[e]);
        in_order();
      }
    }
  }
  copies_done();
  if constexpr (kRanged<T>) {
#pragma unroll
    for (int t = 0; t < D / 32; ++t) dka[t] *= 1.f / f, dva[t] *= 0x1p-12f;
  }
  if (a.splits > 1) {
    if (key < n) {  // the join reads no more
      const int64_t part = static_cast<int64_t>(a.B) * a.S * a.Hk * D;
      float* w = a.partial + split * 2 * part + ((static_cast<int64_t>(b) * a.S + key) * a.Hk + hk) * D;
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4 x, y;
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = dka[t][g * 4 + j], y[j] = dva[t][g * 4 + j];
          const int e = t * 32 + g * 8 + (lane >> 5) * 4;
          *reinterpret_cast<f32x4*>(w + e) = x;
          *reinterpret_cast<f32x4*>(w + part + e) = y;
        }
    }
    return;
  }
  if (key >= n)
#pragma unroll
    for (int t = 0; t < D / 32; ++t) dka[t] = dva[t] = f32x16{};
  char* const own = smem + wave * 32 * Tl::kRow;  // the wave's rows of v, which no other reads
  store_rows<T, D>(dka, a.scale, own, const_cast<char*>(at<T>(a.dk, a.dk_st, b, kw, hk)), a.dk_st[1], a.S - kw, lane);
  store_rows<T, D>(dva, 1.f, own, const_cast<char*>(at<T>(a.dv, a.dv_st, b, kw, hk)), a.dv_st[1], a.S - kw, lane);
}

// Adds the parts of a split walk, in their order: 4 elements a thread of dk, then of dv.
template <class T, int D>
__global__ __launch_bounds__(256) void attention_join_kernel(KgsAttention a) {
  using x4 = typename El<T>::x4;
  const int64_t part = static_cast<int64_t>(a.B) * a.S * a.Hk * D;
  const int64_t i = (blockIdx.x * 256ll + threadIdx.x) * 4;  // under 2^28 parts of 4: splits are of few keys
  if (i >= 2 * part) return;
  const bool v = i >= part;
  const int64_t e = v ? i - part : i;
  const int d = static_cast<int>(e % D), hk = static_cast<int>(e / D % a.Hk);
  const int64_t bs = e / D / a.Hk;
  const int s = static_cast<int>(bs % a.S), b = static_cast<int>(bs / a.S);
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (s < (a.lengths ? min(a.lengths[b], a.S) : a.S))
    for (int p = 0; p < a.splits; ++p) sum += *reinterpret_cast<const f32x4*>(a.partial + p * 2 * part + i);
  x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = static_cast<T>(v ? sum[j] : sum[j] * a.scale);
  char* to = const_cast<char*>(v ? at<T>(a.dv, a.dv_st, b, s, hk) : at<T>(a.dk, a.dk_st, b, s, hk));
  *reinterpret_cast<x4*>(to + d * 2) = r;
}

int check(const KgsAttention* a, bool backward) {
  const char* w = "attention";
  if (!a || !a->q || !a->k || !a->v || !a->out) return fail(w, "a tensor is missing");
  if (a->B < 0 || a->S < 0 || a->H <= 0 || a->Hk <= 0 || a->H % a->Hk) return fail(w, "bad sizes");
  if (a->D != 64 && a->D != 128) return fail(w, "head dimension must be 64 or 128");
  if (a->type != 0 && a->type != 1) return fail(w, "type must be bfloat16 or float16");
  if (backward && (!a->dout || !a->lse || !a->low || !a->delta || !a->dq || !a->dk || !a->dv)) return fail(w, "a tensor is missing");
  if (backward && (a->splits < 1 || (a->splits > 1 && !a->partial))) return fail(w, "bad split");
  const int64_t* st[] = {a->q_st, a->k_st, a->v_st, a->o_st, a->g_st, a->dq_st, a->dk_st, a->dv_st};
  for (int i = 0; i < (backward ? 8 : 4); ++i)
    for (int j = 0; j < 3; ++j)
      // rows behind the last lie past the descriptor's end; offsets inside a tile stay under 2^30
      if (st[i][j] < 0 || st[i][j] % 8 || (j == 1 && (st[i][j] < a->D || st[i][j] > (1 << 22)))) return fail(w, "unsupported strides");
  if (a->H > (1 << 18)) return fail(w, "too many heads");  // offsets inside a tile of low
  // a launch has under 2^32 threads; the products of counts that head_item forms, 16 times
  // a head's pieces at most, stay under 2^31 with that
  const int64_t tiles = (a->S + kRows - 1) / kRows, most = (1 << 24) - 8;
  if (a->B * static_cast<int64_t>(a->H) * tiles > most || (backward && a->B * static_cast<int64_t>(a->Hk) * tiles * a->splits > most))
    return fail(w, "too many workgroups");
  return 0;
}

template <class T, int D, bool CAUSAL> int forward(const KgsAttention& a, hipStream_t s) {
  const int64_t tiles = (a.S + kRows - 1) / kRows;
  attention_fwd_kernel<T, D, CAUSAL><<<static_cast<unsigned>(head_items(a.B * static_cast<int64_t>(a.H), tiles, a.lengths)), kThreads, 0, s>>>(a);
  return launched("attention forward");
}

template <class T, int D, bool CAUSAL> int backward(const KgsAttention& a, hipStream_t s) {
  const int64_t tiles = (a.S + kRows - 1) / kRows, b = a.B;
  if constexpr (kRanged<T>) {
    attention_norms_kernel<T, D><<<static_cast<unsigned>(b * a.Hk * tiles), kThreads, 0, s>>>(a);
    if (launched("attention norms")) return -1;
  }
  attention_dq_kernel<T, D, CAUSAL><<<static_cast<unsigned>(head_items(b * a.H, tiles, a.lengths)), kThreads, 0, s>>>(a);
  if (launched("attention dq")) return -1;
  attention_dkv_kernel<T, D, CAUSAL><<<static_cast<unsigned>(head_items(b * a.Hk, tiles * a.splits, a.lengths)), kThreads, 0, s>>>(a);
  if (launched("attention dk, dv")) return -1;
  if (a.splits > 1) {
    const int64_t n = 2 * b * a.S * a.Hk * D / 4;
    attention_join_kernel<T, D><<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(a);
    return launched("attention join");
  }
  return 0;
}

template <class T, int D> int run(const KgsAttention& a, bool back, hipStream_t s) {
  if (back) return a.causal ? backward<T, D, true>(a, s) : backward<T, D, false>(a, s);
  return a.causal ? forward<T, D, true>(a, s) : forward<T, D, false>(a, s);
}

int dispatch(const KgsAttention* a, bool back, void* stream) {
  if (check(a, back)) return -1;
  if (a->B == 0 || a->S == 0) return 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->type == 0) return a->D == 64 ? run<bf16, 64>(*a, back, s) : run<bf16, 128>(*a, back, s);
  return a->D == 64 ? run<f16, 64>(*a, back, s) : run<f16, 128>(*a, back, s);
}

}  // namespace
}  // namespace kgs

extern "C" {
int kgs_attention_fwd(const KgsAttention* a, void* stream) { return kgs::dispatch(a, false, stream); }
int kgs_attention_bwd(const KgsAttention* a, void* stream) { return kgs::dispatch(a, true, stream); }
}
