// The gated half of a feed-forward block, forward and backward, for gfx950.
//
//   g = x Wg^T, u = x Wu^T, h = silu(g) u            x [T, K], W = [Wg; Wu] [2F, K]
//   dg = dh u silu'(g), du = dh silu(g)
//   dx = dg Wg + du Wu = [dg du] W,   dW = [dg du]^T x
//
// One matrix product kernel serves the three products.  A workgroup's tile of the
// forward product takes the same columns of Wg and Wu, so that a wave holds g and u of
// the same elements and the activation and the product are its epilogue: h is written
// once, and g and u only if a backward pass will want them.
//
// Tiles of both operands go from memory straight to LDS, two steps of 64 of the summed
// index deep, as they lie in memory; an operand whose summed index is not the
// contiguous one is transposed by the LDS read.  Accumulators are 32 bits; g and u are
// saved with 24 of them: rounded to 16 they would add as much error to dx and dw as the
// rounding of dg and du, operands of the two products, which is not to be avoided, and
// 32 cost a third more traffic.  Rounded besides those: the outputs.
//
// Bound by the matrix units (busy 56 % of the time, at the clock the power limit leaves),
// by memory for few rows.  8192 x 4096, F = 11008, bf16: forward 1230 us (1200 TFLOP/s),
// saving the projections 1320 us, dx 1290 us (1140), dW 1500 us (980: both operands read
// transposed take about as many cycles at a lower clock), dg and du 205 us (5.3 TB/s).
// 5 rows of the same, weights from memory: 38 us (4.8 TB/s), two launches.
#include "decoder.h"
#include "decoder_common.h"

namespace kgs {
namespace {

constexpr int kK = 64;  // summed index a step

struct Product {
  const void *a, *b;   // a: [M, K] or, transposed, [K, M]; b: [N, K] or, transposed, [K, N]
  int64_t a_ld, b_ld;  // elements
  void* c;             // [M, N] contiguous (pairs: [M, N / 2])
  uint8_t* saved;      // [M, 3 N] (Saved) or null
  float* partial;      // splits > 1: [splits, M, N]
  int M, N, K, splits;
};

// One operand's tile of ROWS indexes by kK of the sum, and its fragments.
template <class T, int ROWS, bool TR, int NW> struct Operand;

template <class T, int ROWS, int NW> struct Operand<T, ROWS, false, NW> {
  using Tl = Tile<kK>;
  using Cp = typename Tl::template Copy<ROWS, NW>;
  static constexpr int kBytes = ROWS * kK * 2;
  Cp copy;
  i32x4 d;
  int k0, K;
  // rows r0.. (rows - r0 of them), sum indexes from k of K.  The descriptor is that of the
  // whole rows and stands; the sum index is the scalar offset.  Whether that is part of
  // the range check or not, rows past the last are out of range and the others in it.
  __device__ __forceinline__ void init(const void* p, int64_t ld, int r0, int rows, int k, int sum, int wave, int lane) {
    copy.init(wave, lane, ld * 2);
    d = buffer(static_cast<const T*>(p) + r0 * ld, rows > r0 ? ((rows - 1 - r0) * ld + sum) * 2 : 0);
    k0 = k;
    K = sum;
  }
  // the next kK of the sum; chunks past K are read as zero
  __device__ __forceinline__ void go(uint32_t lds, int wave, int lane) {
    const int k = k0;
    k0 += kK;
    if (k0 <= K) return copy.go(d, lds, wave, k * 2);
#pragma unroll
    for (int i = 0; i < Cp::kN; ++i) {
      const int byte = (wave * Cp::kN + i) * 1024 + lane * 16, row = byte / Tl::kRow;
      const int chunk = ((byte >> 4) & 7) ^ Tl::swizzle(row);
      if (Cp::kAll % NW == 0 || wave * Cp::kN + i < Cp::kAll)
        copy16(d, k + chunk * 8 < K ? copy.voff[i] : static_cast<int>(kFar), lds + (wave * Cp::kN + i) * 1024, k * 2);
    }
  }
  static __device__ __forceinline__ typename El<T>::x8 read(const char* t, int r0, int kk, int lane) {
    return Tl::template rows<T>(t, r0, kk, lane);
  }
};

template <class T, int ROWS, int NW> struct Operand<T, ROWS, true, NW> {
  static constexpr int W = ROWS >= 128 ? 128 : 64, kSub = ROWS / W, kSubBytes = kK * W * 2;
  using Tl = Tile<W>;
  using Cp = typename Tl::template Copy<kK, NW>;
  static constexpr int kBytes = kSub * kSubBytes;
  Cp copy;
  Walk walk[kSub];
  int64_t step;
  __device__ __forceinline__ void init(const void* p, int64_t ld, int r0, int rows, int k, int sum, int wave, int lane) {
    copy.init(wave, lane, ld * 2);
    step = kK * ld * 2;
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      const int r = r0 + s * W;
      walk[s] = Walk(static_cast<const T*>(p) + k * ld + r, rows > r ? ((sum - 1 - k) * ld + (rows - r)) * 2 : 0);
    }
  }
  __device__ __forceinline__ void go(uint32_t lds, int wave, int) {
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      copy.go(walk[s].descriptor(), lds + s * kSubBytes, wave);
      walk[s].go(step);
    }
  }
  static __device__ __forceinline__ typename El<T>::x8 read(const char* t, int r0, int kk, int lane) {
    return Tl::template columns_in_order<T>(t + r0 / W * kSubBytes, kk * 16, r0 % W, lane);
  }
};

// A row of n saved values: their upper 16 bits, then the 8 below, rounded.
struct Saved {
  uint8_t* row;
  int n;
  __device__ __forceinline__ Saved(uint8_t* base, int64_t m, int n) : row(base + m * 3 * n), n(n) {}
  __device__ __forceinline__ uint16_t* high(int i) const { return reinterpret_cast<uint16_t*>(row) + i; }
  __device__ __forceinline__ uint8_t* low(int i) const { return row + 2 * static_cast<int64_t>(n) + i; }
  // 4 values from i, a multiple of 4
  __device__ __forceinline__ f32x4 load(int i) const {
    const u32x2 h = *reinterpret_cast<const u32x2*>(high(i));
    const uint32_t l = *reinterpret_cast<const uint32_t*>(low(i));
    f32x4 x;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      x[j] = __builtin_bit_cast(float, ((h[j >> 1] >> (16 * (j & 1))) << 16) | (((l >> (8 * j)) & 0xFF) << 8));
    return x;
  }
  static __device__ __forceinline__ void split(f32x4 x, u32x2& h, uint32_t& l) {
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float e = x[j];  // (of an element itself, bit_cast takes the first)
      const uint32_t v = __builtin_bit_cast(uint32_t, e);
      // half a step up; not across the exponent of infinities and NaNs, whose payload stays above
      b[j] = (v & 0x7F800000u) == 0x7F800000u ? v : v + 0x80u;
    }
    h[0] = __builtin_amdgcn_perm(b[1], b[0], 0x07060302);
    h[1] = __builtin_amdgcn_perm(b[3], b[2], 0x07060302);
    l = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0501) | (__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0501) << 16);
  }
  __device__ __forceinline__ void store(int i, f32x4 x) const {
    u32x2 h;
    uint32_t l;
    split(x, h, l);
    *reinterpret_cast<u32x2*>(high(i)) = h;
    *reinterpret_cast<uint32_t*>(low(i)) = l;
  }
};

// silu(g) = g / (1 + 2^(-g log2 e)): an overflowing power makes the quotient 0.
__device__ __forceinline__ float sigmoid(float g) { return 1.f / (1.f + __builtin_amdgcn_exp2f(-g * kLog2e)); }

__device__ __forceinline__ f32x4 quarter(const f32x16& x, int g) {
  return f32x4{x[g * 4], x[g * 4 + 1], x[g * 4 + 2], x[g * 4 + 3]};
}

// c = a b over tiles of BM x BN, WM x WN waves.  PAIR: the columns of a tile are BN / 2
// of the first half of N and the same of the second.
template <class T, int BM, int BN, int WM, int WN, bool TA, bool TB, bool PAIR>
__global__ __launch_bounds__(WM * WN * 64, 2) void product_kernel(Product p) {
  using E = El<T>;
  constexpr int NW = WM * WN, MT = BM / WM / 32, NT = BN / WN / 32, HALF = BN / 2;
  using OA = Operand<T, BM, TA, NW>;
  using OB = Operand<T, PAIR ? HALF : BN, TB, NW>;
  constexpr int kB = PAIR ? 2 * OB::kBytes : OB::kBytes, kStage = OA::kBytes + kB;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int N = PAIR ? p.N / 2 : p.N;  // columns of c
  const int tm = (p.M + BM - 1) / BM, tn = (N + (PAIR ? HALF : BN) - 1) / (PAIR ? HALF : BN);
  const int64_t total = static_cast<int64_t>(tm) * tn * p.splits;
  const int64_t item = xcd_item(blockIdx.x, total);
  if ((blockIdx.x >> 3) >= (total + 7) / 8 || item >= total) return;
  // Items in bands of 4 tiles of rows: the workgroups of an XCD share 4 row tiles and few
  // column tiles through their L2.
  const int split = static_cast<int>(item / (static_cast<int64_t>(tm) * tn));
  const int t = static_cast<int>(item % (static_cast<int64_t>(tm) * tn));
  const int band = t / (4 * tn), high = min(4, tm - band * 4), in = t - band * 4 * tn;
  const int m0 = (band * 4 + in % high) * BM, n0 = in / high * (PAIR ? HALF : BN);
  const int steps_all = (p.K + kK - 1) / kK;
  const int lo = static_cast<int>(static_cast<int64_t>(steps_all) * split / p.splits);
  const int hi = static_cast<int>(static_cast<int64_t>(steps_all) * (split + 1) / p.splits);

  OA oa;
  OB ob, ou;  // ou: the columns of the second half
  oa.init(p.a, p.a_ld, m0, p.M, lo * kK, p.K, wave, lane);
  ob.init(p.b, p.b_ld, n0, N, lo * kK, p.K, wave, lane);
  if (PAIR) ou.init(static_cast<const T*>(p.b) + N * p.b_ld, p.b_ld, n0, N, lo * kK, p.K, wave, lane);
  const uint32_t lds = lds_address(smem);
  auto fetch = [&](int j) {
    const uint32_t to = lds + (j & 1) * kStage;
    oa.go(to, wave, lane);
    ob.go(to + OA::kBytes, wave, lane);
    if (PAIR) ou.go(to + OA::kBytes + OB::kBytes, wave, lane);
  };

  // The fragments of a sixteenth of the sum, read while the products of the one before
  // run: without that order, which the compiler would undo, a wave waits for LDS before
  // every other product.
  typename E::x8 fa[2][MT], fb[2][NT];
  auto read = [&](int j, int kk, int into) {
    const char* at = smem + (j & 1) * kStage;
    const char* bt = at + OA::kBytes;
#pragma unroll
    for (int i = 0; i < NT; ++i)
      fb[into][i] = PAIR ? OB::read(bt + (i < NT / 2 ? 0 : OB::kBytes), wn * NT * 16 + i % (NT / 2 ? NT / 2 : 1) * 32, kk, lane)
                         : OB::read(bt, wn * NT * 32 + i * 32, kk, lane);
#pragma unroll
    for (int i = 0; i < MT; ++i) fa[into][i] = OA::read(at, wm * MT * 32 + i * 32, kk, lane);
  };
  f32x16 acc[MT][NT] = {};
  auto multiply = [&](int from) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int k = 0; k < NT; ++k) acc[i][k] = E::mfma(fb[from][k], fa[from][i], acc[i][k]);
    __builtin_amdgcn_sched_barrier(0);
  };
  if (lo < hi) {
    fetch(lo);
    copies_done();
    barrier();
    if (lo + 1 < hi) fetch(lo + 1);
    read(lo, 0, 0);
    for (int j = lo; j < hi; ++j) {
#pragma unroll
      for (int kk = 0; kk + 1 < kK / 16; ++kk) {
        read(j, kk + 1, (kk + 1) & 1);
        multiply(kk & 1);
      }
      if (j + 1 < hi) {
        copies_done();
        barrier();  // step j + 1 has landed for every wave, and everyone has read step j
        if (j + 2 < hi) fetch(j + 2);
        read(j + 1, 0, 0);
      }
      multiply(1);
    }
  }

  // Lane % 32 = row of c, registers = columns, 4 in a row each.  A split's parts go out as
  // they lie; results by way of LDS, which the wave leaves in whole stretches of rows.
  constexpr int CT = PAIR ? NT / 2 : NT, W = CT * 32;  // a wave's columns of c
  const int nw = n0 + wn * W;
  if (p.splits > 1) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = m0 + wm * MT * 32 + i * 32 + (lane & 31);
      if (m >= p.M) continue;
#pragma unroll
      for (int k = 0; k < CT; ++k)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int n = nw + k * 32 + g * 8 + (lane >> 5) * 4;
          if (n >= N) continue;  // N is a multiple of 8
          float* to = p.partial + (static_cast<int64_t>(split) * p.M + m) * p.N + n;
          *reinterpret_cast<f32x4*>(to) = quarter(acc[i][k], g);
          if (PAIR) *reinterpret_cast<f32x4*>(to + N) = quarter(acc[i][(CT + k) % NT], g);
        }
    }
    return;
  }
  barrier();  // everyone has read the last step
  constexpr int kRow = W * 2, kRows = 64 * 16 / kRow, kArea = 32 * kRow;  // bytes a row, rows a store
  char* const own = smem + wave * (PAIR ? 4 : 1) * kArea;
  const int row = lane & 31, half = lane >> 5;
  // 16-byte chunk c of row r; 8 (or 4) rows lie side by side in the banks
  const auto place = [](int r, int c) { return r * kRow + ((c ^ ((r >> (W == 128 ? 0 : W == 64 ? 1 : 2)) & (W / 8 - 1))) << 4); };
  const auto out = [&](const char* from, char* base, int64_t stride, int m, int n) {
#pragma unroll
    for (int i = 0; i < 32 / kRows; ++i) {
      const int r = i * kRows + lane / (W / 8), c = lane % (W / 8);
      const i32x4 v = *reinterpret_cast<const i32x4*>(from + place(r, c));
      if (m + r < p.M && n + c * 8 < N) *reinterpret_cast<i32x4*>(base + (m + r) * stride + (n + c * 8) * 2) = v;
    }
  };
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + wm * MT * 32 + i * 32;
#pragma unroll
    for (int k = 0; k < CT; ++k)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 x = quarter(acc[i][k], g);
        f32x4 c = x;
        const int at = place(row, k * 4 + g) + half * 8;
        if constexpr (PAIR) {
          const f32x4 y = quarter(acc[i][(CT + k) % NT], g);
#pragma unroll
          for (int j = 0; j < 4; ++j) c[j] = x[j] * sigmoid(x[j]) * y[j];
          if (p.saved) {
            u32x2 h;
            uint32_t l;
            Saved::split(x, h, l);
            *reinterpret_cast<u32x2*>(own + kArea + at) = h;
            *reinterpret_cast<uint32_t*>(own + 3 * kArea + at / 2) = l;
            Saved::split(y, h, l);
            *reinterpret_cast<u32x2*>(own + 2 * kArea + at) = h;
            *reinterpret_cast<uint32_t*>(own + 3 * kArea + kArea / 2 + at / 2) = l;
          }
        }
        typename E::x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = static_cast<T>(c[j]);
        *reinterpret_cast<typename E::x4*>(own + at) = r;
      }
    wave_order();
    out(own, static_cast<char*>(p.c), static_cast<int64_t>(N) * 2, m, nw);
    if constexpr (PAIR) {
      if (p.saved) {
        const int64_t stride = 3ll * p.N;
        char* const base = reinterpret_cast<char*>(p.saved);
        out(own + kArea, base, stride, m, nw);
        out(own + 2 * kArea, base + 2 * N, stride, m, nw);
        // the low bytes, 8 a lane
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int s = 0; s < 32 / kRows; ++s) {
            const int r = s * kRows + lane / (W / 8), c = lane % (W / 8);
            const u32x2 x = *reinterpret_cast<const u32x2*>(own + 3 * kArea + v * (kArea / 2) + place(r, c) / 2);
            if (m + r < p.M && nw + c * 8 < N)
              *reinterpret_cast<u32x2*>(base + (m + r) * stride + 2 * p.N + v * N + nw + c * 8) = x;
          }
      }
    }
    wave_order();
  }
}

// The parts of a split product, added in their order, 4 columns a thread.
template <class T, bool PAIR> __global__ __launch_bounds__(256) void join_kernel(Product p) {
  using x4 = typename El<T>::x4;
  const int N = PAIR ? p.N / 2 : p.N;
  for (int64_t i = (blockIdx.x * 256ll + threadIdx.x) * 4; i < static_cast<int64_t>(p.M) * N; i += gridDim.x * 1024ll) {
    const int64_t m = i / N, n = i % N, part = static_cast<int64_t>(p.M) * p.N;
    f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
    const float* from = p.partial + m * p.N + n;
    for (int s = 0; s < p.splits; ++s) {
      x += *reinterpret_cast<const f32x4*>(from + s * part);
      if (PAIR) y += *reinterpret_cast<const f32x4*>(from + s * part + N);
    }
    x4 h;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = static_cast<T>(PAIR ? x[j] * sigmoid(x[j]) * y[j] : x[j]);
    *reinterpret_cast<x4*>(static_cast<T*>(p.c) + i) = h;
    if (PAIR && p.saved) {
      const Saved to(p.saved, m, p.N);
      to.store(n, x);
      to.store(N + n, y);
    }
  }
}

// [dg du] from dh and the saved [g u], 4 columns a thread.
template <class T> __global__ __launch_bounds__(256) void gate_bwd_kernel(const T* dh, int64_t dh_ld, uint8_t* saved, T* d,
                                                                         int M, int F) {
  using x4 = typename El<T>::x4;
  for (int64_t i = (blockIdx.x * 256ll + threadIdx.x) * 4; i < static_cast<int64_t>(M) * F; i += gridDim.x * 1024ll) {
    const int64_t m = i / F, n = i % F;
    const x4 a = *reinterpret_cast<const x4*>(dh + m * dh_ld + n);
    const Saved from(saved, m, 2 * F);
    const f32x4 g = from.load(n), u = from.load(F + n);
    x4 dg, du;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float grad = static_cast<float>(a[j]), s = sigmoid(g[j]);
      dg[j] = static_cast<T>(grad * u[j] * s * (1.f + g[j] * (1.f - s)));
      du[j] = static_cast<T>(grad * g[j] * s);
    }
    *reinterpret_cast<x4*>(d + m * 2 * F + n) = dg;
    *reinterpret_cast<x4*>(d + m * 2 * F + F + n) = du;
  }
}

// Workgroups of 256 threads for n items, of which a thread takes more than one if they are
// over 2^28 (a launch has under 2^32 threads).
unsigned blocks(int64_t n) { return static_cast<unsigned>(n < (1 << 28) ? (n + 255) / 256 : 1 << 20); }

template <class T, int BM, int BN, int WM, int WN, bool TA, bool TB, bool PAIR>
int product_tiled(const Product& p, hipStream_t s) {
  constexpr int kLds = 2 * (BM + BN) * kK * 2;
  const auto kernel = product_kernel<T, BM, BN, WM, WN, TA, TB, PAIR>;
  // more than the default 64 KiB: once a device, and harmless when repeated
  if (kLds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess) return fail("swiglu LDS", hipGetErrorString(e));
  }
  const int N = PAIR ? p.N / 2 : p.N, bn = PAIR ? BN / 2 : BN;
  const int64_t total = static_cast<int64_t>((p.M + BM - 1) / BM) * ((N + bn - 1) / bn) * p.splits;
  if (total > (1ll << 32) / (WM * WN * 64) - 8) return fail("swiglu", "too many workgroups");  // under 2^32 threads
  kernel<<<static_cast<unsigned>((total + 7) / 8 * 8), WM * WN * 64, kLds, s>>>(p);
  if (launched("swiglu product")) return -1;
  if (p.splits > 1) {
    const int64_t n = static_cast<int64_t>(p.M) * N / 4;
    join_kernel<T, PAIR><<<blocks(n), 256, 0, s>>>(p);
    return launched("swiglu join");
  }
  return 0;
}

template <class T, bool TA, bool TB, bool PAIR> int product(const Product& p, int tile, hipStream_t s) {
  switch (tile) {
    case 0: return product_tiled<T, 128, 128, 2, 2, TA, TB, PAIR>(p, s);
    case 1: return product_tiled<T, 256, 256, 2, 4, TA, TB, PAIR>(p, s);
    case 2:  // few rows, forward
      if constexpr (PAIR) return product_tiled<T, 32, 256, 1, 4, TA, TB, PAIR>(p, s);
  }
  return fail("swiglu", "unknown tile");
}

template <class T> int forward(const KgsSwiglu& a, hipStream_t s) {
  const Product p{a.x, a.w, a.x_ld, a.w_ld, a.h, static_cast<uint8_t*>(a.saved), a.partial, a.T, 2 * a.F, a.K, a.splits[0]};
  return product<T, false, false, true>(p, a.tile[0], s);
}

template <class T> int backward(const KgsSwiglu& a, hipStream_t s) {
  const int64_t n = static_cast<int64_t>(a.T) * a.F / 4;
  gate_bwd_kernel<T><<<blocks(n), 256, 0, s>>>(
      static_cast<const T*>(a.dh), a.dh_ld, static_cast<uint8_t*>(a.saved), static_cast<T*>(a.dgu), a.T, a.F);
  if (launched("swiglu gate backward")) return -1;
  if (a.dx) {
    const Product p{a.dgu, a.w, 2ll * a.F, a.w_ld, a.dx, nullptr, a.partial, a.T, a.K, 2 * a.F, a.splits[1]};
    if (product<T, false, true, false>(p, a.tile[1], s)) return -1;
  }
  if (a.dw) {
    const Product p{a.dgu, a.x, 2ll * a.F, a.x_ld, a.dw, nullptr, a.partial, 2 * a.F, a.K, a.T, a.splits[2]};
    if (product<T, true, true, false>(p, a.tile[2], s)) return -1;
  }
  return 0;
}

int check(const KgsSwiglu* a, bool back) {
  const char* w = "swiglu";
  if (!a || !a->x || !a->w || (!back && !a->h)) return fail(w, "a tensor is missing");
  if (back && (!a->dh || !a->saved || !a->dgu)) return fail(w, "a tensor is missing");
  if (a->T <= 0 || a->K <= 0 || a->F <= 0 || a->K % 8 || a->F % 8) return fail(w, "bad sizes");
  // offsets inside a tile of 256 rows stay under 2^30
  if (a->K > (1 << 20) || a->F > (1 << 20)) return fail(w, "too wide");
  if (a->x_ld < a->K || a->w_ld < a->K || a->x_ld % 8 || a->w_ld % 8 || a->x_ld > (1 << 21) || a->w_ld > (1 << 21))
    return fail(w, "unsupported strides");
  if (back && (a->dh_ld < a->F || a->dh_ld % 8)) return fail(w, "unsupported strides");
  if (a->type != 0 && a->type != 1) return fail(w, "type must be bfloat16 or float16");
  for (int i = back ? 1 : 0; i < (back ? 3 : 1); ++i)
    if ((i == 1 && !a->dx) || (i == 2 && !a->dw)) continue;
    else if (a->splits[i] < 1 || (a->splits[i] > 1 && !a->partial)) return fail(w, "bad split");
  return 0;
}

}  // namespace
}  // namespace kgs

extern "C" {
int kgs_swiglu_fwd(const KgsSwiglu* a, void* stream) {
  if (kgs::check(a, false)) return -1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->type == 0 ? kgs::forward<kgs::bf16>(*a, s) : kgs::forward<kgs::f16>(*a, s);
}
int kgs_swiglu_bwd(const KgsSwiglu* a, void* stream) {
  if (kgs::check(a, true)) return -1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->type == 0 ? kgs::backward<kgs::bf16>(*a, s) : kgs::backward<kgs::f16>(*a, s);
}
}
