// The norms around a residual connection, forward and backward, for gfx950.
//
//   n = post_weight b rb  (rb = 1 / sqrt(mean b^2 + eps); n = b without post_weight)
//   s = r + scale gate n,   y = weight s rs  (rs = 1 / sqrt(mean s^2 + eps))
//   ds = dS + rs (w dy - s rs^2 mean(w dy s)),   dr = ds,   t = scale ds
//   dn = gate t,   db = rb (pw dn - b rb^2 mean(pw dn b))  (db = dn without post_weight)
//   dweight = sum dy s rs,  dpost_weight = sum dn b rb,  dgate = sum t n   over the rows
//
// Bound by memory: each row is read once and stays in its threads' registers between
// the two means; the weights stay there from row to row.  A workgroup takes rows in
// turn; for the backward's column sums each thread adds its columns in registers over
// its rows, the workgroups' sums are joined by a second kernel in a fixed order (no
// atomics, so equal calls give equal bits).
//
// Everything is computed in 32 bits and rounded once, as an output.  The forward
// normalises the unrounded stream; the backward sees it as it was stored.
#include "decoder.h"
#include "decoder_common.h"

namespace kgs {
namespace {

constexpr int kV = 8;  // elements of a row a thread handles at a time

// 8 elements whose address is aligned to one element only: an odd width moves rows off
// every wider boundary, which global memory instructions allow.
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Loose { T v[kV]; };

template <class T> __device__ __forceinline__ void load(float (&x)[kV], const T* p, int left) {
  if (left >= kV) {
    const Loose<T> r = *reinterpret_cast<const Loose<T>*>(p);
#pragma unroll
    for (int i = 0; i < kV; ++i) x[i] = static_cast<float>(r.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) x[i] = i < left ? static_cast<float>(p[i]) : 0.f;
  }
}

template <class T> __device__ __forceinline__ void store(const float (&x)[kV], T* p, int left) {
  if (left >= kV) {
    Loose<T> r;
#pragma unroll
    for (int i = 0; i < kV; ++i) r.v[i] = static_cast<T>(x[i]);
    *reinterpret_cast<Loose<T>*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i)
      if (i < left) p[i] = static_cast<T>(x[i]);
  }
}

// Sum over a row's threads.  One wave a row: no LDS.  More: one slot a wave, and two
// sets of slots in turn so that one barrier a sum is enough.
template <int TPR> __device__ __forceinline__ float row_sum(float x, float* slots, int& turn) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m, 64);
  if constexpr (TPR > 64) {
    float* s = slots + turn * (TPR / 64);
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) x += s[i];
  }
  return x;
}

template <int TPR> struct Shape {
  static constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR;
};

// FULL: with post_weight or gate (or a scale).  NV: chunks of 8 a thread.
template <class T, int TPR, int NV, bool FULL>
__global__ __launch_bounds__(Shape<TPR>::kThreads) void add_norm_fwd_kernel(KgsAddNorm a) {
  __shared__ float slots[2 * (TPR > 64 ? TPR / 64 : 1)];
  int turn = 0;
  const int t = threadIdx.x % TPR, C = a.width;
  const T *residual = static_cast<const T*>(a.residual), *branch = static_cast<const T*>(a.branch);
  float w[NV][kV], pw[FULL ? NV : 1][kV], gate[FULL ? NV : 1][kV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * kV;
    load(w[i], static_cast<const T*>(a.weight) + c, C - c);
    if constexpr (FULL) {
      if (a.post_weight) load(pw[i], static_cast<const T*>(a.post_weight) + c, C - c);
      else for (float& x : pw[i]) x = 1.f;
      if (a.gate) load(gate[i], static_cast<const T*>(a.gate) + c, C - c);
      else for (float& x : gate[i]) x = 1.f;
      for (float& x : gate[i]) x *= a.scale;
    }
  }
  const int step = gridDim.x * Shape<TPR>::kRows;
  for (int row = blockIdx.x * Shape<TPR>::kRows + threadIdx.x / TPR; row < a.rows; row += step) {
    float s[NV][kV], b[NV][kV];
    float sq = 0.f, rb = 1.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * TPR) * kV;
      load(b[i], branch + row * a.branch_ld + c, C - c);
      load(s[i], residual + row * a.residual_ld + c, C - c);
    }
    if constexpr (FULL) {
      if (a.post_weight) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < kV; ++j) sq = fmaf(b[i][j], b[i][j], sq);
        rb = 1.f / sqrtf(row_sum<TPR>(sq, slots, turn) / C + a.eps);
        sq = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * TPR) * kV;
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        if constexpr (FULL) s[i][j] = fmaf(gate[i][j], b[i][j] * rb * pw[i][j], s[i][j]);
        else s[i][j] += b[i][j];
        sq = fmaf(s[i][j], s[i][j], sq);
      }
      store(s[i], static_cast<T*>(a.stream) + row * a.stream_ld + c, C - c);
    }
    const float rs = 1.f / sqrtf(row_sum<TPR>(sq, slots, turn) / C + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * TPR) * kV;
#pragma unroll
      for (int j = 0; j < kV; ++j) s[i][j] *= rs * w[i][j];
      store(s[i], static_cast<T*>(a.out) + static_cast<int64_t>(row) * C + c, C - c);
    }
    if (a.rstd && t == 0) {
      a.rstd[row] = rs;
      a.rstd[a.rows + row] = rb;
    }
  }
}

template <class T, int TPR, int NV, bool FULL>
__global__ __launch_bounds__(Shape<TPR>::kThreads) void add_norm_bwd_kernel(KgsAddNorm a) {
  constexpr int kRows = Shape<TPR>::kRows;
  __shared__ float slots[2 * (TPR > 64 ? TPR / 64 : 1)];
  int turn = 0;
  const int t = threadIdx.x % TPR, C = a.width;
  float w[NV][kV], pw[FULL ? NV : 1][kV], gate[FULL ? NV : 1][kV];
  float dw[NV][kV] = {}, dpw[FULL ? NV : 1][kV] = {}, dgate[FULL ? NV : 1][kV] = {};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * kV;
    load(w[i], static_cast<const T*>(a.weight) + c, C - c);
    if constexpr (FULL) {
      if (a.post_weight) load(pw[i], static_cast<const T*>(a.post_weight) + c, C - c);
      else for (float& x : pw[i]) x = 1.f;
      if (a.gate) load(gate[i], static_cast<const T*>(a.gate) + c, C - c);
      else for (float& x : gate[i]) x = 1.f;
    }
  }
  const int step = gridDim.x * kRows;
  for (int row = blockIdx.x * kRows + threadIdx.x / TPR; row < a.rows; row += step) {
    const float rs = a.rstd[row];
    float s[NV][kV], dy[NV][kV], ds[NV][kV], b[FULL ? NV : 1][kV];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * TPR) * kV;
      load(s[i], static_cast<const T*>(a.stream) + row * a.stream_ld + c, C - c);
      if (a.dout) load(dy[i], static_cast<const T*>(a.dout) + row * a.dout_ld + c, C - c);
      else for (float& x : dy[i]) x = 0.f;
      if (a.dstream) load(ds[i], static_cast<const T*>(a.dstream) + row * a.dstream_ld + c, C - c);
      else for (float& x : ds[i]) x = 0.f;
      if constexpr (FULL) load(b[i], static_cast<const T*>(a.branch) + row * a.branch_ld + c, C - c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        s[i][j] *= rs;
        dw[i][j] = fmaf(dy[i][j], s[i][j], dw[i][j]);
        dy[i][j] *= w[i][j];
        dot = fmaf(dy[i][j], s[i][j], dot);
      }
    const float mean = row_sum<TPR>(dot, slots, turn) / C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * TPR) * kV;
#pragma unroll
      for (int j = 0; j < kV; ++j) ds[i][j] = fmaf(rs, dy[i][j] - s[i][j] * mean, ds[i][j]);
      store(ds[i], static_cast<T*>(a.dresidual) + static_cast<int64_t>(row) * C + c, C - c);
    }
    if constexpr (FULL) {
      const float rb = a.rstd[a.rows + row];
      float dot2 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < kV; ++j) {
          const float bh = b[i][j] * rb, g = ds[i][j] * a.scale, dn = g * gate[i][j];
          dgate[i][j] = fmaf(g, bh * pw[i][j], dgate[i][j]);
          dpw[i][j] = fmaf(dn, bh, dpw[i][j]);
          b[i][j] = bh;
          ds[i][j] = dn * pw[i][j];
          dot2 = fmaf(ds[i][j], bh, dot2);
        }
      const float mean2 = a.post_weight ? row_sum<TPR>(dot2, slots, turn) / C : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * kV;
#pragma unroll
        for (int j = 0; j < kV; ++j) ds[i][j] = rb * (ds[i][j] - b[i][j] * mean2);
        store(ds[i], static_cast<T*>(a.dbranch) + static_cast<int64_t>(row) * C + c, C - c);
      }
    }
  }
  // this workgroup's column sums; with several rows in flight, one part a row of them
  float* part = a.partial + (static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR) * 3 * C;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * kV;
    store(dw[i], part + c, C - c);
    if constexpr (FULL) {
      store(dpw[i], part + C + c, C - c);
      store(dgate[i], part + 2 * C + c, C - c);
    }
  }
}

// Column sums of the parts: 64 columns a workgroup, 16 threads a column.
template <class T> __global__ __launch_bounds__(1024) void add_norm_join_kernel(KgsAddNorm a) {
  __shared__ float sums[16][64];
  const int C = a.width, col = threadIdx.x & 63, group = threadIdx.x >> 6, c = blockIdx.x * 64 + col;
  T* const to = static_cast<T*>(blockIdx.y == 0 ? a.dweight : blockIdx.y == 1 ? a.dpost_weight : a.dgate);
  if (!to) return;
  float sum = 0.f;
  if (c < C) {
    const float* p = a.partial + static_cast<int64_t>(blockIdx.y) * C + c;
#pragma unroll 8
    for (int i = group; i < a.parts; i += 16) sum += p[static_cast<int64_t>(i) * 3 * C];
  }
  sums[group][col] = sum;
  __syncthreads();
  if (group == 0 && c < C) {
    for (int i = 1; i < 16; ++i) sum += sums[i][col];
    to[c] = static_cast<T>(sum);
  }
}

template <class T, int TPR, int NV> int launch(const KgsAddNorm& a, bool back, hipStream_t s) {
  constexpr int kRows = Shape<TPR>::kRows, kThreads = Shape<TPR>::kThreads;
  const bool full = a.post_weight || a.gate || a.scale != 1.f;
  if (!back) {
    const int want = (a.rows + kRows - 1) / kRows, grid = want < 8192 ? want : 8192;
    if (full) add_norm_fwd_kernel<T, TPR, NV, true><<<grid, kThreads, 0, s>>>(a);
    else add_norm_fwd_kernel<T, TPR, NV, false><<<grid, kThreads, 0, s>>>(a);
    return launched("add_norm forward");
  }
  // one part of the column sums a row of threads; the caller's partial has room for that
  const int grid = a.parts / kRows;
  if (grid < 1 || grid * kRows != a.parts) return fail("add_norm", "parts do not fit the rows of a workgroup");
  if (full) add_norm_bwd_kernel<T, TPR, NV, true><<<grid, kThreads, 0, s>>>(a);
  else add_norm_bwd_kernel<T, TPR, NV, false><<<grid, kThreads, 0, s>>>(a);
  if (launched("add_norm backward")) return -1;
  add_norm_join_kernel<T><<<dim3((a.width + 63) / 64, full ? 3 : 1), 1024, 0, s>>>(a);
  return launched("add_norm join");
}

template <class T> int run(const KgsAddNorm& a, bool back, hipStream_t s) {
  // At most 16 elements of a row a thread: the three column sums and the row fit the
  // registers of four waves a SIMD.
  if (a.width <= 512) return launch<T, 64, 1>(a, back, s);
  if (a.width <= 2048) return launch<T, 256, 1>(a, back, s);
  if (a.width <= 4096) return launch<T, 256, 2>(a, back, s);
  if (a.width <= 8192) return launch<T, 512, 2>(a, back, s);
  return launch<T, 1024, 2>(a, back, s);
}

int dispatch(const KgsAddNorm* a, bool back, void* stream) {
  const char* w = "add_norm";
  if (!a || !a->branch || !a->weight || !a->stream) return fail(w, "a tensor is missing");
  if (!back && (!a->residual || !a->out)) return fail(w, "a tensor is missing");
  if (back && (!a->rstd || !a->dresidual || !a->dbranch || !a->dweight || !a->partial)) return fail(w, "a tensor is missing");
  if (back && ((a->post_weight && !a->dpost_weight) || (a->gate && !a->dgate))) return fail(w, "a tensor is missing");
  if (a->rows <= 0 || a->width <= 0 || a->width > 16384) return fail(w, "bad sizes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->type) {
    case 0: return run<bf16>(*a, back, s);
    case 1: return run<f16>(*a, back, s);
    case 2: return run<float>(*a, back, s);
  }
  return fail(w, "type must be bfloat16, float16 or float32");
}

}  // namespace
}  // namespace kgs

extern "C" {
int kgs_add_norm_fwd(const KgsAddNorm* a, void* stream) { return kgs::dispatch(a, false, stream); }
int kgs_add_norm_bwd(const KgsAddNorm* a, void* stream) { return kgs::dispatch(a, true, stream); }
}
