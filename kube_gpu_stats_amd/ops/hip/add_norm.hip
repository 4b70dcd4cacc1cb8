// The norms around a residual connection, forward and backward, for gfx950.
//
//   n = post_weight b rb  (rb = 1 / sqrt(mean b^2 + eps); n = b without post_weight)
//   s = r + scale gate n,   y = weight s rs  (rs = 1 / sqrt(mean s^2 + eps))
//   ds = dS + rs (w dy - s rs^2 mean(w dy s)),   dr = ds,   t = scale ds
//   dn = gate t,   db = rb (pw dn - b rb^2 mean(pw dn b))  (db = dn without post_weight)
//   dweight = sum dy s rs,  with A = sum ds b rb over the rows:
//   dpost_weight = scale gate A,  dgate = scale post_weight A
//
// Bound by memory: each row is read once and stays in its threads' registers between
// the two means; the weights stay there from row to row.  Rows up to 512 wide take a
// power of two of lanes, 8 elements each, so that a wave works on several; wider ones a
// workgroup.  Workgroups take rows in turn; for the backward's column sums each thread
// adds its columns in registers over its rows, the workgroups' sums are joined by a
// second kernel in a fixed order (no atomics, so equal calls give equal bits).
//
// Everything is computed in 32 bits and rounded once, as an output.  Both passes use the
// unrounded stream.  The backward adds it up again from residual and branch, or reads the
// stream that the forward wrote with 8 more bits of each element beside it.  (The 16-bit
// stream alone would add half as much error again to dweight.)
#include "decoder.h"
#include "decoder_common.h"

namespace kgs {
namespace {

constexpr int kV = 8;  // elements of a row a thread handles at a time

// 8 elements whose address is aligned to one element only: an odd width moves rows off
// every wider boundary, which global memory instructions allow.
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Loose { T v[kV]; };

// (a row of fewer than 8 elements: zeros behind them)
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

// Element `start` of p, the same in the whole workgroup where a row is one's, and a
// thread's bytes from there: one scalar address and 32 bits a thread.
template <class T> __device__ __forceinline__ const T* place(const void* p, int64_t start, uint32_t bytes) {
  return reinterpret_cast<const T*>(reinterpret_cast<const char*>(static_cast<const T*>(p) + start) + bytes);
}
template <class T> __device__ __forceinline__ T* place(void* p, int64_t start, uint32_t bytes) {
  return const_cast<T*>(place<T>(static_cast<const void*>(p), start, bytes));
}

// The same as it lies in memory.
template <class T> __device__ __forceinline__ void load_raw(Loose<T>& r, const T* p, int left) {
  if (left >= kV) {
    r = *reinterpret_cast<const Loose<T>*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) r.v[i] = i < left ? p[i] : static_cast<T>(0.f);
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

// Sum over the threads of a row: `lanes` of a wave (a power of two), or the workgroup,
// by way of one slot a wave in two sets used in turn, so that one barrier is enough.
template <bool WAVES> __device__ __forceinline__ float row_sum(float x, int lanes, float* slots, int& turn) {
  if constexpr (WAVES) {
    for (int m = 1; m < lanes; m <<= 1) x += __shfl_xor(x, m, 64);
  } else {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m, 64);
    float* s = slots + turn * 16;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.f;
    for (unsigned i = 0; i < blockDim.x / 64; ++i) x += s[i];
  }
  return x;
}

// What rounding took from 8 elements of a 16-bit stream, a byte each.  With no byte below
// it an infinity is read back as a NaN: so is an element that rounding made infinite, whose
// difference would make it a finite one.
template <class T> __device__ __forceinline__ void store_low(const float (&x)[kV], uint8_t* p, int left) {
  u32x2 bytes;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float e = x[g * 4 + j];
      q[j] = __builtin_isinf(static_cast<float>(static_cast<T>(e))) ? 0 : low_of<T>(e);
    }
    bytes[g] = __builtin_amdgcn_perm(q[1], q[0], 0x0C0C0501) | (__builtin_amdgcn_perm(q[3], q[2], 0x0C0C0501) << 16);
    __builtin_amdgcn_sched_barrier(0);  // four at a time: over 64 registers half as many waves run
  }
  if (left >= kV) {
    __builtin_memcpy(p, &bytes, kV);
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i)
      if (i < left) p[i] = static_cast<uint8_t>(bytes[i >> 2] >> (8 * (i & 3)));
  }
}

__host__ __device__ __forceinline__ int lanes_of_row(int width) {
  int n = 1;
  while (n * kV < width) n *= 2;
  return n;
}

// Where a thread stands: the first column chunk of its row, the row of its workgroup's
// turn, and the rows a turn.  WAVES: widths up to 512.
//
// A width that is no multiple of 8 has its last chunk moved back to end with the row, so
// that it too is loaded and stored at once; the first skip() of its elements are the
// chunk's before it as well: both threads write the same there, and the last leaves them
// out of the sums.  A thread past the end skips all 8.  (Element by element at the end of
// each row 20000 x 1501 with all weights took 64 us forward and 111 us back, so 41 us and
// 95 us.)
enum Fit { kWhole, kRagged, kTiny };  // a multiple of 8; another width; fewer than 8
template <bool WAVES> struct Place {
  int lanes, t, row, rows;
  __device__ __forceinline__ int column(int i, int C) const {
    const int c = (t + i * lanes) * kV;
    return c < C ? max(0, min(c, C - kV)) : 0;
  }
  __device__ __forceinline__ int skip(int i, int C) const {
    const int c = (t + i * lanes) * kV;
    return c >= C ? kV : max(0, c - max(0, C - kV));
  }
  __device__ __forceinline__ explicit Place(int width) {
    lanes = WAVES ? lanes_of_row(width) : blockDim.x;
    t = WAVES ? threadIdx.x & (lanes - 1) : threadIdx.x;
    row = WAVES ? threadIdx.x / lanes : 0;
    rows = WAVES ? 256 / lanes : 1;
  }
};

// FULL: with post_weight, gate or a scale.  NV: chunks of 8 a thread.  LOW: writes the low
// bytes too.
template <class T, bool WAVES, int NV, bool FULL, bool LOW, Fit FIT>
__global__ __launch_bounds__(WAVES ? 256 : 1024, LOW && NV == 1 ? 8 : 1) void add_norm_fwd_kernel(KgsAddNorm a) {
  __shared__ float slots[2 * 16];
  int turn = 0;
  const Place<WAVES> at(a.width);
  const int C = a.width;
  const int size = FIT == kTiny ? C : kV;  // elements a chunk has
  int skip[NV];
  uint32_t column[NV];  // in bytes
  float w[NV][kV], pw[FULL ? NV : 1][kV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = at.column(i, C);
    column[i] = c * sizeof(T);
    skip[i] = at.skip(i, C);
    load(w[i], static_cast<const T*>(a.weight) + c, size);
    if constexpr (FULL) {  // what the normalised branch is multiplied by
      for (float& x : pw[i]) x = a.scale;
      float f[kV];
      if (a.post_weight) {
        load(f, static_cast<const T*>(a.post_weight) + c, size);
        for (int j = 0; j < kV; ++j) pw[i][j] *= f[j];
      }
      if (a.gate) {
        load(f, static_cast<const T*>(a.gate) + c, size);
        for (int j = 0; j < kV; ++j) pw[i][j] *= f[j];
      }
    }
  }
  // an element's part in a sum
  const auto part = [&](int i, int j, float x) { return (FIT == kWhole ? skip[i] : j < skip[i]) ? 0.f : x; };
  const int step = gridDim.x * at.rows;
  for (int row = blockIdx.x * at.rows + at.row; row < a.rows; row += step) {
    float s[NV][kV], b[NV][kV];
    float sq = 0.f, rb = 1.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      load(b[i], place<T>(a.branch, row * a.branch_ld, column[i]), size);
      load(s[i], place<T>(a.residual, row * a.residual_ld, column[i]), size);
    }
    if constexpr (FULL) {
      if (a.post_weight) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < kV; ++j) sq = fmaf(b[i][j], part(i, j, b[i][j]), sq);
        rb = 1.f / sqrtf(row_sum<WAVES>(sq, at.lanes, slots, turn) / C + a.eps);
        sq = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        if constexpr (FULL) s[i][j] = fmaf(pw[i][j], b[i][j] * rb, s[i][j]);
        else s[i][j] += b[i][j];
        sq = fmaf(s[i][j], part(i, j, s[i][j]), sq);
      }
      if (skip[i] < kV) {
        store(s[i], place<T>(a.stream, row * a.stream_ld, column[i]), size);
        if constexpr (LOW) store_low<T>(s[i], a.low + static_cast<int64_t>(row) * C + column[i] / sizeof(T), size);
      }
    }
    const float rs = 1.f / sqrtf(row_sum<WAVES>(sq, at.lanes, slots, turn) / C + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < kV; ++j) s[i][j] *= rs * w[i][j];
      if (skip[i] < kV) store(s[i], place<T>(a.out, static_cast<int64_t>(row) * C, column[i]), size);
    }
    if (a.rstd && at.t == 0) {
      a.rstd[row] = rs;
      a.rstd[a.rows + row] = rb;
    }
  }
}

// A column's finished sum: v 0 is dweight's, v 1 is A.
template <class T> __device__ __forceinline__ void finish(const KgsAddNorm& a, int v, int c, float sum) {
  if (v == 0) {
    static_cast<T*>(a.dweight)[c] = static_cast<T>(sum);
    return;
  }
  sum *= a.scale;
  const float pw = a.post_weight ? static_cast<float>(static_cast<const T*>(a.post_weight)[c]) : 1.f;
  const float gate = a.gate ? static_cast<float>(static_cast<const T*>(a.gate)[c]) : 1.f;
  if (a.dpost_weight) static_cast<T*>(a.dpost_weight)[c] = static_cast<T>(sum * gate);
  if (a.dgate) static_cast<T*>(a.dgate)[c] = static_cast<T>(sum * pw);
}

// The next row's loads are under way while this one is reduced; with one chunk a thread
// that fits the registers of 16 waves a CU.  Two chunks (rows over 8192 wide) do without,
// and read the weights again for every row.  STORED: from the stream and its low bytes, one
// byte an element less to read than residual and branch, with FULL one more (8192 x 4096:
// 57 us, 63 us from the residual; 16384 x 8192 with all weights 310 us, 287 us; the forward,
// which writes them, 5 and 28 us more).
template <class T, bool WAVES, int NV, bool FULL, bool STORED, Fit FIT, int THREADS>
__global__ __launch_bounds__(THREADS) void add_norm_bwd_kernel(KgsAddNorm a) {
  __shared__ float slots[2 * 16];
  __shared__ float sums[WAVES ? (FULL ? 2 : 1) * 4 * 512 : 1];
  constexpr bool kAhead = NV == 1;
  int turn = 0;
  const Place<WAVES> at(a.width);
  const int C = a.width;
  const int size = FIT == kTiny ? C : kV;
  int skip[NV];
  uint32_t column[NV];  // in bytes
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    column[i] = at.column(i, C) * sizeof(T);
    skip[i] = at.skip(i, C);
  }
  // an element's part in a sum; of whole chunks zero weights leave out a thread past the end
  const auto part_of = [&](int i, int j, float x) { return FIT != kWhole && j < skip[i] ? 0.f : x; };
  const auto get = [&](Loose<T>& r, const void* p, int64_t start, uint32_t column) {
    load_raw(r, place<T>(p, start, column), size);
  };
  // For residual and branch: last read by the forward pass, they are not in a cache, and
  // are not kept in one (8192 x 4096: 69 us to 61 us, all weights 88 us to 75 us; with the
  // gradients read so too, which the pass before has just written, 47 us for 45 us at a
  // size that the caches hold).  Ragged rows share lines with their neighbours, which are
  // better kept (30000 x 537: 56 us, kept 43 us).
  const auto get_once = [&](Loose<T>& r, const void* p, int64_t start, uint32_t column) {
    if constexpr (FIT == kWhole) {
      typedef T V8 __attribute__((ext_vector_type(kV), aligned(sizeof(T))));
      const V8 x = __builtin_nontemporal_load(reinterpret_cast<const V8*>(place<T>(p, start, column)));
#pragma unroll
      for (int j = 0; j < kV; ++j) r.v[j] = x[j];
    } else {
      get(r, p, start, column);
    }
  };
  // weight, and scale post_weight gate
  float w[NV][kV], full[FULL ? NV : 1][kV];
  const auto weights = [&] {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = at.column(i, C);
      load(w[i], static_cast<const T*>(a.weight) + c, FIT == kWhole && skip[i] ? 0 : size);
      if constexpr (FULL) {
        float f[kV];
#pragma unroll
        for (int j = 0; j < kV; ++j) full[i][j] = FIT == kWhole && skip[i] ? 0.f : a.scale;
        if (a.post_weight) {
          load(f, static_cast<const T*>(a.post_weight) + c, size);
#pragma unroll
          for (int j = 0; j < kV; ++j) full[i][j] *= f[j];
        }
        if (a.gate) {
          load(f, static_cast<const T*>(a.gate) + c, size);
#pragma unroll
          for (int j = 0; j < kV; ++j) full[i][j] *= f[j];
        }
      }
    }
  };
  if (kAhead) weights();
  constexpr bool kLow = STORED && sizeof(T) == 2;
  struct Row {
    Loose<T> s[NV], dy[NV], ds[NV], b[STORED && !FULL ? 1 : NV];  // s: the residual, or the stream
    u32x2 low[kLow ? NV : 1];  // 8 bytes (as bytes they would take a register each)
    float rs, rb;
  } next;
  const auto fetch = [&](int row) {
    next.rs = a.rstd[row];
    next.rb = FULL ? a.rstd[a.rows + row] : 1.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (STORED) get_once(next.s[i], a.stream, row * a.stream_ld, column[i]);
      else get_once(next.s[i], a.residual, row * a.residual_ld, column[i]);
      if constexpr (kLow) {
        const uint8_t* p = a.low + static_cast<int64_t>(row) * C + column[i] / sizeof(T);
        if constexpr (FIT == kWhole) {
          next.low[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
        } else if constexpr (FIT == kRagged) {
          __builtin_memcpy(&next.low[i], p, kV);
        } else {
          next.low[i] = u32x2{0, 0};
#pragma unroll
          for (int j = 0; j < kV; ++j)
            if (j < C) next.low[i][j >> 2] |= static_cast<uint32_t>(p[j]) << (8 * (j & 3));
        }
      }
      if constexpr (FULL || !STORED) get_once(next.b[i], a.branch, row * a.branch_ld, column[i]);
      if (a.dout) get(next.dy[i], a.dout, row * a.dout_ld, column[i]);
      if (a.dstream) get(next.ds[i], a.dstream, row * a.dstream_ld, column[i]);
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < kV; ++j) next.dy[i].v[j] = next.ds[i].v[j] = static_cast<T>(0.f);  // absent
  float dw[NV][kV] = {}, sum[FULL ? NV : 1][kV] = {};  // column sums: dweight, A
  const int step = gridDim.x * at.rows;
  int row = blockIdx.x * at.rows + at.row;
  if (kAhead && row < a.rows) fetch(row);
  for (; row < a.rows; row += step) {
    if (!kAhead) {
      fetch(row);
      weights();
    }
    float s[NV][kV], dy[NV][kV], ds[NV][kV], b[FULL ? NV : 1][kV];
    const float rs = next.rs, rb = next.rb;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const float g = static_cast<float>(next.dy[i].v[j]);
        ds[i][j] = static_cast<float>(next.ds[i].v[j]);
        float r;
        if constexpr (kLow) r = with_low<T>(next.s[i].v[j], static_cast<int8_t>(next.low[i][j >> 2] >> (8 * (j & 3))));
        else r = static_cast<float>(next.s[i].v[j]);
        if constexpr (FULL) b[i][j] = static_cast<float>(next.b[i].v[j]) * rb;
        if constexpr (STORED) s[i][j] = r * rs;
        else if constexpr (FULL) s[i][j] = fmaf(full[i][j], b[i][j], r) * rs;
        else s[i][j] = (r + static_cast<float>(next.b[i].v[j])) * rs;
        dw[i][j] = fmaf(g, s[i][j], dw[i][j]);
        dy[i][j] = g * w[i][j];
        dot = fmaf(dy[i][j], part_of(i, j, s[i][j]), dot);
      }
    if (kAhead && row + step < a.rows) fetch(row + step);
    const float mean = row_sum<WAVES>(dot, at.lanes, slots, turn) / C;
    float dot2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < kV; ++j) ds[i][j] = fmaf(rs, dy[i][j] - s[i][j] * mean, ds[i][j]);
      if (skip[i] < kV) store(ds[i], place<T>(a.dresidual, static_cast<int64_t>(row) * C, column[i]), size);
      if constexpr (FULL) {
#pragma unroll
        for (int j = 0; j < kV; ++j) {
          sum[i][j] = fmaf(ds[i][j], b[i][j], sum[i][j]);
          ds[i][j] *= full[i][j];
          dot2 = fmaf(ds[i][j], part_of(i, j, b[i][j]), dot2);
        }
      }
    }
    if constexpr (FULL) {
      const float mean2 = a.post_weight ? row_sum<WAVES>(dot2, at.lanes, slots, turn) / C : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < kV; ++j) ds[i][j] = rb * (ds[i][j] - b[i][j] * mean2);
        if (skip[i] < kV) store(ds[i], place<T>(a.dbranch, static_cast<int64_t>(row) * C, column[i]), size);
      }
    }
  }
  // This workgroup's column sums: a part, and if it is the only one, the results.
  float* part = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * C;
  if constexpr (WAVES) {
    // over the wave's rows, then over the four waves
    const int wave = threadIdx.x >> 6, c = at.column(0, C);
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      for (int m = at.lanes; m < 64; m <<= 1) {
        dw[0][j] += __shfl_xor(dw[0][j], m, 64);
        if constexpr (FULL) sum[0][j] += __shfl_xor(sum[0][j], m, 64);
      }
      if ((threadIdx.x & 63) < at.lanes && skip[0] < kV) {
        sums[wave * 512 + c + j] = dw[0][j];
        if constexpr (FULL) sums[(4 + wave) * 512 + c + j] = sum[0][j];
      }
    }
    __syncthreads();
    for (int v = 0; v < (FULL ? 2 : 1); ++v)
      for (int c = threadIdx.x; c < C; c += 256) {
        const float* x = sums + v * 4 * 512 + c;
        part[v * C + c] = (x[0] + x[512]) + (x[1024] + x[1536]);
      }
  } else {
    // (where chunks overlap, two threads have summed the same and write the same)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = at.column(i, C);
      if (skip[i] == kV) continue;
      store(dw[i], part + c, size);
      if constexpr (FULL) store(sum[i], part + C + c, size);
    }
  }
  if (gridDim.x > 1) return;
  __syncthreads();
  for (int v = 0; v < (FULL && (a.dpost_weight || a.dgate) ? 2 : 1); ++v)
    for (int c = threadIdx.x; c < C; c += blockDim.x) finish<T>(a, v, c, part[v * C + c]);
}

// Column sums of the parts: 16 columns a workgroup, 64 threads a column.
template <class T> __global__ __launch_bounds__(1024) void add_norm_join_kernel(KgsAddNorm a) {
  __shared__ float sums[64][16];
  const int C = a.width, col = threadIdx.x & 15, group = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  float sum = 0.f;
  if (c < C) {
    const float* p = a.partial + static_cast<int64_t>(blockIdx.y) * C + c;
#pragma unroll 8
    for (int i = group; i < a.parts; i += 64) sum += p[static_cast<int64_t>(i) * 2 * C];
  }
  sums[group][col] = sum;
  __syncthreads();
  if (group == 0 && c < C) {
    sum = 0.f;
    for (int i = 0; i < 64; ++i) sum += sums[i][col];
    finish<T>(a, blockIdx.y, c, sum);
  }
}

bool is_full(const KgsAddNorm& a) { return a.post_weight || a.gate || a.scale != 1.f; }

// Threads and rows a turn of a workgroup.
template <bool WAVES, int NV> void shape(const KgsAddNorm& a, int& threads, int& rows) {
  threads = WAVES ? 256 : (a.width + 64 * kV * NV - 1) / (64 * kV * NV) * 64;
  rows = WAVES ? 256 / lanes_of_row(a.width) : 1;
}

template <class T, bool WAVES, int NV, bool LOW> int forward_and(const KgsAddNorm& a, hipStream_t s) {
  int threads, rows;
  shape<WAVES, NV>(a, threads, rows);
  const int want = (a.rows + rows - 1) / rows, grid = want < 8192 ? want : 8192;
  const auto go = [&](auto kernel) { kernel<<<grid, threads, 0, s>>>(a); };
  const bool full = is_full(a);
  if (a.width % kV == 0) full ? go(add_norm_fwd_kernel<T, WAVES, NV, true, LOW, kWhole>) : go(add_norm_fwd_kernel<T, WAVES, NV, false, LOW, kWhole>);
  else if (a.width > kV) full ? go(add_norm_fwd_kernel<T, WAVES, NV, true, LOW, kRagged>) : go(add_norm_fwd_kernel<T, WAVES, NV, false, LOW, kRagged>);
  else if constexpr (WAVES) full ? go(add_norm_fwd_kernel<T, WAVES, NV, true, LOW, kTiny>) : go(add_norm_fwd_kernel<T, WAVES, NV, false, LOW, kTiny>);
  return launched("add_norm forward");
}

template <class T, bool WAVES, int NV> int forward(const KgsAddNorm& a, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (a.low) return forward_and<T, WAVES, NV, true>(a, s);
  }
  return forward_and<T, WAVES, NV, false>(a, s);
}

template <class T, bool WAVES, int NV, bool STORED, int THREADS> int backward_from(const KgsAddNorm& a, hipStream_t s) {
  int threads, rows;
  shape<WAVES, NV>(a, threads, rows);
  const auto go = [&](auto kernel) { kernel<<<a.parts, threads, 0, s>>>(a); };
  const bool full = is_full(a);
  if (a.width % kV == 0) full ? go(add_norm_bwd_kernel<T, WAVES, NV, true, STORED, kWhole, THREADS>) : go(add_norm_bwd_kernel<T, WAVES, NV, false, STORED, kWhole, THREADS>);
  else if (a.width > kV) full ? go(add_norm_bwd_kernel<T, WAVES, NV, true, STORED, kRagged, THREADS>) : go(add_norm_bwd_kernel<T, WAVES, NV, false, STORED, kRagged, THREADS>);
  else if constexpr (WAVES) full ? go(add_norm_bwd_kernel<T, WAVES, NV, true, STORED, kTiny, THREADS>) : go(add_norm_bwd_kernel<T, WAVES, NV, false, STORED, kTiny, THREADS>);
  if (launched("add_norm backward")) return -1;
  if (a.parts == 1) return 0;
  const bool second = a.dpost_weight || a.dgate;
  add_norm_join_kernel<T><<<dim3((a.width + 15) / 16, second ? 2 : 1), 1024, 0, s>>>(a);
  return launched("add_norm join");
}

template <class T, bool WAVES, int NV, int THREADS> int backward(const KgsAddNorm& a, hipStream_t s) {
  return a.residual ? backward_from<T, WAVES, NV, false, THREADS>(a, s) : backward_from<T, WAVES, NV, true, THREADS>(a, s);
}

template <class T> int run(const KgsAddNorm& a, bool back, hipStream_t s) {
  if (a.width <= 512) return back ? backward<T, true, 1, 256>(a, s) : forward<T, true, 1>(a, s);
  // (forward of 16384 x 8192 with all weights: 197 us with one chunk a thread, 227 us with two)
  if (!back) return a.width <= 8192 ? forward<T, false, 1>(a, s) : forward<T, false, 2>(a, s);
  if (a.width <= 8192) return backward<T, false, 1, 1024>(a, s);
  // two chunks a thread need more than the 128 registers of 16 waves, and have them with 12
  if (a.width <= 12288) return backward<T, false, 2, 768>(a, s);
  return backward<T, false, 2, 1024>(a, s);
}

int dispatch(const KgsAddNorm* a, bool back, void* stream) {
  const char* w = "add_norm";
  if (!a || !a->branch || !a->weight) return fail(w, "a tensor is missing");
  if (!a->residual && (!back || !a->stream || (a->type != 2 && !a->low))) return fail(w, "a tensor is missing");
  if (!back && (!a->stream || !a->out)) return fail(w, "a tensor is missing");
  if (back && (!a->rstd || !a->dresidual || !a->dbranch || !a->dweight)) return fail(w, "a tensor is missing");
  if (back && ((a->post_weight && !a->dpost_weight) || (a->gate && !a->dgate))) return fail(w, "a tensor is missing");
  if (a->rows <= 0 || a->rows >= 1 << 30 || a->width <= 0 || a->width > 16384) return fail(w, "bad sizes");
  if (back && (a->parts < 1 || a->parts > 65536 || !a->partial)) return fail(w, "bad parts");
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
