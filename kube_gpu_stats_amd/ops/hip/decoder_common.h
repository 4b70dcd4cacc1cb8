// What the decoder block's kernels share on gfx950: element types and their matrix
// instruction, buffer descriptors whose range check keeps every load in bounds, copies
// from memory straight into LDS, and the swizzled tile that both row-wise and
// transposed fragment reads walk without bank conflicts.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace kgs {

using bf16 = __bf16;
using f16 = _Float16;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using i32x4 = __attribute__((ext_vector_type(4))) int;
using u32x2 = __attribute__((ext_vector_type(2))) unsigned;

constexpr int kWave = 64;
constexpr float kLog2e = 1.44269504088896340736f;

template <class T> struct El;
template <> struct El<bf16> {
  using x2 = __attribute__((ext_vector_type(2))) bf16;
  using x4 = __attribute__((ext_vector_type(4))) bf16;
  using x8 = __attribute__((ext_vector_type(8))) bf16;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ x4 read_tr(const char* lds) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) x4*)lds);
  }
};
template <> struct El<f16> {
  using x2 = __attribute__((ext_vector_type(2))) f16;
  using x4 = __attribute__((ext_vector_type(4))) f16;
  using x8 = __attribute__((ext_vector_type(8))) f16;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ x4 read_tr(const char* lds) {
    using i16x4 = __attribute__((ext_vector_type(4))) short;
    return __builtin_bit_cast(x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)lds));
  }
};

template <class T> __device__ __forceinline__ typename El<T>::x8 join(typename El<T>::x4 a, typename El<T>::x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A raw buffer descriptor over [base, base + bytes): a lane's access past it reads 0 or
// stores nothing, dword by dword.  Offsets are 32 bits, so callers move the base (64
// bits) from tile to tile and keep offsets inside one tile (under 2^30); an offset of
// kFar is past the end of any.
constexpr uint32_t kFar = 0x7FFFFFE0u;
__device__ __forceinline__ i32x4 buffer(const void* base, int64_t bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  bytes = bytes < 0 ? 0 : bytes;
  const uint32_t n = bytes > kFar ? kFar : static_cast<uint32_t>(bytes);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(p));
  r[1] = __builtin_amdgcn_readfirstlane(static_cast<int>(p >> 32) & 0xFFFF);
  r[2] = __builtin_amdgcn_readfirstlane(static_cast<int>(n));
  r[3] = 0x00027000;
  return r;
}

// A descriptor that walks through a matrix: `step` bytes further each time, and as many
// fewer to the end.  Few scalar instructions: they stand between a workgroup's products.
struct Walk {
  uint64_t base;
  int64_t left;
  __device__ __forceinline__ Walk() {}
  __device__ __forceinline__ Walk(const void* p, int64_t bytes) : base(reinterpret_cast<uint64_t>(p)), left(bytes) {}
  __device__ __forceinline__ void go(int64_t step) {
    base += step;
    left -= step;
  }
  __device__ __forceinline__ i32x4 descriptor() const {
    const int high = static_cast<int>(left >> 32);
    const uint32_t low = static_cast<uint32_t>(left);
    const uint32_t some = high > 0 || low > kFar ? kFar : low;
    return i32x4{static_cast<int>(base), static_cast<int>(base >> 32) & 0xFFFF, high < 0 ? 0 : static_cast<int>(some),
                 0x00027000};
  }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(i32x4 d) {
  const uint64_t p = static_cast<uint32_t>(d[0]) | (static_cast<uint64_t>(static_cast<uint32_t>(d[1])) << 32);
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(p), 0, d[2], 0x00027000);
}

template <class V> __device__ __forceinline__ V load16(i32x4 d, int voff) {
  return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(rsrc(d), voff, 0, 0));
}

// 16 bytes a lane; past the descriptor's end nothing.  (A test of the row instead keeps the
// compiler from reading several rows out of LDS before the first is stored.)
__device__ __forceinline__ void store16(i32x4 v, i32x4 d, int voff) {
  using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rsrc(d), voff, 0, 0);
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p));
}

// 16 (or 4) bytes a lane from memory to LDS at lds + lane * 16 (or 4); lds must be the
// same in the whole wave.  Written as assembly because the compiler, which cannot tell
// the buffer being filled from the one being read, would wait for the copy before the
// next LDS read; there is no result register, and copies_done() is the wait.  The s_nop
// covers what the compiler would: a scalar register written by a vector instruction (the
// descriptor's readfirstlane) is not read by a memory instruction within 5 states.
__device__ __forceinline__ void copy16(i32x4 d, int voff, uint32_t lds, int soff = 0) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(d), "s"(soff)
               : "memory", "m0");
}
__device__ __forceinline__ void copy4(i32x4 d, int voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(d)
               : "memory", "m0");
}
// Waits until none of the wave's copies is under way.
__device__ __forceinline__ void copies_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// The same wait in a form the compiler knows: what it loaded before is there, and it puts
// no wait of its own for that into the loop that follows.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }

__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Between a wave's writes to LDS and the reads of them by its other lanes, and before it writes
// there again.  The hardware does one wave's LDS operations in order; this keeps the
// compiler, which looks at one lane's addresses, from changing the order.  No instruction.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A tile of rows of W elements (W = 64 or 128) in LDS, in 16-byte chunks, chunk c of a
// row at c ^ swizzle(row).  256 bytes (all 64 banks) are one row of 128 or two of 64.
// Row-wise reads take the same chunk of 32 rows: 16 rows in turn land on 16 places.
// Transposed reads take 64 bytes of 4 rows in turn: the swizzle's high bits come from
// the row's low ones, so that the four lie in different quarters of the 256 bytes.
template <int W> struct Tile {
  static constexpr int kRow = W * 2;
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (W == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    else return ((row & 2) << 1) | ((row >> 2) & 3);
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * kRow + ((chunk ^ swizzle(row)) << 4); }

  // Lane's fragment of rows r0..r0+31, elements 16 kk..16 kk + 15: row lane % 32,
  // 8 elements from 16 kk + 8 (lane / 32).
  template <class T> static __device__ __forceinline__ typename El<T>::x8 rows(const char* t, int r0, int kk, int lane) {
    return *reinterpret_cast<const typename El<T>::x8*>(t + r0 * kRow + at(lane & 31, kk * 2 + (lane >> 5)));
  }
  // The transposed fragment in the order of rows(): lane holds element e0 + lane % 32 of
  // rows r0 + 8 (lane / 32) + {0..7}.
  template <class T> static __device__ __forceinline__ typename El<T>::x8 columns_in_order(const char* t, int r0, int e0,
                                                                                           int lane) {
    const int i = lane & 15, row = (lane >> 5) * 8 + (i >> 2);
    const int chunk = (e0 >> 3) + ((lane >> 4) & 1) * 2 + ((i >> 1) & 1);
    const char* p = t + r0 * kRow + (i & 1) * 8;
    return join<T>(El<T>::read_tr(p + at(row, chunk)), El<T>::read_tr(p + at(row + 4, chunk)));
  }
  // The transposed fragment: lane holds element e0 + lane % 32 of 8 rows, the rows
  // that an accumulator of the 32x32 product keeps in its registers 8 h .. 8 h + 7:
  // r0 + 4 (lane / 32) + {0..3} and 8 more.  r0 a multiple of 16.
  template <class T> static __device__ __forceinline__ typename El<T>::x8 columns(const char* t, int r0, int e0, int lane) {
    const int i = lane & 15, row = (lane >> 5) * 4 + (i >> 2);
    const int chunk = (e0 >> 3) + ((lane >> 4) & 1) * 2 + ((i >> 1) & 1);
    const char* p = t + r0 * kRow + (i & 1) * 8;
    return join<T>(El<T>::read_tr(p + at(row, chunk)), El<T>::read_tr(p + at(row + 8, chunk)));
  }
  // Wave w of NW copies its part of ROWS rows, stride bytes apart in memory, to LDS.
  template <int ROWS, int NW> struct Copy {
    static constexpr int kAll = ROWS * kRow / 1024, kN = (kAll + NW - 1) / NW;
    int voff[kN];
    __device__ __forceinline__ void init(int wave, int lane, int64_t stride) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int byte = (wave * kN + i) * 1024 + lane * 16, row = byte / kRow, pc = (byte >> 4) & (W / 8 - 1);
        voff[i] = static_cast<int>(row * stride) + ((pc ^ swizzle(row)) << 4);
      }
    }
    __device__ __forceinline__ void go(i32x4 d, uint32_t lds, int wave, int soff = 0) const {
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (kAll % NW == 0 || wave * kN + i < kAll) copy16(d, voff[i], lds + (wave * kN + i) * 1024, soff);
    }
  };
};

// A 32-bit value x as a result keeps it, r rounded to T, and a byte: how many
// 256ths of r's last place x is above r, rounded down.  As numbers of 32 bits they differ
// by an integer of up to half a last place, 2^15 for bf16 and 2^12 for fp16; the upper
// half is left out (a tie rounded down), and what fp16 rounds off below its normal range
// is cut to that.  (In place of the difference times its exponent: attention forward of 4 x
// 2048, 32 heads, 164.6 us to 163.1 us, of which the bytes cost 11 us.)
template <class T> constexpr int kLowShift = __is_same(T, bf16) ? 8 : 5;
template <class T> __device__ __forceinline__ uint32_t low_of(float x) {  // in bits 8 to 15
  const int d = __builtin_bit_cast(int, x) - __builtin_bit_cast(int, static_cast<float>(static_cast<T>(x)));
  constexpr int most = 128 << kLowShift<T>;
  return static_cast<uint32_t>(min(max(d, -most), most - 1)) << (8 - kLowShift<T>);
}
// x again, to half of a 256th
template <class T> __device__ __forceinline__ float with_low(T r, int low) {
  return __builtin_bit_cast(float, __builtin_bit_cast(int, static_cast<float>(r)) + (low << kLowShift<T>) +
                                       (1 << (kLowShift<T> - 1)));
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

// Workgroup id -> work item so that neighbouring items run on one of the 8 XCDs (ids
// go round them in turn) and share its L2.  Returns total or more for no work.
__device__ __forceinline__ int64_t xcd_item(int64_t id, int64_t total) {
  const int64_t per = (total + 7) / 8;
  return (id & 7) * per + (id >> 3);
}

// The same for `heads` heads of `ranks` pieces each, the longest piece first (rank 0).
// An XCD takes whole heads: their pieces read the same keys.  It goes through `group`
// heads at a time rank by rank: where pieces differ in length (causal) the short ones of
// 16 heads fill up the end (forward of 4 x 32 heads, 2048 positions: 192 us, 208 us head
// by head); where they do not, head by head keeps fewer keys in the L2 in use (280 us,
// 297 us by 16).  The heads that are left when 8 do not divide them are dealt to the
// XCDs piece by piece, so that none has more than its share; so are all of them (deal)
// where sequences differ in length, or an XCD could hold the long ones' heads.
__host__ __device__ __forceinline__ int64_t head_items(int64_t heads, int64_t ranks, bool deal) {
  const int64_t left = deal ? heads : heads % 8;
  return 8 * ((left * ranks + 7) / 8 + (heads - left) / 8 * ranks);
}
__device__ __forceinline__ bool head_item(int id, int heads, int ranks, int group, bool deal, int& head, int& rank) {
  const int x = id & 7, left = deal ? heads : heads & 7, own = (heads - left) >> 3, dealt = (left * ranks + 7) / 8;
  int k = id >> 3;
  if (k < dealt) {
    const int i = k * 8 + x;
    if (i >= left * ranks) return false;
    rank = i / left;
    head = heads - left + i % left;
    return true;
  }
  k -= dealt;
  const int g = k / (group * ranks), size = min(group, own - g * group), in = k - g * group * ranks;
  rank = in / size;
  head = x * own + g * group + in % size;
  return true;
}

// Error text of the calling thread's last failed entry, and its setter.
extern thread_local char g_decoder_error[256];
int fail(const char* what, const char* why);
int launched(const char* what);

}  // namespace kgs
