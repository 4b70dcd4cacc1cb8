// C interface of libkgs_decoder.so (loaded with ctypes by kube_gpu_stats_amd/ops/decoder.py,
// whose struct formats repeat these layouts field by field; none has padding at its end,
// which a packed block would lack and an entry copy).  Every entry launches on `stream`,
// returns 0, or -1 with kgs_decoder_last_error() set.
#pragma once
#include <cstddef>
#include <cstdint>

extern "C" {

// Tensors [B, S, heads, D]; strides in elements of (B, S, heads), D contiguous; pointers
// 16-byte aligned, strides multiples of 8.  lse: float [B, H, S],
// delta: float [B, H, ceil(S / 32), 2, 32], for float16 then [B, Hk, ceil(S / 128)] and
// [B, H, ceil(S / 32)] (workspace).  low: [B, S, H, D], what rounding
// took from out, a signed byte of 256ths of its last place.  The forward pass writes lse and low if they
// are not null.
struct KgsAttention {
  const void *q, *k, *v;
  void* out;
  const void* dout;
  void *dq, *dk, *dv;
  float *lse, *delta, *partial;  // partial: float [splits, 2, B, S, Hk, D]
  uint8_t* low;
  const int32_t* lengths;        // [B] or null
  int64_t q_st[3], k_st[3], v_st[3], o_st[3], g_st[3], dq_st[3], dk_st[3], dv_st[3];
  int32_t B, S, H, Hk, D, type, causal, splits, unused;  // type: 0 bfloat16, 1 float16
  float scale;
};
static_assert(sizeof(KgsAttention) == offsetof(KgsAttention, scale) + 4, "padding at the end");

// x [T, K] and w [2F, K] with row strides, h [T, F], saved [T, 6F] bytes (null: not kept), dh [T, F]
// with a row stride, dgu [T, 2F], dx [T, K], dw [2F, K] (either null: not wanted).  Pointers
// 16-byte aligned; K, F and strides multiples of 8.  tile, splits: of the forward product,
// of dx and of dw.  partial: float [splits, rows, columns] of the largest split product.
struct KgsSwiglu {
  const void *x, *w;
  void *h, *saved;
  const void* dh;
  void *dgu, *dx, *dw;
  float* partial;
  int64_t x_ld, w_ld, dh_ld;
  int32_t T, K, F, type;
  int32_t tile[3], splits[3];
};
static_assert(sizeof(KgsSwiglu) == offsetof(KgsSwiglu, splits) + 12, "padding at the end");

// Rows of `width` elements; row strides in elements.  rstd float [2, rows] (of the stream, of
// the branch); dstream and dout may be null (zero).  post_weight and gate may be null.
// partial: float [parts, 2, width], parts the workgroups of the backward.
// dbranch may equal dresidual where they are the same.
// The backward starts from residual and branch or, where residual is null, from the stream
// (contiguous, as the forward wrote it) and low [rows, width]: what rounding took from the
// stream of a 16-bit type, bytes as attention's.  The forward writes low if it is not null.
struct KgsAddNorm {
  const void *residual, *branch, *weight, *post_weight, *gate;
  void *stream, *out;
  float* rstd;
  const void *dstream, *dout;
  void *dresidual, *dbranch, *dweight, *dpost_weight, *dgate;
  float* partial;
  int64_t residual_ld, branch_ld, stream_ld, dstream_ld, dout_ld;
  int32_t rows, width, type, parts;  // type: 0 bfloat16, 1 float16, 2 float32
  uint8_t* low;
  float scale, eps;
};
static_assert(sizeof(KgsAddNorm) == offsetof(KgsAddNorm, eps) + 4, "padding at the end");

const char* kgs_decoder_last_error();
int kgs_swiglu_fwd(const KgsSwiglu* a, void* stream);
int kgs_swiglu_bwd(const KgsSwiglu* a, void* stream);
int kgs_add_norm_fwd(const KgsAddNorm* a, void* stream);
int kgs_add_norm_bwd(const KgsAddNorm* a, void* stream);
int kgs_attention_fwd(const KgsAttention* a, void* stream);
int kgs_attention_bwd(const KgsAttention* a, void* stream);
}
