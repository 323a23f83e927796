// attn.cuh — what the cache and attention kernels share: the device view of a cache and a batch,
// element types, argument checks and int8 -> fp16 conversion.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "api_export.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace acf {

// ------------------------------------------------------------------ device views
struct KvView {
  int8_t* k;
  int8_t* v;
  float* ks;
  float* vs;
  int pages, heads, page, dim, page_log2;
};

struct BatchView {
  const int32_t* table;
  const int32_t* start;
  const int32_t* length;
  int seqs, cols, tokens, max_new, max_len;
};

// One sequence of a batch.  A sequence whose entries are out of range is reported in the error
// word and comes out as empty (n = 0 when its rows are unusable, len = 0 when its length is).
struct SeqView {
  int row0, n, len;
};
__device__ __forceinline__ SeqView seq_view(const BatchView& b, int i, unsigned* err) {
  SeqView s;
  s.row0 = b.start[i];
  s.n = b.start[i + 1] - s.row0;
  s.len = b.length[i];
  if (s.row0 < 0 || s.n < 0 || s.n > b.max_new || s.row0 > b.tokens - s.n) {
    atomicOr(err, ACF_DEV_ERR_BADARG);
    s.n = 0;
  }
  if (s.len < 0 || s.len > b.max_len) {
    atomicOr(err, ACF_DEV_ERR_BADARG);
    s.len = 0;
  }
  return s;
}
// The page of token block g (of `page` tokens) of sequence i, or -1 (reported).
__device__ __forceinline__ int seq_page(const BatchView& b, int i, int g, int pages, unsigned* err) {
  const int p = b.table[(size_t)i * b.cols + g];
  if ((unsigned)p >= (unsigned)pages) {
    atomicOr(err, ACF_DEV_ERR_BADARG);
    return -1;
  }
  return p;
}

// ------------------------------------------------------------------ element types
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// Eight consecutive elements.  vec: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8]) {
  if (vec) {
    constexpr int W = 16 / sizeof(T);
    union {
      uint4 u;
      T t[W];
    } w;
#pragma unroll
    for (int i = 0; i < 8; i += W) {
      w.u = *reinterpret_cast<const uint4*>(p + i);
#pragma unroll
      for (int j = 0; j < W; ++j) x[i + j] = to_f(w.t[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f(p[i]);
  }
}
// The same in two steps, so that a load can be under way while other work is done.
template <typename T>
struct Raw8 {
  union {
    uint4 u[sizeof(T) / 2];
    T t[8];
  };
};
template <typename T>
__device__ __forceinline__ void load8_raw(const T* p, bool vec, Raw8<T>& r) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.t[i] = p[i];
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float (&x)[8]) {
  if (vec) {
    constexpr int W = 16 / sizeof(T);
    union {
      uint4 u;
      T t[W];
    } w;
#pragma unroll
    for (int i = 0; i < 8; i += W) {
#pragma unroll
      for (int j = 0; j < W; ++j) w.t[j] = from_f<T>(x[i + j]);
      *reinterpret_cast<uint4*>(p + i) = w.u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_f<T>(x[i]);
  }
}

// cos and sin of pos * f.  The product of a 31-bit integer and a 24-bit significand is taken in
// 64 bits and reduced by whole turns there, so a late position loses nothing; what is left is
// within half a turn and goes to the 32-bit functions.
__device__ __forceinline__ float2 rope_cs(int pos, float f, float amp) {
  const double a = (double)pos * (double)f;
  const double turns = rint(a * 0.15915494309189533577);
  const float r = (float)(a - turns * 6.28318530717958647693);
  float s, c;
  sincosf(r, &s, &c);
  return make_float2(c * amp, s * amp);
}

// Place of pair i in a token's row of cosines and sines: 8 pairs (a thread's) stay together, their four
// 16-byte quarters exchanged so that eight neighbouring threads read 128 different bytes at a time.
__device__ __forceinline__ int cs_place(int i) { return (i & ~6) | ((((i >> 1) ^ (i >> 4)) & 3) << 1); }

// ------------------------------------------------------------------ int8 -> fp16
// Four signed bytes, XORed with 0x80808080, are u = code + 128; a byte u put under the exponent
// byte 0x64 is the fp16 number 1024 + u, and subtracting 1152 is exact.
__device__ __forceinline__ uint32_t f16_from_u8(uint32_t w, uint32_t sel) {
  const uint32_t h = __byte_perm(w, 0x64646464u, sel);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// ------------------------------------------------------------------ host checks (kv8.cu)
inline size_t dtype_size(int dtype) { return dtype == ACFUN_F32 ? 4 : 2; }
// Each returns 0 or sets the error and returns its code.
int check_dtype(const char* what, int dtype, bool f32_ok);
int check_cache(const char* what, const AcfunKvCache8* c);
int check_batch(const char* what, const AcfunKvBatch* b, int page);
int check_rope(const char* what, const AcfunRope* r, int dim);
// Strides of a [tokens, heads, dim] tensor; an output's rows must not overlap.
int check_strides(const char* what, long long token, long long head, int tokens, int heads, int dim, bool output);
// Bytes from a tensor's address to its last element.
inline size_t span_bytes(long long token, long long head, int tokens, int heads, int dim, int dtype) {
  return (size_t)((tokens - 1) * token + (heads - 1) * head + dim) * dtype_size(dtype);
}
KvView cache_view(const AcfunKvCache8* c);
BatchView batch_view(Call& c, const AcfunKvBatch* b);  // index arrays resolved to device memory

// ------------------------------------------------------------------ attention (attn_kv8*.cu)
struct AttnArgs {
  KvView kv;
  BatchView b;
  const void* q;
  void* out;
  float* lse;
  long long q_token, q_head, o_token, o_head;
  int dtype, q_heads, group;  // group = q_heads / kv.heads
  float scale;
  int causal, window;
  // sequences whose rows (new tokens * group) are within [rows_least, rows_most] are this launch's
  long long rows_least, rows_most;
  bool beside;  // the launch before in the stream is k_attn_tc of the same call
};
__device__ __forceinline__ bool rows_taken(const AttnArgs& a, int rows) {
  return rows >= a.rows_least && rows <= a.rows_most;
}
bool attn_stream_dev(Call& c, const AttnArgs& a);  // any shape
// dim 64 or 128; *last_is_main: whether its last launch is k_attn_tc
bool attn_tc_dev(Call& c, const AttnArgs& a, bool* last_is_main);

}  // namespace acf
