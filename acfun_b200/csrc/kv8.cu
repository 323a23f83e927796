// kv8.cu — the int8 key / value cache: tokens quantised into their pages (acfun_kv8_append), read
// back as values (acfun_kv8_read), and the argument checks the cache's functions share.
//
// A scale covers the `page` tokens of one page and head, so one block sees all the new tokens of
// a (page, head) and nothing is exchanged between blocks:
//   s = max(max|x|, 127 * 2^-60) / 127, code = rint(x * (1 / s)) clamped to +-127;
// in a page that holds older tokens s does not shrink, and when it grows, their codes are moved
// to it in the same block.  The values wait in registers between the maximum and the coding, so they
// are read once; the next head's are requested meanwhile.  1 / s is rounded once and multiplied by, as
// the definition says, not divided by: a tie may fall to the other side of it, by half a code.
//
// Measured (B200, bf16, 8 heads of 128): append of 65551 tokens with rotation 99 us, 4.1 TB/s of what
// it has to move, 62 % of the measured copy rate: bound by instructions (18 per value; a page of 128
// tokens takes a block of 1024 threads, whose barrier per head shows, and whose 64 registers per thread
// hold for the smaller blocks too: 16 to 44 bytes are spilled, and 208 to 496 with heads of 256).  The same
// in fp32 145 us (its bytes take 103), with heads of 256 270 us in bf16 (123) and 450 in fp32 (206).  Read of 24 prefixes of 500 to
// 8191 tokens 84 us, 6.0 TB/s, 92 % of the measured copy rate.
#include <algorithm>

#include "attn.cuh"

namespace acf {

// ------------------------------------------------------------------ host checks
int check_dtype(const char* what, int dtype, bool f32_ok) {
  if (dtype == ACFUN_F16 || dtype == ACFUN_BF16 || (f32_ok && dtype == ACFUN_F32)) return 0;
  set_error(kInvalid, "%s: dtype %d is not %sfp16 or bf16", what, dtype, f32_ok ? "fp32, " : "");
  return kInvalid;
}

int check_cache(const char* what, const AcfunKvCache8* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) {
    set_error(kInvalid, "%s: the cache or one of its arrays is NULL", what);
    return kInvalid;
  }
  if (c->pages <= 0 || c->heads <= 0 || c->heads > 4096) {
    set_error(kInvalid, "%s: pages %d must be positive and heads %d within [1, 4096]", what, c->pages, c->heads);
    return kInvalid;
  }
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) {
    set_error(kInvalid, "%s: page %d is not 16, 32, 64 or 128", what, c->page);
    return kInvalid;
  }
  if (c->dim != 64 && c->dim != 128 && c->dim != 256) {
    set_error(kInvalid, "%s: dim %d is not 64, 128 or 256", what, c->dim);
    return kInvalid;
  }
  if (!aligned16(c->k) || !aligned16(c->v) || ((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3) {
    set_error(kInvalid, "%s: codes must be 16-byte aligned, scales 4-byte aligned", what);
    return kInvalid;
  }
  if (ptr_kind(c->k) != PtrKind::Device || ptr_kind(c->v) != PtrKind::Device ||
      ptr_kind(c->k_scale) != PtrKind::Device || ptr_kind(c->v_scale) != PtrKind::Device) {
    set_error(kInvalid, "%s: the cache must be device memory", what);
    return kInvalid;
  }
  return 0;
}

int check_batch(const char* what, const AcfunKvBatch* b, int page) {
  if (!b || b->seqs < 0 || b->tokens < 0 || b->max_new < 0 || b->max_len < 0 || b->table_cols < 0) {
    set_error(kInvalid, "%s: the batch is NULL or has a negative size", what);
    return kInvalid;
  }
  if (b->seqs > 65535) {
    set_error(kInvalid, "%s: %d sequences, at most 65535", what, b->seqs);
    return kInvalid;
  }
  if (b->seqs > 0 && (!b->start || !b->length || (!b->table && b->table_cols > 0))) {
    set_error(kInvalid, "%s: an index array of the batch is NULL", what);
    return kInvalid;
  }
  if ((long long)b->table_cols * page < b->max_len) {
    set_error(kInvalid, "%s: %d table columns of %d tokens do not reach max_len %d", what, b->table_cols, page,
              b->max_len);
    return kInvalid;
  }
  if (b->max_len > (1 << 30) || b->max_new > (1 << 30)) {
    set_error(kInvalid, "%s: max_len and max_new are at most 2^30", what);
    return kInvalid;
  }
  return 0;
}

int check_strides(const char* what, long long token, long long head, int tokens, int heads, int dim, bool output) {
  const long long lim = 1LL << 46;
  bool ok = token >= 0 && head >= 0 && token < lim && head < lim && (long long)heads * dim < (1LL << 27);
  if (ok && output) {
    const bool token_major = (tokens <= 1 || token >= (long long)(heads - 1) * head + dim) && (heads <= 1 || head >= dim);
    const bool head_major = (heads <= 1 || head >= (long long)(tokens - 1) * token + dim) && (tokens <= 1 || token >= dim);
    ok = token_major || head_major;
  }
  if (ok) return 0;
  set_error(kInvalid, "%s: strides %lld (token) and %lld (head) of [%d, %d, %d] are negative, too large or overlap", what,
            token, head, tokens, heads, dim);
  return kInvalid;
}

KvView cache_view(const AcfunKvCache8* c) {
  const int lg = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
  return {c->k, c->v, c->k_scale, c->v_scale, c->pages, c->heads, c->page, c->dim, lg};
}

BatchView batch_view(Call& c, const AcfunKvBatch* b) {
  BatchView v = {};
  v.table = (const int32_t*)c.in(b->table, (size_t)b->seqs * b->table_cols * 4);
  v.start = (const int32_t*)c.in(b->start, ((size_t)b->seqs + 1) * 4);
  v.length = (const int32_t*)c.in(b->length, (size_t)b->seqs * 4);
  v.seqs = b->seqs, v.cols = b->table_cols, v.tokens = b->tokens, v.max_new = b->max_new, v.max_len = b->max_len;
  return v;
}

namespace {

// ------------------------------------------------------------------ append
struct AppendArgs {
  KvView kv;
  BatchView b;
  const void* k;
  const void* v;
  long long k_token, k_head, v_token, v_head;
  int vec;  // k and v can be read 16 bytes at a time
  const float* freq;
  int rot, interleaved;
  float amp;
  int head_block;  // heads of one block
  int per_head;    // threads of one head: whole warps, enough for the new tokens that a page can get
};

// The larger of |a| and |b|, of either sign; NaN when either is.
__device__ __forceinline__ float amax_nan(float a, float b) {
  float d;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// x / 127 rounded to nearest: the quotient by the rounded reciprocal, corrected once by its exact
// remainder (Markstein's theorem on division with fused multiply-add; x is far from both ends of
// the range).
__device__ __forceinline__ float div127(float x) {
  constexpr float y = 1.0f / 127.0f;
  const float q = __fmul_rn(x, y);
  return __fmaf_rn(__fmaf_rn(-127.0f, q, x), y, q);
}
// The largest over a warp.
__device__ __forceinline__ float warp_max_nan(float a) {
  float d;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(a));
  return d;
}
constexpr float kFinite = 3.4028234663852886e38f;

// rint(x * unit) of eight values, |x * unit| < 127.5, as bytes: adding 1.5 * 2^23 rounds to an integer
// (ties to even, as rint) that stands in the sum's low byte.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float unit) {
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], unit), 12582912.0f));
  return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// n words of 8 codes, coded under `before`, moved to `scale`.  Out of line, so that what it needs is not
// prepared for every head.
__device__ __noinline__ void move_codes(int8_t* codes, int n, float before, float scale, int tid, int threads) {
  const float f = __fdiv_rn(before, scale);
  uint2* w = reinterpret_cast<uint2*>(codes);
  for (int i = tid; i < n; i += threads) {
    const uint2 v = w[i];
    float y[8];
#pragma unroll
    for (int b = 0; b < 4; ++b) y[b] = (float)(int8_t)(v.x >> (8 * b)), y[4 + b] = (float)(int8_t)(v.y >> (8 * b));
    w[i] = codes8(y, f);
  }
}

template <int DIM>
constexpr int kUnits = DIM == 256 ? 2 : 1;

// One block: page slot blockIdx.x of the new tokens of sequence blockIdx.z, heads
// [blockIdx.y / 2 * head_block, ...), keys (blockIdx.y even) or values (odd).  A head takes the threads
// that a page's share of max_new tokens needs, so that small pages and single tokens have several
// heads in a block at a time.  A thread holds a
// unit of 16 elements of the tile (two of them when dim is 256) in registers between the maximum and
// the coding: two runs of 8 elements, which in the half layout are the two sides of 8 pairs.
template <typename T, int DIM, bool VEC>
__global__ void __launch_bounds__(1024) k_kv8_append(const AppendArgs a, unsigned* err) {
  extern __shared__ __align__(16) float2 cs[];  // [tokens in this page][rot / 2], keys only
  __shared__ float warp_max[2][2][32];
  constexpr int UPR = DIM / 16;  // units per row
  constexpr int UN = kUnits<DIM>;
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  const int seq = blockIdx.z, page = a.kv.page;
  const bool is_v = blockIdx.y & 1;
  const SeqView sv = seq_view(a.b, seq, err);
  const int first = sv.len - sv.n;  // position of the first new token
  if (sv.n <= 0) return;
  if (first < 0) {  // more new tokens than the sequence holds (or a length out of range)
    if (threadIdx.x == 0) atomicOr(err, ACF_DEV_ERR_BADARG);
    return;
  }
  const int g = first / page + blockIdx.x;           // this block's page of the sequence
  if (g * (long long)page >= sv.len) return;
  const int lo = max(first - g * page, 0), hi = min(sv.len - g * page, page);  // new slots [lo, hi)
  const int row_of_slot0 = sv.row0 + g * page - first;  // packed row of slot 0 (may be before row0)
  const int h0 = (blockIdx.y >> 1) * a.head_block, h1 = min(h0 + a.head_block, a.kv.heads);
  const int half = a.rot / 2;
  const bool turn = !is_v && a.rot > 0;
  const int per_head = a.per_head, group = threadIdx.x / per_head, groups = blockDim.x / per_head;
  const int tid = threadIdx.x - group * per_head;
  // this thread's units: slot and the element offsets of their two runs
  int slot[UN], at0[UN], at1[UN], cs_at[UN], cs_x[UN];
#pragma unroll
  for (int j = 0; j < UN; ++j) {
    const int idx = tid + j * per_head;
    const int u = idx % UPR;
    slot[j] = lo + idx / UPR;
    cs_at[j] = -1, cs_x[j] = (u >> 1) & 3;
    if (turn && !a.interleaved) {
      const int pairs = a.rot / 16;
      if (u < pairs) {
        at0[j] = 8 * u, at1[j] = 8 * u + half;
        cs_at[j] = (slot[j] - lo) * half + 8 * u;
      } else {
        at0[j] = a.rot + 16 * (u - pairs), at1[j] = at0[j] + 8;
      }
    } else {
      at0[j] = 16 * u, at1[j] = 16 * u + 8;
      if (turn && at0[j] < a.rot) cs_at[j] = (slot[j] - lo) * half + 8 * u;
    }
  }
  const T* src = static_cast<const T*>(is_v ? a.v : a.k);
  const long long tok_stride = is_v ? a.v_token : a.k_token, head_stride = is_v ? a.v_head : a.k_head;
  int8_t* codes = is_v ? a.kv.v : a.kv.k;
  float* scales = is_v ? a.kv.vs : a.kv.ks;

  const int w0 = group * per_head / 32, w1 = w0 + per_head / 32;  // the head's warps
  Raw8<T> raw[UN][2];
  bool in[UN];
  const T* from[UN];  // of the next head to request
  int8_t* to[UN];     // of the head at hand
  const long long from_step = groups * head_stride, to_step = (long long)groups * page * DIM;
#pragma unroll
  for (int j = 0; j < UN; ++j) {
    in[j] = slot[j] >= lo && slot[j] < hi;
    from[j] = src + (long long)(row_of_slot0 + slot[j]) * tok_stride + (h0 + group) * head_stride;
  }
  auto request = [&](int h) {
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      if (h < h1 && in[j]) {
        load8_raw(from[j] + at0[j], VEC, raw[j][0]);
        load8_raw(from[j] + at1[j], VEC, raw[j][1]);
      } else {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[j][0].u[i] = raw[j][1].u[i] = make_uint4(0, 0, 0, 0);
      }
      from[j] += from_step;
    }
  };
  // the first values, the page's number and the angles are on their way together
  request(h0 + group);
  const int pid = seq_page(a.b, seq, g, a.kv.pages, err);
  if (pid < 0) return;
  size_t sc = (size_t)pid * a.kv.heads + h0 + group;
#pragma unroll
  for (int j = 0; j < UN; ++j) to[j] = codes + sc * page * DIM + slot[j] * DIM;
  if (turn) {
    // A thread takes a pair's run of consecutive tokens: the first angle is computed, the others
    // are turned on from it by one position's angle (at most 127 turns, each within 2^-23).
    const int n = hi - lo, runs = max(1, (int)blockDim.x / half), len = (n + runs - 1) / runs;
    for (int i = threadIdx.x; i < half * runs; i += blockDim.x) {
      const int t0 = i / half * len, pair = i % half;
      if (t0 >= n) continue;
      const float f = a.freq[pair];
      float2 w = rope_cs(g * page + lo + t0, f, a.amp);
      const float2 one = len > 1 ? rope_cs(1, f, 1.0f) : make_float2(1.0f, 0.0f);
      for (int t = t0; t < min(t0 + len, n); ++t) {
        cs[t * half + cs_place(pair)] = w;
        w = make_float2(w.x * one.x - w.y * one.y, w.y * one.x + w.x * one.y);
      }
    }
    __syncthreads();
  }
  for (int hb = h0, buf = 0; hb < h1; hb += groups, buf ^= 1) {
    const bool mine = hb + group < h1;  // a group without a head of its own only keeps the barriers
    float x[UN][2][8];
    float top = 127.0f * 0x1p-60f;
#pragma unroll
    for (int j = 0; j < UN; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][r][i] = to_f(raw[j][r].t[i]);
    request(hb + groups + group);  // the next head's values, while this one's are worked on
    const float before = lo > 0 && mine ? scales[sc] : 0.0f;
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      if (in[j] && cs_at[j] >= 0) {
        const float4* w = reinterpret_cast<const float4*>(cs + cs_at[j]);  // 8 pairs from a multiple of 8
        if (a.interleaved) {
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float4 c = w[((4 * r + i) / 2) ^ cs_x[j]];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float cc = k ? c.z : c.x, ss = k ? c.w : c.y;
                const float p = x[j][r][2 * (i + k)], q = x[j][r][2 * (i + k) + 1];
                x[j][r][2 * (i + k)] = p * cc - q * ss;
                x[j][r][2 * (i + k) + 1] = q * cc + p * ss;
              }
            }
        } else {
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float4 c = w[(i / 2) ^ cs_x[j]];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float cc = k ? c.z : c.x, ss = k ? c.w : c.y;
              const float p = x[j][0][i + k], q = x[j][1][i + k];
              x[j][0][i + k] = p * cc - q * ss;
              x[j][1][i + k] = q * cc + p * ss;
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = amax_nan(top, x[j][r][i]);
    }
    // the head's maximum; the buffers alternate so that one barrier per round is enough
    top = warp_max_nan(fabsf(top));
    if ((threadIdx.x & 31) == 0) warp_max[0][buf][threadIdx.x >> 5] = top;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const float m = lane < (int)blockDim.x / 32 ? warp_max[0][buf][lane] : 0.0f;  // at most 32 warps
    const bool finite = __all_sync(0xffffffffu, m <= kFinite);
    top = warp_max_nan(lane >= w0 && lane < w1 ? m : 0.0f);
    if (__builtin_expect(!finite, 0)) {  // somewhere in the block: all look for their finite maximum
      top = 127.0f * 0x1p-60f;
#pragma unroll
      for (int j = 0; j < UN; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (x[j][r][i] != x[j][r][i]) x[j][r][i] = 0.0f;
            if (fabsf(x[j][r][i]) <= kFinite) top = fmaxf(top, fabsf(x[j][r][i]));
          }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if ((threadIdx.x & 31) == 0) warp_max[1][buf][threadIdx.x >> 5] = top;
      __syncthreads();
      for (int w = w0; w < w1; ++w) top = fmaxf(top, warp_max[1][buf][w]);
    }
    const float scale = fmaxf(before, div127(top));
    const float unit = __frcp_rn(scale);
    if (__builtin_expect(!finite, 0)) {
#pragma unroll
      for (int j = 0; j < UN; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (fabsf(x[j][r][i]) > kFinite) x[j][r][i] = copysignf(scale * 127.0f, x[j][r][i]);
    }
    if (__builtin_expect(lo > 0, 0)) {  // older tokens of the page move to a larger scale
      if (mine && scale > before) move_codes(to[0] - slot[0] * DIM, lo * (DIM / 8), before, scale, tid, per_head);
    }
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      int8_t* o = to[j];
      to[j] += to_step;
      if (!mine || !in[j]) continue;
      const uint2 c0 = codes8(x[j][0], unit), c1 = codes8(x[j][1], unit);
      if (at1[j] == at0[j] + 8) {
        *reinterpret_cast<uint4*>(o + at0[j]) = make_uint4(c0.x, c0.y, c1.x, c1.y);
      } else {
        *reinterpret_cast<uint2*>(o + at0[j]) = c0;
        *reinterpret_cast<uint2*>(o + at1[j]) = c1;
      }
    }
    // every thread has read the old scale before the barrier above
    if (mine && tid == 0) scales[sc] = scale;
    sc += groups;
  }
  // new tokens past the last page slot of the grid
  if (threadIdx.x == 0 && blockIdx.x == gridDim.x - 1 && (g + 1) * (long long)page < sv.len)
    atomicOr(err, ACF_DEV_ERR_BADARG);
}

template <typename T, int DIM, bool VEC>
bool append_run(Call& c, AppendArgs a) {
  const int page = a.kv.page;
  const int per_head = (std::min(page, a.b.max_new) * DIM / (16 * kUnits<DIM>) + 31) / 32 * 32;
  a.per_head = per_head;
  // pages that a run of max_new tokens can touch
  const int slots = std::max(1, (std::min(a.b.max_new, a.b.max_len) + page - 2) / page + 1);
  // All heads of a page in one block share its cosines and sines; with few pages the heads go to
  // blocks of their own, which recompute them but fill the machine.
  const long long pages = (long long)slots * a.b.seqs;
  int parts = (int)std::min<long long>(a.kv.heads, std::max<long long>(1, 4LL * c.sm_count() / std::max<long long>(1, pages)));
  a.head_block = std::min(a.kv.heads, std::max((a.kv.heads + parts - 1) / parts, 128 / per_head));
  parts = (a.kv.heads + a.head_block - 1) / a.head_block;
  const int threads = per_head * std::max(1, std::min(a.head_block, 256 / per_head));
  const size_t smem = (size_t)std::min(page, a.b.max_new) * (a.rot / 2) * sizeof(float2);
  // The most that any call takes is asked for at the first one: 48 KiB hold without asking, but for the
  // static arrays too.
  static bool attr_done[64] = {false};
  const int dv = current_device() & 63;
  if (!attr_done[dv]) {
    if (!ACF_CUDA_OK(cudaFuncSetAttribute(k_kv8_append<T, DIM, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          128 * (DIM / 2) * (int)sizeof(float2))))
      return false;
    attr_done[dv] = true;
  }
  if (!ACF_CUDA_OK(launch_pdl(k_kv8_append<T, DIM, VEC>, dim3(slots, 2 * parts, a.b.seqs), dim3(threads), smem, c.stream(), a,
                              c.err())))
    return false;
  return c.launched("k_kv8_append");
}
template <typename T, int DIM>
bool append_launch(Call& c, const AppendArgs& a) {
  return a.vec ? append_run<T, DIM, true>(c, a) : append_run<T, DIM, false>(c, a);
}

// ------------------------------------------------------------------ read
// Byte i of a word of codes, each XORed with 0x80, as a float: under the exponent of 2^23 it is
// 2^23 + code + 128, and the difference is exact.
__device__ __forceinline__ float code_value(uint32_t w, int i) {
  return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650 | i)) - 8388736.0f;
}
struct ReadArgs {
  KvView kv;
  BatchView b;
  void* k;
  void* v;
  int head_block;
};

// One block: page slot blockIdx.x of the tokens wanted of sequence blockIdx.z, `head_block` heads
// of it.  Codes of neighbouring heads are contiguous; a thread turns 16 codes into values.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) k_kv8_read(const ReadArgs a, unsigned* err) {
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  const int seq = blockIdx.z, page = a.kv.page;
  const SeqView sv = seq_view(a.b, seq, err);
  const int first = sv.len - sv.n;
  if (sv.n <= 0) return;
  if (first < 0) {
    if (threadIdx.x == 0) atomicOr(err, ACF_DEV_ERR_BADARG);
    return;
  }
  const int g = first / page + blockIdx.x;
  if (g * (long long)page >= sv.len) return;
  const int lo = max(first - g * page, 0), hi = min(sv.len - g * page, page);
  const int pid = seq_page(a.b, seq, g, a.kv.pages, err);
  if (pid < 0) return;
  if (threadIdx.x == 0 && blockIdx.x == gridDim.x - 1 && (g + 1) * (long long)page < sv.len)
    atomicOr(err, ACF_DEV_ERR_BADARG);
  const int h0 = blockIdx.y * a.head_block, nh = min(a.head_block, a.kv.heads - h0);
  constexpr int CPR = DIM / 16;  // 16-code runs per row
  const int rows = hi - lo, total = nh * rows * CPR;
  const size_t head0 = (size_t)pid * a.kv.heads + h0;
  const long long out0 = (long long)(sv.row0 + g * page + lo - first) * a.kv.heads + h0;
  constexpr int U = 2;  // runs under way per thread, of K and of V each
  const bool wide = ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 31) == 0;
  for (int i0 = threadIdx.x; i0 < total; i0 += U * blockDim.x) {
    uint4 w[U][2];
    float scale[U][2];
    size_t to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * (int)blockDim.x, total - 1);
      const int c = i % CPR, rest = i / CPR, h = nh == 1 ? 0 : rest / rows, r = rest - h * rows;
      const size_t from = (((head0 + h) * page) + lo + r) * DIM + 16 * c;
      to[u] = (size_t)(out0 + (long long)r * a.kv.heads + h) * DIM + 16 * c;
      if (a.k) w[u][0] = __ldg(reinterpret_cast<const uint4*>(a.kv.k + from)), scale[u][0] = a.kv.ks[head0 + h];
      if (a.v) w[u][1] = __ldg(reinterpret_cast<const uint4*>(a.kv.v + from)), scale[u][1] = a.kv.vs[head0 + h];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * (int)blockDim.x >= total) break;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        T* o = static_cast<T*>(which ? a.v : a.k);
        if (!o) continue;
        const uint32_t words[4] = {w[u][which].x, w[u][which].y, w[u][which].z, w[u][which].w};
        if (wide) {  // 32 bytes per store: a whole sector per lane
          union {
            T t[32 / sizeof(T)];
            uint32_t w[8];
          } y;
          constexpr int E = 32 / (int)sizeof(T);
#pragma unroll
          for (int e = 0; e < 16; e += E) {
#pragma unroll
            for (int j = 0; j < E; ++j)
              y.t[j] = from_f<T>(code_value(words[(e + j) / 4] ^ 0x80808080u, j % 4) * scale[u][which]);
            dev::st_global_v8(o + to[u] + e, y.w);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = code_value(words[(e + j) / 4] ^ 0x80808080u, j % 4) * scale[u][which];
            store8(o + to[u] + e, true, x);
          }
        }
      }
    }
  }
}

template <typename T, int DIM>
bool read_launch(Call& c, ReadArgs a) {
  const int page = a.kv.page;
  const int slots = std::max(1, (std::min(a.b.max_new, a.b.max_len) + page - 2) / page + 1);
  // a block takes the heads that make about two passes of its 256 threads
  a.head_block = std::max(1, std::min(a.kv.heads, 512 * 16 / (page * DIM)));
  const int parts = (a.kv.heads + a.head_block - 1) / a.head_block;
  if (!ACF_CUDA_OK(launch_pdl(k_kv8_read<T, DIM>, dim3(slots, parts, a.b.seqs), dim3(256), 0, c.stream(), a, c.err())))
    return false;
  return c.launched("k_kv8_read");
}

template <typename F16, typename BF16, typename F32>
bool by_dtype(int dtype, F16 f16, BF16 bf16, F32 f32) {
  return dtype == ACFUN_F16 ? f16() : dtype == ACFUN_BF16 ? bf16() : f32();
}

}  // namespace
}  // namespace acf

using namespace acf;

#define ACF_BY_DIM(fn, T, args) \
  (args.kv.dim == 64 ? fn<T, 64>(c, args) : args.kv.dim == 128 ? fn<T, 128>(c, args) : fn<T, 256>(c, args))
#define ACF_BY_DTYPE(fn, dtype, args)                        \
  by_dtype(dtype, [&] { return ACF_BY_DIM(fn, __half, args); }, \
           [&] { return ACF_BY_DIM(fn, __nv_bfloat16, args); }, [&] { return ACF_BY_DIM(fn, float, args); })

extern "C" int acfun_kv8_append(const AcfunKvCache8* cache, const AcfunKvBatch* batch, const void* k, const void* v,
                                int dtype, long long k_token, long long k_head, long long v_token, long long v_head,
                                const AcfunRope* rope) {
  const char* what = "acfun_kv8_append";
  if (int e = check_dtype(what, dtype, true)) return e;
  if (int e = check_cache(what, cache)) return e;
  if (int e = check_batch(what, batch, cache->page)) return e;
  if (rope) {
    if (int e = check_rope(what, rope, cache->dim)) return e;
    if (rope->rot % 16) {
      set_error(kInvalid, "%s: rope.rot %d is not a multiple of 16 (rotate such keys with acfun_rope first)", what,
                rope->rot);
      return kInvalid;
    }
  }
  const int heads = cache->heads, dim = cache->dim, tokens = batch->tokens;
  if (int e = check_strides(what, k_token, k_head, tokens, heads, dim, false)) return e;
  if (int e = check_strides(what, v_token, v_head, tokens, heads, dim, false)) return e;
  if (batch->seqs == 0 || tokens == 0 || batch->max_new == 0) return 0;
  if (!k || !v) {
    set_error(kInvalid, "%s: k or v is NULL", what);
    return kInvalid;
  }
  Call c(what, true);
  if (!c.ok()) return last_error_code();
  AppendArgs a = {};
  a.kv = cache_view(cache);
  a.b = batch_view(c, batch);
  a.k = c.in(k, span_bytes(k_token, k_head, tokens, heads, dim, dtype));
  a.v = c.in(v, span_bytes(v_token, v_head, tokens, heads, dim, dtype));
  if (rope && rope->rot) {
    a.freq = (const float*)c.in(rope->freq, (size_t)rope->rot / 2 * 4);
    a.rot = rope->rot, a.interleaved = rope->interleaved != 0, a.amp = rope->amplitude;
  }
  if (!c.ok()) return last_error_code();
  const long long per16 = 16 / (long long)dtype_size(dtype);
  a.vec = aligned16(a.k) && k_token % per16 == 0 && k_head % per16 == 0 && aligned16(a.v) && v_token % per16 == 0 &&
          v_head % per16 == 0;
  a.k_token = k_token, a.k_head = k_head, a.v_token = v_token, a.v_head = v_head;
  if (!ACF_BY_DTYPE(append_launch, dtype, a)) c.fail();
  return c.finish() ? 0 : last_error_code();
}

extern "C" int acfun_kv8_read(const AcfunKvCache8* cache, const AcfunKvBatch* batch, void* k, void* v, int dtype) {
  const char* what = "acfun_kv8_read";
  if (int e = check_dtype(what, dtype, true)) return e;
  if (int e = check_cache(what, cache)) return e;
  if (int e = check_batch(what, batch, cache->page)) return e;
  if (batch->seqs == 0 || batch->tokens == 0 || batch->max_new == 0 || (!k && !v)) return 0;
  Call c(what, true);
  if (!c.ok()) return last_error_code();
  ReadArgs a = {};
  a.kv = cache_view(cache);
  a.b = batch_view(c, batch);
  const size_t bytes = (size_t)batch->tokens * cache->heads * cache->dim * dtype_size(dtype);
  // rows of a sequence that is skipped keep what they held
  a.k = c.inout(k, bytes);
  a.v = c.inout(v, bytes);
  if (!c.ok()) return last_error_code();
  if ((a.k && !aligned16(a.k)) || (a.v && !aligned16(a.v))) {
    set_error(kInvalid, "%s: k and v must be 16-byte aligned", what);
    c.fail();
  } else if (!ACF_BY_DTYPE(read_launch, dtype, a)) {
    c.fail();
  }
  return c.finish() ? 0 : last_error_code();
}
