// rope.cu — rotary positions on [tokens, heads, dim] (acfun_rope) and the frequencies for them.
//
//   y_a = amp * (x_a cos(p f_i) - x_b sin(p f_i)),  y_b = amp * (x_b cos(p f_i) + x_a sin(p f_i))
//
// with (a, b) = (i, i + rot/2), or (2i, 2i + 1) when interleaved; elements from rot on are copied.
// Bound by memory: every element is read and written once.  A block takes a few tokens, computes
// their cosines and sines once into shared memory (the angle in 64 bits, attn.cuh) and applies
// them to all heads, 16 bytes per load.  Measured (B200): fp32, 20 heads of 64: 4099 tokens, 42 MB, 9.2 us,
// 4.6 TB/s, 70 % of the measured copy rate; 65536 tokens, 671 MB, 107 us, 6.3 TB/s, 96 %: the smaller call
// pays for its start and end.  65536 tokens of 40 bf16 heads of 128 264 us, 5.1 TB/s.  One token each of 48
// sequences, 40 bf16 heads of 128, 8.6 us, which is the host's time for a call.  Requesting the first values
// before the cosines and sines took 9.8 us for the former: it costs registers, and other blocks already
// fill the wait.
#include <math.h>

#include <algorithm>

#include "attn.cuh"

namespace acf {
namespace {

struct RopeArgs {
  const void* x;
  void* y;
  const int32_t* pos;
  const float* freq;
  long long x_token, x_head, y_token, y_head;
  int tokens, heads, dim, rot, interleaved;
  float amp;
  int tok_block, head_block, items;  // items of one (token, head)
};

// VEC: 16-byte loads.  An item is 8 pairs (half layout, two runs of 8 elements) or 8 consecutive
// elements (interleaved, and what is copied); without VEC a pair or one copied element.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_rope(const RopeArgs a) {
  extern __shared__ __align__(16) float2 cs[];  // [tok_block][rot / 2 rounded up to 8], cs_place
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  const int half = a.rot / 2, row = (half + 7) & ~7;
  const int t0 = blockIdx.x * a.tok_block, nt = min(a.tok_block, a.tokens - t0);
  const int h0 = blockIdx.y * a.head_block, nh = min(a.head_block, a.heads - h0);
  for (int i = threadIdx.x; i < nt * half; i += blockDim.x) {
    const int t = i / half;
    cs[t * row + cs_place(i - t * half)] = rope_cs(a.pos[t0 + t], a.freq[i - t * half], a.amp);
  }
  __syncthreads();
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  const int per_token = nh * a.items, total = nt * per_token;
  if constexpr (VEC) {
    constexpr int U = 2;  // items in flight per thread
    const int pairs = a.interleaved ? 0 : a.rot / 16;
    for (int base = threadIdx.x; base < total; base += U * blockDim.x) {
      float lo[U][8], hi[U][8];
      long long dst[U];
      int tok[U], at[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int it = base + u * blockDim.x;
        at[u] = -1;
        if (it < total) {
          const int t = it / per_token, r = it - t * per_token, h = r / a.items, j = r - h * a.items;
          tok[u] = t;
          at[u] = j < pairs ? j * 8 : a.interleaved ? j * 8 : a.rot + (j - pairs) * 8;
          const T* p = x + (t0 + t) * a.x_token + (h0 + h) * a.x_head + at[u];
          dst[u] = (t0 + t) * a.y_token + (h0 + h) * a.y_head + at[u];
          load8(p, true, lo[u]);
          if (j < pairs) load8(p + half, true, hi[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (at[u] < 0) continue;
        if (at[u] < a.rot) {
          // 8 pairs from a multiple of 8 (half), or 4 from a multiple of 4: quarters of a run of 8
          const int p0 = a.interleaved ? at[u] / 2 : at[u], x = (p0 >> 4) & 3;
          const float4* w = reinterpret_cast<const float4*>(cs + tok[u] * row + (p0 & ~7));
          if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float4 c = w[(((p0 & 7) >> 1) + i) ^ x];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float cc = k ? c.z : c.x, ss = k ? c.w : c.y;
                const float p = lo[u][4 * i + 2 * k], q = lo[u][4 * i + 2 * k + 1];
                lo[u][4 * i + 2 * k] = p * cc - q * ss;
                lo[u][4 * i + 2 * k + 1] = q * cc + p * ss;
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 c = w[i ^ x];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float cc = k ? c.z : c.x, ss = k ? c.w : c.y;
                const float p = lo[u][2 * i + k], q = hi[u][2 * i + k];
                lo[u][2 * i + k] = p * cc - q * ss;
                hi[u][2 * i + k] = q * cc + p * ss;
              }
            }
            store8(y + dst[u] + half, true, hi[u]);
          }
        }
        store8(y + dst[u], true, lo[u]);
      }
    }
  } else {
    for (int it = threadIdx.x; it < total; it += blockDim.x) {
      const int t = it / per_token, r = it - t * per_token, h = r / a.items, j = r - h * a.items;
      const T* p = x + (t0 + t) * a.x_token + (h0 + h) * a.x_head;
      T* o = y + (t0 + t) * a.y_token + (h0 + h) * a.y_head;
      if (j < half) {
        const float2 c = cs[t * row + cs_place(j)];
        const int ia = a.interleaved ? 2 * j : j, ib = a.interleaved ? 2 * j + 1 : j + half;
        const float u = to_f(p[ia]), v = to_f(p[ib]);
        o[ia] = from_f<T>(u * c.x - v * c.y);
        o[ib] = from_f<T>(v * c.x + u * c.y);
      } else {
        o[j + half] = p[j + half];
      }
    }
  }
}

template <typename T>
bool rope_launch(Call& c, RopeArgs a) {
  const long long per16 = 16 / sizeof(T);
  const bool vec = a.dim % 8 == 0 && a.rot % (a.interleaved ? 8 : 16) == 0 && aligned16(a.x) && aligned16(a.y) &&
                   a.x_token % per16 == 0 && a.x_head % per16 == 0 && a.y_token % per16 == 0 && a.y_head % per16 == 0;
  a.items = vec ? (a.interleaved ? a.dim / 8 : a.rot / 16 + (a.dim - a.rot) / 8) : a.rot / 2 + a.dim - a.rot;
  // tokens per block: enough blocks for about eight per SM; few tokens share their heads out
  const int want = 8 * c.sm_count();
  int smem_cap = a.rot ? (40 * 1024) / (a.rot * 4 + 64) : 8;
  a.tok_block = std::max(1, std::min({a.tokens / want, 8, std::max(1, smem_cap)}));
  const int blocks = (a.tokens + a.tok_block - 1) / a.tok_block;
  int parts = std::max(1, std::min(a.heads, 2 * c.sm_count() / blocks));
  // no block with less than a pass of its 256 threads
  while (parts > 1 && (long long)(a.heads / parts) * a.items < 256) --parts;
  a.head_block = (a.heads + parts - 1) / parts;
  parts = (a.heads + a.head_block - 1) / a.head_block;
  if (parts > 65535) {
    set_error(kInvalid, "acfun_rope: too many heads");
    return false;
  }
  const size_t smem = (size_t)a.tok_block * ((a.rot / 2 + 7) / 8 * 8) * sizeof(float2);
  if (!ACF_CUDA_OK(launch_pdl(vec ? k_rope<T, true> : k_rope<T, false>, dim3(blocks, parts), dim3(256), smem, c.stream(), a)))
    return false;
  return c.launched("k_rope");
}

}  // namespace

int check_rope(const char* what, const AcfunRope* r, int dim) {
  if (!r->freq && r->rot > 0) {
    set_error(kInvalid, "%s: rope.freq is NULL", what);
    return kInvalid;
  }
  if (r->rot < 0 || r->rot % 2 || r->rot > dim || r->rot > 8192) {
    set_error(kInvalid, "%s: rope.rot %d must be even, at most dim (%d) and at most 8192", what, r->rot, dim);
    return kInvalid;
  }
  return 0;
}

}  // namespace acf

using namespace acf;

extern "C" int acfun_rope_frequencies(int rot, double base, int scaling, double factor, double trained,
                                      double fast, double slow, float* freq, float* amplitude) {
  const char* bad = nullptr;
  if (rot <= 0 || rot % 2) bad = "rot must be positive and even";
  else if (!(base > 1.0) || !isfinite(base)) bad = "base must be above 1";
  else if (!freq) bad = "freq is NULL";
  else if (scaling < 0 || scaling > 5) bad = "scaling must be 0 to 5";
  else if (scaling && (!(factor >= 1.0) || !isfinite(factor))) bad = "factor must be at least 1";
  else if (scaling == 2 && rot < 4) bad = "scaling 2 needs rot of at least 4";
  else if (scaling >= 3 && (!(trained > 0.0) || !isfinite(trained) || !(slow > 0.0) || !(fast > slow) || !isfinite(fast)))
    bad = "trained, slow and fast must be positive, and fast above slow";
  if (bad) {
    set_error(kInvalid, "acfun_rope_frequencies: %s", bad);
    return kInvalid;
  }
  const double tau = 6.28318530717958647693;
  const double b = scaling == 2 ? base * pow(factor, (double)rot / (rot - 2)) : base;
  // the (real) pair index at which a pair makes `turns` turns in the trained length
  auto index_of = [&](double turns) { return rot * log(trained / (turns * tau)) / (2.0 * log(base)); };
  for (int i = 0; i < rot / 2; ++i) {
    double f = pow(b, -2.0 * i / rot);
    if (scaling == 1) f /= factor;
    if (scaling >= 3) {
      double keep;  // the share of the unscaled frequency
      if (scaling != 4) {
        double lo = index_of(fast), hi = index_of(slow);
        if (scaling == 5) {
          lo = fmax(floor(lo), 0.0), hi = fmin(ceil(hi), rot - 1.0);
          if (hi <= lo) hi = lo + 1e-3;  // both ends past the last pair
        }
        keep = (hi - i) / (hi - lo);
      } else {
        keep = (trained * f / tau - slow) / (fast - slow);
      }
      keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
      f = f * keep + f / factor * (1.0 - keep);
    }
    freq[i] = (float)f;
  }
  if (amplitude) *amplitude = scaling == 3 || scaling == 5 ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
  return 0;
}

extern "C" int acfun_rope(const void* x, void* y, int dtype, int tokens, int heads, int dim, long long x_token,
                          long long x_head, long long y_token, long long y_head, const int32_t* pos,
                          const AcfunRope* rope) {
  const char* what = "acfun_rope";
  if (int e = check_dtype(what, dtype, true)) return e;
  if (tokens < 0 || heads <= 0 || dim <= 0) {
    set_error(kInvalid, "%s: tokens %d, heads %d and dim %d must be positive", what, tokens, heads, dim);
    return kInvalid;
  }
  if (!rope) {
    set_error(kInvalid, "%s: rope is NULL", what);
    return kInvalid;
  }
  if (int e = check_rope(what, rope, dim)) return e;
  if (int e = check_strides(what, x_token, x_head, tokens, heads, dim, false)) return e;
  if (int e = check_strides(what, y_token, y_head, tokens, heads, dim, true)) return e;
  if (tokens == 0) return 0;
  if (!x || !y || !pos) {
    set_error(kInvalid, "%s: a tensor is NULL", what);
    return kInvalid;
  }
  if (x == y && (x_token != y_token || x_head != y_head)) {
    set_error(kInvalid, "%s: in place needs equal strides", what);
    return kInvalid;
  }
  Call c(what, true);
  if (!c.ok()) return last_error_code();
  RopeArgs a = {};
  const size_t yb = span_bytes(y_token, y_head, tokens, heads, dim, dtype);
  // a host output is staged with its present contents: strides may leave gaps
  a.y = c.inout(y, yb);
  a.x = x == y ? a.y : c.in(x, span_bytes(x_token, x_head, tokens, heads, dim, dtype));
  a.pos = (const int32_t*)c.in(pos, (size_t)tokens * 4);
  a.freq = rope->rot ? (const float*)c.in(rope->freq, (size_t)rope->rot / 2 * 4) : nullptr;
  if (!c.ok()) return last_error_code();
  a.x_token = x_token, a.x_head = x_head, a.y_token = y_token, a.y_head = y_head;
  a.tokens = tokens, a.heads = heads, a.dim = dim, a.rot = rope->rot, a.interleaved = rope->interleaved != 0;
  a.amp = rope->amplitude;
  const bool ok = dtype == ACFUN_F32   ? rope_launch<float>(c, a)
                  : dtype == ACFUN_F16 ? rope_launch<__half>(c, a)
                                       : rope_launch<__nv_bfloat16>(c, a);
  if (!ok) c.fail();
  return c.finish() ? 0 : last_error_code();
}
