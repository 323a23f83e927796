// attn_kv8.cu — attention over the int8 cache (acfun_kv8_attention): the entry point and the
// streaming kernel, whose warps turn codes straight into matrix-instruction fragments.  It takes any
// shape; attention with few rows per cache head (decode steps, drafts) is bound by the codes it
// reads, and that is what it is built for.
//
// Rows: the new tokens of a sequence times the query heads that share a cache head, row = token *
// group + head, in tiles of 8, 16 or 32.  A block of four warps takes one (sequence, cache head, row
// tile, chunk of keys); its warps take 32 keys in turn, each with its own running offset, sum and
// output, which are joined in shared memory at the end.  A long sequence is split over blocks; the
// last of them to finish joins their parts in the order of the chunks, so the result does not
// depend on who was last.
//
// Mathematics.  With q scaled per row by a power of two to fp16 range (elements below 2^-14 of the row's
// largest keep bits down to 2^-24 of it: an absolute error far below that of 11 bits in the largest),
// codes c exact in fp16, S = q.c_k in fp32,
//   t = S * (scale * s_k[page]) log2 e + log2 s_v[page],  w = 2^(t - m) in fp16,  O += w c_v,
//   l += (sum of w over the page's keys, in fp32 before rounding) / s_v[page],  out = O / l.
// The V scale rides in the exponent, so O needs no per-page scaling and w stays within fp16 range
// whatever the scales are; m moves only when a weight would pass 2^15.
//
// Fragments.  The products are transposed, S^T = K Q^T and O^T = V^T w^T, so that keys and elements
// take the 16 places of m16n8k16 and the rows the 8: a decode step's few rows leave none of them
// idle (with the rows in the 16 places, half of the products were of nothing, and the board's
// power limit, which this kernel reaches, made that time).  K is the A operand with its contraction
// index (the element of a head) permuted so that a thread's share of a key is 16 consecutive bytes;
// V^T is the A operand with its row index permuted so that a thread's share of each of its four keys
// is 16 consecutive bytes (8 when dim is 64); the weights change from C to B operand by movmatrix.
// The codes pass through a ring in shared memory of two steps of 32 keys per warp, copied
// asynchronously; nothing is shared between warps.
//
// Measured (B200): one fp16 token of 64 query heads over 262145 keys of 8 cache heads of 128 elements
// 100.6 us, 5.3 TB/s, 81 % of the measured copy rate, at 1.65 GHz under the board's power limit; one
// token each of 48 sequences of 33 to 16000 keys, 32 query and 8 cache heads, 56 us, 4.0 TB/s, where
// blocks that find no chunk of their own and the joins of short chunks cost the rest.  16 sequences of
// 4096 keys with 8 drafted tokens each (32 rows) 56 us where the codes take 20.6; heads of 256, a prompt of
// 4096 tokens of 16 query and 8 cache heads 986 us.  The keys are divided by max_len, not by the window: one
// token with a window of 16384 over 262144 keys keeps 32 blocks busy and takes 57 us.
#include <math.h>

#include <algorithm>

#include "attn_tile.cuh"

namespace acf {
namespace {

constexpr int kWarps = 4;
constexpr int kUnit = 16;          // keys that share a page entry
constexpr int kPair = 2;           // units per step of a warp: two chains to hide each other's latencies
constexpr int kMaxPages = 1024;    // most pages of one chunk (their scales are staged in shared memory)
constexpr int kTickets = 1 << 16;

struct StreamArgs {
  AttnArgs a;
  int chunk;                 // keys per block, a multiple of kUnit
  int splits;                // chunks of max_len keys (the stride of the partial results)
  int part_rows;             // rows that a (sequence, head) of this launch can have
  float* part_o;             // [seqs][heads][part_rows][splits][DIM], null when splits == 1
  float2* part_ml;           // [seqs][heads][part_rows][splits]
  unsigned* tickets;         // [seqs][heads][row tiles], zero between calls
  int row_tiles;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// over the eight lanes that hold the same rows
__device__ __forceinline__ float rows_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}
__device__ __forceinline__ float rows_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 4);
  x += __shfl_xor_sync(0xffffffffu, x, 8);
  return x + __shfl_xor_sync(0xffffffffu, x, 16);
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // of an 8 x 8 matrix of 16-bit elements
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// What a page needs in the loop: its place, and its scales in the forms used.
struct __align__(16) PageEntry {
  int pid;          // -1: out of range (reported), its keys are not seen
  float ks;         // scale * k scale * log2 e
  float lv, rv;     // log2 and reciprocal of the v scale
};

template <typename T>
__device__ __forceinline__ void store2(T* p, float a, float b) {
  p[0] = from_f<T>(a);
  p[1] = from_f<T>(b);
}

// A warp's codes on their way: two steps, each kPair units of 16 keys of K and V.  16-byte chunk ch
// of a row is kept at chunk_at(row, ch), so that the fragment reads below (two rows x 4 chunks of K,
// four alternate rows x 2 chunks of V at a time) meet no bank twice.
template <int DIM>
struct alignas(128) Ring {
  uint8_t kv[2][2][kPair * kUnit * DIM];  // [step][K, V]
};
template <int DIM>
__device__ __forceinline__ int chunk_at(int row, int ch) {
  if constexpr (DIM == 64) {
    const int unit = ((row & 1) * 4 + ch) ^ (row & 6);
    return (row >> 1) * 128 + unit * 16;
  } else {
    return row * DIM + (ch >> 3) * 128 + (((ch & 7) ^ (row & 6) ^ ((row & 1) << 2)) << 4);
  }
}
__device__ __forceinline__ void cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dev::smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int DIM, int R8>
struct StreamSmem {
  float2 ml[kWarps][8 * R8];
  float row_ml[8 * R8][2];
  int last;
  uint2 q[R8 > 1 ? DIM / 16 : 1][R8][32];  // Q fragments, the same for the four warps
  union {
    Ring<DIM> ring[kWarps];
    float o[kWarps][8 * R8][DIM + 4];
  };
  PageEntry pages[1];  // as many as a chunk can touch: the launch sizes the block's memory by them
};
static_assert(alignof(StreamSmem<64, 1>) == 128 && alignof(Ring<64>) == 128 && sizeof(Ring<64>) % 128 == 0,
              "16-byte copies into the ring");

// DIM / 64 runs of 16 bytes per key for K; DIM / 8 bytes per key for V.
template <typename T, int DIM, int R8>
__device__ __forceinline__ void attn_stream(const StreamArgs& p, unsigned* err) {
  constexpr int KR = DIM / 64;          // 16-byte runs of a thread per key (K)
  constexpr int MT = DIM / 16;          // output m-tiles
  constexpr int VW = DIM / 32;          // 32-bit words of a thread per key (V)
  constexpr int RT = 8 * R8;            // rows of a tile
  extern __shared__ __align__(128) uint8_t smem_raw[];
  using Smem = StreamSmem<DIM, R8>;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const AttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int head = blockIdx.x % a.kv.heads, rt = blockIdx.x / a.kv.heads, seq = blockIdx.y, chunk_i = blockIdx.z;
  const int lg = a.kv.page_log2;
  // without a window the chunk's pages do not depend on the length: their numbers come with it
  const int guess = (int)(((long long)chunk_i * p.chunk) >> lg) + threadIdx.x;
  const int early = a.window == 0 && guess < a.b.cols ? __ldg(a.b.table + (size_t)seq * a.b.cols + guess) : -1;
  const SeqView sv = seq_view(a.b, seq, err);
  const int rows = sv.n * a.group;
  const int r0 = rt * RT;
  if (r0 >= rows || !rows_taken(a, rows)) return;
  const int nr = min(RT, rows - r0);
  const int t_first = r0 / a.group, t_last = (r0 + nr - 1) / a.group;
  const int pos0 = sv.len - sv.n;  // position of new token 0 (negative: it sees nothing)
  const KeyRange kr = key_range(a, sv, r0, nr, kUnit);
  const int unit0 = kr.first, units = kr.n;
  const int per = p.chunk / kUnit;
  const int nsplit = max(1, (units + per - 1) / per);
  if (chunk_i >= nsplit) return;
  const int ub = unit0 + chunk_i * per, ue = min(unit0 + units, ub + per);

  // the chunk's pages
  const int pg0 = (ub * kUnit) >> lg;
  const int npg = ue > ub ? (((ue * kUnit - 1) >> lg) - pg0 + 1) : 0;
  for (int i = threadIdx.x; i < npg; i += blockDim.x) {
    int pid = a.window == 0 && i == (int)threadIdx.x ? early : a.b.table[(size_t)seq * a.b.cols + pg0 + i];
    if ((unsigned)pid >= (unsigned)a.kv.pages) {
      atomicOr(err, ACF_DEV_ERR_BADARG);
      pid = -1;
    }
    sm.pages[i].pid = pid;
  }
  __syncthreads();

  const size_t head_at = (size_t)head * a.kv.page, page_step = (size_t)a.kv.heads * a.kv.page;
  Ring<DIM>& ring = sm.ring[warp];
  // Requests the units from u on as step `at`; past the chunk's end the last one again (masked below).
  auto request = [&](int u, int at) {
    constexpr int CH = DIM / 16, RPP = 32 / CH;  // chunks per row, rows per pass
    const int row0 = lane / CH, ch = lane % CH;
#pragma unroll
    for (int p = 0; p < kPair; ++p) {
      const int key = min(u + p, ue - 1) * kUnit;
      const int pid = sm.pages[(key >> lg) - pg0].pid;
      const size_t from = (max(pid, 0) * page_step + head_at + (key & (a.kv.page - 1)) + row0) * DIM + ch * 16;
#pragma unroll
      for (int r = 0; r < kUnit; r += RPP) {
        const int to = chunk_at<DIM>(p * kUnit + r + row0, ch);
        cp16(&ring.kv[at][0][to], a.kv.k + from + r * DIM);
        cp16(&ring.kv[at][1][to], a.kv.v + from + r * DIM);
      }
    }
  };
  int u = ub + warp * kPair;
  constexpr int kStride = kWarps * kPair;
  // two steps on their way while the scales and Q are
  if (u < ue) request(u, 0);
  cp_commit();
  if (u + kStride < ue) request(u + kStride, 1);
  cp_commit();
  for (int i = threadIdx.x; i < npg; i += blockDim.x) {
    PageEntry e = {sm.pages[i].pid, 0.0f, 0.0f, 0.0f};
    if (e.pid >= 0) {
      const size_t sc = (size_t)e.pid * a.kv.heads + head;
      const float vs = fmaxf(a.kv.vs[sc], 0x1p-100f);
      e.ks = a.scale * a.kv.ks[sc] * 1.4426950408889634f;
      e.lv = log2f(vs);
      e.rv = 1.0f / vs;
    }
    sm.pages[i] = e;  // by the thread that wrote its pid
  }

  // Q fragments of row g of each eight, scaled by a power of two per row.  With one eight they stay in
  // registers; with more, every warp reads the rows for their maxima and writes its share.
  uint2 qf[DIM / 16];
  float q_unit[R8][2];  // of rows 2 c, 2 c + 1 of each eight
  {
    const T* q = static_cast<const T*>(a.q);
    const bool vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && a.q_token % 8 == 0 && a.q_head % 8 == 0;
#pragma unroll
    for (int n = 0; n < R8; ++n) {
      const int r = r0 + 8 * n + g;
      const bool in = 8 * n + g < nr;
      const int t = r / a.group, hq = head * a.group + r - t * a.group;
      const T* src = q + (long long)(sv.row0 + t) * a.q_token + (long long)hq * a.q_head + c * 16;
      float x[KR][2][8], top = 0.0f;  // 16 elements of each run of 64
#pragma unroll
      for (int i = 0; i < KR; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[i][h][e] = 0.0f;
          if (in) load8(src + i * 64 + 8 * h, vec, x[i][h]);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][h][e]));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const Pow2 w = row_pow2(top);
#pragma unroll
      for (int i = 0; i < DIM / 16; ++i) {
        if (R8 > 1 && i % kWarps != warp) continue;
        const float* y = &x[i / 4][(i % 4) >> 1][4 * (i & 1)];
        qf[i] = make_uint2(pack_f16(y[0] * w.down, y[1] * w.down), pack_f16(y[2] * w.down, y[3] * w.down));
        if constexpr (R8 > 1) sm.q[i][n][lane] = qf[i];
      }
      q_unit[n][0] = __shfl_sync(0xffffffffu, w.up, 8 * c);
      q_unit[n][1] = __shfl_sync(0xffffffffu, w.up, 8 * c + 4);
    }
  }
  // the keys rows 2 c, 2 c + 1 of each eight see: [lo, hi)
  int see_lo[R8][2], see_hi[R8][2];
#pragma unroll
  for (int n = 0; n < R8; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int pos = pos0 + (r0 + 8 * n + 2 * c + i) / a.group;
      see_hi[n][i] = a.causal ? min(sv.len, pos + 1) : sv.len;
      see_lo[n][i] = a.window > 0 ? max(0, pos - a.window + 1) : 0;
      if (pos < 0) see_hi[n][i] = 0;
    }
  // units that every row of the tile sees whole
  const int all_lo = a.window > 0 ? max(0, pos0 + t_last - a.window + 1) : 0;
  const int all_hi = pos0 + t_first < 0 ? 0 : a.causal ? min(sv.len, pos0 + t_first + 1) : sv.len;

  float o[MT][R8][4];
  float m[R8][2], l[R8][2];
#pragma unroll
  for (int n = 0; n < R8; ++n) {
#pragma unroll
    for (int j = 0; j < MT; ++j) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.0f;
    m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;
  }
  __syncthreads();

  for (int at = 0; u < ue; u += kStride, at ^= 1) {
    cp_wait<1>();
    __syncwarp();
    const uint8_t *ks = ring.kv[at][0], *vs = ring.kv[at][1];
    float s[kPair][R8][4];  // keys g (0, 1) and g + 8 (2, 3) of a unit, rows 2 c and 2 c + 1
#pragma unroll
    for (int p = 0; p < kPair; ++p)
#pragma unroll
      for (int n = 0; n < R8; ++n) s[p][n][0] = s[p][n][1] = s[p][n][2] = s[p][n][3] = 0.0f;
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      uint4 kc[kPair][2];
#pragma unroll
      for (int p = 0; p < kPair; ++p)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          kc[p][t] = *reinterpret_cast<const uint4*>(ks + chunk_at<DIM>(p * kUnit + t * 8 + g, r * 4 + c));
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int p = 0; p < kPair; ++p) {
          const uint4 &lo = kc[p][0], &hi = kc[p][1];
          const uint32_t x = (i == 0 ? lo.x : i == 1 ? lo.y : i == 2 ? lo.z : lo.w) ^ 0x80808080u;
          const uint32_t y = (i == 0 ? hi.x : i == 1 ? hi.y : i == 2 ? hi.z : hi.w) ^ 0x80808080u;
          const uint32_t a0 = f16_from_u8(x, 0x4140), a2 = f16_from_u8(x, 0x4342);
          const uint32_t a1 = f16_from_u8(y, 0x4140), a3 = f16_from_u8(y, 0x4342);
#pragma unroll
          for (int n = 0; n < R8; ++n) {
            const uint2 b = R8 > 1 ? sm.q[R8 > 1 ? r * 4 + i : 0][n][lane] : qf[r * 4 + i];
            mma_f16(s[p][n], a0, a1, a2, a3, b.x, b.y);
          }
        }
    }
    // scores in powers of two, masked where the step crosses an edge of what some row sees
    const int k0 = u * kUnit;
    float rv[kPair];
    bool whole = k0 >= all_lo && k0 + kPair * kUnit <= all_hi && u + kPair <= ue;
#pragma unroll
    for (int p = 0; p < kPair; ++p) {
      const PageEntry e = sm.pages[((min(u + p, ue - 1) * kUnit) >> lg) - pg0];
      rv[p] = e.rv;
      whole = whole && e.pid >= 0;
      const float lv = e.pid >= 0 && u + p < ue ? e.lv : -INFINITY;
#pragma unroll
      for (int n = 0; n < R8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[p][n][i] = fmaf(s[p][n][i], e.ks * q_unit[n][i & 1], lv);
    }
    if (__builtin_expect(!whole, 0)) {
#pragma unroll
      for (int p = 0; p < kPair; ++p)
#pragma unroll
        for (int n = 0; n < R8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = k0 + p * kUnit + g + 8 * (i >> 1);
            if (key < see_lo[n][i & 1] || key >= see_hi[n][i & 1]) s[p][n][i] = -INFINITY;
          }
    }
    // a thread's own scores say whether an offset has to move; the rows' maxima are looked up only then
    bool over = false;
#pragma unroll
    for (int n = 0; n < R8; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int p = 0; p < kPair; ++p) top = fmaxf(top, fmaxf(s[p][n][i], s[p][n][2 + i]));
        over = over || top > m[n][i] + kMost;
      }
    if (__builtin_expect(__any_sync(0xffffffffu, over), 0)) {
#pragma unroll
      for (int n = 0; n < R8; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = -INFINITY;
#pragma unroll
          for (int p = 0; p < kPair; ++p) top = fmaxf(top, fmaxf(s[p][n][i], s[p][n][2 + i]));
          top = rows_max(top);
          const float to = top > m[n][i] + kMost ? top - kTop : m[n][i];
          const float b = m[n][i] == to ? 1.0f : ex2(m[n][i] - to);
          m[n][i] = to;
          l[n][i] *= b;
#pragma unroll
          for (int j = 0; j < MT; ++j) o[j][n][i] *= b, o[j][n][2 + i] *= b;
        }
    }
#pragma unroll
    for (int p = 0; p < kPair; ++p) {
      uint32_t b0[R8], b1[R8];
#pragma unroll
      for (int n = 0; n < R8; ++n) {
        // a row that has seen nothing yet has m = -inf and only -inf scores
        const float m0 = m[n][0] == -INFINITY ? 0.0f : m[n][0], m1 = m[n][1] == -INFINITY ? 0.0f : m[n][1];
        const float w0 = ex2(s[p][n][0] - m0), w1 = ex2(s[p][n][1] - m1);
        const float w2 = ex2(s[p][n][2] - m0), w3 = ex2(s[p][n][3] - m1);
        l[n][0] = fmaf(w0 + w2, rv[p], l[n][0]);
        l[n][1] = fmaf(w1 + w3, rv[p], l[n][1]);
        b0[n] = transpose8(pack_f16(w0, w1));
        b1[n] = transpose8(pack_f16(w2, w3));
      }
      uint32_t vr[4][VW];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = p * kUnit + 2 * c + (k & 1) + 8 * (k >> 1);
        if constexpr (DIM == 64) {
          const uint2 w2 = *reinterpret_cast<const uint2*>(vs + chunk_at<DIM>(row, g >> 1) + 8 * (g & 1));
          vr[k][0] = w2.x, vr[k][1] = w2.y;
        } else {
#pragma unroll
          for (int r = 0; r < VW / 4; ++r) {
            const uint4 w4 = *reinterpret_cast<const uint4*>(vs + chunk_at<DIM>(row, g * (VW / 4) + r));
            vr[k][4 * r] = w4.x, vr[k][4 * r + 1] = w4.y, vr[k][4 * r + 2] = w4.z, vr[k][4 * r + 3] = w4.w;
          }
        }
      }
      // O^T: m-tile j holds elements (lane / 4) * DIM / 8 + 2 j and the next of the head
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        const uint32_t x0 = vr[0][i] ^ 0x80808080u, x1 = vr[1][i] ^ 0x80808080u;
        const uint32_t x2 = vr[2][i] ^ 0x80808080u, x3 = vr[3][i] ^ 0x80808080u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t p0 = __byte_perm(x0, x1, h ? 0x7362 : 0x5140), p1 = __byte_perm(x2, x3, h ? 0x7362 : 0x5140);
          const uint32_t a0 = f16_from_u8(p0, 0x4140), a1 = f16_from_u8(p0, 0x4342);
          const uint32_t a2 = f16_from_u8(p1, 0x4140), a3 = f16_from_u8(p1, 0x4342);
#pragma unroll
          for (int n = 0; n < R8; ++n) mma_f16(o[2 * i + h][n], a0, a1, a2, a3, b0[n], b1[n]);
        }
      }
    }
    __syncwarp();
    if (u + 2 * kStride < ue) request(u + 2 * kStride, at);
    cp_commit();
  }
  cp_wait<0>();

  // ---- the four warps' parts joined (the outputs take the place of the codes)
#pragma unroll
  for (int n = 0; n < R8; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[n][i] = rows_sum(l[n][i]);
      if (g == 0) sm.ml[warp][8 * n + 2 * c + i] = make_float2(m[n][i], l[n][i]);
    }
  __syncthreads();  // also: no warp reads codes any more
#pragma unroll
  for (int n = 0; n < R8; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 8 * n + 2 * c + i;
      float top = -INFINITY;
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.ml[w][r].x);
      const float b = m[n][i] == top ? 1.0f : ex2(m[n][i] - top);
      if (r < nr) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
          *reinterpret_cast<float2*>(&sm.o[warp][r][g * (DIM / 8) + 2 * j]) = make_float2(o[j][n][i] * b, o[j][n][2 + i] * b);
      }
      if (warp == 0 && g == 0) {
        float sum = 0.0f;
        for (int w = 0; w < kWarps; ++w) {
          const float2 x = sm.ml[w][r];
          sum += x.x == top ? x.y : x.y * ex2(x.x - top);
        }
        sm.row_ml[r][0] = top, sm.row_ml[r][1] = sum;
      }
    }
  __syncthreads();
  T* out = static_cast<T*>(a.out);
  for (int i = threadIdx.x; i < nr * (DIM / 2); i += blockDim.x) {
    const int r = i / (DIM / 2), d = 2 * (i % (DIM / 2));
    float x = 0.0f, y = 0.0f;
    for (int w = 0; w < kWarps; ++w) x += sm.o[w][r][d], y += sm.o[w][r][d + 1];
    const int t = (r0 + r) / a.group, hq = head * a.group + (r0 + r) - t * a.group;
    const float top = sm.row_ml[r][0], sum = sm.row_ml[r][1];
    if (nsplit == 1) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      store2(out + (long long)(sv.row0 + t) * a.o_token + (long long)hq * a.o_head + d, x * inv, y * inv);
      if (d == 0 && a.lse)
        a.lse[(long long)(sv.row0 + t) * a.q_heads + hq] =
            sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
    } else {
      const size_t at = (((size_t)seq * a.kv.heads + head) * p.part_rows + r0 + r) * p.splits + chunk_i;
      *reinterpret_cast<float2*>(p.part_o + at * DIM + d) = make_float2(x, y);
      if (d == 0) p.part_ml[at] = make_float2(top, sum);
    }
  }
  if (nsplit == 1) return;

  // ---- the last block of this row tile joins the chunks
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned* ticket = p.tickets + ((size_t)seq * a.kv.heads + head) * p.row_tiles + rt;
    const unsigned before = atomicAdd(ticket, 1u);
    sm.last = before == (unsigned)nsplit - 1;
    if (sm.last) *ticket = 0;
  }
  __syncthreads();
  if (!sm.last) return;
  __threadfence();
  // All (row, chunk) offsets and sums are requested at once and kept in shared memory, in blocks of
  // chunks if they are many; then a thread takes 4 elements of some rows, all chunks of which are
  // again independent loads.  A round trip to L2 takes longer than everything else here.
  float2* ml = reinterpret_cast<float2*>(sm.o);  // [row][chunk of the block]
  const int kb = min(nsplit, (int)(sizeof(sm.o) / sizeof(float2)) / nr);
  auto row_at = [&](int r) -> size_t {
    return (((size_t)seq * a.kv.heads + head) * p.part_rows + r0 + r) * p.splits;
  };
  auto fetch_ml = [&](int k0) {
    __syncthreads();
    for (int i = threadIdx.x; i < nr * kb; i += blockDim.x) {
      const int r = i / kb, k = k0 + i - r * kb;
      ml[i] = k < nsplit ? __ldcg(&p.part_ml[row_at(r) + k]) : make_float2(-INFINITY, 0.0f);
    }
    __syncthreads();
  };
  for (int r = threadIdx.x; r < RT; r += blockDim.x) sm.row_ml[r][0] = -INFINITY, sm.row_ml[r][1] = 0.0f;
  for (int k0 = 0; k0 < nsplit; k0 += kb) {  // the rows' largest offsets
    fetch_ml(k0);
    for (int r = warp; r < nr; r += kWarps) {
      float top = sm.row_ml[r][0];
      for (int k = lane; k < kb; k += 32) top = fmaxf(top, ml[r * kb + k].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) sm.row_ml[r][0] = top;
    }
  }
  constexpr int kItems = RT * DIM / 4 / (kWarps * 32);
  float4 acc[kItems];
  const float* from[kItems];
  int row[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int i = threadIdx.x + j * kWarps * 32;
    row[j] = i / (DIM / 4);
    from[j] = p.part_o + row_at(min(row[j], nr - 1)) * DIM + 4 * (i % (DIM / 4));
    acc[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  for (int k0 = 0; k0 < nsplit; k0 += kb) {
    if (kb < nsplit)
      fetch_ml(k0);
    else
      __syncthreads();
    for (int r = warp; r < nr; r += kWarps) {  // the sums make way for the chunks' factors
      const float top = sm.row_ml[r][0];
      float sum = 0.0f;
      for (int k = lane; k < kb; k += 32) {
        float2& x = ml[r * kb + k];
        const float b = x.x == top ? 1.0f : ex2(x.x - top);
        sum = fmaf(x.y, b, sum);
        x.y = b;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) sm.row_ml[r][1] += sum;
    }
    __syncthreads();
    const int n = min(kb, nsplit - k0);
#pragma unroll(kItems >= 8 ? 2 : 16 / kItems)
    for (int k = 0; k < n; ++k) {
#pragma unroll
      for (int j = 0; j < kItems; ++j) {
        if (row[j] < nr) {
          const float b = ml[row[j] * kb + k].y;
          const float4 v = __ldcg(reinterpret_cast<const float4*>(from[j] + (size_t)(k0 + k) * DIM));
          acc[j].x = fmaf(v.x, b, acc[j].x), acc[j].y = fmaf(v.y, b, acc[j].y);
          acc[j].z = fmaf(v.z, b, acc[j].z), acc[j].w = fmaf(v.w, b, acc[j].w);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int i = threadIdx.x + j * kWarps * 32, r = i / (DIM / 4), d = 4 * (i % (DIM / 4));
    if (r >= nr) continue;
    const int t = (r0 + r) / a.group, hq = head * a.group + (r0 + r) - t * a.group;
    const float of = sm.row_ml[r][1], inv = of == 0.0f ? 0.0f : 1.0f / of;
    T* dst = out + (long long)(sv.row0 + t) * a.o_token + (long long)hq * a.o_head + d;
    store2(dst, acc[j].x * inv, acc[j].y * inv);
    store2(dst + 2, acc[j].z * inv, acc[j].w * inv);
    if (d == 0 && a.lse)
      a.lse[(long long)(sv.row0 + t) * a.q_heads + hq] =
          of == 0.0f ? -INFINITY : (sm.row_ml[r][0] + log2f(of)) * 0.69314718055994531f;
  }
}

template <typename T, int DIM, int R8>
__global__ void __launch_bounds__(kWarps * 32, DIM * R8 >= 512 ? 2 : 3) k_attn_stream(const StreamArgs p, unsigned* err) {
  // Beside k_attn_tc the kernel before is not a producer but the other half of the same call: what it
  // waited for is complete, and only the end waits for it, so that completion stays in order.
  if (!p.a.beside) dev::grid_dep_wait();
  dev::grid_dep_launch();
  attn_stream<T, DIM, R8>(p, err);
  if (p.a.beside) dev::grid_dep_wait();
}

// Zeroed once per device, in the stream of the call that needs it first (a call on another stream waits
// for the calls before it, as for their scratch); the kernel leaves it zero.  *zeroed: by this call.
unsigned* tickets_of(Call& c, int device, bool* zeroed) {
  static unsigned* buf[64] = {};
  if (!buf[device]) {
    unsigned* d = nullptr;
    if (!ACF_CUDA_OK(cudaMalloc(&d, kTickets * sizeof(unsigned)))) return nullptr;
    if (!ACF_CUDA_OK(cudaMemsetAsync(d, 0, kTickets * sizeof(unsigned), c.stream()))) {
      cudaFree(d);
      return nullptr;
    }
    buf[device] = d;
    *zeroed = true;
  }
  return buf[device];
}

template <typename T, int DIM, int R8>
bool stream_launch(Call& c, const AttnArgs& a) {
  constexpr int kBase = (int)sizeof(StreamSmem<DIM, R8>), kMost = kBase + kMaxPages * (int)sizeof(PageEntry);
  static int per_sm[64] = {};  // blocks per SM with few pages, which is the case where it counts
  const int dv = current_device() & 63;
  if (!per_sm[dv]) {
    int n = 0;
    if (!ACF_CUDA_OK(cudaFuncSetAttribute(k_attn_stream<T, DIM, R8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost)) ||
        !ACF_CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_attn_stream<T, DIM, R8>, kWarps * 32, kBase + 1024)))
      return false;
    per_sm[dv] = std::max(1, n);
  }
  StreamArgs p = {};
  p.a = a;
  const long long tiles = (std::min(std::min(a.b.max_new, a.b.tokens) * (long long)a.group, a.rows_most) + 8 * R8 - 1) / (8 * R8);
  if (tiles * a.kv.heads > 0x7fffffffLL) {
    set_error(kInvalid, "acfun_kv8_attention: too many rows");
    return false;
  }
  p.row_tiles = (int)tiles;
  // Split the keys so that one wave of resident blocks covers the batch.  Sequences of a batch may
  // differ in length: chunks of at most about 2048 keys keep the longest from being the last (48 ragged
  // sequences: 512 keys 73 us, 1024 and 2048 59 us), longer ones only where these would make more
  // than 16 waves of blocks.  Blocks that walk a list of the chunks there are, made from the lengths
  // in the kernel, took 61 us: their start has to wait for the list.
  const long long work = tiles * a.kv.heads * a.b.seqs;
  const long long slots = (long long)per_sm[dv] * c.sm_count();
  const long long want = std::max<long long>(1, slots / std::max<long long>(1, work));
  long long chunk = (a.b.max_len + want - 1) / want;
  if (a.b.seqs > 1) chunk = std::min(chunk, std::max<long long>(2048, work * a.b.max_len / (16 * slots)));
  chunk = std::max<long long>(chunk, kUnit * kPair * kWarps);
  chunk = std::min<long long>((chunk + kUnit - 1) / kUnit * kUnit, (long long)(kMaxPages - 1) * a.kv.page);
  p.chunk = (int)chunk;
  p.splits = (int)((a.b.max_len + 2 * kUnit + chunk - 1) / chunk);
  if (a.b.max_len <= chunk) p.splits = 1;
  if (p.splits > 65535) {
    set_error(kInvalid, "acfun_kv8_attention: max_len %d is too long for this page size", a.b.max_len);
    return false;
  }
  if (p.splits > 1) {
    // by sequence, not by token: beside a prompt only the rows of the short sequences are here
    p.part_rows = (int)std::min(std::min(a.b.max_new, a.b.tokens) * (long long)a.group, a.rows_most);
    const size_t n = (size_t)a.b.seqs * a.kv.heads * p.part_rows * p.splits;
    p.part_o = (float*)c.scratch(n * DIM * sizeof(float));
    p.part_ml = (float2*)c.scratch(n * sizeof(float2));
    bool zeroed = false;
    if (work <= kTickets && !c.capturing()) {
      p.tickets = tickets_of(c, dv, &zeroed);
    } else {
      p.tickets = (unsigned*)c.scratch((size_t)work * sizeof(unsigned));
      if (p.tickets && !ACF_CUDA_OK(cudaMemsetAsync(p.tickets, 0, (size_t)work * sizeof(unsigned), c.stream())))
        return false;
      zeroed = true;
    }
    if (zeroed) p.a.beside = false;  // the operation before in the stream is the memset, and is waited for
    if (!c.ok() || !p.tickets) return false;
  }
  const int smem = kBase + (int)std::min<long long>(chunk / a.kv.page + 2, kMaxPages) * (int)sizeof(PageEntry);
  if (!ACF_CUDA_OK(launch_pdl(k_attn_stream<T, DIM, R8>, dim3(p.row_tiles * a.kv.heads, a.b.seqs, p.splits), dim3(kWarps * 32), (size_t)smem, c.stream(), p, c.err())))
    return false;
  return c.launched("k_attn_stream");
}

template <typename T, int DIM>
bool stream_rows(Call& c, const AttnArgs& a) {
  // the widest tile that the rows fill: each tile reads (from L2, after the first) and converts the
  // keys again.  32 rows of 256 elements do not fit in the registers.
  const long long rows = std::min(std::min(a.b.max_new, a.b.tokens) * (long long)a.group, a.rows_most);
  if (rows <= 8) return stream_launch<T, DIM, 1>(c, a);
  if (rows <= 16 || DIM == 256) return stream_launch<T, DIM, 2>(c, a);
  return stream_launch<T, DIM, DIM == 256 ? 2 : 4>(c, a);
}

}  // namespace

bool attn_stream_dev(Call& c, const AttnArgs& a) {
  const int d = a.kv.dim;
  if (a.dtype == ACFUN_F16)
    return d == 64 ? stream_rows<__half, 64>(c, a) : d == 128 ? stream_rows<__half, 128>(c, a) : stream_rows<__half, 256>(c, a);
  return d == 64    ? stream_rows<__nv_bfloat16, 64>(c, a)
         : d == 128 ? stream_rows<__nv_bfloat16, 128>(c, a)
                    : stream_rows<__nv_bfloat16, 256>(c, a);
}

}  // namespace acf

using namespace acf;

extern "C" int acfun_kv8_attention(const AcfunKvCache8* cache, const AcfunKvBatch* batch, const void* q, void* out,
                                   int dtype, int q_heads, long long q_token, long long q_head, long long o_token,
                                   long long o_head, float scale, int causal, int window, float* lse) {
  const char* what = "acfun_kv8_attention";
  if (int e = check_dtype(what, dtype, false)) return e;
  if (int e = check_cache(what, cache)) return e;
  if (int e = check_batch(what, batch, cache->page)) return e;
  const int tokens = batch->tokens, dim = cache->dim;
  if (q_heads <= 0 || q_heads % cache->heads) {
    set_error(kInvalid, "%s: q_heads %d is not a positive multiple of the cache's %d heads", what, q_heads, cache->heads);
    return kInvalid;
  }
  if (!isfinite(scale)) {
    set_error(kInvalid, "%s: scale is not finite", what);
    return kInvalid;
  }
  if (window < 0 || (window > 0 && !causal)) {
    set_error(kInvalid, "%s: window %d must not be negative and needs causal", what, window);
    return kInvalid;
  }
  if ((long long)std::min(batch->max_new, tokens) * (q_heads / cache->heads) > 0x3fffffffLL) {
    set_error(kInvalid, "%s: max_new %d new tokens of %d heads are too many rows", what, batch->max_new, q_heads);
    return kInvalid;
  }
  if (int e = check_strides(what, q_token, q_head, tokens, q_heads, dim, false)) return e;
  if (int e = check_strides(what, o_token, o_head, tokens, q_heads, dim, true)) return e;
  if (batch->seqs == 0 || tokens == 0 || batch->max_new == 0) return 0;
  if (!q || !out) {
    set_error(kInvalid, "%s: q or out is NULL", what);
    return kInvalid;
  }
  Call c(what, true);
  if (!c.ok()) return last_error_code();
  AttnArgs a = {};
  a.kv = cache_view(cache);
  a.b = batch_view(c, batch);
  a.q = c.in(q, span_bytes(q_token, q_head, tokens, q_heads, dim, dtype));
  a.out = c.inout(out, span_bytes(o_token, o_head, tokens, q_heads, dim, dtype));
  a.lse = (float*)c.inout(lse, (size_t)tokens * q_heads * 4);
  if (!c.ok()) return last_error_code();
  a.q_token = q_token, a.q_head = q_head, a.o_token = o_token, a.o_head = o_head;
  a.dtype = dtype, a.q_heads = q_heads, a.group = q_heads / cache->heads;
  a.scale = scale, a.causal = causal != 0;
  // a window that holds any sequence hides nothing (and in the kernels position - window stays in range)
  a.window = window < batch->max_len ? window : 0;
  // Sequences with more than 32 rows per cache head go to the tensor cores' tiles of 128, the others are
  // streamed.  Measured with 32 query and 8 cache heads, 16 sequences of 4096 keys, bf16: heads of 128,
  // 16 rows 38 us streamed and 71 us tiled, 32 rows 56 and 71, 48 rows 97 and 71, 64 rows 99 and 71;
  // heads of 64, 39 and 60 at 32 rows, 66 and 60 at 48.  (One sequence of 32768 keys is even at about 20
  // rows: 16 rows 35 and 46, 32 rows 57 and 49.)  A batch may hold both kinds (decode steps beside
  // prompts); where every sequence has max_new tokens it does not.
  constexpr long long kStreamRows = 32;
  const long long most = std::min(batch->max_new, tokens) * (long long)a.group;
  const bool tiled = most > kStreamRows && dim != 256;
  const bool streamed = !tiled || (batch->seqs > 1 && a.group <= kStreamRows && tokens < (long long)batch->seqs * batch->max_new);
  bool ok = true;
  if (tiled) {
    a.rows_least = streamed ? kStreamRows + 1 : 0, a.rows_most = 0x7fffffffLL;
    ok = attn_tc_dev(c, a, &a.beside);
  }
  if (ok && streamed) {
    a.rows_least = 0, a.rows_most = tiled ? kStreamRows : 0x7fffffffLL;
    ok = attn_stream_dev(c, a);
  }
  if (!ok) c.fail();
  return c.finish() ? 0 : last_error_code();
}
