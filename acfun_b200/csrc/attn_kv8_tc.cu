// attn_kv8_tc.cu — attention over the int8 cache on the tcgen05 tensor cores, for calls with many
// rows per cache head (prompts, chunks of prompts, batches of drafts).
//
// Rows are packed as in attn_kv8.cu (row = token * group + head of the group), 256 to a block: two
// tiles of 128, A and B, against the same keys.  Per 64 keys and tile
//   S = Q K^T  (M = 128, N = 64, both operands in shared memory)  -> TMEM
//   w = 2^(S f + log2 s_v - m) in registers, one row per thread, rounded to fp16 -> TMEM, over S
//   O += w V   (A operand from TMEM, V's codes as fp16 in shared memory, N = dim)  -> TMEM
// so the tensor cores work on one tile while the other is in its softmax.  Codes are exact in fp16
// (and bf16); K and V scales enter the exponent as in attn_kv8.cu, and the running offset m moves
// only when a weight would pass 2^15, so O is rescaled a few times per row at most.
//
//   warps 0-3, 4-7  Q of tile A / B to shared memory, then its softmax and output (a TMEM lane and
//                   a row per thread)
// The codes become 16-bit operands in the MMA's 128-byte swizzled layout in one of two places:
//   in the kernel   warps 8-11 convert the block's keys one tile of 128 ahead (two stages each for K and
//                   V), warps 12 and 13 issue the MMAs; the cache is read once per 256 rows, at a byte
//                   a code.  K is fp16, and q is brought to fp16 by a power of two per row.
//   before it       k_kv8_tiles writes each key tile's image to scratch once, warp 10 only copies images
//                   (cp.async.bulk), warps 8 and 9 issue the MMAs.  K takes q's type.  Conversion costs the
//                   softmax's issue slots and registers, and with many row tiles it is repeated for each.
// TMEM: two buffers of S of A and of B (64 columns each; the fp16 weights overlay their first half),
// O of A and B.  With one buffer of 128 keys a softmax waited a third of its time for the products
// between its weights and its next scores.
//
// Measured (B200, 32 query and 8 cache heads of 128 elements, bf16, causal): a prompt of 8192 tokens
// 515-536 us, 1.0 PFLOP/s of what the mask leaves, 63 % of the measured bf16 peak, at 1.65 GHz under the
// board's power limit.  A step of 64 keys of both tiles takes about 1650 cycles; its products need 1280
// (their arithmetic alone 1024: the operands of S, both from shared memory, 48 cycles of its bandwidth per
// instruction of 32), its 2^x 770 of the special function units (a quarter of them on the FMA units: none
// 1.22 and half 1.11 times as long per softmax), and it issues 890 instructions per scheduler.  Two threads per
// row, with four softmax warps per scheduler instead of two, took 565 us: the exchange of maxima cost
// more than the latencies it hid.
// Every wait is bounded (ptx.cuh); on expiry the error word is set and all roles leave.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "attn_tile.cuh"

namespace acf {
namespace {

// Threads, and the registers (per thread) of the softmax warps, of the converters, and of the warps that
// issue; per warpgroup their sum is what the block is launched with.
template <bool PRE>
struct Roles;
template <>
struct Roles<false> {
  static constexpr int kThreads = 512, kMmaWarp = 12, kMmaWarpB = 13;  // 2 x 144 + 128 + 96 = 4 x 128
};
template <>
struct Roles<true> {
  static constexpr int kThreads = 384, kMmaWarp = 8, kMmaWarpB = 9, kCopyWarp = 10;  // 2 x 192 + 120 = 3 x 168
};
constexpr int kRows = 256;     // packed rows of a block
constexpr int kKeys = 128;     // keys per stage of K and V
constexpr int kStep = 64;      // keys of one S product and its softmax
constexpr int kUnits = kKeys / 16;
constexpr int kFmaOf4 = 1;      // pairs of four whose 2^x the FMA units compute instead of the special function unit
// A factor never underflows to 0: a masked score stays -inf under it.  With q's rows within [2^-40, 2^40] no
// score that matters has a smaller one.
constexpr float kLeast = 1e-37f;
// The offset from which a row's weights are taken from its rounded scores.  The common form, one fused
// operation on S, sees the rounding of the offset: below this within 2 powers of two, which kTop leaves
// room for, but from 2^27 on past fp16.
constexpr float kFar = 0x1p24f;
// Row tiles of a sequence from which the key tiles are converted before the kernel, and the most scratch
// that this may take.  Measured, one causal bf16 prompt, in the kernel and before it: 32 query and 8 cache
// heads of 128, 16 row tiles 28.6 and 28.9 us, 24 tiles 37.0 and 37.1, 32 tiles 52.1 and 49.5; 12 and 4
// heads of 64, 31.4 and 35.1, 43.3 and 43.8, 56.6 and 51.5; 8 and 8 heads of 128, where more blocks wait
// their turn, 81.5 and 73.9 at 16 tiles already.
constexpr int kPreRowTiles = 24;
constexpr size_t kPreBytes = size_t(1) << 30;
constexpr int kScaleRing = 4;  // the converters are at most two tiles ahead of a softmax

struct TcArgs {
  AttnArgs a;
  int chunk;       // key tiles per block
  int splits;
  float* part_o;   // [tokens][q_heads][splits][DIM], null when splits == 1
  float2* part_ml;
  // images of the key tiles made before the kernel: [seqs][heads][tiles] of K, V and their scales
  uint8_t* k_img;
  uint8_t* v_img;
  float4* scale_img;
  int tiles;
};

template <int DIM>
struct TcSmem {
  static constexpr int kChunks = DIM / 64;               // 128-byte column chunks
  static constexpr int kQTile = 128 * DIM * 2;
  static constexpr int kTile = kKeys * DIM * 2;          // one stage of K or V
  static constexpr int kQ = 0, kK = 2 * kQTile, kV = kK + 2 * kTile, kBars = kV + 2 * kTile;
  static constexpr int kScales = kBars + 256;
  static constexpr int kBytes = kScales + kScaleRing * kUnits * 16 + 1024;  // + alignment
  static_assert(kBytes <= 232448, "shared memory");
};

struct TcBars {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2][2], p_full[2][2], o_step[2], o_full, drain[2];  // [tile][buffer of S]
  uint32_t tmem;
  volatile int abort;
};
static_assert(sizeof(TcBars) <= 256, "barrier block");

__device__ __forceinline__ void umma_ts_f16(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// 32 consecutive columns of this warp's lanes; r points into a register array.
__device__ __forceinline__ void tmem_ld32p(uint32_t t, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(t));
}
__device__ __forceinline__ void tmem_ld16p(uint32_t t, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(t));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(t)
      : "memory");
}
// Two 32-bit operations per instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// 2^x of two values with the FMA units, for x >= -126: a fourth-degree minimax polynomial of the
// fraction (relative error 2.6e-6; one degree less would show in the sums, and so in lse) and the
// integer part added to its exponent.
__device__ __forceinline__ float2 ex2_fma2(float2 x) {
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
  x.x = fmaxf(x.x, -126.0f), x.y = fmaxf(x.y, -126.0f);
  const float2 r = add2(x, make_float2(kMagic, kMagic));
  const float2 n = add2(r, make_float2(-kMagic, -kMagic));
  const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
  float2 y = fma2(f, make_float2(0.009570102f, 0.009570102f), make_float2(0.05591786f, 0.05591786f));
  y = fma2(y, f, make_float2(0.24024744f, 0.24024744f));
  y = fma2(y, f, make_float2(0.6931218f, 0.6931218f));
  y = fma2(y, f, make_float2(0.9999993f, 0.9999993f));
  y.x = __uint_as_float(__float_as_uint(y.x) + (__float_as_uint(r.x) << 23));
  y.y = __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(r.y) << 23));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Eight codes (already XORed with 0x80 each) to fp16, one 16-byte unit.
__device__ __forceinline__ void put8(uint8_t* p, uint32_t w0, uint32_t w1) {
  uint4 o;
  o.x = f16_from_u8(w0, 0x4140), o.y = f16_from_u8(w0, 0x4342);
  o.z = f16_from_u8(w1, 0x4140), o.w = f16_from_u8(w1, 0x4342);
  *reinterpret_cast<uint4*>(p) = o;
}

// What a softmax needs of 16 keys' page: factor of S, log2 and reciprocal of the V scale.  Keys of a
// missing page are masked (past the length) or not seen (out of range): weight 0.
__device__ __forceinline__ float4 scale_entry(float2 ks_vs, bool there, float scale) {
  const float vs = fmaxf(ks_vs.y, 0x1p-100f);
  return there ? make_float4(fabsf(scale) * ks_vs.x * 1.4426950408889634f, log2f(vs), 1.0f / vs, 0.0f)
               : make_float4(1.0f, -INFINITY, 0.0f, 0.0f);
}

// Eight codes as T (exact in either type), one 16-byte unit; negated where `flip` is 0x80008000.
template <typename T>
__device__ __forceinline__ void put8_as(uint8_t* p, uint32_t w0, uint32_t w1, uint32_t flip) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (i < 2 ? w0 : w1) >> (16 * (i & 1));
    const T lo = from_f<T>((float)(int8_t)w), hi = from_f<T>((float)(int8_t)(w >> 8));
    o[i] = ((uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16) ^ flip;
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(o[0], o[1], o[2], o[3]);
}

// Images of the key tiles that some row of a sequence sees: block (tile, head, sequence), 256
// threads, half of them for K and half for V.  K takes q's type, so that q is used as it is, and the
// sign of the scale; V is fp16 as the weights are.  Bound by the write of two bytes per code.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) k_kv8_tiles(const TcArgs p, unsigned* err) {
  const AttnArgs& a = p.a;
  const int tile = blockIdx.x, head = blockIdx.y, seq = blockIdx.z;
  const SeqView sv = seq_view(a.b, seq, err);
  if (sv.n == 0 || !rows_taken(a, sv.n * a.group)) return;
  const KeyRange kr = key_range(a, sv, 0, sv.n * a.group, kKeys);
  if (tile < kr.first || tile >= kr.first + kr.n) return;
  const int v = threadIdx.x >> 7, t = threadIdx.x & 127;
  const int8_t* codes = v ? a.kv.v : a.kv.k;
  const size_t at = ((size_t)seq * a.kv.heads + head) * p.tiles + tile;
  uint8_t* img = (v ? p.v_img : p.k_img) + at * (kKeys * DIM * 2);
  auto page_of = [&](int key) -> int {
    return key < kr.hi && key + 15 >= kr.lo ? seq_page(a.b, seq, key >> a.kv.page_log2, a.kv.pages, err) : -1;
  };
  if (threadIdx.x < kUnits) {
    const int pg = page_of(tile * kKeys + threadIdx.x * 16);
    const size_t sc = (size_t)max(pg, 0) * a.kv.heads + head;
    p.scale_img[at * kUnits + threadIdx.x] =
        scale_entry(pg >= 0 ? make_float2(a.kv.ks[sc], a.kv.vs[sc]) : make_float2(0.f, 0.f), pg >= 0, a.scale);
  }
  constexpr int CPR = DIM / 16;  // 16-code chunks per row
  constexpr int STEP = 128 / CPR, N = kKeys / STEP;  // rows per pass: 16 (dim 128) or 32 (dim 64); passes
  const int c = t % CPR, r0 = t / CPR;
  int pg[N];
  uint4 w[N];
#pragma unroll
  for (int r = 0; r < N; ++r) {
    const int key = tile * kKeys + r * STEP + r0;
    pg[r] = (key & ~15) < kr.hi && key + 15 >= kr.lo ? __ldg(a.b.table + (size_t)seq * a.b.cols + (key >> a.kv.page_log2)) : -1;
  }
#pragma unroll
  for (int r = 0; r < N; ++r) {
    const int slot = (tile * kKeys + r * STEP + r0) & (a.kv.page - 1);
    w[r] = make_uint4(0, 0, 0, 0);
    if ((unsigned)pg[r] < (unsigned)a.kv.pages)  // what is not is reported with the scales above
      w[r] = __ldg(reinterpret_cast<const uint4*>(codes + (((size_t)pg[r] * a.kv.heads + head) * a.kv.page + slot) * DIM + c * 16));
  }
#pragma unroll
  for (int r = 0; r < N; ++r) {
    const int row = r * STEP + r0;
    uint8_t* o = img + (c >> 2) * (kKeys * 128) + row * 128;
    const int x = row & 7, u = 2 * (c & 3);
    if (v) {
      put8(o + ((u ^ x) << 4), w[r].x ^ 0x80808080u, w[r].y ^ 0x80808080u);
      put8(o + (((u + 1) ^ x) << 4), w[r].z ^ 0x80808080u, w[r].w ^ 0x80808080u);
    } else {
      const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
      put8_as<T>(o + ((u ^ x) << 4), w[r].x, w[r].y, flip);
      put8_as<T>(o + (((u + 1) ^ x) << 4), w[r].z, w[r].w, flip);
    }
  }
}

// Row tile `slot` of the batch's sequences in their order, the last rows of a sequence first (when causal
// they see the most keys); seq is -1 past the end.  The host does not know the lengths: a grid of
// [seqs][row tiles of max_new] left most blocks of a ragged batch without rows, and as a block takes an
// SM, the full ones came late (this kernel, 11 sequences of 2 to 1300 tokens, 12 query and 4 cache heads of
// 64, window 1000: 38.9 us, so 35.1).  Each warp scans the starts, 128 sequences at a time.
struct Slot {
  int seq, rt;
  SeqView sv;
};
__device__ __forceinline__ Slot find_slot(const AttnArgs& a, int slot, unsigned* err) {
  constexpr int K = 4;  // sequences per lane
  const int lane = threadIdx.x & 31;
  Slot s = {-1, 0, {0, 0, 0}};
  for (int s0 = 0; s0 < a.b.seqs; s0 += 32 * K) {
    SeqView v[K];
    int tiles[K], mine = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = s0 + lane * K + k;
      tiles[k] = 0;
      if (i < a.b.seqs) {
        v[k] = seq_view(a.b, i, err);
        const int rows = v[k].n * a.group;
        if (rows_taken(a, rows)) tiles[k] = (rows + kRows - 1) / kRows;
      }
      mine += tiles[k];
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, slot < upto);
    if (past) {
      const int owner = __ffs(past) - 1;
      int left = slot - (upto - mine);
      bool found = false;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!found && left < tiles[k]) {
          found = true;
          s.seq = s0 + lane * K + k, s.rt = tiles[k] - 1 - left, s.sv = v[k];
        }
        left -= tiles[k];
      }
      s.seq = __shfl_sync(0xffffffffu, s.seq, owner);
      s.rt = __shfl_sync(0xffffffffu, s.rt, owner);
      s.sv.row0 = __shfl_sync(0xffffffffu, s.sv.row0, owner);
      s.sv.n = __shfl_sync(0xffffffffu, s.sv.n, owner);
      s.sv.len = __shfl_sync(0xffffffffu, s.sv.len, owner);
      return s;
    }
    slot -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return s;
}

template <typename T, int DIM, bool PRE>
__global__ void __launch_bounds__(Roles<PRE>::kThreads, 1) k_attn_tc(const TcArgs p, unsigned* err) {
  using L = TcSmem<DIM>;
  extern __shared__ uint8_t smem_raw[];
  // Once every block is past the wait, everything before this kernel in the stream is complete, and the
  // streaming kernel of the same call may run on the SMs that are free.
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcBars& bar = *reinterpret_cast<TcBars*>(smem + L::kBars);
  float4* scales = reinterpret_cast<float4*>(smem + L::kScales);  // [ring][unit]: k factor, log2 v, 1 / v
  const AttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.x % a.kv.heads, part = blockIdx.y;
  const Slot slot = find_slot(a, blockIdx.x / a.kv.heads, err);
  const int seq = slot.seq;
  if (seq < 0) return;
  const SeqView sv = slot.sv;
  const int rows = sv.n * a.group, r0 = slot.rt * kRows;
  const int nr = min(kRows, rows - r0);
  const KeyRange kr = key_range(a, sv, r0, nr, kKeys);
  const int nsplit = max(1, (kr.n + p.chunk - 1) / p.chunk);
  if (part >= nsplit) return;
  const int tile0 = kr.first + part * p.chunk, ntiles = min(kr.n - part * p.chunk, p.chunk);
  // steps of 64 keys; the last key tile may need its first half only
  const int steps = ntiles > 0 ? min(2 * ntiles, (kr.hi - tile0 * kKeys + kStep - 1) / kStep) : 0;
  const bool two = nr > 128;

  if (threadIdx.x == 0) {
    dev::mbar_init(&bar.q_full, 8);
    for (int i = 0; i < 2; ++i) {
      dev::mbar_init(&bar.k_full[i], PRE ? 1 : 4);
      dev::mbar_init(&bar.k_empty[i], two ? 2 : 1);
      dev::mbar_init(&bar.v_full[i], PRE ? 1 : 4);
      dev::mbar_init(&bar.v_empty[i], two ? 2 : 1);
      dev::mbar_init(&bar.s_full[i][0], 1);
      dev::mbar_init(&bar.s_full[i][1], 1);
      dev::mbar_init(&bar.o_step[i], 1);
      dev::mbar_init(&bar.p_full[i][0], 4);
      dev::mbar_init(&bar.p_full[i][1], 4);
    }
    dev::mbar_init(&bar.o_full, two ? 2 : 1);
    dev::mbar_init(&bar.drain[0], 1);
    dev::mbar_init(&bar.drain[1], 1);
    bar.abort = 0;
    dev::fence_mbar_init();
  }
  if (warp == Roles<PRE>::kMmaWarp) {
    dev::tmem_alloc(&bar.tmem, 512);
    dev::tmem_relinquish();
  }
  dev::tc_fence_before();
  __syncthreads();
  dev::tc_fence_after();
  const uint32_t tmem = bar.tmem;
  const uint32_t tS0 = tmem, tO0 = tmem + 256;  // tile t: S at tS0 + 128 t, O at tO0 + DIM t
  auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
    if (dev::mbar_try_wait(dev::smem_u32(b), parity)) return true;
    if (bar.abort) return false;
    if (dev::mbar_wait(b, parity, err)) return true;
    bar.abort = 1;
    return false;
  };
  // one arrival for the warp, after what its lanes did
  auto arrive = [&](uint64_t* b) {
    __syncwarp();
    if (lane == 0) dev::mbar_arrive(b);
  };

  if (warp >= (PRE ? 8 : 12)) {
    // ---------------------------------------------------------------- MMA issuer, image copies
    if constexpr (PRE)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
    else
      asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if constexpr (PRE) {
      if (warp == Roles<PRE>::kCopyWarp && dev::elect_one()) {
        const size_t at = ((size_t)seq * a.kv.heads + head) * p.tiles + tile0;
        for (int j = 0; j < ntiles; ++j) {
          const int st = j & 1;
          const uint32_t eph = ((j >> 1) & 1) ^ 1;
          if (!wait(&bar.k_empty[st], eph)) break;
          dev::mbar_arrive_expect_tx(&bar.k_full[st], L::kTile + kUnits * 16);
          dev::bulk_load(smem + L::kK + st * L::kTile, p.k_img + (at + j) * L::kTile, L::kTile, &bar.k_full[st]);
          dev::bulk_load(scales + (j % kScaleRing) * kUnits, p.scale_img + (at + j) * kUnits, kUnits * 16, &bar.k_full[st]);
          // the first product needs Q and the first K tile: what follows waits until Q is there
          if (j == 0 && !wait(&bar.q_full, 0)) break;
          if (!wait(&bar.v_empty[st], eph)) break;
          dev::mbar_arrive_expect_tx(&bar.v_full[st], L::kTile);
          dev::bulk_load(smem + L::kV + st * L::kTile, p.v_img + (at + j) * L::kTile, L::kTile, &bar.v_full[st]);
        }
        // no copy may be in flight when the block leaves: the last stages' are waited for (an
        // aborted block's too)
        for (int j = max(0, ntiles - 2); j < ntiles; ++j) {
          dev::mbar_wait(&bar.k_full[j & 1], (j >> 1) & 1, nullptr, 200000000ull);
          dev::mbar_wait(&bar.v_full[j & 1], (j >> 1) & 1, nullptr, 200000000ull);
        }
      }
    }
    // The issuing thread is one that elect.sync names: with a thread picked by its lane number the
    // compiler has to move every operand to uniform registers by itself, and next to busy softmax
    // warps an instruction then took 116 cycles to issue instead of the 64 that it runs.
    // Each tile has an issuer of its own: a wait costs one 100 cycles and more even when it is over,
    // and the other's products run meanwhile.
    const int t = warp == Roles<PRE>::kMmaWarpB;
    if ((warp == Roles<PRE>::kMmaWarp || (t && two)) && steps > 0 && dev::elect_one()) {
      constexpr uint32_t kQType = PRE && std::is_same<T, __nv_bfloat16>::value ? 1 : 0;  // of Q and K: bf16 or f16
      constexpr uint32_t idS = dev::umma_idesc(1, kQType, kQType, 0, 0, 128, kStep), idO = dev::umma_idesc(1, 0, 0, 0, 1, 128, DIM);
      const uint32_t base = dev::smem_u32(smem);
      const uint64_t dQ = dev::umma_sdesc(base + L::kQ + t * L::kQTile, 16, 1024, dev::UMMA_SW128);
      const uint64_t dK = dev::umma_sdesc(base + L::kK, 16, 1024, dev::UMMA_SW128);
      const uint64_t dV = dev::umma_sdesc(base + L::kV, kKeys * 128, 1024, dev::UMMA_SW128);
      const uint32_t tS = tS0 + t * 128, tO = tO0 + t * DIM;
      // Descriptors are formed anew for each group of products: left to itself the compiler keeps all
      // of them across the loop, which in this role's registers means local memory, and a load from it
      // per instruction made the products of S four times as long as the tensor cores take.
      auto fresh = [](uint64_t d) {
        uint64_t r;
        asm volatile("mov.b64 %0, %1;" : "=l"(r) : "l"(d));
        return r;
      };
      // S for the 64 keys of step i, into the buffer of the step's parity
      auto mma_s = [&](int i) {
        const uint64_t q = fresh(dQ);
        const uint64_t k = fresh(dK + ((((i >> 1) & 1) * L::kTile + (i & 1) * kStep * 128) >> 4));
#pragma unroll
        for (int ks = 0; ks < DIM / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * (kKeys * 128) + (ks & 3) * 32) >> 4;
          dev::umma<dev::MmaKind::F16>(tS + (i & 1) * kStep, q + off, k + off, idS, ks != 0);
        }
        dev::umma_commit(&bar.s_full[t][i & 1]);
      };
      bool ok = wait(&bar.q_full, 0) && wait(&bar.k_full[0], 0);
      dev::tc_fence_after();
      for (int i = 0; i < min(steps, 2) && ok; ++i) {
        mma_s(i);
        if (i == 1) dev::umma_commit(&bar.k_empty[0]);
      }
      // S runs two steps ahead of O, so a softmax finds its next scores when it is done with the last
      for (int i = 0; i < steps; ++i) {
        const int n = i + 2, j = i >> 1, jn = n >> 1;
        if (ok && !(i & 1)) ok = wait(&bar.v_full[j & 1], (j >> 1) & 1);
        if (ok && n < steps && !(n & 1)) ok = wait(&bar.k_full[jn & 1], (jn >> 1) & 1);
        if (!(ok = ok && wait(&bar.p_full[t][i & 1], j & 1))) break;
        dev::tc_fence_after();
        const uint64_t v = fresh(dV + (((j & 1) * L::kTile + (i & 1) * kStep * 128) >> 4));
#pragma unroll
        for (int ks = 0; ks < kStep / 16; ++ks)
          umma_ts_f16(tO, tS + (i & 1) * kStep + ks * 8, v + ((ks * 2048) >> 4), idO, (i | ks) != 0);
        dev::umma_commit(&bar.o_step[t]);
        if (i & 1) dev::umma_commit(&bar.v_empty[j & 1]);
        if (n < steps) {
          mma_s(n);
          if (n & 1) dev::umma_commit(&bar.k_empty[jn & 1]);
        }
      }
      if (ok) {
        dev::umma_commit(&bar.o_full);
      } else {
        bar.abort = 1;
        dev::umma_commit(&bar.drain[t]);
        dev::mbar_wait(&bar.drain[t], 0, nullptr, 200000000ull);
      }
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- converters
    if constexpr (!PRE) {
        constexpr int N = DIM / 16;  // 16-code loads per thread, tile and operand
      const int cw = warp - 8, ct = threadIdx.x - 256;
      const int lg = a.kv.page_log2;
      // Lanes take 4 chunks x 8 rows at a time: 64-byte segments from memory and, as neighbouring
      // rows swizzle to the other parity of 16-byte units, shared-memory stores without conflicts.
      // Load i: rows cw * 32 + (i / (DIM / 64)) * 8 + lane / 4, chunk (i % (DIM / 64)) * 4 + lane % 4.
      // Page numbers are fetched two tiles ahead of their use and looked at only then: a check right
      // after the load would wait for memory twice per tile.
      int next_pid[2], next_sc = -1;
      float2 sc = {0.f, 0.f};
      int sc_ok = 0;
      // page of the 16 keys from `key` on; -1 where no row of the block sees them
      auto fetch_pid = [&](int key) -> int {
        return key < kr.hi && key + 15 >= kr.lo ? __ldg(a.b.table + (size_t)seq * a.b.cols + (key >> lg)) : -1;
      };
      // a page number that is out of range is reported, and its keys are not seen
      auto good = [&](int pid, int key) -> int {
        if ((unsigned)pid < (unsigned)a.kv.pages) return pid;
        if (key < kr.hi && key + 15 >= kr.lo) atomicOr(err, ACF_DEV_ERR_BADARG);
        return -1;
      };
      auto fetch = [&](int j) {
        const int key = (tile0 + j) * kKeys;
        next_pid[0] = fetch_pid(key + cw * 32);
        next_pid[1] = fetch_pid(key + cw * 32 + 16);
        if (ct < kUnits) next_sc = fetch_pid(key + ct * 16);
      };
      int pid[2];
      auto take = [&](int j) {  // the fetched numbers become tile j's; its scales are requested
        const int key = (tile0 + j) * kKeys;
        pid[0] = good(next_pid[0], key + cw * 32);
        pid[1] = good(next_pid[1], key + cw * 32 + 16);
        if (ct < kUnits) {
          const int pg = good(next_sc, key + ct * 16);
          sc_ok = pg >= 0;
          if (sc_ok) {
            const size_t at = (size_t)pg * a.kv.heads + head;
            sc = make_float2(a.kv.ks[at], a.kv.vs[at]);
          }
        }
      };
      const int key_in_unit = lane >> 2;
      auto load_tile = [&](const int8_t* codes, uint4 (&r)[N]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int slot = (cw * 32 + u * 16 + key_in_unit) & (a.kv.page - 1);  // tiles start at multiples of every page size
          const int8_t* src = codes + (((size_t)max(pid[u], 0) * a.kv.heads + head) * a.kv.page + slot) * DIM + (lane & 3) * 16;
#pragma unroll
          for (int i = u * N / 2; i < (u + 1) * N / 2; ++i) {
            r[i] = make_uint4(0, 0, 0, 0);
            if (pid[u] >= 0)
              r[i] = __ldg(reinterpret_cast<const uint4*>(src + ((i / L::kChunks) & 1) * 8 * DIM + (i % L::kChunks) * 64));
          }
        }
      };
      // this thread's two 16-byte units of row cw * 32 + lane / 4; its other rows are 8 apart
      const int unit0 = (cw * 32 + key_in_unit) * 128 + (((2 * (lane & 3)) ^ key_in_unit) << 4);
      const int unit1 = (cw * 32 + key_in_unit) * 128 + (((2 * (lane & 3) + 1) ^ key_in_unit) << 4);
      auto put_tile = [&](uint8_t* tile, const uint4 (&r)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int off = (i / L::kChunks) * 8 * 128 + (i % L::kChunks) * (kKeys * 128);
          put8(tile + unit0 + off, r[i].x ^ 0x80808080u, r[i].y ^ 0x80808080u);
          put8(tile + unit1 + off, r[i].z ^ 0x80808080u, r[i].w ^ 0x80808080u);
        }
      };
      uint4 kreg[N], vreg[N];
      if (ntiles > 0) {
        fetch(0);
        take(0);
        if (ntiles > 1) fetch(1);
        load_tile(a.kv.k, kreg);
        load_tile(a.kv.v, vreg);
      }
      for (int j = 0; j < ntiles; ++j) {
        const int st = j & 1;
        const uint32_t eph = ((j >> 1) & 1) ^ 1;
        const bool more = j + 1 < ntiles;
        if (!wait(&bar.k_empty[st], eph)) break;
        put_tile(smem + L::kK + st * L::kTile, kreg);
        if (ct < kUnits) {
          scales[(j % kScaleRing) * kUnits + ct] = scale_entry(sc, sc_ok, a.scale);
        }
        dev::fence_proxy_async_smem();
        arrive(&bar.k_full[st]);
        if (more) {
          take(j + 1);
          if (j + 2 < ntiles) fetch(j + 2);
          load_tile(a.kv.k, kreg);
        }
        if (!wait(&bar.v_empty[st], eph)) break;
        put_tile(smem + L::kV + st * L::kTile, vreg);
        dev::fence_proxy_async_smem();
        arrive(&bar.v_full[st]);
        if (more) load_tile(a.kv.v, vreg);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax, one row per thread
    if constexpr (PRE)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    else
      asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    const int t = warp >> 2, row = threadIdx.x & 127;
    const int r = r0 + t * 128 + row;
    const bool in = r < rows;
    const int tok = r / a.group, hq = head * a.group + r - tok * a.group;
    float q_unit = 1.0f;
    {
      // Q to shared memory: a warp copies its 32 rows as they are, all in flight at once, DIM / 8 lanes
      // with 16 bytes of a row each; a row's place in memory comes from the lane that owns the row.
      constexpr int LPR = DIM / 8, RPP = 32 / LPR, N = 32 / RPP;  // lanes per row, rows per pass, passes
      const int sub = lane / LPR, c = lane % LPR;
      const T* q = static_cast<const T*>(a.q);
      const bool vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && a.q_token % 8 == 0 && a.q_head % 8 == 0;
      const long long own = in ? (long long)(sv.row0 + tok) * a.q_token + (long long)hq * a.q_head : -1;
      uint8_t* tile = smem + L::kQ + t * L::kQTile;
      uint8_t* at = tile + (c >> 3) * (128 * 128) + ((warp & 3) * 32 + sub) * 128;
#pragma unroll 8
      for (int i = 0; i < N; ++i) {
        const long long from = __shfl_sync(0xffffffffu, own, i * RPP + sub);
        uint8_t* to = at + i * RPP * 128 + (((c & 7) ^ ((i * RPP + sub) & 7)) << 4);
        if (from < 0) {
          *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
        } else if (vec) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dev::smem_u32(to)), "l"(q + from + c * 8) : "memory");
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(to)[e] = q[from + c * 8 + e];
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      // Where K is fp16 and q is not (or the scale's sign has to go somewhere), each thread converts its
      // row in place, scaled by a power of two.
      if (!PRE && (!std::is_same<T, __half>::value || a.scale < 0.0f)) {
        __syncwarp();
        uint8_t* mine = tile + row * 128;
        float top = 0.0f;
#pragma unroll 4
        for (int k = 0; k < DIM / 8; ++k) {
          float x[8];
          load8(reinterpret_cast<const T*>(mine + (k >> 3) * (128 * 128) + (((k & 7) ^ (row & 7)) << 4)), true, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
        }
        const Pow2 f = row_pow2(top);
        const float down = copysignf(f.down, a.scale);
        q_unit = f.up;
#pragma unroll 4
        for (int k = 0; k < DIM / 8; ++k) {
          uint8_t* p16 = mine + (k >> 3) * (128 * 128) + (((k & 7) ^ (row & 7)) << 4);
          float x[8];
          load8(reinterpret_cast<const T*>(p16), true, x);
          uint4 o;
          o.x = pack_f16(x[0] * down, x[1] * down), o.y = pack_f16(x[2] * down, x[3] * down);
          o.z = pack_f16(x[4] * down, x[5] * down), o.w = pack_f16(x[6] * down, x[7] * down);
          *reinterpret_cast<uint4*>(p16) = o;
        }
      }
      // Where K takes bf16 as q does, a row's products with codes can pass 2^128 although its scores do not:
      // such a row is brought down by a power of two, in place and exactly, and so is one so small that
      // its products would be subnormal brought up.
      if constexpr (PRE && std::is_same<T, __nv_bfloat16>::value) {
        __syncwarp();
        uint8_t* mine = tile + row * 128;
        auto part = [&](int k) { return reinterpret_cast<uint4*>(mine + (k >> 3) * (128 * 128) + (((k & 7) ^ (row & 7)) << 4)); };
        __nv_bfloat162 most = __float2bfloat162_rn(0.0f);
#pragma unroll 4
        for (int k = 0; k < DIM / 8; ++k) {
          const uint4 w = *part(k);
          const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
          for (int e = 0; e < 4; ++e) most = __hmax2(most, __habs2(x[e]));
        }
        const float top = fmaxf(__low2float(most), __high2float(most));
        if (top > 0x1p40f || (top > 0.0f && top < 0x1p-40f)) {
          const Pow2 f = row_pow2(top);
          q_unit = f.up;
#pragma unroll 1
          for (int k = 0; k < DIM / 8; ++k) {
            float x[8];
            load8(reinterpret_cast<const T*>(part(k)), true, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= f.down;
            store8(reinterpret_cast<T*>(part(k)), true, x);
          }
        }
      }
      dev::fence_proxy_async_smem();
      arrive(&bar.q_full);
    }
    const int pos = sv.len - sv.n + tok;
    // a thread without a row masks nothing (its zeros of Q give results that are not written): the
    // masking of a ragged end's warps made its block a quarter longer
    const int see_hi = !in ? 0x7fffffff : pos < 0 ? 0 : a.causal ? min(sv.len, pos + 1) : sv.len;
    const int see_lo = in && a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    const bool active = t == 0 || two;
    // Rows that the common form of a weight does not serve (`odd`: those with a factor of their own beside K
    // in bf16, and those whose offset has passed kFar) go by their scores, formed in place of S before the
    // maximum, and turned back after it into what that form makes the same weights of.  A warp with such a
    // row takes a loop of its own: in the one loop this took 3 % of a long prompt (488 against 473 us in a
    // burst).
    bool odd = PRE && q_unit != 1.0f;
    auto factor = [&](const float4& f) { return fmaxf(PRE ? f.x : f.x * q_unit, kLeast); };
    // Steps from i on; the first one that was not done.
    auto softmax = [&](int i, auto with_odd) -> int {
      constexpr bool ODD = decltype(with_odd)::value;
      for (; i < steps; ++i) {
        const uint32_t tS = tS0 + t * 128 + (i & 1) * kStep + lanes;
        if (!(ok = wait(&bar.s_full[t][i & 1], (i >> 1) & 1))) return i;
        dev::tc_fence_after();
        float s[kStep];
        tmem_ld32p(tS, s);
        tmem_ld32p(tS + 32, s + 32);
        dev::tmem_ld_wait();
        const float4* sc = scales + ((i >> 1) % kScaleRing) * kUnits + (i & 1) * (kUnits / 2);
        const int k0 = tile0 * kKeys + i * kStep;
        const int lo = see_lo - k0, hi = see_hi - k0;
        if (__any_sync(0xffffffffu, lo > 0 || hi < kStep)) {
          // opaque bounds: the comparisons stay inside this branch instead of running for every step
          int from = lo, to = hi;
          asm volatile("" : "+r"(from), "+r"(to));
#pragma unroll
          for (int e = 0; e < kStep; ++e)
            if (e < from || e >= to) s[e] = -INFINITY;
        }
        float top = -INFINITY;
        auto scores = [&] {
          top = -INFINITY;
#pragma unroll
          for (int u = 0; u < kStep / 16; ++u) {
            const float4 f = sc[u];
            const float fx = fmaxf(f.x * q_unit, kLeast);
#pragma unroll
            for (int e = 16 * u; e < 16 * u + 16; ++e) s[e] = fmaf(s[e], fx, f.y), top = fmaxf(top, s[e]);
          }
        };
        if (ODD && odd) {
          scores();
        } else {
#pragma unroll
          for (int u = 0; u < kStep / 16; ++u) {
            const float* v = s + 16 * u;
            const float x0 = max3(max3(v[0], v[1], v[2]), v[3], v[4]), x1 = max3(max3(v[5], v[6], v[7]), v[8], v[9]);
            const float x2 = max3(max3(v[10], v[11], v[12]), v[13], v[14]);
            const float4 f = sc[u];
            top = fmaxf(top, fmaf(max3(fmaxf(x0, v[15]), x1, x2), factor(f), f.y));
          }
        }
        if (__any_sync(0xffffffffu, top > m + kMost)) {
          const float n = fmaxf(m, top - kTop);
          if constexpr (ODD) {
            if (!odd && fabsf(n) >= kFar && n != -INFINITY) odd = true, scores();
            __syncwarp();
          } else {
            if (__any_sync(0xffffffffu, fabsf(n) >= kFar && n != -INFINITY)) return i;  // again, in the other loop
          }
          const float b = m == n ? 1.0f : ex2(m - n);
          m = n;
          l *= b;
          if (i > 0) {  // O holds the steps before this one, once the last of them is done
            if (!(ok = wait(&bar.o_step[t], (i - 1) & 1))) return i;
            dev::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < DIM / 16; ++c) {
              float o[16];
              tmem_ld16p(tO0 + t * DIM + lanes + c * 16, o);
              dev::tmem_ld_wait();
              uint32_t x[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(o[e] * b);
              tmem_st16(tO0 + t * DIM + lanes + c * 16, x);
            }
          }
        }
        float m0 = m == -INFINITY ? 0.0f : m;
        if constexpr (ODD) {
          if (odd) {  // s * factor + (f.y - 0) is to be score - m0
#pragma unroll
            for (int u = 0; u < kStep / 16; ++u) {
              const float4 f = sc[u];
              const float r = 1.0f / factor(f);
#pragma unroll
              for (int e = 16 * u; e < 16 * u + 16; ++e) s[e] = s[e] == -INFINITY ? s[e] : ((s[e] - m0) - f.y) * r;
            }
            m0 = 0.0f;
          }
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < kStep / 32; ++h) {  // 32 keys: 16 registers of weights
          uint32_t w[16];
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int u = 2 * h + v;
            const float4 f = sc[u];
            const float fx = factor(f), off = f.y - m0;
            const float2 fx2 = make_float2(fx, fx), off2 = make_float2(off, off);
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float2 x = fma2(make_float2(s[16 * u + e], s[16 * u + e + 1]), fx2, off2);
              if ((e / 2) % 4 >= kFmaOf4) {
                x.x = ex2(x.x), x.y = ex2(x.y);
              } else {
                x = ex2_fma2(x);
              }
              sum = add2(sum, x);
              w[8 * v + e / 2] = pack_f16(x.x, x.y);
            }
            l = fmaf(sum.x + sum.y, f.z, l);
          }
          tmem_st16(tS + 16 * h, w);
        }
        tmem_st_wait();
        dev::tc_fence_before();
        arrive(&bar.p_full[t][i & 1]);
      }
      return steps;
    };
    if (active) {
      const int i = __any_sync(0xffffffffu, odd) ? 0 : softmax(0, std::false_type());
      if (ok && i < steps) softmax(i, std::true_type());
    }
    if (ok && ntiles > 0) ok = wait(&bar.o_full, 0);
    dev::tc_fence_after();
    if (active) {
      // no key seen: m is -inf and l holds at most the least powers of two (a NaN has m = -inf too)
      const bool none = ntiles == 0 || (m == -INFINITY && l == l);
      const float inv = none ? 0.0f : 1.0f / l;
      const bool whole = nsplit == 1;
      const size_t at = ((size_t)(sv.row0 + tok) * a.q_heads + hq) * p.splits + part;
      // A thread has a row, but 32 rows at a time are 32 places in memory: the rows go through this
      // tile's part of Q, which no product needs any more, and leave DIM / 8 lanes to a row.
      uint8_t* stage = smem + L::kQ + t * L::kQTile + row * 128;
#pragma unroll 2
      for (int i = 0; i < DIM / 32; ++i) {
        float o[32];
        if (ntiles > 0) {
          tmem_ld32p(tO0 + t * DIM + lanes + i * 32, o);
          dev::tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.0f;
        }
        if (!ok) continue;
        if (whole) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = none ? 0.0f : o[e + k] * inv;
            const int k16 = i * 4 + e / 8;
            store8(reinterpret_cast<T*>(stage + (k16 >> 3) * (128 * 128) + (((k16 & 7) ^ (row & 7)) << 4)), true, x);
          }
        } else if (in) {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(p.part_o + at * DIM + i * 32 + e) =
                none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
      if (whole && ok) {
        constexpr int LPR = DIM / 8, RPP = 32 / LPR;
        const int sub = lane / LPR, c = lane % LPR;
        T* out = static_cast<T*>(a.out);
        const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && a.o_token % 8 == 0 && a.o_head % 8 == 0;
        const long long own = in ? (long long)(sv.row0 + tok) * a.o_token + (long long)hq * a.o_head : -1;
        const uint8_t* from = smem + L::kQ + t * L::kQTile + (c >> 3) * (128 * 128) + ((warp & 3) * 32 + sub) * 128;
        __syncwarp();
#pragma unroll 8
        for (int i = 0; i < 32 / RPP; ++i) {
          const long long to = __shfl_sync(0xffffffffu, own, i * RPP + sub);
          if (to < 0) continue;
          const uint4 w = *reinterpret_cast<const uint4*>(from + i * RPP * 128 + (((c & 7) ^ ((i * RPP + sub) & 7)) << 4));
          if (vec) {
            *reinterpret_cast<uint4*>(out + to + c * 8) = w;
          } else {
            const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int e = 0; e < 8; ++e) out[to + c * 8 + e] = x[e];
          }
        }
      }
      if (in && ok) {
        if (!whole)
          p.part_ml[at] = make_float2(m, none ? 0.0f : l);
        else if (a.lse)
          a.lse[(long long)(sv.row0 + tok) * a.q_heads + hq] =
              none ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
      }
    }
  }
  dev::tc_fence_before();
  __syncthreads();
  if (warp == Roles<PRE>::kMmaWarp) {
    dev::tc_fence_after();
    dev::tmem_dealloc(tmem, 512);
  }
}

// Joins the key parts of split rows, in the order of the parts: one warp per (token, head).
template <typename T, int DIM>
__global__ void __launch_bounds__(128) k_attn_join(const TcArgs p, unsigned* err) {
  const AttnArgs& a = p.a;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, seq = blockIdx.y;
  dev::grid_dep_wait();
  dev::grid_dep_launch();
  const SeqView sv = seq_view(a.b, seq, err);
  if (item >= (long long)sv.n * a.q_heads || !rows_taken(a, sv.n * a.group)) return;
  const int tok = (int)(item / a.q_heads), hq = (int)(item - (long long)tok * a.q_heads);
  const int r = tok * a.group + hq % a.group, r0 = r / kRows * kRows;
  const KeyRange kr = key_range(a, sv, r0, min(kRows, sv.n * a.group - r0), kKeys);
  const int nsplit = max(1, (kr.n + p.chunk - 1) / p.chunk);
  if (nsplit == 1) return;  // written whole
  const size_t at = ((size_t)(sv.row0 + tok) * a.q_heads + hq) * p.splits;
  float top = -INFINITY, sum = 0.0f;
  for (int k = 0; k < nsplit; ++k) top = fmaxf(top, p.part_ml[at + k].x);
  float o[DIM / 32] = {};
  for (int k = 0; k < nsplit; ++k) {
    const float2 ml = p.part_ml[at + k];
    const float b = ml.x == top ? 1.0f : ex2(ml.x - top);
    sum = fmaf(ml.y, b, sum);
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i) o[i] = fmaf(p.part_o[(at + k) * DIM + i * 32 + lane], b, o[i]);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  T* dst = static_cast<T*>(a.out) + (long long)(sv.row0 + tok) * a.o_token + (long long)hq * a.o_head;
#pragma unroll
  for (int i = 0; i < DIM / 32; ++i) dst[i * 32 + lane] = from_f<T>(sum == 0.0f ? 0.0f : o[i] * inv);
  if (lane == 0 && a.lse)
    a.lse[(long long)(sv.row0 + tok) * a.q_heads + hq] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

template <typename T, int DIM, bool PRE>
bool tc_launch(Call& c, TcArgs p, dim3 grid) {
  using L = TcSmem<DIM>;
  static bool attr_done[64] = {false};
  const int dv = current_device() & 63;
  if (!attr_done[dv]) {
    if (!ACF_CUDA_OK(cudaFuncSetAttribute(k_attn_tc<T, DIM, PRE>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes)))
      return false;
    attr_done[dv] = true;
  }
  if (!ACF_CUDA_OK(launch_pdl(k_attn_tc<T, DIM, PRE>, grid, dim3(Roles<PRE>::kThreads), (size_t)L::kBytes, c.stream(), p, c.err()))) return false;
  return c.launched("k_attn_tc");
}

template <typename T, int DIM>
bool tc_run(Call& c, const AttnArgs& a, bool* last_is_main) {
  TcArgs p = {};
  p.a = a;
  const long long max_new = std::min(a.b.max_new, a.b.tokens);
  const long long row_tiles = (max_new * a.group + kRows - 1) / kRows;  // of one sequence
  const long long slots = std::min(row_tiles * a.b.seqs, (long long)a.b.tokens * a.group / kRows + a.b.seqs);
  const long long work = slots * a.kv.heads;
  if (work > 0x7fffffffLL) {
    set_error(kInvalid, "acfun_kv8_attention: too many rows");
    return false;
  }
  // few blocks: the keys are split so that every SM gets one, in parts of at least 4 key tiles
  const int tiles = (a.b.max_len + kKeys - 1) / kKeys;
  const long long want = std::max<long long>(1, c.sm_count() / std::max<long long>(1, work));
  // most key tiles that a block's rows see; a window's can start and end inside a tile
  const int most = a.window > 0 ? (int)std::min<long long>(tiles, ((long long)a.window + kRows / a.group + 1) / kKeys + 2) : tiles;
  p.chunk = (int)std::max<long long>(4, (most + want - 1) / want);
  p.splits = (most + p.chunk - 1) / p.chunk;
  if (p.splits > 1) {
    const size_t n = (size_t)a.b.tokens * a.q_heads * p.splits;
    p.part_o = (float*)c.scratch(n * DIM * sizeof(float));
    p.part_ml = (float2*)c.scratch(n * sizeof(float2));
    if (!c.ok()) return false;
  }
  // tile images before the kernel: where the conversion would be repeated, and they fit
  const size_t images = (size_t)a.b.seqs * a.kv.heads * tiles;
  const bool pre = row_tiles >= kPreRowTiles && images * (2 * kKeys * DIM * 2) <= kPreBytes;
  const dim3 grid((unsigned)work, p.splits);
  if (pre) {
    p.tiles = tiles;
    p.k_img = (uint8_t*)c.scratch(images * kKeys * DIM * 2);
    p.v_img = (uint8_t*)c.scratch(images * kKeys * DIM * 2);
    p.scale_img = (float4*)c.scratch(images * kUnits * sizeof(float4));
    if (!c.ok()) return false;
    k_kv8_tiles<T, DIM><<<dim3(tiles, a.kv.heads, a.b.seqs), 256, 0, c.stream()>>>(p, c.err());
    if (!c.launched("k_kv8_tiles") || !tc_launch<T, DIM, true>(c, p, grid)) return false;
  } else if (!tc_launch<T, DIM, false>(c, p, grid)) {
    return false;
  }
  *last_is_main = p.splits == 1;
  if (p.splits > 1) {
    const long long items = (max_new * a.q_heads + 3) / 4;
    const dim3 each((unsigned)items, a.b.seqs);
    if (!ACF_CUDA_OK(launch_pdl(k_attn_join<T, DIM>, each, dim3(128), (size_t)0, c.stream(), p, c.err()))) return false;
    return c.launched("k_attn_join");
  }
  return true;
}

}  // namespace

bool attn_tc_dev(Call& c, const AttnArgs& a, bool* last_is_main) {
  if (a.dtype == ACFUN_F16) return a.kv.dim == 64 ? tc_run<__half, 64>(c, a, last_is_main) : tc_run<__half, 128>(c, a, last_is_main);
  return a.kv.dim == 64 ? tc_run<__nv_bfloat16, 64>(c, a, last_is_main) : tc_run<__nv_bfloat16, 128>(c, a, last_is_main);
}

}  // namespace acf
