// The paged 8-bit KV cache on gfx950: rows of K and V quantized as they are
// written, read back, and attended over, with their C-ABI entry points
// (include/kvdec_paged8.h).

#include <algorithm>

#include "kvdec_device.h"
#include "kvdec_paged8.h"

using namespace kvdec;

namespace {

typedef __attribute__((address_space(4))) const int32_t cint32;

constexpr int kCodeRow = kHeadDim;      // bytes of a row of codes
constexpr int kLowest = -100;           // least exponent of a scale the writer makes
enum { kInt8 = 0, kE4m3 = 1 };

// A cache and the new tokens' offsets, as the kernels take them.
struct Cache8 {
  char* k;
  char* v;
  float* ks;
  float* vs;
  const int32_t* bt;
  const int32_t* lens;
  const int32_t* cu;          // [B + 1], or null: one new token a sequence
  int64_t page_bytes, head_bytes, num_pages;
  int64_t B, T;
  uint32_t row_bytes;
  int ps_log2, blk_log2;      // page and block sizes
  int max_blocks, max_len;    // table entries of a sequence, and their tokens
  int KVH;
};

// New tokens [c0, c0 + n) of the call are the last n of a sequence's len.
struct Seq8 {
  int b, c0, n, len;
};

// Offset of sequence b's first new token (sequence 0's is 0), inside [0, T]
// whatever the tensor holds.
__device__ __forceinline__ int offset8(const Cache8& C, int64_t b) {
  if (b == 0) return 0;
  return (int)min(max((int64_t)((cint32*)C.cu)[b], (int64_t)0), C.T);
}

// Sequence b, or (b == B) the rows past the last one's, as tokens before the
// start of an empty sequence.
__device__ __forceinline__ Seq8 seq8(const Cache8& C, int64_t b) {
  Seq8 s;
  s.b = (int)b;
  if (C.cu == nullptr) {
    s.c0 = (int)b;
    s.n = 1;
  } else {
    s.c0 = offset8(C, b);
    s.n = (b < C.B ? offset8(C, b + 1) : (int)C.T) - s.c0;
  }
  s.len = b < C.B ? min(max((int)((cint32*)C.lens)[b], 0), C.max_len) : 0;
  return s;
}

// Units of work without a count on the host: sequence b starts at a unit
// first(b) that grows with the rows before it by what a unit holds, and by as
// many more a sequence as its rows can touch beyond that.  The sequence of unit
// u is the last with first(b) <= u; first(0) is 0.
template <class First>
__device__ __forceinline__ int64_t seq_of_unit(int64_t B, int64_t u, First&& first) {
  int64_t lo = 0, hi = B;   // B: the rows past the last sequence
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (first(mid) <= u) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// The tokens of unit u that lie in one block of one sequence: rows [r0, r1) of
// the block that starts at position `start`, whose row r is token c + r of the
// call.  page < 0: no page holds them (also positions below 0).
struct Run8 {
  int64_t start, c;
  int r0, r1;
  int64_t page;
};

__device__ __forceinline__ Run8 run8(const Cache8& C, int64_t u) {
  int64_t b, j;
  if (C.cu == nullptr) {
    b = u;
    j = 0;
  } else {
    auto first = [&](int64_t s) { return ((int64_t)offset8(C, s) >> C.blk_log2) + 2 * s; };
    b = seq_of_unit(C.B, u, first);
    j = u - first(b);
  }
  const Seq8 s = seq8(C, b);
  const int64_t p0 = (int64_t)s.len - s.n, block = (int64_t)1 << C.blk_log2;
  Run8 r;
  r.start = ((p0 >> C.blk_log2) + j) << C.blk_log2;
  r.c = (int64_t)s.c0 + r.start - p0;
  r.r0 = (int)min(max(p0 - r.start, (int64_t)0), block);
  r.r1 = s.n > 0 ? (int)max(min((int64_t)s.len - r.start, block), (int64_t)0) : 0;
  r.page = -1;
  if (r.r1 > r.r0 && r.start >= 0) {   // then start < len <= max_len
    const int64_t id = ((cint32*)C.bt)[b * C.max_blocks + (r.start >> C.ps_log2)];
    if (id >= 0 && id < C.num_pages) r.page = id;
  }
  return r;
}

// Units of a call over all blocks of its tokens (and of the rows past them).
int64_t block_units(const Cache8& C) { return C.cu ? (C.T >> C.blk_log2) + 2 * (C.B + 1) : C.B; }

__device__ __forceinline__ int64_t scale_index(const Cache8& C, int64_t page, int head, int64_t tok) {
  const int nb_log2 = C.ps_log2 - C.blk_log2;
  return (((page * C.KVH + head) << nb_log2)) + ((tok & ((1 << C.ps_log2) - 1)) >> C.blk_log2);
}
__device__ __forceinline__ int64_t row_offset(const Cache8& C, int64_t page, int head, int64_t tok) {
  return page * C.page_bytes + head * C.head_bytes + (tok & ((1 << C.ps_log2) - 1)) * (int64_t)C.row_bytes;
}

// ---------------------------------------------------------------------------
// Codes
// ---------------------------------------------------------------------------

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight codes as eight fp16 or bf16 (every code is exact in both): e4m3 two an
// instruction; int8 as the fp16 1024 + (code + 128) put together from bytes,
// less 1152, or through fp32 for bf16, whose high half holds it.
template <int CODE, int E>
__device__ __forceinline__ u32x4 widen8(u32x2 c) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (CODE == kE4m3 && E == kEltF16) {
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, false));
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, true));
    } else if constexpr (CODE == kE4m3) {
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.f, false));
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], 1.f, true));
    } else if constexpr (E == kEltF16) {
      const uint32_t x = c[i] ^ 0x80808080u;
      const half2v off = {(_Float16)1152.f, (_Float16)1152.f};
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - off);
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - off);
    } else {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = (float)(int8_t)(c[i] >> (8 * j));
      r[2 * i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[1]), __builtin_bit_cast(uint32_t, f[0]), 0x07060302u);
      r[2 * i + 1] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[3]), __builtin_bit_cast(uint32_t, f[2]), 0x07060302u);
    }
  }
  return r;
}

// Four codes of a dword as floats.
template <int CODE>
__device__ __forceinline__ float4v code_values(uint32_t c) {
  if constexpr (CODE == kE4m3) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    return float4v{a[0], a[1], b[0], b[1]};
  } else {
    return float4v{(float)(int8_t)c, (float)(int8_t)(c >> 8), (float)(int8_t)(c >> 16), (float)(int8_t)(c >> 24)};
  }
}

__device__ __forceinline__ bool finite32(float x) { return __builtin_fabsf(x) <= 3.402823466e38f; }

// Four values in the codes' range, rounded to codes (ties to even).  e4m3:
// anything not finite becomes the NaN code.
template <int CODE>
__device__ __forceinline__ uint32_t to_codes(float4v x) {
  if constexpr (CODE == kE4m3) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], c, true);
    uint32_t r = (uint32_t)c;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!finite32(x[j])) r = (r & ~(0xffu << (8 * j))) | (0x7fu << (8 * j));
    return r;
  } else {
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) r |= ((uint32_t)(int)__builtin_rintf(x[j]) & 0xffu) << (8 * j);
    return r;
  }
}

// The high bit of every byte of c that is a NaN of e4m3.
__device__ __forceinline__ uint32_t nan_codes(uint32_t c) {
  return ((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// The least power of two s >= 2^kLowest with amax <= s * (448 or 127).
template <int CODE>
__device__ __forceinline__ float need_scale(float amax) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
  const int ex = (int)(bits >> 23);
  const uint32_t mant = bits & 0x7fffffu;
  // amax = (1 + mant / 2^23) 2^(ex - 127) against 448 = 1.75 * 2^8 and 127 = 1.984375 * 2^6
  const int e = CODE == kE4m3 ? ex - 135 + (mant > 0x600000u ? 1 : 0) : ex - 133 + (mant > 0x7e0000u ? 1 : 0);
  return __builtin_bit_cast(float, (uint32_t)(max(e, kLowest) + 127) << 23);
}

// ---------------------------------------------------------------------------
// Writing
// ---------------------------------------------------------------------------

struct Write8Args {
  Cache8 C;
  const void* x[2];                       // K, V
  int64_t tok_stride[2], head_stride[2];  // in elements
  int64_t tasks;                          // units * 2 * KVH
};

// Eight elements of a row as floats.
template <class T>
__device__ __forceinline__ void load_row8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4v a = *reinterpret_cast<const float4v*>(p), b = *reinterpret_cast<const float4v*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = a[j];
      x[4 + j] = b[j];
    }
  } else {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint16_t h = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
      if constexpr (std::is_same<T, _Float16>::value)
        x[j] = (float)__builtin_bit_cast(_Float16, h);
      else
        x[j] = __builtin_bit_cast(float, (uint32_t)h << 16);
    }
  }
}

constexpr int kWriteWaves = 4;

// One task quantizes the call's rows of one block of one KV head, of K or of
// V: at most 32 rows a wave (kept in registers between the search for the
// largest value and the rounding), 1 to 4 waves a task.
template <int CODE, class T, int BLOCK>
__global__ __launch_bounds__(64 * kWriteWaves) void write8_kernel(Write8Args A) {
  constexpr int kRows = BLOCK < 32 ? BLOCK : 32, kPer = BLOCK / kRows, kLoads = kRows / 4;
  const Cache8& C = A.C;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave % kPer;
  const int64_t task = (int64_t)blockIdx.x * (kWriteWaves / kPer) + wave / kPer;
  const int t = lane & 15, g = lane >> 4;

  Run8 run;
  run.page = -1;
  run.r0 = run.r1 = 0;
  int head = 0, kv = 0;
  if (task < A.tasks) {
    const int64_t rest = task / C.KVH;
    head = (int)(task - rest * C.KVH);
    kv = (int)(rest & 1);
    run = run8(C, rest >> 1);
  }
  const bool live = run.page >= 0;   // (uniform over a task's waves)
  const int base = part * kRows;

  float x[kLoads][8];
  float amax = 0.f;
  bool bad = false;
  float old = 0.f;
  float* scale = nullptr;
  char* codes = nullptr;
  if (live) {
    scale = (kv ? C.vs : C.ks) + scale_index(C, run.page, head, run.start);
    codes = (kv ? C.v : C.k) + row_offset(C, run.page, head, run.start);
    if (run.r0 > 0) old = *scale;
    const T* src = (const T*)A.x[kv] + run.c * A.tok_stride[kv] + head * A.head_stride[kv] + 8 * t;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = base + 4 * i + g;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = 0.f;
      if (r >= run.r0 && r < run.r1) load_row8(src + r * A.tok_stride[kv], x[i]);
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool ok = finite32(x[i][j]);
        bad = bad || !ok;
        amax = ok ? fmaxf(amax, __builtin_fabsf(x[i][j])) : amax;
      }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
    bad = __any(bad);
  }
  if constexpr (kPer > 1) {
    __shared__ float wave_max[kWriteWaves];
    __shared__ int wave_bad[kWriteWaves];
    if (lane == 0) {
      wave_max[wave] = amax;
      wave_bad[wave] = bad;
    }
    __syncthreads();   // also: every wave has read the old scale
#pragma unroll
    for (int w = 0; w < kPer; ++w) {
      amax = fmaxf(amax, wave_max[wave - part + w]);
      bad = bad || wave_bad[wave - part + w];
    }
  }
  if (!live) return;

  const bool kept = run.r0 > 0;   // the block has earlier tokens
  float s = need_scale<CODE>(amax);
  if (kept) s = fmaxf(old, s);
  bool poison = false;            // int8: a NaN or infinity in the block
  if (CODE == kInt8) {
    poison = bad || (kept && !(old == old));
    if (poison) s = __builtin_nanf("");
  }

  // earlier tokens, on a scale that grew
  if (kept && !poison && s != old) {
    const float ratio = old / s;
    const int row8 = lane >> 3, col = 16 * (lane & 7);
    for (int r = base + row8; r < min(run.r0, base + kRows); r += 8) {
      u32x4* p = reinterpret_cast<u32x4*>(codes + (int64_t)r * C.row_bytes + col);
      u32x4 c = *p;
#pragma unroll
      for (int d = 0; d < 4; ++d) c[d] = to_codes<CODE>(code_values<CODE>(c[d]) * ratio);
      *p = c;
    }
  }

  // A power of two divides by its inverse, exactly; a scale that some other
  // program put there may be any.
  const uint32_t sb = __builtin_bit_cast(uint32_t, s);
  const bool pow2 = (sb & 0x7fffffu) == 0 && sb < 0x7f000000u;
  const float inv = __builtin_bit_cast(float, 0x7f000000u - sb);
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = base + 4 * i + g;
    if (r < run.r0 || r >= run.r1) continue;
    u32x2 c;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      float4v y;
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = pow2 ? x[i][4 * d + j] * inv : x[i][4 * d + j] / s;
      c[d] = poison ? 0u : to_codes<CODE>(y);
    }
    *reinterpret_cast<u32x2*>(codes + (int64_t)r * C.row_bytes + 8 * t) = c;
  }
  if (part == 0 && lane == 0) *scale = s;
}

// ---------------------------------------------------------------------------
// Reading back
// ---------------------------------------------------------------------------

struct Read8Args {
  Cache8 C;
  void* out[2];
  int64_t tasks;
};

template <class T>
__device__ __forceinline__ void store_values4(T* p, float4v v) {
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4v*>(p) = v;
  else
    *reinterpret_cast<u32x2*>(p) = round_elt4<std::is_same<T, _Float16>::value ? kEltF16 : kEltBf16>(v);
}

// One wave reads the call's rows of one block of one KV head, of K or of V,
// eight rows an instruction.
template <int CODE, class T>
__global__ __launch_bounds__(64 * kWriteWaves) void read8_kernel(Read8Args A) {
  const Cache8& C = A.C;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t task = (int64_t)blockIdx.x * kWriteWaves + wave;
  if (task >= A.tasks) return;
  const int64_t rest = task / C.KVH;
  const int head = (int)(task - rest * C.KVH), kv = (int)(rest & 1);
  const Run8 run = run8(C, rest >> 1);
  const int row8 = lane >> 3, col = 16 * (lane & 7);
  float scale = 0.f;
  const char* codes = nullptr;
  if (run.page >= 0) {
    scale = (kv ? C.vs : C.ks)[scale_index(C, run.page, head, run.start)];
    codes = (kv ? C.v : C.k) + row_offset(C, run.page, head, run.start) + col;
  }
  T* out = (T*)A.out[kv] + (run.c * C.KVH + head) * kHeadDim + col;
  for (int r = run.r0 + row8; r < run.r1; r += 8) {
    u32x4 c = {0u, 0u, 0u, 0u};
    if (run.page >= 0) c = *reinterpret_cast<const u32x4*>(codes + (int64_t)r * C.row_bytes);
    T* p = out + (int64_t)r * C.KVH * kHeadDim;
#pragma unroll
    for (int d = 0; d < 4; ++d) store_values4(p + 4 * d, code_values<CODE>(c[d]) * scale);
  }
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
//
// The query rows of a sequence and KV head are its new tokens' heads of the
// group, token-major: row r is head r % G of new token r / G.  Sequences of at
// most kRowsA rows (single tokens, mostly) are read by the narrow kernel, whose
// work is the reading of the cache, those of more by the wide one, whose work
// is the products.
//
// Softmax over scaled codes.  With x = log2(e) sm_scale (q . k) per token, the
// scale of V's block enters as x + log2(vs): w = exp2(x + log2(vs) - m) is the
// token's weight times vs, so the product with the codes needs no scale, and
// the sum of the weights takes w / vs.  m is the running maximum of
// x + log2(vs), so that w stays in fp16's range whatever the scales.

constexpr int kRowsA = 16;
constexpr int kWavesA = 4;
constexpr int kThreadsA = 64 * kWavesA;
constexpr int kSlotA = 2 * kTile * kCodeRow;        // K and V codes of a tile
constexpr int kGroupsA = 1024;                      // workgroups of a launch, at most
static_assert(kRowsA * kHeadDim * 4 <= kSlotA, "a wave's partial rows fit its slot");

constexpr int kRowsB = 128;                         // query rows of a workgroup, 32 a wave
constexpr int kThreadsB = 256;
constexpr int kTileB = 64;                          // tokens of its tiles
constexpr int kPairsB = 512;                        // workgroups that fill the GPU

struct Attn8Args {
  Cache8 C;
  const void* q;
  void* o;
  float* part;                // partial rows, then their maxima and sums
  int64_t q_tok, q_head;      // in elements
  int64_t units;
  int32_t G, H, window, sink;
  int32_t groups;             // narrow: workgroups
  int32_t splits;             // wide: workgroups a pair
  float scale_log2;
};

// A unit: query rows [row0, row0 + rows) of a sequence's n * G, at positions
// pos0 .. pos1, and its tiles: [0, ts) of the sink and [tw, te).
struct Unit8 {
  Seq8 s;
  int row0, rows, pos0, pos1;
  int ts, tw, te;
  __device__ __forceinline__ int tiles() const { return ts + te - tw; }
  __device__ __forceinline__ int tile(int j) const { return j < ts ? j : tw + j - ts; }
};

template <int TILE>
__device__ __forceinline__ void unit_tiles(const Attn8Args& A, Unit8& U) {
  U.ts = U.tw = U.te = 0;
  U.pos0 = U.pos1 = -1;
  if (U.rows <= 0) {
    U.rows = 0;
    return;
  }
  U.pos0 = U.s.len - U.s.n + U.row0 / A.G;
  U.pos1 = U.s.len - U.s.n + (U.row0 + U.rows - 1) / A.G;
  if (U.pos1 < 0) return;
  U.te = U.pos1 / TILE + 1;
  if (A.window > 0) {
    U.ts = min((int)(((int64_t)A.sink + TILE - 1) / TILE), U.te);
    U.tw = min(max(U.ts, max(U.pos0 - A.window + 1, 0) / TILE), U.te);
  }
}

// The narrow kernel's unit: a sequence, if its rows fit.
__device__ __forceinline__ Unit8 unit_a(const Attn8Args& A, int64_t b) {
  Unit8 U;
  U.s = seq8(A.C, b);
  const int64_t rows = (int64_t)U.s.n * A.G;
  U.row0 = 0;
  U.rows = rows <= kRowsA ? (int)rows : 0;
  unit_tiles<kTile>(A, U);
  return U;
}

// The wide kernel's unit u: kRowsB rows of a sequence of more than kRowsA, or of
// the rows past the last sequence (which attend to nothing).
__device__ __forceinline__ Unit8 unit_b(const Attn8Args& A, int64_t u) {
  const Cache8& C = A.C;
  Unit8 U;
  int64_t b, first;
  if (C.cu == nullptr) {
    const int per = (A.G + kRowsB - 1) / kRowsB;
    b = u / per;
    first = b * per;
  } else {
    auto start = [&](int64_t s) { return (int64_t)offset8(C, s) * A.G / kRowsB + s; };
    b = seq_of_unit(C.B, u, start);
    first = start(b);
  }
  U.s = seq8(C, b);
  const int64_t rows = (int64_t)U.s.n * A.G, row0 = (u - first) * kRowsB;
  U.row0 = (int)min(row0, rows);
  U.rows = rows > kRowsA || b == C.B ? (int)min(rows - U.row0, (int64_t)kRowsB) : 0;
  unit_tiles<kTileB>(A, U);
  return U;
}

// Where a token of a tile stands against a row's position.
__device__ __forceinline__ bool sees(int p, int pos, int window, int sink) {
  return p <= pos && (window <= 0 || p < sink || p > pos - window);
}

// Every token of [tok, tok + n) is seen by every row of the unit.
__device__ __forceinline__ bool all_seen(const Attn8Args& A, const Unit8& U, int tok, int n) {
  return tok + n - 1 <= U.pos0 && (A.window <= 0 || tok + n <= A.sink || tok > U.pos1 - A.window);
}

// What a token of the pair's rows weighs by: kf turns q . k into x, lv is
// log2 of V's scale and inv its inverse.  No page: keys and values of zero.
struct Meta8 {
  int page;
  float kf, lv, inv;
};

__device__ __forceinline__ Meta8 meta8(const Attn8Args& A, int b, int head, int tok, bool live) {
  const Cache8& C = A.C;
  Meta8 m = {-1, 0.f, 0.f, 1.f};
  if (live) {
    const int id = C.bt[(int64_t)b * C.max_blocks + (tok >> C.ps_log2)];
    if (id >= 0 && id < C.num_pages) {
      m.page = id;
      const int64_t at = scale_index(C, id, head, tok);
      m.kf = C.ks[at] * A.scale_log2;
      const float vs = C.vs[at];
      // a scale that is hardly one counts as the writer's least
      const float s = vs < 0x1p-100f ? 0x1p-100f : vs;
      m.lv = __builtin_amdgcn_logf(s);
      m.inv = s == s ? 1.f / s : 1.f;   // a NaN arrives through lv, where masks hold
    }
  }
  return m;
}

// Place of row `row` of a pair in the output.
__device__ __forceinline__ int64_t out_row(const Attn8Args& A, const Unit8& U, int head, int row) {
  const int r = U.row0 + row, tok = r / A.G;
  return ((int64_t)(U.s.c0 + tok) * A.H + head * A.G + (r - tok * A.G)) * kHeadDim;
}

template <int E>
__device__ __forceinline__ void store_out(const Attn8Args& A, int64_t at, float4v acc, float l) {
  const float d = l == 0.f ? 1.f : l;
  *reinterpret_cast<u32x2*>((uint16_t*)A.o + at) = round_elt4<E>(float4v{acc[0] / d, acc[1] / d, acc[2] / d, acc[3] / d});
}

// ---- the narrow kernel ----
//
// The tiles (32 tokens) of all pairs of a sequence and a KV head, in order, are
// dealt to the launch's workgroups in equal runs, whatever the sequences'
// lengths: each finds its run from the lengths on the device.  A pair that
// falls to several workgroups leaves partial rows in the workspace, which a
// second kernel joins.

__device__ __forceinline__ uint32_t wave_total(uint32_t x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off);
  return __builtin_amdgcn_readfirstlane(x);
}

// Tiles of all sequences, and of those before sequence u (one KV head's).
struct Counts8 {
  int64_t all, before;
};
__device__ __forceinline__ Counts8 count8(const Attn8Args& A, int64_t u, int lane) {
  Counts8 c = {0, 0};
  for (int64_t u0 = 0; u0 < A.C.B; u0 += 64) {
    const int64_t v = u0 + lane;
    const uint32_t n = v < A.C.B ? (uint32_t)unit_a(A, v).tiles() : 0u;
    c.all += wave_total(n);
    if (u0 < u) c.before += wave_total(v < u ? n : 0u);
  }
  return c;
}

__device__ __forceinline__ int64_t group_share(const Attn8Args& A, int64_t all) {
  return max((all * A.C.KVH + A.groups - 1) / A.groups, (int64_t)kWavesA);
}

// A wave's running softmax: lane (n, g) has row n; O[cb][r] is channel
// 16 cb + 4 g + r; l is the lane's share of the sum.
struct State8 {
  float4v O[8];
  float m, l;
};

struct Raw8 {
  u32x4 k[4], v[4];
};

template <int CODE, int E>
__global__ __launch_bounds__(kThreadsA, 2) void attn8_kernel(Attn8Args A) {
  __shared__ __align__(16) char lds[kWavesA * kSlotA];
  __shared__ float lds_m[kWavesA][kRowsA], lds_l[kWavesA][kRowsA];
  const Cache8& C = A.C;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = lane & 15, g = lane >> 4;
  char* slot = lds + wave * kSlotA;

  const int64_t all = count8(A, 0, lane).all;
  const int64_t share = group_share(A, all);
  int64_t cur = (int64_t)blockIdx.x * share;
  const int64_t end = min(cur + share, all * C.KVH);
  if (cur >= end) return;

  // the sequence of tile `cur`
  int64_t u = 0, base = 0;   // base: tiles of all heads before unit u
  for (int64_t u0 = 0; u0 < C.B; u0 += 64) {
    const int64_t v = u0 + lane;
    const uint32_t n = v < C.B ? (uint32_t)unit_a(A, v).tiles() : 0u;
    uint32_t upto = n;       // inclusive prefix
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t y = __shfl_up(upto, off);
      if (lane >= off) upto += y;
    }
    const uint64_t past = __ballot(base + (int64_t)upto * C.KVH > cur);
    if (past) {
      const int first = __builtin_ctzll(past);
      u = u0 + first;
      base += (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(upto - n), first) * C.KVH;
      break;
    }
    base += (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)upto, 63) * C.KVH;
  }

  while (cur < end) {
    const Unit8 U = unit_a(A, u);
    const int nt = U.tiles();
    if (nt == 0) {
      ++u;
      continue;
    }
    const int head = (int)((cur - base) / nt);
    if (head >= C.KVH) {   // the unit's pairs are done
      base += (int64_t)nt * C.KVH;
      ++u;
      continue;
    }
    const int j0 = (int)((cur - base) - (int64_t)head * nt);
    const int j1 = (int)min((int64_t)nt, j0 + (end - cur));
    cur += j1 - j0;

    // this lane's query row
    const int my_row = U.row0 + t;
    const int my_tok = my_row / A.G, my_head = my_row - my_tok * A.G;
    const int pos = t < U.rows ? U.s.len - U.s.n + my_tok : -1;
    half8 qB[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u32x4 w = {0u, 0u, 0u, 0u};
      if (t < U.rows)
        w = *reinterpret_cast<const u32x4*>((const uint16_t*)A.q + (int64_t)(U.s.c0 + my_tok) * A.q_tok +
                                            (int64_t)(head * A.G + my_head) * A.q_head + 64 * (c >> 1) + 16 * g +
                                            8 * (c & 1));
      qB[c] = as_h8(w);
    }

    State8 st;
#pragma unroll
    for (int i = 0; i < 8; ++i) st.O[i] = float4v{0.f, 0.f, 0.f, 0.f};
    st.m = kMaxSentinel;
    st.l = 0.f;

    const int hi = U.pos1 + 1, lo = A.window > 0 ? max(U.pos0 - A.window + 1, 0) : 0;
    const int sink = A.window > 0 ? A.sink : 0;
    const char* kbase = C.k + head * C.head_bytes;
    const char* vbase = C.v + head * C.head_bytes;
    const int own = (j1 - j0 - wave + kWavesA - 1) / kWavesA;   // this wave's tiles: j0 + wave, + kWavesA, ...
    const uint32_t off0 = (uint32_t)(lane >> 3) * C.row_bytes + 16u * (lane & 7);

    for (int i0 = 0; i0 < own; i0 += 32) {
      const int n = min(own - i0, 32);
      // lane 2i + h: half h of the wave's tile i: its page, scales
      const int mi = lane >> 1;
      const int mtok = kTile * U.tile(j0 + wave + kWavesA * (i0 + min(mi, n - 1))) + 16 * (lane & 1);
      const Meta8 meta = meta8(A, U.s.b, head, mtok, mi < n && mtok < hi);
      auto lane_f = [](float x, int l) {
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
      };
      auto tok_of = [&](int i) { return kTile * U.tile(j0 + wave + kWavesA * (i0 + i)); };
      auto load = [&](int i, Raw8& X) {
        const bool live = i < n;
        const int tok = tok_of(live ? i : 0);
        const bool full = all_seen(A, U, tok, kTile);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int id = live ? __builtin_amdgcn_readlane(meta.page, 2 * i + h) : -1;
          const uint32_t bytes = id >= 0 ? 15u * C.row_bytes + kCodeRow : 0u;
          const int64_t off = id >= 0 ? row_offset(C, id, 0, tok + 16 * h) : 0;
          const rsrc_t rk = make_rsrc(kbase + off, bytes), rv = make_rsrc(vbase + off, bytes);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t o = off0 + 8u * r * C.row_bytes;
            if (!full) {   // rows that no query row sees read as zeros
              const int p = tok + 16 * h + 8 * r + (lane >> 3);
              if (!(p < hi && (p >= lo || p < sink))) o = kOOB;
            }
            X.k[2 * h + r] = bload16(rk, o);
            X.v[2 * h + r] = bload16(rv, o);
          }
        }
      };
      auto step = [&](int i, Raw8& X) {
        const int tok = tok_of(i);
        const bool full = all_seen(A, U, tok, kTile);
        // staged: K rows' 16-byte chunks turned by the row, V's by its place
        // among the eight rows that a transposed read takes
        const int r8 = lane >> 3, ch = lane & 7;
        bool nans = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 8 * k + r8;
          *reinterpret_cast<u32x4*>(slot + r * kCodeRow + ((ch ^ r8) << 4)) = X.k[k];
          *reinterpret_cast<u32x4*>(slot + kTile * kCodeRow + r * kCodeRow + ((ch ^ ((r8 & 3) | ((k >> 1) << 2))) << 4)) = X.v[k];
        }
        if (CODE == kE4m3 && !full) {
          uint32_t any = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int d = 0; d < 4; ++d) any |= nan_codes(X.v[k][d]);
          nans = __any(any != 0);
        }
        load(i + 2, X);

        float4v s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
          const u32x4 a = *reinterpret_cast<const u32x4*>(slot + t * kCodeRow + (((g + 4 * h2) ^ (t & 7)) << 4));
          const u32x4 b = *reinterpret_cast<const u32x4*>(slot + (16 + t) * kCodeRow + (((g + 4 * h2) ^ (t & 7)) << 4));
          s0 = mfma16x16x32<E>(widen8<CODE, E>(u32x2{a[0], a[1]}), qB[2 * h2], s0);
          s0 = mfma16x16x32<E>(widen8<CODE, E>(u32x2{a[2], a[3]}), qB[2 * h2 + 1], s0);
          s1 = mfma16x16x32<E>(widen8<CODE, E>(u32x2{b[0], b[1]}), qB[2 * h2], s1);
          s1 = mfma16x16x32<E>(widen8<CODE, E>(u32x2{b[2], b[3]}), qB[2 * h2 + 1], s1);
        }
        const float kf0 = lane_f(meta.kf, 2 * i), kf1 = lane_f(meta.kf, 2 * i + 1);
        const float lv0 = lane_f(meta.lv, 2 * i), lv1 = lane_f(meta.lv, 2 * i + 1);
        const float inv0 = lane_f(meta.inv, 2 * i), inv1 = lane_f(meta.inv, 2 * i + 1);
        float x[8];
        uint32_t seen = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = __builtin_fmaf(j < 4 ? s0[j & 3] : s1[j & 3], j < 4 ? kf0 : kf1, j < 4 ? lv0 : lv1);
          if (!full) {
            const bool ok = sees(tok + tau(g, j), pos, A.window, sink);
            seen |= (uint32_t)ok << j;
            x[j] = ok ? x[j] : -INFINITY;
          }
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
        if (__any(top > st.m + kRescaleSlack)) {
          const float m = fmaxf(st.m, group_max(top));
          const float f = __builtin_amdgcn_exp2f(st.m - m);
          st.l *= f;
#pragma unroll
          for (int cb = 0; cb < 8; ++cb) st.O[cb] = st.O[cb] * f;
          st.m = m;
        }
        // weights as an fp16 and the fp16 of its remainder: good to 2^-22
        half8 pB, pL;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = __builtin_amdgcn_exp2f(x[j] - st.m);
          st.l = __builtin_fmaf(w, j < 4 ? inv0 : inv1, st.l);
          pB[j] = (_Float16)w;
          pL[j] = (_Float16)(w - (float)pB[j]);
        }
        const char* vt = slot + kTile * kCodeRow + tau(g, t >> 1) * kCodeRow + 8 * (t & 1);
#pragma unroll
        for (int cb = 0; cb < 8; ++cb) {
          u32x2 c = lds_read_tr8(vt + ((cb ^ (t >> 1)) << 4));
          if (CODE == kE4m3 && nans) {
            // a NaN reaches the rows that see its token: marked as ones, and
            // multiplied with what each row sees; the others count it as 0
            u32x4 marks;
            half8 eyes;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              const uint32_t bad = nan_codes(c[d]) >> 7;   // 0 or 1 a byte
              c[d] &= ~(bad * 0xffu);
              marks[2 * d] = (bad & 1u) * 0x3c00u | ((bad >> 8) & 1u) * 0x3c000000u;
              marks[2 * d + 1] = ((bad >> 16) & 1u) * 0x3c00u | ((bad >> 24) & 1u) * 0x3c000000u;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) eyes[j] = (seen >> j) & 1u ? (_Float16)1.f : (_Float16)0.f;
            const float4v hit = mfma16x16x32<kEltF16>(marks, eyes, float4v{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int r = 0; r < 4; ++r) st.O[cb][r] = hit[r] > 0.f ? __builtin_nanf("") : st.O[cb][r];
          }
          const u32x4 a = widen8<CODE, kEltF16>(c);
          st.O[cb] = mfma16x16x32<kEltF16>(a, pB, st.O[cb]);
          st.O[cb] = mfma16x16x32<kEltF16>(a, pL, st.O[cb]);
        }
      };
      Raw8 X0, X1;
      load(0, X0);
      load(1, X1);
      for (int i = 0; i < n; i += 2) {
        step(i, X0);
        if (i + 1 < n) step(i + 1, X1);
      }
    }

    // join the waves: each parks its rows in its slot
    const float l = group_sum(st.l);
    if (g == 0) {
      lds_m[wave][t] = st.m;
      lds_l[wave][t] = l;
    }
#pragma unroll
    for (int cb = 0; cb < 8; ++cb)
      *reinterpret_cast<float4v*>(slot + t * (kHeadDim * 4) + (((4 * cb + g) ^ t) << 4)) = st.O[cb];
    __syncthreads();
    {
      const int row = threadIdx.x >> 4;   // kThreadsA / 16 == kRowsA
      float M = lds_m[0][row], f[kWavesA], L = 0.f;
#pragma unroll
      for (int w = 1; w < kWavesA; ++w) M = fmaxf(M, lds_m[w][row]);
#pragma unroll
      for (int w = 0; w < kWavesA; ++w) {
        f[w] = __builtin_amdgcn_exp2f(lds_m[w][row] - M);
        L = __builtin_fmaf(lds_l[w][row], f[w], L);
      }
      const bool whole = j1 - j0 == nt;
      const int64_t place = 2 * (int64_t)blockIdx.x + (j0 == 0 ? 1 : 0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int chunk = (threadIdx.x & 15) + 16 * h;
        float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWavesA; ++w)
          acc += *reinterpret_cast<const float4v*>(lds + w * kSlotA + row * (kHeadDim * 4) + ((chunk ^ row) << 4)) * f[w];
        if (row < U.rows) {
          if (whole) {
            store_out<E>(A, out_row(A, U, head, row) + 4 * chunk, acc, L);
          } else {
            *reinterpret_cast<float4v*>(A.part + (place * kRowsA + row) * kHeadDim + 4 * chunk) = acc;
          }
        }
      }
      if (!whole && row < U.rows && (threadIdx.x & 15) == 0) {
        float* ml = A.part + (int64_t)2 * A.groups * kRowsA * kHeadDim;
        ml[place * kRowsA + row] = M;
        ml[(int64_t)2 * A.groups * kRowsA + place * kRowsA + row] = L;
      }
    }
    __syncthreads();   // the slots are free again
  }
}

// One workgroup a pair's row: the rows that several workgroups share, and
// zeros for those that attend to nothing.
template <int E>
__global__ __launch_bounds__(256) void join8_kernel(Attn8Args A) {
  const Cache8& C = A.C;
  const int lane = threadIdx.x & 63;
  const int64_t id = blockIdx.x;
  const int row = (int)(id % kRowsA);
  const int64_t pair = id / kRowsA, u = pair / C.KVH;
  const int head = (int)(pair - u * C.KVH);
  const Unit8 U = unit_a(A, u);
  if (row >= U.rows) return;
  const int64_t out = out_row(A, U, head, row);
  const int nt = U.tiles();
  if (nt == 0) {
    if (threadIdx.x < 32) store_out<E>(A, out + 4 * threadIdx.x, float4v{0.f, 0.f, 0.f, 0.f}, 0.f);
    return;
  }
  const Counts8 c = count8(A, u, lane);
  const int64_t share = group_share(A, c.all);
  const int64_t begin = c.before * C.KVH + (int64_t)head * nt;
  const int64_t w0 = begin / share, w1 = (begin + nt - 1) / share;
  if (w0 == w1) return;   // written whole
  const float* pm = A.part + (int64_t)2 * A.groups * kRowsA * kHeadDim;
  const float* pl = pm + (int64_t)2 * A.groups * kRowsA;
  auto place = [&](int64_t w) { return (2 * w + (w == w0 ? 1 : 0)) * kRowsA + row; };
  float M = kMaxSentinel;
  for (int64_t w = w0; w <= w1; ++w) M = fmaxf(M, pm[place(w)]);
  const int grp = threadIdx.x >> 5, chunk = threadIdx.x & 31;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  float L = 0.f;
  for (int64_t w = w0 + grp; w <= w1; w += 8) {
    const int64_t p = place(w);
    const float f = __builtin_amdgcn_exp2f(pm[p] - M);
    L = __builtin_fmaf(pl[p], f, L);
    acc += *reinterpret_cast<const float4v*>(A.part + p * kHeadDim + 4 * chunk) * f;
  }
  __shared__ float4v parts[8][32];
  __shared__ float sums[8];
  parts[grp][chunk] = acc;
  if (chunk == 0) sums[grp] = L;
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) {
    acc += parts[w][chunk];
    L += sums[w];
  }
  store_out<E>(A, out + 4 * chunk, acc, L);
}

// ---- the wide kernel ----
//
// One workgroup a pair (unit, KV head) and split: four waves of 32 query rows
// each share a tile of 64 tokens, widened to fp16 (K: the query's type) in LDS
// once for all, two tiles in turn.  K's rows are staged with their 16-byte
// chunks turned by the row, V's with their 64-byte quarters turned by it, so
// that neither the operand reads nor V's transposed ones collide in a bank.
// The products are v_mfma_f32_32x32x16: S = K Q^T leaves lane (n, hf) row n's
// tokens 8 (r / 4) + 4 hf + r % 4, which is the order that the transposed
// reads give V^T's operand in.
// Weights are rounded to fp16 once here (2^-11 of each, as the output itself
// in fp16): a second product for the remainder would cost half as much again
// of the kernel's bound.

typedef float float16v __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));

template <int E>
__device__ __forceinline__ float16v mfma32x32x16(u32x4 a, u32x4 b, float16v c) {
  if constexpr (E == kEltBf16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(a), as_h8(b), c, 0, 0, 0);
}

// Transposed LDS read (ds_read_b64_tr_b16): in each group of 16 lanes, lane
// 4j + h supplies row j's columns 4h .. 4h + 3 and lane i receives column i.
__device__ __forceinline__ u32x2 lds_read_tr16(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(p)));
}

// The two halves' values of a row (lanes n and n + 32) joined.
__device__ __forceinline__ float half_max(float x) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x);
  const auto s = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)s[0]), __builtin_bit_cast(float, (uint32_t)s[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x);
  const auto s = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
}

constexpr int kRowB = 2 * kHeadDim;                 // bytes of a widened row
constexpr int kTileBytesB = kTileB * kRowB;         // of K or of V
constexpr int kChunkB = 64;                         // tiles whose Meta8 are held at once
constexpr int kSegs = kTileB / 16;                  // 16-token segments of a tile
static_assert(kChunkB * kSegs == kThreadsB, "a thread a segment");

// The tiles of split s of a pair.
__device__ __forceinline__ void split_tiles(const Attn8Args& A, int nt, int s, int& j0, int& j1) {
  const int per = max((nt + A.splits - 1) / A.splits, 4);
  j0 = min(s * per, nt);
  j1 = min(j0 + per, nt);
}

template <int CODE, int E>
__global__ __launch_bounds__(kThreadsB, 2) void wide8_kernel(Attn8Args A) {
  __shared__ __align__(16) char ks[2][kTileBytesB], vs[2][kTileBytesB];
  __shared__ Meta8 metas[kThreadsB];
  // e4m3, tiles that not every row sees whole: whether V tile i & 3 has a NaN,
  // and which channels of each token
  __shared__ int nan_seen[4];
  __shared__ __align__(16) uint8_t nan_map[2][kTileB][kHeadDim / 8];
  const Cache8& C = A.C;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, hf = lane >> 5;
  // KV heads fastest (they go to different XCDs' caches), then splits; the last
  // rows of a sequence, which have the most tiles, first
  uint32_t id = blockIdx.x;
  const int head = (int)(id % (uint32_t)C.KVH);
  id /= (uint32_t)C.KVH;
  const int split = (int)(id % (uint32_t)A.splits);
  const int64_t u = A.units - 1 - (int64_t)(id / (uint32_t)A.splits);
  const Unit8 U = unit_b(A, u);
  if (U.rows == 0) return;
  const int nt = U.tiles();
  int j0, j1;
  split_tiles(A, nt, split, j0, j1);
  const bool whole = j1 - j0 == nt;
  if (j0 == j1 && !(whole && split == 0)) return;

  const int my_row = 32 * wave + n;
  const int my_tok = (U.row0 + my_row) / A.G, my_head = U.row0 + my_row - my_tok * A.G;
  const bool mine = my_row < U.rows;
  const int pos = mine ? U.s.len - U.s.n + my_tok : -1;
  const bool busy = 32 * wave < U.rows;   // the wave has rows
  u32x4 qB[8];
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    qB[s] = u32x4{0u, 0u, 0u, 0u};
    if (mine)
      qB[s] = *reinterpret_cast<const u32x4*>((const uint16_t*)A.q + (int64_t)(U.s.c0 + my_tok) * A.q_tok +
                                              (int64_t)(head * A.G + my_head) * A.q_head + 16 * s + 8 * hf);
  }
  float16v O[4];
#pragma unroll
  for (int cb = 0; cb < 4; ++cb)
#pragma unroll
    for (int r = 0; r < 16; ++r) O[cb][r] = 0.f;
  float m = -INFINITY, l = 0.f;   // no token seen yet; the lane's share of the sum

  const int hi = U.pos1 + 1, lo = A.window > 0 ? max(U.pos0 - A.window + 1, 0) : 0;
  const int sink = A.window > 0 ? A.sink : 0;
  const char* kbase = C.k + head * C.head_bytes;
  const char* vbase = C.v + head * C.head_bytes;
  const int r4 = lane >> 4, ch = lane & 15;   // staging: row 16 i + 4 wave + r4, 8 codes from 8 ch

  for (int i0 = j0; i0 < j1; i0 += kChunkB) {
    const int cnt = min(j1 - i0, kChunkB);
    __syncthreads();
    {
      const int i = threadIdx.x / kSegs;
      const int tok = kTileB * U.tile(i0 + min(i, cnt - 1)) + 16 * (threadIdx.x % kSegs);
      metas[threadIdx.x] = meta8(A, U.s.b, head, tok, i < cnt && tok < hi);
      if (threadIdx.x < 4) nan_seen[threadIdx.x] = 0;
    }
    __syncthreads();

    u32x2 kc[kSegs], vc[kSegs];   // codes on their way: of the tile after the next
    auto load = [&](int i) {
      const bool live = i < cnt;
      const int tok = kTileB * U.tile(i0 + (live ? i : 0));
      const bool full = all_seen(A, U, tok, kTileB);
#pragma unroll
      for (int g = 0; g < kSegs; ++g) {
        const int page = live ? __builtin_amdgcn_readfirstlane(metas[kSegs * i + g].page) : -1;
        const uint32_t bytes = page >= 0 ? 15u * C.row_bytes + kCodeRow : 0u;
        const int64_t off = page >= 0 ? row_offset(C, page, 0, tok + 16 * g) : 0;
        uint32_t o = (uint32_t)(4 * wave + r4) * C.row_bytes + 8u * ch;
        if (!full) {   // rows that no query row sees read as zeros
          const int p = tok + 16 * g + 4 * wave + r4;
          if (!(p < hi && (p >= lo || p < sink))) o = kOOB;
        }
        typedef int v2i __attribute__((ext_vector_type(2)));
        kc[g] = __builtin_bit_cast(u32x2, (v2i)__builtin_amdgcn_raw_buffer_load_b64(make_rsrc(kbase + off, bytes), o, 0, 0));
        vc[g] = __builtin_bit_cast(u32x2, (v2i)__builtin_amdgcn_raw_buffer_load_b64(make_rsrc(vbase + off, bytes), o, 0, 0));
      }
    };
    auto stage = [&](int i) {
      const int buf = i & 1;
      // a NaN of V must not meet the weight 0 of a row that does not see it: it
      // is staged as 0 and noted
      if (CODE == kE4m3 && i < cnt && !all_seen(A, U, kTileB * U.tile(i0 + i), kTileB)) {
        uint32_t any = 0;
#pragma unroll
        for (int g = 0; g < kSegs; ++g) {
          uint32_t bits = 0;
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            const uint32_t bad = nan_codes(vc[g][d]) >> 7;   // 0 or 1 a byte
            vc[g][d] &= ~(bad * 0xffu);
            bits |= ((bad * 0x01020408u) >> 24) << (4 * d);
          }
          nan_map[buf][16 * g + 4 * wave + r4][ch] = (uint8_t)bits;
          any |= bits;
        }
        if (__any(any != 0)) nan_seen[i & 3] = 1;
      }
#pragma unroll
      for (int g = 0; g < kSegs; ++g) {
        const int r = 16 * g + 4 * wave + r4;
        *reinterpret_cast<u32x4*>(ks[buf] + r * kRowB + ((ch ^ (r & 15)) << 4)) = widen8<CODE, E>(kc[g]);
        *reinterpret_cast<u32x4*>(vs[buf] + r * kRowB + ((ch ^ ((r & 3) << 2)) << 4)) = widen8<CODE, kEltF16>(vc[g]);
      }
    };

    load(0);
    stage(0);
    load(1);
    __syncthreads();
    for (int i = 0; i < cnt; ++i) {
      const int tok = kTileB * U.tile(i0 + i);
      const bool full = all_seen(A, U, tok, kTileB);
      const bool nans = CODE == kE4m3 && !full && nan_seen[i & 3];
      if (CODE == kE4m3 && threadIdx.x == 0) nan_seen[(i + 2) & 3] = 0;
      stage(i + 1);   // (past the last tile: zeros)
      load(i + 2);
      if (busy) {
        float16v S[2];
        const char* kt = ks[i & 1];
        const char* vt = vs[i & 1];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
          for (int r = 0; r < 16; ++r) S[b][r] = 0.f;
#pragma unroll
          for (int s = 0; s < 8; ++s)
            S[b] = mfma32x32x16<E>(*reinterpret_cast<const u32x4*>(kt + (32 * b + n) * kRowB + (((2 * s + hf) ^ (n & 15)) << 4)),
                                   qB[s], S[b]);
        }
        // logits against the running maximum (0 while there is none)
        const float ref = m == -INFINITY ? 0.f : m;
        float inv[kSegs], top = -INFINITY;
#pragma unroll
        for (int g = 0; g < kSegs; ++g) {
          const Meta8 mt = metas[kSegs * i + g];
          inv[g] = mt.inv;
          const float add = mt.lv - ref;
#pragma unroll
          for (int r = 8 * (g & 1); r < 8 * (g & 1) + 8; ++r) {
            float x = __builtin_fmaf(S[g >> 1][r], mt.kf, add);
            if (!full) {
              x = sees(tok + 32 * (g >> 1) + 8 * (r >> 2) + 4 * hf + (r & 3), pos, A.window, A.sink) ? x : -INFINITY;
            }
            top = fmaxf(top, x);
            S[g >> 1][r] = x;
          }
        }
        if (__any(top > (m == -INFINITY ? -INFINITY : kRescaleSlack))) {
          const float t = half_max(top);
          const float now = m == -INFINITY ? t : fmaxf(m, m + t);
          const float to = now == -INFINITY ? 0.f : now;
          const float f = __builtin_amdgcn_exp2f(m - to);   // 0 while there was none
          const float d = ref - to;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) S[b][r] += d;
          l *= f;
#pragma unroll
          for (int cb = 0; cb < 4; ++cb)
#pragma unroll
            for (int r = 0; r < 16; ++r) O[cb][r] *= f;
          m = now;
        }
        u32x4 P[kSegs];
#pragma unroll
        for (int g = 0; g < kSegs; ++g) {
          half8 h;
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const float w = __builtin_amdgcn_exp2f(S[g >> 1][8 * (g & 1) + r]);
            sum += w;
            h[r] = (_Float16)w;
          }
          l = __builtin_fmaf(sum, inv[g], l);
          P[g] = as_u4(h);
        }
        // lane (group of 16 lanes, 4j + h): row 4 hf + j, channel 16 (group & 1) + 4 h
        const int j = (lane >> 2) & 3;
        const char* vl = vt + (4 * hf + j) * kRowB + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
        auto values = [&](int g, int cb) {
          const u32x2 a = lds_read_tr16(vl + 16 * g * kRowB + ((cb ^ j) << 6));
          const u32x2 b = lds_read_tr16(vl + (16 * g + 8) * kRowB + ((cb ^ j) << 6));
          return u32x4{a[0], a[1], b[0], b[1]};
        };
#pragma unroll
        for (int cb = 0; cb < 4; ++cb)
#pragma unroll
          for (int g = 0; g < kSegs; ++g) O[cb] = mfma32x32x16<kEltF16>(values(g, cb), P[g], O[cb]);
        if (nans) {   // and reaches the rows that do
          u32x4 hit = {0u, 0u, 0u, 0u};   // this row's channels
          for (int p = 0; p < kTileB; ++p)
            if (sees(tok + p, pos, A.window, A.sink)) hit |= *reinterpret_cast<const u32x4*>(nan_map[i & 1][p]);
#pragma unroll
          for (int cb = 0; cb < 4; ++cb) {
            const uint32_t w = hit[cb] >> (4 * hf);
#pragma unroll
            for (int r = 0; r < 16; ++r)
              O[cb][r] = w >> (8 * (r >> 2) + (r & 3)) & 1u ? __builtin_nanf("") : O[cb][r];
          }
        }
      }
      __syncthreads();
    }
  }

  if (!mine) return;
  l = half_sum(l);
  const int64_t at = whole ? out_row(A, U, head, my_row) : (((u * C.KVH + head) * A.splits + split) * kRowsB + my_row) * kHeadDim;
#pragma unroll
  for (int cb = 0; cb < 4; ++cb)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int64_t c = at + 32 * cb + 2 * r + 4 * hf;
      const float4v v = {O[cb][r], O[cb][r + 1], O[cb][r + 2], O[cb][r + 3]};
      if (whole)
        store_out<E>(A, c, v, l);
      else
        *reinterpret_cast<float4v*>(A.part + c) = v;
    }
  if (!whole && hf == 0) {
    float* ml = A.part + A.units * C.KVH * A.splits * kRowsB * kHeadDim;
    ml[at / kHeadDim] = m;
    ml[A.units * C.KVH * A.splits * kRowsB + at / kHeadDim] = l;
  }
}

// Joins the splits of the wide kernel's rows, 32 threads a row.
template <int E>
__global__ __launch_bounds__(256) void wide_join8_kernel(Attn8Args A) {
  const Cache8& C = A.C;
  const int64_t pair = blockIdx.x / (kRowsB / 8);
  const int row = 8 * (int)(blockIdx.x % (kRowsB / 8)) + (threadIdx.x >> 5), chunk = threadIdx.x & 31;
  const int64_t u = pair / C.KVH;
  const int head = (int)(pair - u * C.KVH);
  const Unit8 U = unit_b(A, u);
  const int nt = U.tiles();
  int j0, j1;
  split_tiles(A, nt, 0, j0, j1);
  if (row >= U.rows || j1 == nt) return;
  const int64_t rows = A.units * C.KVH * A.splits * kRowsB;
  const float* pm = A.part + rows * kHeadDim;
  const float* pl = pm + rows;
  const int64_t first = pair * A.splits * kRowsB + row;
  const int splits = (nt + j1 - 1) / j1;
  float M = -INFINITY;
  for (int s = 0; s < splits; ++s) M = fmaxf(M, pm[first + s * kRowsB]);
  const float ref = M == -INFINITY ? 0.f : M;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  float L = 0.f;
  for (int s = 0; s < splits; ++s) {
    const int64_t p = first + s * kRowsB;
    const float f = __builtin_amdgcn_exp2f(pm[p] - ref);
    L = __builtin_fmaf(pl[p], f, L);
    acc += *reinterpret_cast<const float4v*>(A.part + p * kHeadDim + 4 * chunk) * f;
  }
  store_out<E>(A, out_row(A, U, head, row) + 4 * chunk, acc, L);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

int launch_status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? KVDEC_OK : (int)e;
}

bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Checks a cache and the call's tokens and fills the kernels' form of them.
int take_cache(const kvdec_paged8_cache* c, const int32_t* cu, int64_t B, int64_t T, Cache8& C) {
  if (!c || !c->k_pages || !c->v_pages || !c->k_scales || !c->v_scales || !c->block_table || !c->seq_lens)
    return KVDEC_E_NULL;
  if (c->code != KVDEC_I8 && c->code != KVDEC_E4M3) return KVDEC_E_DTYPE;
  if (c->D != kHeadDim || c->KVH < 1 || c->num_pages < 1 || c->max_blocks < 1) return KVDEC_E_SHAPE;
  if (B < 1 || T < 1 || B >= ((int64_t)1 << 24) || T >= ((int64_t)1 << 30) || c->KVH > (1 << 16)) return KVDEC_E_SHAPE;
  if (!cu && T != B) return KVDEC_E_SHAPE;
  const int32_t ps = c->page_size, blk = c->block_size;
  if (ps < 16 || ps > (1 << 20) || (ps & (ps - 1))) return KVDEC_E_UNSUPPORTED;
  if (blk < 16 || blk > 128 || (blk & (blk - 1)) || blk > ps) return KVDEC_E_GROUP;
  if ((int64_t)c->max_blocks * ps >= ((int64_t)1 << 30) || c->num_pages >= ((int64_t)1 << 31)) return KVDEC_E_SHAPE;
  if (c->page_stride < 0 || c->row_stride < 0 || c->head_stride < 0 || c->row_stride >= ((int64_t)1 << 27))
    return KVDEC_E_SHAPE;
  if (!on16(c->k_pages) || !on16(c->v_pages) || ((c->page_stride | c->row_stride | c->head_stride) & 15))
    return KVDEC_E_UNSUPPORTED;
  C.k = (char*)c->k_pages;
  C.v = (char*)c->v_pages;
  C.ks = c->k_scales;
  C.vs = c->v_scales;
  C.bt = c->block_table;
  C.lens = c->seq_lens;
  C.cu = cu;
  C.page_bytes = c->page_stride;
  C.head_bytes = c->head_stride;
  C.row_bytes = (uint32_t)c->row_stride;
  C.num_pages = c->num_pages;
  C.B = B;
  C.T = T;
  C.ps_log2 = __builtin_ctz((unsigned)ps);
  C.blk_log2 = __builtin_ctz((unsigned)blk);
  C.max_blocks = c->max_blocks;
  C.max_len = c->max_blocks * ps;
  C.KVH = c->KVH;
  return KVDEC_OK;
}

template <int CODE, class T>
int launch_write(const Write8Args& A, hipStream_t stream) {
  auto go = [&](auto block) {
    constexpr int kBlock = decltype(block)::value, kTasks = kWriteWaves / (kBlock <= 32 ? 1 : kBlock / 32);
    const int64_t n = (A.tasks + kTasks - 1) / kTasks;
    if (n > 0x7fffffff) return (int)KVDEC_E_SHAPE;
    write8_kernel<CODE, T, kBlock><<<dim3((unsigned)n), dim3(64 * kWriteWaves), 0, stream>>>(A);
    return launch_status();
  };
  switch (A.C.blk_log2) {
    case 4: return go(std::integral_constant<int, 16>());
    case 5: return go(std::integral_constant<int, 32>());
    case 6: return go(std::integral_constant<int, 64>());
    default: return go(std::integral_constant<int, 128>());
  }
}

template <int CODE>
int launch_write(const Write8Args& A, int dtype, hipStream_t stream) {
  switch (dtype) {
    case KVDEC_F16: return launch_write<CODE, _Float16>(A, stream);
    case KVDEC_BF16: return launch_write<CODE, uint16_t>(A, stream);
    default: return launch_write<CODE, float>(A, stream);
  }
}

template <int CODE>
int launch_read(const Read8Args& A, int dtype, hipStream_t stream) {
  const int64_t n = (A.tasks + kWriteWaves - 1) / kWriteWaves;
  if (n > 0x7fffffff) return KVDEC_E_SHAPE;
  const dim3 grid((unsigned)n), block(64 * kWriteWaves);
  switch (dtype) {
    case KVDEC_F16: read8_kernel<CODE, _Float16><<<grid, block, 0, stream>>>(A); break;
    case KVDEC_BF16: read8_kernel<CODE, uint16_t><<<grid, block, 0, stream>>>(A); break;
    default: read8_kernel<CODE, float><<<grid, block, 0, stream>>>(A); break;
  }
  return launch_status();
}

// Narrow kernel: workgroups, no more than there can be runs of one tile a wave;
// none if no sequence can have so few rows.
int narrow_groups(bool offsets, int64_t B, int32_t KVH, int32_t G, int64_t max_len) {
  if (G > kRowsA) return 0;
  const int64_t tiles = B * KVH * ((max_len + kTile - 1) / kTile);
  return (int)std::min<int64_t>(kGroupsA, std::max<int64_t>(1, (tiles + kWavesA - 1) / kWavesA));
}
size_t narrow_bytes(int groups) { return (size_t)2 * groups * kRowsA * (kHeadDim + 2) * sizeof(float); }

// Wide kernel: units of a call (with those of the rows past the last sequence),
// and splits a pair where the pairs do not fill the GPU.
int64_t wide_units(bool offsets, int64_t B, int64_t T, int32_t G) {
  if (!offsets) return G > kRowsA ? B * ((G + kRowsB - 1) / kRowsB) : 0;
  return T * G / kRowsB + B + 1;
}
int wide_splits(int64_t units, int32_t KVH, int64_t max_len) {
  const int64_t pairs = std::max<int64_t>(units * KVH, 1), tiles = (max_len + kTileB - 1) / kTileB;
  return (int)std::max<int64_t>(1, std::min((kPairsB + pairs - 1) / pairs, tiles / 4));
}
size_t wide_bytes(int64_t units, int32_t KVH, int splits) {
  return splits <= 1 ? 0 : (size_t)units * KVH * splits * kRowsB * (kHeadDim + 2) * sizeof(float);
}

size_t attn_bytes(bool offsets, int64_t B, int64_t T, int32_t G, int32_t KVH, int64_t max_len) {
  const int64_t units = wide_units(offsets, B, T, G);
  return std::max(narrow_bytes(narrow_groups(offsets, B, KVH, G, max_len)),
                  wide_bytes(units, KVH, wide_splits(units, KVH, max_len)));
}

template <int CODE, int E>
int launch_attn8(Attn8Args A, hipStream_t stream) {
  // one after the other: both kernels' partial rows go to the same workspace
  if (A.groups > 0) {
    attn8_kernel<CODE, E><<<dim3((unsigned)A.groups), dim3(kThreadsA), 0, stream>>>(A);
    join8_kernel<E><<<dim3((unsigned)(A.C.B * A.C.KVH * kRowsA)), dim3(256), 0, stream>>>(A);
    const int rc = launch_status();
    if (rc) return rc;
  }
  if (A.units > 0) {
    wide8_kernel<CODE, E><<<dim3((unsigned)(A.units * A.C.KVH * A.splits)), dim3(kThreadsB), 0, stream>>>(A);
    if (A.splits > 1)
      wide_join8_kernel<E><<<dim3((unsigned)(A.units * A.C.KVH * (kRowsB / 8))), dim3(256), 0, stream>>>(A);
  }
  return launch_status();
}

bool bad_dtype(int dtype) { return dtype != KVDEC_F16 && dtype != KVDEC_BF16 && dtype != KVDEC_F32; }

}  // namespace

extern "C" {

int kvdec_paged8_write(const kvdec_paged8_cache* cache, const void* k, const void* v, int dtype,
                       int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                       int64_t v_head_stride, const int32_t* cu_seqlens, int64_t B, int64_t T, void* stream) {
  if (!k || !v) return KVDEC_E_NULL;
  if (bad_dtype(dtype)) return KVDEC_E_DTYPE;
  Write8Args A{};
  const int rc = take_cache(cache, cu_seqlens, B, T, A.C);
  if (rc) return rc;
  const int per16 = dtype == KVDEC_F32 ? 4 : 8;   // elements of 16 bytes
  if (!on16(k) || !on16(v) || k_token_stride % per16 || k_head_stride % per16 || v_token_stride % per16 || v_head_stride % per16)
    return KVDEC_E_UNSUPPORTED;
  A.x[0] = k;
  A.x[1] = v;
  A.tok_stride[0] = k_token_stride;
  A.tok_stride[1] = v_token_stride;
  A.head_stride[0] = k_head_stride;
  A.head_stride[1] = v_head_stride;
  A.tasks = block_units(A.C) * 2 * A.C.KVH;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return cache->code == KVDEC_I8 ? launch_write<kInt8>(A, dtype, s) : launch_write<kE4m3>(A, dtype, s);
}

int kvdec_paged8_read(const kvdec_paged8_cache* cache, const int32_t* cu_seqlens, int64_t B, int64_t T,
                      void* k_out, void* v_out, int dtype, void* stream) {
  if (!k_out || !v_out) return KVDEC_E_NULL;
  if (bad_dtype(dtype)) return KVDEC_E_DTYPE;
  Read8Args A{};
  const int rc = take_cache(cache, cu_seqlens, B, T, A.C);
  if (rc) return rc;
  if (!on16(k_out) || !on16(v_out)) return KVDEC_E_UNSUPPORTED;
  A.out[0] = k_out;
  A.out[1] = v_out;
  A.tasks = block_units(A.C) * 2 * A.C.KVH;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return cache->code == KVDEC_I8 ? launch_read<kInt8>(A, dtype, s) : launch_read<kE4m3>(A, dtype, s);
}

size_t kvdec_paged8_workspace_bytes(int64_t B, int64_t T, int32_t H, int32_t KVH, int64_t max_len) {
  if (B < 1 || T < 1 || H < 1 || KVH < 1 || H % KVH || max_len < 1 || max_len >= ((int64_t)1 << 30)) return 0;
  if (B >= ((int64_t)1 << 24) || T * (H / KVH) >= ((int64_t)1 << 30)) return 0;
  return std::max(attn_bytes(true, B, T, H / KVH, KVH, max_len), T == B ? attn_bytes(false, B, T, H / KVH, KVH, max_len) : 0);
}

int kvdec_paged8_attention(const kvdec_paged8_cache* cache, const void* q, void* o, int dtype,
                           int64_t q_token_stride, int64_t q_head_stride, const int32_t* cu_seqlens,
                           int64_t B, int64_t T, int32_t H, int32_t window, int32_t sink, float sm_scale,
                           void* ws, size_t ws_bytes, void* stream) {
  if (!q || !o) return KVDEC_E_NULL;
  if (dtype != KVDEC_F16 && dtype != KVDEC_BF16) return KVDEC_E_DTYPE;
  Attn8Args A{};
  const int rc = take_cache(cache, cu_seqlens, B, T, A.C);
  if (rc) return rc;
  if (H < 1 || H % A.C.KVH) return KVDEC_E_SHAPE;
  A.G = H / A.C.KVH;
  if (T * A.G >= ((int64_t)1 << 30)) return KVDEC_E_SHAPE;
  if (window < 0 || sink < 0 || (window == 0 && sink > 0)) return KVDEC_E_WINDOW;
  if (!on16(q) || !on16(o) || q_token_stride % 8 || q_head_stride % 8) return KVDEC_E_UNSUPPORTED;
  const bool offsets = cu_seqlens != nullptr;
  A.groups = narrow_groups(offsets, B, A.C.KVH, A.G, A.C.max_len);
  A.units = wide_units(offsets, B, T, A.G);
  A.splits = wide_splits(A.units, A.C.KVH, A.C.max_len);
  if (B * A.C.KVH * kRowsA > 0x7fffffff || A.units * A.C.KVH * std::max(A.splits, kRowsB / 8) > 0x7fffffff)
    return KVDEC_E_SHAPE;
  if (!ws || !on16(ws) || ws_bytes < attn_bytes(offsets, B, T, A.G, A.C.KVH, A.C.max_len)) return KVDEC_E_WORKSPACE;
  A.q = q;
  A.o = o;
  A.part = static_cast<float*>(ws);
  A.q_tok = q_token_stride;
  A.q_head = q_head_stride;
  A.H = H;
  A.window = window;
  A.sink = sink;
  A.scale_log2 = (float)((double)sm_scale * 1.4426950408889634);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->code == KVDEC_I8)
    return dtype == KVDEC_F16 ? launch_attn8<kInt8, kEltF16>(A, s) : launch_attn8<kInt8, kEltBf16>(A, s);
  return dtype == KVDEC_F16 ? launch_attn8<kE4m3, kEltF16>(A, s) : launch_attn8<kE4m3, kEltBf16>(A, s);
}

}  // extern "C"
