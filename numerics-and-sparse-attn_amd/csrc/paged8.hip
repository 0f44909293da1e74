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
  s.len = b < C.B ? max((int)((cint32*)C.lens)[b], 0) : 0;
  return s;
}

// Units of work without a count on the host: sequence b, whose first new token
// is c0, starts at unit first(c0, b), which grows with the rows before it by what
// a unit holds, and by as many more a sequence as its rows can touch beyond that;
// first(0, 0) is 0.  The sequence of unit u is the last with first <= u: 64 are
// tried at once, a lane each, so that a search among 64 is one load's latency.
struct Found8 {
  Seq8 s;
  int64_t first;
};

// (Sequence B: the rows past the last.)  Where `first` grows by `each` a sequence
// and by at most `rows` for all rows of the call, only sequences from
// (u - rows) / each to u / each can be it.
template <class First>
__device__ __forceinline__ Found8 find8(const Cache8& C, int64_t u, int64_t rows, int each, int lane, First&& first) {
  int64_t lo = max(u - rows, (int64_t)0) / each, n = min(u / each, C.B) - lo + 1;
  while (n > 64) {
    const int64_t step = (n + 63) / 64, s = lo + lane * step;
    const bool ok = s < lo + n && first(offset8(C, s), s) <= u;
    const int cnt = max((int)__builtin_popcountll(__ballot(ok)), 1);
    const int64_t to = lo + (cnt - 1) * step;
    n = min(step, lo + n - to);
    lo = to;
  }
  const int64_t s = lo + lane;
  int c0 = 0, c1 = 0, len = 0;
  if (lane < n) {
    c0 = offset8(C, s);
    c1 = s < C.B ? offset8(C, s + 1) : (int)C.T;
    if (s < C.B) len = max(((const int32_t*)C.lens)[s], 0);
  }
  const bool ok = lane < n && first(c0, s) <= u;
  const int at = __builtin_amdgcn_readfirstlane(max((int)__builtin_popcountll(__ballot(ok)), 1) - 1);
  Found8 f;
  f.s.b = __builtin_amdgcn_readfirstlane((int)lo) + at;
  f.s.c0 = __builtin_amdgcn_readlane(c0, at);
  f.s.n = __builtin_amdgcn_readlane(c1, at) - f.s.c0;
  f.s.len = __builtin_amdgcn_readlane(len, at);
  f.first = first(f.s.c0, (int64_t)f.s.b);
  return f;
}

// The tokens of unit u that lie in one block of one sequence: rows [r0, r1) of
// the block that starts at position `start`, whose row r is token c + r of the
// call.  page < 0: no page holds them (also positions below 0 and past the table).
struct Run8 {
  int64_t start, c;
  int r0, r1;
  int64_t page;
};

__device__ __forceinline__ Run8 run8(const Cache8& C, int64_t u, int lane) {
  Seq8 s;
  int64_t j = 0;
  if (C.cu == nullptr) {
    s = seq8(C, u);
  } else {
    const Found8 f = find8(C, u, C.T >> C.blk_log2, 2, lane, [&](int c0, int64_t b) { return ((int64_t)c0 >> C.blk_log2) + 2 * b; });
    s = f.s;
    j = u - f.first;
  }
  const int64_t p0 = (int64_t)s.len - s.n, block = (int64_t)1 << C.blk_log2;
  Run8 r;
  r.start = ((p0 >> C.blk_log2) + j) << C.blk_log2;
  r.c = (int64_t)s.c0 + r.start - p0;
  r.r0 = (int)min(max(p0 - r.start, (int64_t)0), block);
  r.r1 = s.n > 0 ? (int)max(min((int64_t)s.len - r.start, block), (int64_t)0) : 0;
  r.page = -1;
  if (r.r1 > r.r0 && r.start >= 0 && r.start < C.max_len) {
    const int64_t id = ((cint32*)C.bt)[(int64_t)s.b * C.max_blocks + (r.start >> C.ps_log2)];
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

// The high bit of every byte of c that is a NaN of e4m3.
__device__ __forceinline__ uint32_t nan_codes(uint32_t c) {
  return ((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// Four values x * m in the codes' range, rounded to codes, ties to even, in one
// rounding where x * m is exact (m a power of two).  e4m3: a NaN is the code
// 0x7f.  int8: added to 1.5 * 2^23, whose last bits are units, it is rounded to
// the byte that the sum ends in.
template <int CODE>
__device__ __forceinline__ uint32_t to_codes(float4v x, float m) {
  if constexpr (CODE == kE4m3) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * m, x[1] * m, 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * m, x[3] * m, c, true);
    return (uint32_t)c & ~nan_codes((uint32_t)c);
  } else {
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = __builtin_bit_cast(uint32_t, __builtin_fmaf(x[j], m, 12582912.f));
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u),
                                 __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
  }
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

constexpr float kFloatMax = 3.402823466e38f;

// Eight elements of a row as they are loaded.  The largest |element| of several
// is kept as bits (of all NaN and infinities above the rest): `Top` in the
// loaded form, and then as those of a float.
template <class T>
struct Row8 {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  typedef u16x2 Top;
  u32x4 w = {0u, 0u, 0u, 0u};
  __device__ __forceinline__ void load(const T* p) { w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)); }
  __device__ __forceinline__ float get(int j) const {
    const uint16_t h = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    if constexpr (std::is_same<T, _Float16>::value)
      return (float)__builtin_bit_cast(_Float16, h);
    else
      return __builtin_bit_cast(float, (uint32_t)h << 16);
  }
  __device__ __forceinline__ void top(Top& m) const {
#pragma unroll
    for (int d = 0; d < 4; ++d) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[d] & 0x7fff7fffu));
  }
  __device__ static __forceinline__ uint32_t bits(Top m) {
    const uint16_t h = m[0] > m[1] ? m[0] : m[1];
    if constexpr (std::is_same<T, _Float16>::value)
      return h >= 0x7c00 ? 0x7f800000u : __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, h));
    else
      return (uint32_t)h << 16;
  }
};
template <>
struct Row8<float> {
  typedef uint32_t Top;
  u32x4 w[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
  __device__ __forceinline__ void load(const float* p) {
    w[0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    w[1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + 4));
  }
  __device__ __forceinline__ float get(int j) const { return __builtin_bit_cast(float, (uint32_t)w[j >> 2][j & 3]); }
  __device__ __forceinline__ void top(Top& m) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, w[j >> 2][j & 3] & 0x7fffffffu);
  }
  __device__ static __forceinline__ uint32_t bits(Top m) { return m; }
};

constexpr int kWriteWaves = 4;

// One task quantizes the call's rows of one block of one KV head, of K or of
// V: at most 32 rows a wave (kept in registers between the search for the
// largest value and the rounding), 1 to 4 waves a task.
//
// Bound by memory: bf16 rows of 37008 tokens and 8 heads into e4m3, 227 MB, take
// 40 us (5.7 TB/s).  One token of one sequence takes 4 us, which are the latencies
// of its lengths, table entry, scale and rows, one after the other.  Rows are read
// past the caches; codes written past them: 42 us.
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
    run = run8(C, rest >> 1, lane);
  }
  const bool live = run.page >= 0;   // (uniform over a task's waves)
  const int base = part * kRows;

  Row8<T> x[kLoads];
  uint32_t top = 0;      // the largest |x|: the bits of a float
  float old = 0.f;
  float* scale = nullptr;
  char* codes = nullptr;
  if (live) {
    scale = (kv ? C.vs : C.ks) + scale_index(C, run.page, head, run.start);
    codes = (kv ? C.v : C.k) + row_offset(C, run.page, head, run.start);
    const T* src = (const T*)A.x[kv] + run.c * A.tok_stride[kv] + head * A.head_stride[kv] + 8 * t;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = base + 4 * i + g;
      if (r >= run.r0 && r < run.r1) x[i].load(src + r * A.tok_stride[kv]);
    }
    if (run.r0 > 0) old = *scale;
    typename Row8<T>::Top m{};
#pragma unroll
    for (int i = 0; i < kLoads; ++i) x[i].top(m);
    top = Row8<T>::bits(m);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
    top = (uint32_t)__builtin_amdgcn_readfirstlane((int)top);
  }
  bool bad = top >= 0x7f800000u;
  float amax = __builtin_bit_cast(float, top);
  if (bad) {   // once more, of the finite ones
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = __builtin_fabsf(x[i].get(j));
        amax = a <= kFloatMax ? fmaxf(amax, a) : amax;
      }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
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
      for (int d = 0; d < 4; ++d) c[d] = to_codes<CODE>(code_values<CODE>(c[d]), ratio);
      *p = c;
    }
  }

  auto store = [&](auto&& value, float m) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = base + 4 * i + g;
      u32x2 c;
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        float4v y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = value(x[i].get(4 * d + j));
        c[d] = poison ? 0u : to_codes<CODE>(y, m);
      }
      if (r >= run.r0 && r < run.r1) *reinterpret_cast<u32x2*>(codes + (int64_t)r * C.row_bytes + 8 * t) = c;
    }
  };
  // A power of two divides by its inverse, exactly; a scale that some other
  // program put there may be any.
  const uint32_t sb = (uint32_t)__builtin_amdgcn_readfirstlane((int)__builtin_bit_cast(uint32_t, s));
  const bool pow2 = (sb & 0x7fffffu) == 0 && sb < 0x7f000000u;
  if (pow2 && !bad)
    store([](float v) { return v; }, __builtin_bit_cast(float, 0x7f000000u - sb));
  else
    store([s](float v) { return __builtin_fabsf(v) <= kFloatMax ? v / s : __builtin_nanf(""); }, 1.f);
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

// One wave reads the call's rows of one block of one KV head, of K or of V: a
// lane 8 codes of a row, four rows an instruction, so that 16-bit rows leave as
// whole 256-byte ones.  The codes are read past the caches, which the rows
// written need (101 -> 87 us); the rows written past them too: 73 -> 85 us where they stay in the caches.
//
// Bound by memory: 73728 tokens of 8 heads from e4m3 to bf16, 453 MB, take 78 us
// (5.8 TB/s), 88 us a call in a row of calls with their launches.
template <int CODE, class T>
__global__ __launch_bounds__(64 * kWriteWaves) void read8_kernel(Read8Args A) {
  const Cache8& C = A.C;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t task = (int64_t)blockIdx.x * kWriteWaves + wave;
  if (task >= A.tasks) return;
  const int64_t rest = task / C.KVH;
  const int head = (int)(task - rest * C.KVH), kv = (int)(rest & 1);
  const Run8 run = run8(C, rest >> 1, lane);
  const int g = lane >> 4, col = 8 * (lane & 15);
  float scale = 0.f;
  const char* codes = nullptr;
  if (run.page >= 0) {
    scale = (kv ? C.vs : C.ks)[scale_index(C, run.page, head, run.start)];
    codes = (kv ? C.v : C.k) + row_offset(C, run.page, head, run.start) + col;
  }
  T* out = (T*)A.out[kv] + (run.c * C.KVH + head) * kHeadDim + col;
  for (int r0 = run.r0; r0 < run.r1; r0 += 32) {   // eight loads on their way
    u32x2 c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = r0 + 4 * k + g;
      c[k] = u32x2{0u, 0u};
      if (run.page >= 0 && r < run.r1)
        c[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(codes + (int64_t)r * C.row_bytes));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = r0 + 4 * k + g;
      if (r >= run.r1) continue;
      T* p = out + (int64_t)r * C.KVH * kHeadDim;
      const float4v lo = code_values<CODE>(c[k][0]) * scale, hi = code_values<CODE>(c[k][1]) * scale;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4v*>(p) = lo;
        *reinterpret_cast<float4v*>(p + 4) = hi;
      } else {
        constexpr int kElt = std::is_same<T, _Float16>::value ? kEltF16 : kEltBf16;
        const u32x2 a = round_elt4<kElt>(lo), b = round_elt4<kElt>(hi);
        *reinterpret_cast<u32x4*>(p) = u32x4{a[0], a[1], b[0], b[1]};
      }
    }
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
// the sum of the weights takes w / vs.  m follows the running maximum of
// x + log2(vs), so that w stays in fp16's range whatever the scales: it is
// kLift below the maximum that it was last set from, and set again once that is
// kHighest above it (8 rather than 15 costs the wide kernel 3%).  fp16 rounds a w
// to steps of no less than 2^-24, which the lift makes 2^-31 of the largest: where
// one token outweighs a long cache of equal ones, those are off by no more than
// 2^-32 each.  The sum is kDown of that, so that 2^19 tokens of the largest weight
// and the least V scale, 2^-100, stay under 2^128.

constexpr float kLift = 7.f, kHighest = 15.f, kDown = 0x1p-7f;

constexpr int kRowsA = 16;
constexpr int kWavesA = 4;
constexpr int kThreadsA = 64 * kWavesA;
constexpr int kSlotA = 2 * kTile * kCodeRow;        // K and V codes of a tile
constexpr int kGroupsA = 512;                       // workgroups of a launch, at most: two a CU
static_assert(kRowsA * kHeadDim * 4 <= kSlotA, "a wave's partial rows fit its slot");

constexpr int kRowsB = 128;                         // query rows of a workgroup, 32 a wave
constexpr int kThreadsB = 256;
constexpr int kTileB = 64;                          // tokens of its tiles
constexpr int kPairsB = 512;                        // workgroups that fill the GPU,
constexpr int kJoinsB = 1024;                       // and of a join

struct Attn8Args {
  Cache8 C;
  const void* q;
  void* o;
  float* part;                // the workspace: the narrow kernel's parts,
  int64_t wide_at;            // and (from this float on) the wide one's
  int64_t q_tok, q_head;      // in elements
  int64_t units;
  int32_t G, H, window, sink;
  int32_t groups;             // narrow: workgroups (a power of two),
  int32_t side, pairs;        // KV heads that one may read side by side (1, 2 or 4), and KVH / side
  uint32_t inv_g;             // 65536 / G rounded up: row / G of a narrow row is row * inv_g >> 16
  int32_t slots, few;         // wide: workgroups a KV head that the units are dealt to, and those that
                              // fill the GPU; slots = 0: one a unit
  uint32_t wide_blocks, passes;   // the join's workgroups for them, and the rows of each, by 8
  float scale_log2;
};

// A unit: query rows [row0, row0 + rows) of a sequence's n * G, at positions
// pos0 .. pos1, whose keys end before hi, and its tiles: [0, ts) of the sink and
// [tw, te).
struct Unit8 {
  Seq8 s;
  int row0, rows, pos0, pos1, hi;
  int ts, tw, te;
  __device__ __forceinline__ int tiles() const { return ts + te - tw; }
  __device__ __forceinline__ int tile(int j) const { return j < ts ? j : tw + j - ts; }
};

// The first position of a window that ends at `pos` (any window up to INT32_MAX,
// and positions before the start, which see nothing).
__device__ __forceinline__ int from8(const Attn8Args& A, int pos) { return max(pos, -1) - A.window + 1; }

template <int TILE>
__device__ __forceinline__ void unit_tiles(const Attn8Args& A, Unit8& U, int pos0, int pos1) {
  U.ts = U.tw = U.te = U.hi = 0;
  U.pos0 = U.pos1 = -1;
  if (U.rows <= 0) {
    U.rows = 0;
    return;
  }
  U.pos0 = pos0;
  U.pos1 = pos1;
  if (U.pos1 < 0) return;
  U.hi = min(U.pos1, A.C.max_len - 1) + 1;
  U.te = (U.hi + TILE - 1) / TILE;
  if (A.window > 0) {
    U.ts = min((int)(((int64_t)A.sink + TILE - 1) / TILE), U.te);
    U.tw = min(max(U.ts, max(from8(A, U.pos0), 0) / TILE), U.te);
  }
}

// The narrow kernel's unit: a sequence, if its rows fit.
__device__ __forceinline__ Unit8 unit_a(const Attn8Args& A, const Seq8& s) {
  Unit8 U;
  U.s = s;
  U.row0 = 0;
  U.rows = (int64_t)s.n * A.G <= kRowsA ? s.n * A.G : 0;
  unit_tiles<kTile>(A, U, s.len - s.n, s.len - 1);
  return U;
}
__device__ __forceinline__ Unit8 unit_a(const Attn8Args& A, int64_t b) { return unit_a(A, seq8(A.C, b)); }

// The same by halving, on scalars alone (the wide kernel has no registers for the
// search above: 15% of its time).
template <class First>
__device__ __forceinline__ Found8 find8_scalar(const Cache8& C, int64_t u, int64_t rows, First&& first) {
  int64_t lo = max(u - rows, (int64_t)0), hi = min(u, C.B);
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (first(offset8(C, mid), mid) <= u) lo = mid; else hi = mid - 1;
  }
  const Seq8 s = seq8(C, lo);
  return Found8{s, first(s.c0, lo)};
}

// The wide kernel's units are kRowsB rows of a sequence of more than kRowsA, or
// of the rows past the last sequence (which attend to nothing).
__device__ __forceinline__ int64_t rows_b(const Attn8Args& A, const Seq8& s) {
  const int64_t rows = (int64_t)s.n * A.G;
  return rows > kRowsA || s.b == A.C.B ? rows : 0;
}
__device__ __forceinline__ Unit8 unit_of(const Attn8Args& A, const Seq8& s, int64_t row0) {
  Unit8 U;
  U.s = s;
  const int64_t rows = rows_b(A, s);
  U.row0 = (int)min(row0, rows);
  U.rows = (int)min(rows - U.row0, (int64_t)kRowsB);
  const int p0 = s.len - s.n;
  unit_tiles<kTileB>(A, U, p0 + U.row0 / A.G, p0 + (U.row0 + U.rows - 1) / A.G);
  return U;
}
__device__ __forceinline__ Unit8 unit_b(const Attn8Args& A, int64_t u) {
  const Cache8& C = A.C;
  if (C.cu == nullptr) {
    const int per = (A.G + kRowsB - 1) / kRowsB;
    return unit_of(A, seq8(C, u / per), u % per * kRowsB);
  }
  const Found8 f = find8_scalar(C, u, C.T * A.G / kRowsB, [&](int c0, int64_t b) { return (int64_t)c0 * A.G / kRowsB + b; });
  return unit_of(A, f.s, max(u - f.first, (int64_t)0) * kRowsB);
}

// The positions that a query row sees: up to `upto`, and before `sink` or from
// `from` on.
struct Sight8 {
  int upto, from, sink;
  __device__ __forceinline__ bool sees(int p) const { return (p <= upto) & ((p < sink) | (p >= from)); }
};
__device__ __forceinline__ Sight8 sight8(const Attn8Args& A, const Unit8& U, int pos) {
  return A.window > 0 ? Sight8{min(pos, U.hi - 1), from8(A, pos), A.sink} : Sight8{min(pos, U.hi - 1), 0, 0};
}

// Every token of [tok, tok + n) is seen by every row of the unit.
__device__ __forceinline__ bool all_seen(const Attn8Args& A, const Unit8& U, int tok, int n) {
  return (tok + n - 1 <= min(U.pos0, U.hi - 1)) & ((A.window <= 0) | (tok + n <= A.sink) | (tok > U.pos1 - A.window));
}

// What a token of the pair's rows weighs by: kf turns q . k into x, lv is
// log2 of V's scale and inv its inverse (times kDown).  No page: keys and values of zero.
struct Meta8 {
  int page;
  float kf, lv, inv;
};

// The table's entry of a token (-1: not live), and the page that it names.
__device__ __forceinline__ int entry8(const Cache8& C, int b, int tok, bool live) {
  int id = -1;
  if (live) id = C.bt[(int64_t)b * C.max_blocks + (tok >> C.ps_log2)];
  return id;
}
__device__ __forceinline__ int page8(const Cache8& C, int id) { return id < C.num_pages ? id : -1; }
__device__ __forceinline__ float2v scales8(const Cache8& C, int page, int head, int tok) {
  float2v s = {0.f, 1.f};
  if (page >= 0) {
    const int64_t at = scale_index(C, page, head, tok);
    s = float2v{C.ks[at], C.vs[at]};
  }
  return s;
}
__device__ __forceinline__ Meta8 meta8(const Attn8Args& A, int page, float2v s) {
  const float vs = s[1] < 0x1p-100f ? 0x1p-100f : s[1];   // a scale that is hardly one counts as the writer's least
  return Meta8{page, s[0] * A.scale_log2, __builtin_amdgcn_logf(vs),
               vs == vs ? kDown / vs : 1.f};              // a NaN arrives through lv, where masks hold
}

// Place of row `row` of a pair in the output.
__device__ __forceinline__ int64_t out_row(const Attn8Args& A, const Unit8& U, int head, int row) {
  const int r = U.row0 + row, tok = r / A.G;
  return ((int64_t)(U.s.c0 + tok) * A.H + head * A.G + (r - tok * A.G)) * kHeadDim;
}

template <int E>
__device__ __forceinline__ void store_out(const Attn8Args& A, int64_t at, float4v acc, float l) {
  // one division for all channels (and a 1 / l that stays finite): whole prompts 1.5%
  const float up = l < 0x1p-100f ? 0x1p64f : 1.f;
  const float inv = kDown / (l == 0.f ? 1.f : l * up);
  *reinterpret_cast<u32x2*>((uint16_t*)A.o + at) = round_elt4<E>(acc * up * inv);
}

// ---- the narrow kernel ----
//
// A pair is a sequence and `side` neighbouring KV heads, a wave or more each:
// where the heads' rows of a token are neighbours in memory, the waves read them
// together (NHD pages, B=32, L=32768: 405 -> 350 us).  The tiles (32 tokens) of
// all pairs, in order, are dealt to the launch's workgroups in equal runs,
// whatever the sequences' lengths: each finds its run from the lengths on the
// device.  A pair that falls to several workgroups leaves partial rows in the
// workspace, which a second kernel joins.
//
// Bound by memory where runs are long: 32 sequences of 32768 tokens and 8 heads,
// 2.15 GB, take 347 us with the join's 5 (6.2 TB/s; the same loads alone 6.5).
// Where they are short, by latencies: 2 us to the lengths, 2.4 to deal and to find
// the run, 2.7 for entries, scales and first tiles, 4 for the join of 8 sequences'
// windows of 4096 tokens, which take 26 us of which 12 are the tiles' own.

// The sum of the lanes' x up to this one (DPP: row_shr 1, 2, 4, 8 inside rows of
// 16 lanes, then row_bcast 15 and 31 across them).
__device__ __forceinline__ uint32_t upto_lane(uint32_t x) {
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);
  return x;
}
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }

// Sequence v (none past the last), and its tiles of one KV head.
__device__ __forceinline__ Seq8 seq_a(const Attn8Args& A, int64_t v) {
  return v < A.C.B ? seq8(A.C, v) : Seq8{(int)v, 0, 0, 0};
}
__device__ __forceinline__ uint32_t tiles_a(const Attn8Args& A, int64_t v) {
  return (uint32_t)unit_a(A, seq_a(A, v)).tiles();
}

// a / b rounded up, b > 0; small ones by a reciprocal, put right by one.
__device__ __forceinline__ uint32_t up(uint32_t a, uint32_t b) {
  if ((a | b) >> 21) return a / b + (a % b != 0);
  uint32_t q = (uint32_t)((float)a * __builtin_amdgcn_rcpf((float)b));
  const int left = (int)(a - q * b);
  q = left < 0 ? q - 1 : left >= (int)b ? q + 1 : q;
  return q + (q * b != a);
}
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {   // of numbers >= 0
  return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
// At least a / b, and little more.
__device__ __forceinline__ int64_t about(int64_t a, int64_t b) {
  return (int64_t)((float)a * __builtin_amdgcn_rcpf((float)b) * 1.0001f) + 1;
}

// How a launch's tiles are dealt (all: one KV head's, some: sequences with any).
//   side, pairs  KV heads of a pair, and pairs of a sequence.  Heads side by side
//                where the runs are long, or where a workgroup has several pairs
//                (fewer of them: 256 sequences of up to 300 tokens 118 -> 57 us);
//                else a head's waves, joined in the workgroup.
//   toll         what a pair costs besides its tiles, in tiles, where a
//                workgroup has several: its loads' latencies, 6 us
//   share        a workgroup's run of tiles (and tolls)
//   alone        the pairs are so few that each can be cut into parts of at most
//                `share` tiles, a workgroup each: no workgroup then pays a second
//                pair's latencies (16 sequences of up to 16384 tokens 63 -> 60 us)
struct Deal8 {
  int side, pairs, toll;
  bool alone;
  int64_t share;
  // what a pair of n tiles takes of the runs' common line
  __device__ __forceinline__ int64_t length(uint32_t n) const {
    if (n == 0) return 0;
    return alone ? (int64_t)up(n, (uint32_t)share) * share : (int64_t)n + toll;
  }
};
constexpr int kLongRun = 16, kLeastRounds = 2;
// (n: the lane's sequence's tiles, of the first 64)
__device__ __forceinline__ Deal8 deal8(const Attn8Args& A, int64_t all, int64_t some, uint32_t n) {
  Deal8 d;
  const bool crowd = some * A.C.KVH > A.groups;
  const bool lengthy = all * A.C.KVH >= (int64_t)kLongRun * kWavesA * A.groups;
  const bool far = lengthy && A.C.head_bytes < (int64_t)A.C.row_bytes;
  d.side = (crowd | far) ? A.side : 1;
  d.pairs = (crowd | far) ? A.pairs : A.C.KVH;
  const int phases = (crowd | far) ? kWavesA / A.side : kWavesA;
  const int64_t count = some * d.pairs;
  d.alone = 2 * count <= A.groups;
  d.toll = 2 * count > A.groups ? 4 * phases : 0;
  // runs no shorter than a pair of few tiles, or two tiles for each wave of a head
  const int64_t least = all <= (int64_t)kLeastRounds * phases * some ? about(all, max(some, (int64_t)1)) : kLeastRounds * phases;
  const int64_t even = max(((all + some * d.toll) * d.pairs + A.groups - 1) >> __builtin_ctz(A.groups), least);
  d.share = even;
  if (d.alone) {
    // all / share parts and one a pair are enough workgroups for certain; with
    // 64 sequences at most, the least of some shares between that does
    const int64_t sure = max(about(all * d.pairs, A.groups - count), even);
    d.share = sure;
    if (A.C.B <= 64 && sure > even) {
#pragma unroll
      for (int k = 1; k >= 0; --k) {
        const uint32_t t = (uint32_t)(even + (k ? (sure - even) >> 1 : 0));
        const uint32_t parts = last_lane(upto_lane(up(n, t)));
        if ((int64_t)parts * d.pairs <= A.groups) d.share = t;
      }
    }
  }
  return d;
}

// The workspace: partial rows, of two runs a workgroup can leave (the end of one
// pair, `from` its start the beginning of another), up to A.side heads of
// kRowsA rows each; each row's maximum and sum; and for every sequence and KV
// head how its rows were left.
struct Left8 {
  int first, n;     // workgroups first .. first + n - 1 have parts of the rows; n = 0: written whole
  int side, h;      // their heads side by side, and which this is
};
__device__ __forceinline__ int64_t part_place(int side, int group, bool from, int h, int row) {
  return ((2 * (int64_t)group + (from ? 1 : 0)) * side + h) * kRowsA + row;
}
__host__ __device__ inline int64_t part_rows(int groups, int side) { return (int64_t)2 * groups * side * kRowsA; }
__device__ __forceinline__ float* part_sums(const Attn8Args& A) {
  return A.part + part_rows(A.groups, A.side) * kHeadDim;
}
__device__ __forceinline__ Left8* part_left(const Attn8Args& A) {
  return reinterpret_cast<Left8*>(part_sums(A) + 2 * part_rows(A.groups, A.side));
}

// A wave's running softmax: lane (n, g) has row n; O[cb][r] is channel
// 16 cb + 4 g + r; l is the lane's share of the sum.
struct State8 {
  float4v O[8];
  float m, l;
};

// Tiles whose pages and scales a wave holds.  Two tiles are on their way to it
// (three: 32 sequences of 32768 tokens 2% faster in int8, 64 of 500 35% slower).
constexpr int kAhead = 32;

struct Raw8 {
  u32x4 k[4], v[4];
};

struct NarrowLds {
  char slots[kWavesA * kSlotA];
  float m[kWavesA][kRowsA], l[kWavesA][kRowsA];
};

template <int CODE, int E>
__device__ __forceinline__ void narrow_part(const Attn8Args& A, int group, NarrowLds& L8) {
  char* const lds = L8.slots;
  auto& lds_m = L8.m;
  auto& lds_l = L8.l;
  const Cache8& C = A.C;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = lane & 15, g = lane >> 4;
  char* slot = lds + wave * kSlotA;

  // this workgroup's run of tiles, and the sequence that it starts in
  Seq8 s0 = seq_a(A, lane);
  uint32_t n0 = (uint32_t)unit_a(A, s0).tiles();
  int64_t all = last_lane(upto_lane(n0)), some = __builtin_popcountll(__ballot(n0 != 0));
  for (int64_t u0 = 64; u0 < C.B; u0 += 256) {   // four loads on their way
    uint32_t n = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t mine = tiles_a(A, u0 + 64 * k + lane);
      some += __builtin_popcountll(__ballot(mine != 0));
      n += mine;
    }
    all += last_lane(upto_lane(n));
  }
  const Deal8 deal = deal8(A, all, some, n0);
  const int pairs = deal.pairs, side = deal.side, toll = deal.toll;
  int64_t cur = (int64_t)group * deal.share;
  int64_t end = cur + deal.share;
  int64_t u = 0, base = 0;   // base: where the pair begins that `cur` lies in
  Unit8 U;
  for (;;) {
    const uint32_t mine = (uint32_t)deal.length(n0), upto = upto_lane(mine);
    const uint64_t past = __ballot(base + (int64_t)upto * pairs > cur);
    if (past) {
      const int first = __builtin_ctzll(past);
      base += (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(upto - mine), first) * pairs;
      u += first;
      U = unit_a(A, Seq8{(int)u, __builtin_amdgcn_readlane(s0.c0, first), __builtin_amdgcn_readlane(s0.n, first),
                         __builtin_amdgcn_readlane(s0.len, first)});
      break;
    }
    base += (int64_t)last_lane(upto) * pairs;
    u += 64;
    if (u >= C.B) return;    // no run is left
    s0 = seq_a(A, u + lane);
    n0 = (uint32_t)unit_a(A, s0).tiles();
  }
  int64_t length = deal.length(U.tiles());
  int pair = (int)quotient(cur - base, length);
  base += (int64_t)pair * length;
  const int phases = kWavesA / side, phase = wave / side;   // waves of a head

  for (;;) {
    const int nt = U.tiles();
    const int j0 = (int)max(cur - base - toll, (int64_t)0);
    const int j1 = (int)max(min((int64_t)nt, end - base - toll), (int64_t)0);
    if (j0 < j1) {
    const int head = pair * side + wave % side;

    // this lane's query row
    const int my_tok = (int)((uint32_t)t * A.inv_g >> 16), my_head = t - my_tok * A.G;
    const Sight8 sight = sight8(A, U, t < U.rows ? U.s.len - U.s.n + my_tok : -1);
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

    const int hi = U.hi, lo = A.window > 0 ? max(from8(A, U.pos0), 0) : 0;
    const int sink = A.window > 0 ? A.sink : 0;
    const char* kbase = C.k + head * C.head_bytes;
    const char* vbase = C.v + head * C.head_bytes;
    const int own = (j1 - j0 - phase + phases - 1) / phases;   // this wave's tiles: j0 + phase, + phases, ...
    const uint32_t off0 = (uint32_t)(lane >> 3) * C.row_bytes + 16u * (lane & 7);
    auto tok_of = [&](int i) { return kTile * U.tile(j0 + phase + phases * i); };
    auto lane_f = [](float x, int l) {
      return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
    };
    // Lane 2i + h has half h of the wave's tile i of kAhead: its page and scales;
    // the page, the raw scales of the next kAhead tiles, and the table's entry of
    // those after: each is loaded kAhead tiles before it is used.
    const int my_i = lane >> 1, my_h = 16 * (lane & 1);
    auto my_tok_of = [&](int i0) { return tok_of(min(i0 + my_i, own - 1)) + my_h; };
    auto entries = [&](int i0) {
      const int tok = my_tok_of(i0);
      return entry8(C, U.s.b, tok, i0 + my_i < own && tok < hi);
    };

    if (own > 0) {
      const int first = entries(0), second = entries(kAhead);
      int after = entries(2 * kAhead), next = -1;
      Meta8 meta;
      meta.page = page8(C, first);
      // (whole halves of pages, also where not every row is seen: no branch, so
      // that the waits for the loads stay exact)
      // (c: the tile's place from i0, the first of the held ones)
      int i0 = 0;
      auto load = [&](int c, Raw8& X) {
        const bool live = i0 + c < own;
        const int row = tok_of(live ? i0 + c : 0) & ((1 << C.ps_log2) - 1);
        const int from = c >= kAhead ? next : meta.page, at = c >= kAhead ? c - kAhead : c;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int page = __builtin_amdgcn_readlane(from, 2 * at + h);
          const uint32_t bytes = (live & (page >= 0)) ? 15u * C.row_bytes + kCodeRow : 0u;
          // a tile's second half is the first's page's next rows, or at a page's start
          const int64_t off = max(page, 0) * C.page_bytes + (int64_t)((row + 16 * h) & ((1 << C.ps_log2) - 1)) * C.row_bytes;
          const rsrc_t rk = make_rsrc(kbase + off, bytes), rv = make_rsrc(vbase + off, bytes);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            X.k[2 * h + r] = bload16(rk, off0 + 8u * r * C.row_bytes);
            X.v[2 * h + r] = bload16(rv, off0 + 8u * r * C.row_bytes);
          }
        }
      };
      auto step = [&](int c, Raw8& X) {
        const int tok = tok_of(i0 + c), at = 2 * c;
        const bool full = all_seen(A, U, tok, kTile);
        const int r8 = lane >> 3, ch = lane & 7;
        bool nans = false;
        if (!full) {
          // V rows that no query row sees count as zeros; a NaN that some see
          // takes the longer way below
          uint32_t any = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int p = tok + 8 * k + r8;
            const bool seen = p < hi && (p >= lo || p < sink);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              X.v[k][d] = seen ? X.v[k][d] : 0u;
              any |= nan_codes(X.v[k][d]);
            }
          }
          nans = CODE == kE4m3 && __any(any != 0);
        }
        // staged: K rows' 16-byte chunks turned by the row, V's by its place
        // among the eight rows that a transposed read takes
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 8 * k + r8;
          *reinterpret_cast<u32x4*>(slot + r * kCodeRow + ((ch ^ r8) << 4)) = X.k[k];
          *reinterpret_cast<u32x4*>(slot + kTile * kCodeRow + r * kCodeRow + ((ch ^ ((r8 & 3) | ((k >> 1) << 2))) << 4)) = X.v[k];
        }
        load(c + 2, X);

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
        const float kf0 = lane_f(meta.kf, at), kf1 = lane_f(meta.kf, at + 1);
        const float lv0 = lane_f(meta.lv, at), lv1 = lane_f(meta.lv, at + 1);
        const float inv0 = lane_f(meta.inv, at), inv1 = lane_f(meta.inv, at + 1);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          x[j] = __builtin_fmaf(j < 4 ? s0[j & 3] : s1[j & 3], j < 4 ? kf0 : kf1, j < 4 ? lv0 : lv1);
        uint32_t seen = 0;
        if (!full) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool ok = sight.sees(tok + tau(g, j));
            seen |= (uint32_t)ok << j;
            x[j] = ok ? x[j] : -INFINITY;
          }
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
        if (__any(top > st.m + kHighest)) {
          const float m = fmaxf(st.m, group_max(top) - kLift);
          const float f = __builtin_amdgcn_exp2f(st.m - m);
          st.l *= f;
#pragma unroll
          for (int cb = 0; cb < 8; ++cb) st.O[cb] = st.O[cb] * f;
          st.m = m;
        }
        // weights as an fp16 and the fp16 of its remainder, good to 2^-22 of those
        // that count; a tile's sum is added at once, so that a long cache of small
        // ones is not lost beside a large one
        half8 pB, pL;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = __builtin_amdgcn_exp2f(x[j] - st.m);
          sum[j >> 2] += w;
          pB[j] = (_Float16)w;
          pL[j] = (_Float16)(w - (float)pB[j]);
        }
        st.l += __builtin_fmaf(sum[0], inv0, sum[1] * inv1);
        const char* vt = slot + kTile * kCodeRow + tau(g, t >> 1) * kCodeRow + 8 * (t & 1);
        if (CODE == kE4m3 && nans) {
          // a NaN reaches the rows that see its token: marked as ones, and
          // multiplied with what each row sees; the others count it as 0
          half8 eyes;
#pragma unroll
          for (int j = 0; j < 8; ++j) eyes[j] = (seen >> j) & 1u ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
          for (int cb = 0; cb < 8; ++cb) {
            u32x2 c = lds_read_tr8(vt + ((cb ^ (t >> 1)) << 4));
            u32x4 marks;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              const uint32_t bad = nan_codes(c[d]) >> 7;   // 0 or 1 a byte
              c[d] &= ~(bad * 0xffu);
              marks[2 * d] = (bad & 1u) * 0x3c00u | ((bad >> 8) & 1u) * 0x3c000000u;
              marks[2 * d + 1] = ((bad >> 16) & 1u) * 0x3c00u | ((bad >> 24) & 1u) * 0x3c000000u;
            }
            const float4v hit = mfma16x16x32<kEltF16>(marks, eyes, float4v{0.f, 0.f, 0.f, 0.f});
            const u32x4 a = widen8<CODE, kEltF16>(c);
            st.O[cb] = mfma16x16x32<kEltF16>(a, pB, st.O[cb]);
            st.O[cb] = mfma16x16x32<kEltF16>(a, pL, st.O[cb]);
#pragma unroll
            for (int r = 0; r < 4; ++r) st.O[cb][r] = hit[r] > 0.f ? __builtin_nanf("") : st.O[cb][r];
          }
        } else {
#pragma unroll
          for (int cb = 0; cb < 8; ++cb) {
            const u32x4 a = widen8<CODE, kEltF16>(lds_read_tr8(vt + ((cb ^ (t >> 1)) << 4)));
            st.O[cb] = mfma16x16x32<kEltF16>(a, pB, st.O[cb]);
            st.O[cb] = mfma16x16x32<kEltF16>(a, pL, st.O[cb]);
          }
        }
      };
      const float2v now = scales8(C, meta.page, head, my_tok_of(0));
      Raw8 X[2];
      load(0, X[0]);
      load(1, X[1]);
      next = page8(C, second);
      meta = meta8(A, meta.page, now);
      float2v next_s = scales8(C, next, head, my_tok_of(kAhead));
      for (;;) {
        const int n = min(own - i0, kAhead);
        int c = 0;
        for (; c + 1 < n; c += 2) {
          step(c, X[0]);
          step(c + 1, X[1]);
        }
        if (c < n) step(c, X[0]);   // (the wave's last)
        i0 += kAhead;
        if (i0 >= own) break;
        meta = meta8(A, next, next_s);
        next = page8(C, after);
        next_s = scales8(C, next, head, my_tok_of(i0 + kAhead));
        after = entries(i0 + 2 * kAhead);
      }
    }

    // join the waves of a head: each parks its rows in its slot
    const float l = group_sum(st.l);
    if (g == 0) {
      lds_m[wave][t] = st.m;
      lds_l[wave][t] = l;
    }
#pragma unroll
    for (int cb = 0; cb < 8; ++cb)
      *reinterpret_cast<float4v*>(slot + t * (kHeadDim * 4) + (((4 * cb + g) ^ t) << 4)) = st.O[cb];
    __syncthreads();
    const bool whole = j1 - j0 == nt;
    const int row = threadIdx.x >> 4;   // kThreadsA / 16 == kRowsA
    if (row < U.rows) {
      for (int h = 0; h < side; ++h) {
        float M = lds_m[h][row], L = 0.f;
        for (int w = h + side; w < kWavesA; w += side) M = fmaxf(M, lds_m[w][row]);
        float4v acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        const int chunk = threadIdx.x & 15;
        for (int w = h; w < kWavesA; w += side) {
          const float f = __builtin_amdgcn_exp2f(lds_m[w][row] - M);
          L = __builtin_fmaf(lds_l[w][row], f, L);
          const char* rows = lds + w * kSlotA + row * (kHeadDim * 4);
          acc[0] += *reinterpret_cast<const float4v*>(rows + ((chunk ^ row) << 4)) * f;
          acc[1] += *reinterpret_cast<const float4v*>(rows + (((chunk + 16) ^ row) << 4)) * f;
        }
        const int hd = pair * side + h;
        const int64_t place = part_place(side, group, j0 == 0, h, row);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (whole)
            store_out<E>(A, out_row(A, U, hd, row) + 4 * (chunk + 16 * k), acc[k], L);
          else
            *reinterpret_cast<float4v*>(A.part + place * kHeadDim + 4 * (chunk + 16 * k)) = acc[k];
        }
        if (!whole && chunk == 0) *reinterpret_cast<float2v*>(part_sums(A) + 2 * place) = float2v{M, L};
      }
    }
    if (j0 == 0 && (int)threadIdx.x < side) {   // the pair's first run says where the others are
      Left8 left = {group, 0, side, (int)threadIdx.x};
      if (!whole) left.n = 1 + (int)quotient(nt - j1 + deal.share - 1, deal.share);
      part_left(A)[u * C.KVH + pair * side + threadIdx.x] = left;
    }
    }
    base += length;
    cur = base;
    if (cur >= end) return;
    __syncthreads();   // the slots are free again
    if (++pair == pairs) {
      pair = 0;
      do {
        if (++u >= C.B) return;   // the last run may be short
        U = unit_a(A, u);
      } while (U.tiles() == 0);
      length = deal.length(U.tiles());
    }
  }
}

// Joins the rows that several workgroups share, and writes zeros for those that
// attend to nothing: a workgroup for 16 rows of a sequence and KV head (MANY:
// enough pairs to fill the GPU, and so few parts of each), or for one row, whose
// parts it reads eight at a time.
template <int E, bool MANY>
__device__ __forceinline__ void narrow_join(const Attn8Args& A, uint32_t block) {
  const Cache8& C = A.C;
  const int grp = threadIdx.x >> 5, chunk = threadIdx.x & 31;
  const uint32_t id = MANY ? block : block / (uint32_t)kRowsA;
  const int head = (int)(id % (uint32_t)C.KVH);
  const int64_t u = id / (uint32_t)C.KVH;
  Left8 left = part_left(A)[id];
  // (inside the workspace whatever it holds)
  left.side = left.side == A.side ? A.side : 1;
  left.h = left.h & (left.side - 1);
  left.first = min(max(left.first, 0), A.groups - 1);
  left.n = min(max(left.n, 0), A.groups - left.first);
  const Unit8 U = unit_a(A, u);
  const bool none = U.tiles() == 0;        // (then nothing is said of its rows)
  if (!none && left.n == 0) return;
  // the parts of a row: a first run's is its second place, the others' the first
  auto part = [&](int i, int row) { return part_place(left.side, left.first + i, i == 0, left.h, row); };
  const float2v* sums = reinterpret_cast<const float2v*>(part_sums(A));
  if constexpr (MANY) {
    for (int row = grp; row < U.rows; row += 8) {
      float M = kMaxSentinel, L = 0.f;
      float4v acc = {0.f, 0.f, 0.f, 0.f};
      for (int i0 = 0; !none && i0 < left.n; i0 += 8) {
        float2v ml[8];
        float4v a[8];
        float top = M;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int64_t p = part(min(i0 + k, left.n - 1), row);
          ml[k] = sums[p];
          a[k] = *reinterpret_cast<const float4v*>(A.part + p * kHeadDim + 4 * chunk);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k][0]);
        const float again = __builtin_amdgcn_exp2f(M - top);
        M = top;
        acc = acc * again;
        L *= again;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i0 + k < left.n) {
            const float f = __builtin_amdgcn_exp2f(ml[k][0] - M);
            acc += a[k] * f;
            L = __builtin_fmaf(ml[k][1], f, L);
          }
      }
      store_out<E>(A, out_row(A, U, head, row) + 4 * chunk, acc, L);
    }
  } else {
    const int row = (int)(block % (uint32_t)kRowsA);
    if (row >= U.rows) return;
    float M = kMaxSentinel, L = 0.f;
    float4v acc = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = grp; !none && i0 < left.n; i0 += 32) {   // parts grp, + 8, ..., four on their way
      float2v ml[4];
      float4v a[4];
      float top = M;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t p = part(min(i0 + 8 * k, left.n - 1), row);
        ml[k] = sums[p];
        a[k] = *reinterpret_cast<const float4v*>(A.part + p * kHeadDim + 4 * chunk);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) top = fmaxf(top, ml[k][0]);
      const float again = __builtin_amdgcn_exp2f(M - top);
      M = top;
      acc = acc * again;
      L *= again;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + 8 * k < left.n) {
          const float f = __builtin_amdgcn_exp2f(ml[k][0] - M);
          acc += a[k] * f;
          L = __builtin_fmaf(ml[k][1], f, L);
        }
    }
    __shared__ float4v rows[8][32];
    __shared__ float2v both[8];
    rows[grp][chunk] = acc;
    if (chunk == 0) both[grp] = float2v{M, L};
    __syncthreads();
    if (grp != 0) return;
    float top = M;
#pragma unroll
    for (int w = 1; w < 8; ++w) top = fmaxf(top, both[w][0]);
    acc = float4v{0.f, 0.f, 0.f, 0.f};
    L = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float f = __builtin_amdgcn_exp2f(both[w][0] - top);
      acc += rows[w][chunk] * f;
      L = __builtin_fmaf(both[w][1], f, L);
    }
    store_out<E>(A, out_row(A, U, head, row) + 4 * chunk, acc, L);
  }
}

// ---- the wide kernel ----
//
// One workgroup a unit and KV head, or a part of its tiles: four waves of 32 query rows
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
//
// Bound by the issue of its products and of the weights between them: e4m3, 2048
// new tokens of 64 heads over 8192 take 512 us (481 GFLOP, 940 TFLOP/s; the
// matrix units are busy 45% of the time), int8 prompts of 10501 tokens in 6
// sequences 492 us (373 GFLOP, 760 TFLOP/s, their masked halves of tiles not
// counted).

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
static_assert(kThreadsA == kThreadsB, "one launch for both kernels");

// Where the units are too few to fill the GPU, their tiles are dealt to the
// workgroups in parts of equal size, as the lengths on the device make it: with
// `few` workgroups a KV head, parts of all tiles / (few - units), so that the
// parts that are not whole still find a workgroup each (a sequence's units count
// as having the tiles of its last), or smaller ones if they do too.  Every
// workgroup makes the same deal, and takes the part of its number.  (As many
// parts of each unit, whatever its length: 8 sequences of up to 4000 tokens with
// 5 new ones each 32 us, so 26; more workgroups than fill the GPU: no gain.)
struct DealB {
  Unit8 U;
  int ordinal, units;    // the unit's place among those with rows, and their number
  int first, split, splits;
};
__device__ __forceinline__ bool deal_b(const Attn8Args& A, int slot, int lane, DealB& d) {
  const Cache8& C = A.C;
  const int64_t seqs = C.B + (C.cu != nullptr);   // (with the rows past the last sequence)
  uint32_t units = 0, tiles = 0;
  Seq8 s;
  auto take = [&](int64_t b) {
    s = b < seqs ? seq8(C, b) : Seq8{0, 0, 0, 0};
    units = (uint32_t)((rows_b(A, s) + kRowsB - 1) / kRowsB);
    tiles = units ? (uint32_t)unit_of(A, s, (int64_t)(units - 1) * kRowsB).tiles() : 0u;
  };
  uint64_t all = 0;
  d.units = 0;
  for (int64_t b0 = (seqs - 1) & ~(int64_t)63; b0 >= 0; b0 -= 64) {
    take(b0 + lane);
    const uint64_t mine = (uint64_t)units * tiles;
    all += last_lane(upto_lane((uint32_t)mine & 0xffffu)) + ((uint64_t)last_lane(upto_lane((uint32_t)(mine >> 16))) << 16);
    d.units += (int)last_lane(upto_lane(units));
  }
  const uint32_t parts = (uint32_t)max(A.few - d.units, (A.few + 1) / 2);
  uint32_t per = all >> 31 ? (uint32_t)about((int64_t)all, parts) : max(up((uint32_t)all, parts), 4u);
  if (seqs <= 64 && all >> 31 == 0) {   // or less, if that does too
    const uint32_t even = max(up((uint32_t)all, (uint32_t)A.few), 4u), more = per - min(even, per);
#pragma unroll
    for (int k = 3; k >= 0; --k) {
      const uint32_t t = even + (more * k >> 2);
      if (t < per && (int)last_lane(upto_lane(units * max(up(tiles, t), 1u))) <= A.few) per = t;
    }
  }
  int base = 0, before = 0;
  for (int64_t b0 = 0;;) {
    const uint32_t splits = max(up(tiles, per), 1u), mine = units * splits, upto = upto_lane(mine), counts = upto_lane(units);
    const uint64_t past = __ballot(base + (int)upto > slot);
    if (past) {
      const int at = __builtin_ctzll(past);
      d.splits = __builtin_amdgcn_readlane((int)splits, at);
      const int into = slot - base - __builtin_amdgcn_readlane((int)(upto - mine), at), nth = into / d.splits;
      d.split = into - nth * d.splits;
      d.first = slot - d.split;
      d.ordinal = before + __builtin_amdgcn_readlane((int)(counts - units), at) + nth;
      s = Seq8{__builtin_amdgcn_readlane(s.b, at), __builtin_amdgcn_readlane(s.c0, at),
               __builtin_amdgcn_readlane(s.n, at), __builtin_amdgcn_readlane(s.len, at)};
      d.U = unit_of(A, s, (int64_t)nth * kRowsB);
      return true;
    }
    base += (int)last_lane(upto);
    before += (int)last_lane(counts);
    b0 += 64;
    if (b0 >= seqs) return false;
    take(b0 + lane);
  }
}

// The workspace behind the narrow kernel's: partial rows, their sums, how each
// unit was left, and (behind the last that can be) the units' number.
struct LeftB {
  int first, n;     // slots first .. first + n - 1 have parts of its rows (n = 1: written whole),
  int row, rows;    // rows row .. row + rows - 1 of the call
};
__device__ __forceinline__ float* wide_rows(const Attn8Args& A) { return A.part + A.wide_at; }
__device__ __forceinline__ float* wide_sums(const Attn8Args& A) {
  return wide_rows(A) + (int64_t)A.slots * A.C.KVH * kRowsB * kHeadDim;
}
__device__ __forceinline__ LeftB* wide_left(const Attn8Args& A) {
  return reinterpret_cast<LeftB*>(wide_sums(A) + (int64_t)A.slots * A.C.KVH * kRowsB * 2);
}

struct WideLds {
  char k[2][kTileBytesB], v[2][kTileBytesB];
  Meta8 metas[kThreadsB];
  uint2 places[kThreadsB];   // a segment's bytes from the KV head's first, or (y < 0) none
  // e4m3, tiles that not every row sees whole: whether V tile i & 3 has a NaN,
  // and which channels of each token
  uint8_t nan_map[2][kTileB][kHeadDim / 8];
  int nan_seen[4];
};

// Tiles [j0, j1) of unit U.  HALF: at most half of kRowsB rows; the waves are two
// for the rows and each 32 tokens of a tile, joined at the end (32 sequences of up
// to 4000 tokens with 5 new ones each, 40 rows: 74 -> 57 us).
template <int CODE, int E, bool HALF>
__device__ __forceinline__ void wide_tiles(const Attn8Args& A, const Unit8& U, int head, int j0, int j1, WideLds& L8) {
  auto& ks = L8.k;
  auto& vs = L8.v;
  auto& metas = L8.metas;
  auto& places = L8.places;
  auto& nan_seen = L8.nan_seen;
  auto& nan_map = L8.nan_map;
  const Cache8& C = A.C;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, hf = lane >> 5;
  constexpr int kParts = HALF ? 1 : 2;   // of a tile's tokens, 32 each, that a wave takes,
  const int b0 = HALF ? wave >> 1 : 0;   // from this one on
  const bool whole = j1 - j0 == U.tiles();

  const int my_row = 32 * (HALF ? wave & 1 : wave) + n;
  const int my_tok = (U.row0 + my_row) / A.G, my_head = U.row0 + my_row - my_tok * A.G;
  const bool mine = my_row < U.rows;
  const Sight8 sight = sight8(A, U, mine ? U.s.len - U.s.n + my_tok : -1);
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

  const int hi = U.hi, lo = A.window > 0 ? max(from8(A, U.pos0), 0) : 0;
  const int sink = A.window > 0 ? A.sink : 0;
  const char* kbase = C.k + head * C.head_bytes;
  const char* vbase = C.v + head * C.head_bytes;
  // staging: row 16 g + r16, 8 codes from 8 ch
  const int r16 = 4 * wave + (lane >> 4), ch = lane & 15;
  uint32_t off0 = (uint32_t)r16 * C.row_bytes + 8u * ch;
  uint32_t k_at = r16 * kRowB + ((ch ^ r16) << 4), v_at = r16 * kRowB + ((ch ^ ((r16 & 3) << 2)) << 4);
  uint32_t q_at = n * kRowB + ((hf ^ (n & 15)) << 4);   // row n's chunk 2 s + hf is at q_at ^ (s << 5)
  asm volatile("" : "+v"(off0), "+v"(k_at), "+v"(v_at), "+v"(q_at));   // kept, not computed again for each tile

  for (int i0 = j0; i0 < j1; i0 += kChunkB) {
    const int cnt = min(j1 - i0, kChunkB);
    __syncthreads();
    // a thread a segment: its place, for the loads, and then what its tokens weigh by
    const int my_i = threadIdx.x / kSegs;
    const int my_at = kTileB * U.tile(i0 + min(my_i, cnt - 1)) + 16 * (threadIdx.x % kSegs);
    const int my_page = page8(C, entry8(C, U.s.b, my_at, my_i < cnt && my_at < hi));
    {
      const int page = my_page, tok = my_at;
      const uint64_t off = page >= 0 ? (uint64_t)row_offset(C, page, 0, tok) : ~0ull;
      places[threadIdx.x] = uint2{(uint32_t)off, (uint32_t)(off >> 32)};
      if (threadIdx.x < 4) nan_seen[threadIdx.x] = 0;
    }
    __syncthreads();

    u32x2 kc[kSegs], vc[kSegs];   // codes on their way: of the tile after the next
    // (whole segments, also where not every row is seen: no branch, so that the
    // waits for the loads stay exact)
    auto load = [&](int i, int g) {
      const uint2 at = places[kSegs * min(i, kChunkB - 1) + g];
      const uint32_t lo32 = (uint32_t)__builtin_amdgcn_readfirstlane((int)at.x);
      const int hi32 = __builtin_amdgcn_readfirstlane((int)at.y);
      const uint32_t bytes = ((i < cnt) & (hi32 >= 0)) ? 15u * C.row_bytes + kCodeRow : 0u;
      const uint64_t off = ((uint64_t)(uint32_t)max(hi32, 0) << 32) | lo32;
      typedef int v2i __attribute__((ext_vector_type(2)));
      kc[g] = __builtin_bit_cast(u32x2, (v2i)__builtin_amdgcn_raw_buffer_load_b64(make_rsrc(kbase + off, bytes), off0, 0, 0));
      vc[g] = __builtin_bit_cast(u32x2, (v2i)__builtin_amdgcn_raw_buffer_load_b64(make_rsrc(vbase + off, bytes), off0, 0, 0));
    };
    auto mend = [&](int i) {
      const int tok = kTileB * U.tile(i0 + min(i, cnt - 1));
      if (!all_seen(A, U, tok, kTileB)) {
        // V rows that no query row sees count as zeros; a NaN must not meet the
        // weight 0 of a row that does not see it: it is staged as 0 and noted
        uint32_t any = 0;
#pragma unroll
        for (int g = 0; g < kSegs; ++g) {
          const int r = 16 * g + r16, p = tok + r;
          const bool seen = (p < hi) & ((p >= lo) | (p < sink));
          uint32_t bits = 0;
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            vc[g][d] = seen ? vc[g][d] : 0u;
            if (CODE == kE4m3) {
              const uint32_t bad = nan_codes(vc[g][d]) >> 7;   // 0 or 1 a byte
              vc[g][d] &= ~(bad * 0xffu);
              bits |= ((bad * 0x01020408u) >> 24) << (4 * d);
            }
          }
          if (CODE == kE4m3) nan_map[i & 1][r][ch] = (uint8_t)bits;
          any |= bits;
        }
        if (CODE == kE4m3 && __any(any != 0)) nan_seen[i & 3] = 1;
      }
    };
    auto stage_k = [&](int i, int g) {
      *reinterpret_cast<u32x4*>(ks[i & 1] + k_at + 16 * g * kRowB) = widen8<CODE, E>(kc[g]);
    };
    auto stage_v = [&](int i, int g) {
      *reinterpret_cast<u32x4*>(vs[i & 1] + v_at + 16 * g * kRowB) = widen8<CODE, kEltF16>(vc[g]);
    };

#pragma unroll
    for (int g = 0; g < kSegs; ++g) load(0, g);
    metas[threadIdx.x] = meta8(A, my_page, scales8(C, my_page, head, my_at));
    mend(0);
#pragma unroll
    for (int g = 0; g < kSegs; ++g) {
      stage_k(0, g);
      stage_v(0, g);
      load(1, g);
    }
    __syncthreads();
    for (int i = 0; i < cnt; ++i) {
      const int tok = kTileB * U.tile(i0 + i);
      const bool full = all_seen(A, U, tok, kTileB);
      const bool nans = CODE == kE4m3 && !full && nan_seen[i & 3];
      if (CODE == kE4m3 && threadIdx.x == 0) nan_seen[(i + 2) & 3] = 0;
      mend(i + 1);
      // this tile's S = K Q^T, and meanwhile the next one staged (past the last:
      // zeros) and the one behind it loaded
      float16v S[kParts];
      // (ahead of the SIMD's other wave, so that its weights are made under these
      // products: 2048 new tokens over 8192 519 -> 505 us)
      __builtin_amdgcn_s_setprio(1);
      const char* kt = ks[i & 1];
      uint32_t now_at = q_at;
      asm volatile("" : "+v"(now_at));   // (the eight addresses are not kept: their registers are the operands')
      const char* vt = vs[i & 1];
#pragma unroll
      for (int b = 0; b < kParts; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[b][r] = 0.f;
#pragma unroll
      for (int s = 0; s < 8; ++s) {
#pragma unroll
        for (int b = 0; b < kParts; ++b)
          S[b] = mfma32x32x16<E>(*reinterpret_cast<const u32x4*>(kt + 32 * (b0 + b) * kRowB + (now_at ^ (s << 5))), qB[s], S[b]);
        if (s & 1) {
          stage_v(i + 1, s >> 1);
          load(i + 2, s >> 1);
        } else {
          stage_k(i + 1, s >> 1);
        }
      }
      {
        __builtin_amdgcn_s_setprio(0);
        // logits against the running maximum (0 while there is none)
        const float ref = m == -INFINITY ? 0.f : m;
        float inv[2 * kParts], top = -INFINITY;
#pragma unroll
        for (int g = 0; g < 2 * kParts; ++g) {
          const Meta8 mt = metas[kSegs * i + 2 * b0 + g];
          inv[g] = mt.inv;
          const float add = mt.lv - ref;
#pragma unroll
          for (int r = 8 * (g & 1); r < 8 * (g & 1) + 8; ++r) {
            S[g >> 1][r] = __builtin_fmaf(S[g >> 1][r], mt.kf, add);
          }
        }
        if (!full) {
#pragma unroll
          for (int b = 0; b < kParts; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int p = tok + 32 * (b0 + b) + 8 * (r >> 2) + 4 * hf + (r & 3);
              S[b][r] = sight.sees(p) ? S[b][r] : -INFINITY;
            }
        }
#pragma unroll
        for (int b = 0; b < kParts; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, S[b][r]);
        if (__any(top > (m == -INFINITY ? -INFINITY : kHighest))) {
          const float t = half_max(top) - kLift;
          const float now = m == -INFINITY ? t : fmaxf(m, m + t);
          const float to = now == -INFINITY ? 0.f : now;
          const float f = __builtin_amdgcn_exp2f(m - to);   // 0 while there was none
          const float d = ref - to;
#pragma unroll
          for (int b = 0; b < kParts; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) S[b][r] += d;
          l *= f;
#pragma unroll
          for (int cb = 0; cb < 4; ++cb)
#pragma unroll
            for (int r = 0; r < 16; ++r) O[cb][r] *= f;
          m = now;
        }
        // lane (group of 16 lanes, 4j + h): row 4 hf + j, channel 16 (group & 1) + 4 h
        const int j = (lane >> 2) & 3;
        const char* vl = vt + (32 * b0 + 4 * hf + j) * kRowB + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
        // 16 tokens' weights, then their products, under which the next 16's are made
        float part = 0.f;   // a tile's sum, added at once
#pragma unroll
        for (int g = 0; g < 2 * kParts; ++g) {
          half8 h;
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const float w = __builtin_amdgcn_exp2f(S[g >> 1][8 * (g & 1) + r]);
            sum += w;
            h[r] = (_Float16)w;
          }
          part = __builtin_fmaf(sum, inv[g], part);
#pragma unroll
          for (int cb = 0; cb < 4; ++cb) {
            const u32x2 a = lds_read_tr16(vl + 16 * g * kRowB + ((cb ^ j) << 6));
            const u32x2 b = lds_read_tr16(vl + (16 * g + 8) * kRowB + ((cb ^ j) << 6));
            O[cb] = mfma32x32x16<kEltF16>(u32x4{a[0], a[1], b[0], b[1]}, as_u4(h), O[cb]);
          }
        }
        l += part;
        if (nans) {   // and reaches the rows that do
          u32x4 hit = {0u, 0u, 0u, 0u};   // this row's channels
          for (int p = 32 * b0; p < 32 * (b0 + kParts); ++p)
            if (sight.sees(tok + p)) hit |= *reinterpret_cast<const u32x4*>(nan_map[i & 1][p]);
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

  l = half_sum(l);
  if constexpr (HALF) {   // the tokens' halves joined, through what K's tiles were in
    float4v* const parked = reinterpret_cast<float4v*>(&ks[wave & 1][0]) + lane;
    float2v* const sums = reinterpret_cast<float2v*>(&vs[wave & 1][0]) + lane;
    if (b0) {
#pragma unroll
      for (int cb = 0; cb < 4; ++cb)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          parked[64 * (4 * cb + r / 4)] = float4v{O[cb][r], O[cb][r + 1], O[cb][r + 2], O[cb][r + 3]};
      *sums = float2v{m, l};
    }
    __syncthreads();
    if (b0) return;
    const float2v other = *sums;
    const float top = fmaxf(m, other[0]), ref = top == -INFINITY ? 0.f : top;
    const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(other[0] - ref);
    m = top;
    l = __builtin_fmaf(l, f0, other[1] * f1);
#pragma unroll
    for (int cb = 0; cb < 4; ++cb)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const float4v v = parked[64 * (4 * cb + r / 4)];
#pragma unroll
        for (int k = 0; k < 4; ++k) O[cb][r + k] = __builtin_fmaf(O[cb][r + k], f0, v[k] * f1);
      }
  }
  if (!mine) return;
  const int64_t at = whole ? out_row(A, U, head, my_row) : ((int64_t)blockIdx.x * kRowsB + my_row) * kHeadDim;   // (a slot and KV head's)
#pragma unroll
  for (int cb = 0; cb < 4; ++cb)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int64_t c = at + 32 * cb + 2 * r + 4 * hf;
      const float4v v = {O[cb][r], O[cb][r + 1], O[cb][r + 2], O[cb][r + 3]};
      if (whole)
        store_out<E>(A, c, v, l);
      else
        *reinterpret_cast<float4v*>(wide_rows(A) + c) = v;
    }
  if (!whole && hf == 0) {
    *reinterpret_cast<float2v*>(wide_sums(A) + 2 * (at / kHeadDim)) = float2v{m, l};
  }
}

template <int CODE, int E>
__device__ __forceinline__ void wide_part(const Attn8Args& A, uint32_t id, WideLds& L8) {
  const Cache8& C = A.C;
  const int lane = threadIdx.x & 63;
  // KV heads fastest (they go to different XCDs' caches); the last rows of a
  // sequence, which have the most tiles, first
  const int head = (int)(id % (uint32_t)C.KVH);
  id /= (uint32_t)C.KVH;
  Unit8 U;
  int j0 = 0, j1;
  if (A.slots == 0) {
    U = unit_b(A, A.units - 1 - (int64_t)id);
    if (U.rows == 0) return;
    j1 = U.tiles();
  } else {
    DealB d;
    const bool some = deal_b(A, (int)id, lane, d);
    const bool says = head == 0 && threadIdx.x == 0;
    if (says && id == 0) wide_left(A)[A.units].n = d.units;
    if (!some) return;
    U = d.U;
    const int nt = U.tiles(), per = max((nt + d.splits - 1) / d.splits, 1);
    j0 = min(d.split * per, nt);
    j1 = min(j0 + per, nt);
    if (says && d.split == 0 && d.ordinal < A.units)
      wide_left(A)[d.ordinal] = LeftB{d.first, max((nt + per - 1) / per, 1), U.s.c0 * A.G + U.row0, U.rows};
    if (j0 == j1 && d.split > 0) return;
  }
  if (U.rows > kRowsB / 2) {   // (this one first: the other way round its operands are read too late, 6%)
    wide_tiles<CODE, E, false>(A, U, head, j0, j1, L8);
    return;
  }
  wide_tiles<CODE, E, true>(A, U, head, j0, j1, L8);
}

// Joins the parts of the wide kernel's rows, 32 threads a row, eight parts on
// their way.
template <int E>
__device__ __forceinline__ void wide_join(const Attn8Args& A, uint32_t block) {
  const Cache8& C = A.C;
  const uint32_t per = kRowsB / 8 / A.passes;   // workgroups of a unit and KV head
  const uint32_t pair = block / per;
  const int chunk = threadIdx.x & 31, head = (int)(pair % (uint32_t)C.KVH), u = (int)(pair / (uint32_t)C.KVH);
  const int units = wide_left(A)[A.units].n;
  LeftB left = wide_left(A)[u];
  if (u >= units) return;
  // (inside the workspace and the output whatever it holds)
  left.first = min(max(left.first, 0), A.slots - 1);
  left.n = min(left.n, A.slots - left.first);
  left.row = min(max(left.row, 0), (int)C.T * A.G);
  left.rows = min(min(left.rows, kRowsB), (int)C.T * A.G - left.row);
  if (left.n <= 1) return;
  const float2v* sums = reinterpret_cast<const float2v*>(wide_sums(A));
  for (int row = 8 * (int)(block - pair * per) + (int)(threadIdx.x >> 5); row < left.rows; row += 8 * (int)per) {
    const int64_t first = ((int64_t)left.first * C.KVH + head) * kRowsB + row;
    float M = -INFINITY, L = 0.f;
    float4v acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < left.n; s0 += 8) {
      float2v ml[8];
      float4v a[8];
      float top = M;
  #pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t p = first + (int64_t)min(s0 + k, left.n - 1) * C.KVH * kRowsB;
        ml[k] = sums[p];
        a[k] = *reinterpret_cast<const float4v*>(wide_rows(A) + p * kHeadDim + 4 * chunk);
      }
  #pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k][0]);
      const float ref = top == -INFINITY ? 0.f : top;   // (a row that saw nothing yet)
      const float again = __builtin_amdgcn_exp2f(M - ref);
      M = top;
      acc = acc * again;
      L *= again;
  #pragma unroll
      for (int k = 0; k < 8; ++k)
        if (s0 + k < left.n) {
          const float f = __builtin_amdgcn_exp2f(ml[k][0] - ref);
          acc += a[k] * f;
          L = __builtin_fmaf(ml[k][1], f, L);
        }
    }
    const int r = left.row + row, tok = r / A.G;
    store_out<E>(A, ((int64_t)tok * A.H + head * A.G + (r - tok * A.G)) * kHeadDim + 4 * chunk, acc, L);
  }
}

// ---- launches ----
//
// A call is two launches: the attention of its narrow sequences, of its wide ones
// or of both at once (the wide ones' workgroups first, which have the most to do),
// and the join of what was left in parts.

template <int CODE, int E>
__global__ __launch_bounds__(kThreadsA, 2) void narrow8_kernel(Attn8Args A) {
  __shared__ __align__(16) NarrowLds lds;
  narrow_part<CODE, E>(A, (int)blockIdx.x, lds);
}

template <int CODE, int E>
__global__ __launch_bounds__(kThreadsB, 2) void wide8_kernel(Attn8Args A) {
  __shared__ __align__(16) WideLds lds;
  wide_part<CODE, E>(A, blockIdx.x, lds);
}

template <int CODE, int E>
__global__ __launch_bounds__(kThreadsB, 2) void both8_kernel(Attn8Args A) {
  __shared__ __align__(16) union {
    NarrowLds narrow;
    WideLds wide;
  } lds;
  const uint32_t wide = gridDim.x - A.groups;
  if (blockIdx.x < wide)
    wide_part<CODE, E>(A, blockIdx.x, lds.wide);
  else
    narrow_part<CODE, E>(A, (int)(blockIdx.x - wide), lds.narrow);
}

template <int E, bool MANY>
__global__ __launch_bounds__(256) void join8_kernel(Attn8Args A) {
  if (blockIdx.x < A.wide_blocks)
    wide_join<E>(A, blockIdx.x);
  else
    narrow_join<E, MANY>(A, blockIdx.x - A.wide_blocks);
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
int narrow_groups(int64_t B, int32_t KVH, int32_t G, int64_t max_len) {
  if (G > kRowsA) return 0;
  const int64_t tiles = B * KVH * ((max_len + kTile - 1) / kTile);
  int groups = 1;
  while (groups < kGroupsA && (int64_t)groups * kWavesA < tiles) groups *= 2;
  return groups;
}
size_t narrow_bytes(int groups, int side, int64_t heads) {
  return groups ? (size_t)part_rows(groups, side) * (kHeadDim + 2) * sizeof(float) + (size_t)heads * sizeof(Left8) : 0;
}
// KV heads that a workgroup reads side by side.
int narrow_side(int32_t KVH) { return KVH % 4 == 0 ? 4 : KVH % 2 == 0 ? 2 : 1; }

constexpr int kManyPairs = 64;   // from here on the pairs' parts are few (eight or so)

// Wide kernel: units of a call (with those of the rows past the last sequence),
// and slots a KV head where the units do not fill the GPU (no part is of less
// than 4 tiles).
int64_t wide_units(bool offsets, int64_t B, int64_t T, int32_t G) {
  if (!offsets) return G > kRowsA ? B * ((G + kRowsB - 1) / kRowsB) : 0;
  return T * G / kRowsB + B + 1;
}
int wide_slots(int64_t units, int32_t KVH, int64_t max_len) {
  const int64_t tiles = (max_len + kTileB - 1) / kTileB;
  if (units * KVH >= kPairsB || tiles <= 4) return 0;
  return (int)std::min(kPairsB / KVH + units, units * ((tiles + 3) / 4));
}
size_t wide_bytes(int64_t units, int32_t KVH, int slots) {
  return slots == 0 ? 0 : (size_t)slots * KVH * kRowsB * (kHeadDim + 2) * sizeof(float) + (size_t)(units + 1) * sizeof(LeftB);
}

size_t attn_bytes(bool offsets, int64_t B, int64_t T, int32_t G, int32_t KVH, int64_t max_len) {
  const int64_t units = wide_units(offsets, B, T, G);
  return narrow_bytes(narrow_groups(B, KVH, G, max_len), narrow_side(KVH), B * KVH) +
         wide_bytes(units, KVH, wide_slots(units, KVH, max_len));
}

template <int CODE, int E>
int launch_attn8(Attn8Args A, hipStream_t stream) {
  const unsigned wide = (unsigned)((A.slots ? A.slots : A.units) * A.C.KVH);
  if (A.groups == 0)
    wide8_kernel<CODE, E><<<dim3(wide), dim3(kThreadsB), 0, stream>>>(A);
  else if (wide == 0)
    narrow8_kernel<CODE, E><<<dim3((unsigned)A.groups), dim3(kThreadsA), 0, stream>>>(A);
  else
    both8_kernel<CODE, E><<<dim3(wide + A.groups), dim3(kThreadsB), 0, stream>>>(A);
  const int rc = launch_status();
  if (rc) return rc;
  A.passes = 1;
  while (A.passes < kRowsB / 8 && A.units * A.C.KVH * (kRowsB / 8) / A.passes > kJoinsB) A.passes *= 2;
  A.wide_blocks = A.slots ? (unsigned)(A.units * A.C.KVH * (kRowsB / 8) / A.passes) : 0;
  const int64_t heads = A.groups ? A.C.B * A.C.KVH : 0;
  if (heads / A.side >= kManyPairs)
    join8_kernel<E, true><<<dim3(A.wide_blocks + (unsigned)heads), dim3(256), 0, stream>>>(A);
  else if (A.wide_blocks + heads > 0)
    join8_kernel<E, false><<<dim3(A.wide_blocks + (unsigned)(heads * kRowsA)), dim3(256), 0, stream>>>(A);
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
  const size_t one_each = T == B ? attn_bytes(false, B, T, H / KVH, KVH, max_len) : 0;
  return std::max({attn_bytes(true, B, T, H / KVH, KVH, max_len), one_each, (size_t)16});   // (0 is a refusal)
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
  A.groups = narrow_groups(B, A.C.KVH, A.G, A.C.max_len);
  A.side = narrow_side(A.C.KVH);
  A.pairs = A.C.KVH / A.side;
  A.inv_g = (uint32_t)((65536 + A.G - 1) / A.G);
  A.units = wide_units(offsets, B, T, A.G);
  A.slots = wide_slots(A.units, A.C.KVH, A.C.max_len);
  A.few = kPairsB / A.C.KVH;
  if (B * A.C.KVH * kRowsA + A.units * A.C.KVH + 16 * kPairsB + A.groups > 0x7fffffff)
    return KVDEC_E_SHAPE;
  if (!ws || !on16(ws) || ws_bytes < attn_bytes(offsets, B, T, A.G, A.C.KVH, A.C.max_len)) return KVDEC_E_WORKSPACE;
  A.q = q;
  A.o = o;
  A.part = static_cast<float*>(ws);
  A.wide_at = (int64_t)(narrow_bytes(A.groups, narrow_side(A.C.KVH), B * A.C.KVH) / sizeof(float));
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
