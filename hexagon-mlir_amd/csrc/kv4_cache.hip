// Rows of keys and values into the 4-bit cache (kv4_append) and back (kv4_read);
// numbers and layout: kv4.h.
#include "hxmi_common.h"
#include "hxmi_internal.h"
#include "kv4.h"

namespace hxmi {
namespace {

using namespace kv4;

typedef uint32_t uint1u __attribute__((aligned(2)));  // (rows start anywhere)
typedef int int4u __attribute__((ext_vector_type(4), aligned(2)));

struct CArgs {
  const char* x[2];  // rows of k and of v
  uint8_t* codes[2];
  uint8_t* scale[2];
  const int64_t* slots;
  char* out[2];          // kv4_read
  int64_t ld[2], hs[2];  // row and head strides of x, elements
  int64_t tokens, cells;  // cells: blocks * block size
  int heads, d, dp, lb, span;
};

// ---- kv4_append ------------------------------------------------------------------

// The scale's byte: the smallest one that holds `most` (up to kMost) as six of it.
__device__ __forceinline__ uint32_t scale_byte(float most) {
  const float t = most * 0.16666667f;  // (off by an ulp or two: a byte's step is 2^20 of them)
  const uint32_t normal = (__float_as_uint(t) >> 20) - ((127 - 15) << 3);
  uint32_t b = t < 0x1p-14f ? (uint32_t)(t * 0x1p17f) : normal;  // rounded down
  b = b > 0 ? b - 1 : 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) b += 6.f * scale_value(b) < most;  // (exact: a scale has four bits)
  return b;
}
// x / scale to 16 significant bits (inv: 1 / scale, 0 of 0).  Of a quotient of a 16-bit
// value by a scale, one that is not a border of two numbers is 2^-11 from it, so
// neither the quotient's own error (2^-22) nor this rounding moves it over or onto
// one, and a border itself has four bits: it comes out exact, for the conversion to
// take to the even number.
__device__ __forceinline__ float quotient(float x, float inv) {
  return __uint_as_float((__float_as_uint(x * inv) + 0x80u) & ~0xffu);
}
// What is held for x: infinities and NaN as the largest value.
__device__ __forceinline__ float held(float x) { return x != x ? kMost : fminf(fmaxf(x, -kMost), kMost); }

template <int CTRL, int BANKS = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t old, uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, 0xf, BANKS, false);
}
// Eight lanes l % 8 hold a row of eight 4-bit numbers each: lane j's become the
// numbers j of all of them, lane 0's first.  Halves, quarters and eighths of the words in turn
// go to the lane 4, 2 and 1 away.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t o = dpp<0x104, 0x5>(0, v);  // row_shl:4, for lanes without bit 2
  o = dpp<0x114, 0xa>(o, v);           // row_shr:4, for the others
  v = threadIdx.x & 4 ? __builtin_amdgcn_perm(v, o, 0x07060302u) : __builtin_amdgcn_perm(o, v, 0x05040100u);
  o = dpp<0x4e>(0, v);  // lane l ^ 2
  v = threadIdx.x & 2 ? __builtin_amdgcn_perm(v, o, 0x07030501u) : __builtin_amdgcn_perm(o, v, 0x06020400u);
  o = dpp<0xb1>(0, v);  // lane l ^ 1
  return threadIdx.x & 1 ? (v & 0xf0f0f0f0u) | (o >> 4 & 0x0f0f0f0fu) : (v & 0x0f0f0f0fu) | (o << 4 & 0xf0f0f0f0u);
}

// A wave writes one run (up to 16 rows of the call that go to consecutive slots
// of one piece of 16 tokens) of one head of K or V.  A run is found by its first
// row: the row before it does not go to the slot before, or to another piece.  Lane l takes
// token l % 8 of half a piece and eight dims of 64, so four lanes (l, l + 8, l +
// 16, l + 24) have a scale in common; K's eight numbers are a word of the
// cache, V's become one by an exchange between the eight tokens' lanes.  Nothing that
// is in the cache already changes.
// The code is kept short: a wave meets it cold, and with a run's rows unrolled (two
// dims a lane, 1900 instructions) fetching them cost more than all loads and
// stores: 8900 rows of 4 x 64 17.7 us, 7.5 now.  One row each of 128 requests, 8 x 128,
// takes 5 us: slot, row, and V's word there and back.
template <typename T>
__global__ __launch_bounds__(256) void kv4_append(CArgs a) {
  const int lane = threadIdx.x & 63;
  // item: rows, head, 64 dims, K or V
  const uint32_t item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wide = a.dp > 64;
  const uint32_t parts = 2u * a.heads << wide, group = item / parts, part = item - group * parts;
  const int is_v = part & 1, h = (int)(part >> (1 + wide)), d = (lane & ~7) + (part >> 1 & wide) * 64, token = lane & 7;
  const int64_t t0 = (int64_t)group * a.span;  // (a.span <= 48: a run that begins there ends within 64 rows)
  int64_t slot_l = -1;
  bool begins = false;
  if (t0 + lane < a.tokens) {
    slot_l = a.slots[t0 + lane];
    const int64_t before = t0 + lane > 0 ? a.slots[t0 + lane - 1] : -1;
    begins = slot_l >= 0 && slot_l < a.cells && ((slot_l & 15) == 0 || before != slot_l - 1);
  }
  const int64_t ld = a.ld[is_v];
  const bool mine = d < a.dp;
#pragma unroll 1
  for (uint64_t runs = __ballot(begins && lane < a.span); runs; runs &= runs - 1) {
    const int l = __ffsll((unsigned long long)runs) - 1;
    const int64_t slot = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)slot_l, l) |
                         (int64_t)__builtin_amdgcn_readlane((int)(slot_l >> 32), l) << 32;
    const int off = (int)(slot & 15);
    const uint64_t miss = ~(__ballot(lane >= l && slot_l == slot + (lane - l)) >> l);  // (lane l's own bit is 0)
    const int n = min(16 - off, miss ? __ffsll((unsigned long long)miss) - 1 : 64);
    const int64_t at = (slot & ((1 << a.lb) - 1)) - off, cell = (slot >> a.lb) * a.heads + h;  // the piece
    // (token i of the piece is row i - off of the run)
    const T* const x = (const T*)a.x[is_v] + (t0 + l - off + token) * ld + h * a.hs[is_v] + d;
    uint8_t* const scale = a.scale[is_v] + (((cell * (a.dp >> 5) + (d >> 5)) << a.lb) + at) + token;
    uint8_t* const keys = a.codes[0] + ((cell << a.lb) + at + token) * (a.dp >> 1) + (d >> 1);
    const uint32_t held_by = (uint32_t)(0xffff >> (16 - n) << off);  // a bit a token
    int4v raw[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      raw[i] = int4v{};
      if (d < a.d && held_by >> (8 * i + token) & 1) raw[i] = *(const int4u*)(x + 8 * i * ld);
    }
    uint64_t both = 0;
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      if (!(held_by >> (8 * i) & 0xff)) continue;
      const int4v r = i ? raw[1] : raw[0];
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t b = (uint32_t)r[e] & 0x7fff7fffu;
        top = max(top, max(b & 0xffffu, b >> 16));
      }
      top = max(top, dpp<0x128>(0, top));  // row_ror:8
      const auto r16 = __builtin_amdgcn_permlane16_swap(top, top, false, false);
      top = max((uint32_t)r16[0], (uint32_t)r16[1]);
      const float amax = (float)__builtin_bit_cast(T, (unsigned short)top);
      const bool past = !(amax <= kMost);  // (or no number)
      const uint32_t sb = scale_byte(past ? kMost : amax);
      const float inv = sb ? __builtin_amdgcn_rcpf(scale_value(sb)) : 0.f;
      T f[8];
      __builtin_memcpy(f, &r, 16);
      float q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = (float)f[e];
      if (__any(past)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = held(q[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = quotient(q[e], inv);
      uint32_t word = 0;
      static_for<4>([&](auto e) {
        word = (uint32_t)__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, q[2 * e], q[2 * e + 1], 1.f, e);
      });
      const bool in = mine && held_by >> (8 * i + token) & 1;
      if (in && (lane & 24) == 0) scale[8 * i] = (uint8_t)sb;
      if (!is_v) {
        if (in) *(uint32_t*)(keys + 8 * i * (a.dp >> 1)) = word;
      } else {
        both |= (uint64_t)transpose8(word) << (32 * i);
      }
    }
    if (is_v && mine) {
      // this lane's dim is d + token: sixteen tokens
      const uint64_t mask = (n == 16 ? ~0ull : (1ull << (4 * n)) - 1) << (4 * off);
      uint64_t* const dst = (uint64_t*)(a.codes[1] + (((cell << (a.lb - 4)) + (at >> 4)) * a.dp + d + token) * 8);
      both &= mask;
      // (other runs may write other tokens of the piece meanwhile)
      if (n < 16) __hip_atomic_fetch_xor(dst, both ^ (*dst & mask), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      else *dst = both;
    }
  }
}

// ---- kv4_read --------------------------------------------------------------------

// Outputs [tokens, heads, d], zeros for a slot outside the cache.  A lane takes eight
// dims of a row: of K four bytes, of V their piece's 64 bytes (the other rows of the
// piece take the same ones out of the cache next to the CU), a number of each eight.
// 2^log lanes a row; one row a lane: two or four in flight were slower (4336 rows
// of 8 x 128, 18 MB of results: 8.8 us, 9.4 and 11.0).
template <typename T>
__global__ __launch_bounds__(256) void kv4_read(CArgs a, int log) {
  const int lane = threadIdx.x & 63;
  const uint32_t item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), parts = 2u * a.heads;
  const uint32_t group = item / parts, hv = item - group * parts;
  const int h = (int)(hv >> 1), is_v = hv & 1, d = (lane & ((1 << log) - 1)) * 8;
  const int64_t t = ((int64_t)group << (6 - log)) + (lane >> log);
  if (d >= a.d || t >= a.tokens) return;
  const int64_t slot = a.slots[t];
  T f[8] = {};
  if (slot >= 0 && slot < a.cells) {
    const int64_t cell = (slot >> a.lb) * a.heads + h, at = slot & ((1 << a.lb) - 1);
    const uint32_t sb = a.scale[is_v][((cell * (a.dp >> 5) + (d >> 5)) << a.lb) + at];
    uint32_t word = 0;
    if (!is_v) {
      word = *(const uint32_t*)(a.codes[0] + ((cell << a.lb) + at) * (a.dp >> 1) + (d >> 1));
    } else {
      const int4v* const p = (const int4v*)(a.codes[1] + (((cell << (a.lb - 4)) + (at >> 4)) * a.dp + d) * 8);
      const int o = 4 * ((int)at & 7);
      const bool hi = at & 8;
      int4v v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = p[j];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = (uint32_t)(hi ? v[j][1] : v[j][0]) >> o & 15, y = (uint32_t)(hi ? v[j][3] : v[j][2]) >> o & 15;
        word |= (x | y << 4) << (8 * j);
      }
    }
    const half2v s = scale_twice<0>(sb);
    static_for<4>([&](auto j) {
      const half2v v = numbers<j>(word) * s;
      f[2 * j] = (T)(float)v[0];
      f[2 * j + 1] = (T)(float)v[1];
    });
  }
  int4v bits;
  __builtin_memcpy(&bits, f, 16);
  *(int4u*)((T*)a.out[is_v] + (t * a.heads + h) * a.d + d) = bits;
}

CArgs cache_args(const Kv4CacheProblem& p) {
  CArgs a{};
  a.codes[0] = p.k_codes;
  a.codes[1] = p.v_codes;
  a.scale[0] = p.k_scale;
  a.scale[1] = p.v_scale;
  a.slots = p.slots;
  a.tokens = p.tokens;
  a.cells = p.blocks << p.log2_block;
  a.heads = (int)p.kv_heads;
  a.d = (int)p.d;
  a.dp = (int)((p.d + 31) / 32 * 32);
  a.lb = p.log2_block;
  return a;
}

}  // namespace

hipError_t launch_kv4_append(const Kv4CacheProblem& p, hipStream_t stream) {
  CArgs a = cache_args(p);
  a.x[0] = (const char*)p.k;
  a.x[1] = (const char*)p.v;
  a.ld[0] = p.ldk;
  a.ld[1] = p.ldv;
  a.hs[0] = p.hsk;
  a.hs[1] = p.hsv;
  // a wave looks for runs in `span` rows: one while that leaves at most 8192
  // waves, more for long prompts, whose rows mostly begin none
  const int64_t per_row = p.d > 64 ? 4 * p.kv_heads : 2 * p.kv_heads;
  const int64_t span = p.tokens * per_row / 8192;
  a.span = (int)(span < 1 ? 1 : span < 48 ? span : 48);
  const int64_t blocks = ((p.tokens + a.span - 1) / a.span * per_row + 3) / 4;
  if (blocks >= (1ll << 30)) return hipErrorInvalidValue;
  const auto fn = p.dtype == DT_BF16 ? kv4_append<__bf16> : kv4_append<_Float16>;
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4CacheProblem& p, hipStream_t stream) {
  CArgs a = cache_args(p);
  a.out[0] = (char*)p.k_out;
  a.out[1] = (char*)p.v_out;
  int log = 0;
  while (8 << log < p.d) ++log;
  const int64_t per = 64 >> log, blocks = ((p.tokens + per - 1) / per * 2 * p.kv_heads + 3) / 4;
  if (blocks >= (1ll << 30)) return hipErrorInvalidValue;
  const auto fn = p.dtype == DT_BF16 ? kv4_read<__bf16> : kv4_read<_Float16>;
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), 0, stream, a, log);
  return hipGetLastError();
}

}  // namespace hxmi
