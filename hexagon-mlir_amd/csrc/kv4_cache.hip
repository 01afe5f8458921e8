// Rows of keys and values into the 4-bit cache (kv4_append) and back (kv4_read);
// numbers and layout: kv4.h.
#include "hxmi_common.h"
#include "hxmi_internal.h"
#include "kv4.h"

namespace hxmi {
namespace {

using namespace kv4;

typedef uint32_t uint1u __attribute__((aligned(2)));  // (rows start anywhere)

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

// A wave writes one run (up to 16 rows of the call that go to consecutive slots
// of one piece of 16 tokens) of one head of K or V, two dims a lane: 16 lanes'
// largest magnitude gives a scale, and nothing that is in the cache already
// changes.  A run is found by its first row: the row before it does not go to
// the slot before, or to another piece.
template <typename T>
__global__ __launch_bounds__(256) void kv4_append(CArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int hv = (int)(item % (2 * a.heads)), h = hv >> 1, is_v = hv & 1;
  const int64_t t0 = item / (2 * a.heads) * a.span;  // (a.span <= 48: a run that begins there ends within 64 rows)
  int64_t slot_l = -1;
  bool begins = false;
  if (t0 + lane < a.tokens) {
    slot_l = a.slots[t0 + lane];
    const int64_t before = t0 + lane > 0 ? a.slots[t0 + lane - 1] : -1;
    begins = slot_l >= 0 && slot_l < a.cells && ((slot_l & 15) == 0 || before != slot_l - 1);
  }
  const bool mine = 2 * lane < a.dp, filled = 2 * lane < a.d;
  for (uint64_t runs = __ballot(begins && lane < a.span); runs; runs &= runs - 1) {
    const int l = __ffsll((unsigned long long)runs) - 1;
    const int64_t slot = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)slot_l, l) |
                         (int64_t)__builtin_amdgcn_readlane((int)(slot_l >> 32), l) << 32;
    const int off = (int)(slot & 15);
    const uint64_t miss = ~(__ballot(lane >= l && slot_l == slot + (lane - l)) >> l);  // (lane l's own bit is 0)
    const int n = min(16 - off, miss ? __ffsll((unsigned long long)miss) - 1 : 64);
    const T* const x = (const T*)a.x[is_v] + (t0 + l) * a.ld[is_v] + h * a.hs[is_v] + 2 * lane;
    const int64_t ld = a.ld[is_v], at = slot & ((1 << a.lb) - 1), cell = (slot >> a.lb) * a.heads + h;

    uint32_t raw[16], byte[16], sb = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      raw[i] = 0;
      if (i < n && filled) raw[i] = *(const uint1u*)(x + i * ld);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      byte[i] = 0;
      if (i >= n) continue;  // (uniform)
      T two[2];
      __builtin_memcpy(two, &raw[i], 4);
      const float x0 = held((float)two[0]), x1 = held((float)two[1]);
      const float most = wave_reduce_dpp<16>(fmaxf(fabsf(x0), fabsf(x1)), [](float p, float q) { return fmaxf(p, q); });
      const uint32_t b = scale_byte(most);
      const float inv = b ? 1.f / scale_value(b) : 0.f;
      byte[i] = (uint32_t)__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, quotient(x0, inv), quotient(x1, inv), 1.f, 0) & 0xffu;
      sb = (lane & 15) == i ? b : sb;
    }
    // scales: lane 16 g + i has row i's of group g
    if (mine && (lane & 15) < n) a.scale[is_v][(((cell * (a.dp >> 5) + (lane >> 4)) << a.lb) + at) + (lane & 15)] = (uint8_t)sb;
    if (!is_v) {
      uint8_t* const dst = a.codes[0] + ((cell << a.lb) + at) * (a.dp >> 1) + lane;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < n && mine) dst[i * (a.dp >> 1)] = (uint8_t)byte[i];
    } else if (mine) {
      // row i is token off + i of the piece: two dims' sixteen halves of bytes
      uint64_t d0 = 0, d1 = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        d0 |= (uint64_t)(byte[i] & 15) << (4 * i);
        d1 |= (uint64_t)(byte[i] >> 4) << (4 * i);
      }
      uint64_t* const dst = (uint64_t*)(a.codes[1] + (((cell << (a.lb - 4)) + (at >> 4)) * a.dp + 2 * lane) * 8);
      const uint64_t mask = (n == 16 ? ~0ull : (1ull << (4 * n)) - 1) << (4 * off);
      d0 <<= 4 * off;
      d1 <<= 4 * off;
      if (n < 16) {
        d0 |= dst[0] & ~mask;
        d1 |= dst[1] & ~mask;
      }
      dst[0] = d0;
      dst[1] = d1;
    }
  }
}

// ---- kv4_read --------------------------------------------------------------------

// Outputs [tokens, heads, d], zeros for a slot outside the cache.  A wave takes 16
// rows of a head of K or of V, two dims a lane, piece of 16 tokens by piece: those
// of a piece take their V numbers from one 16-byte load a lane.
template <typename T>
__global__ __launch_bounds__(256) void kv4_read(CArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int hv = (int)(item % (2 * a.heads)), h = hv >> 1, is_v = hv & 1;
  const int64_t t0 = item / (2 * a.heads) * 16;
  const bool mine = 2 * lane < a.d;
  char* const out = a.out[is_v] + ((t0 * a.heads + h) * a.d + 2 * lane) * 2;
  const int64_t step = (int64_t)a.heads * a.d * 2;
  int64_t slot = -1;
  const bool row = lane < 16 && t0 + lane < a.tokens;
  if (row) slot = a.slots[t0 + lane];
  const bool in = row && slot >= 0 && slot < a.cells;
  for (uint64_t left = __ballot(row && !in); left; left &= left - 1)
    if (mine) *(uint32_t*)(out + (__ffsll((unsigned long long)left) - 1) * step) = 0;
  for (uint64_t left = __ballot(in); left;) {
    // the rows whose tokens are in the first one's piece
    const int u0 = __ffsll((unsigned long long)left) - 1;
    const int64_t piece = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(slot >> 4), u0) |
                          (int64_t)__builtin_amdgcn_readlane((int)(slot >> 36), u0) << 32;
    const uint32_t rows = (uint32_t)__ballot(in && slot >> 4 == piece);
    left &= ~(uint64_t)rows;
    const int lp = a.lb - 4;
    const int64_t cell = (piece >> lp) * a.heads + h, at = (piece & ((1 << lp) - 1)) * 16;
    const int off = (int)slot & 15;  // (lane u: row u's token)
    if (!mine) continue;
    const uint8_t* const sc = a.scale[is_v] + (((cell * (a.dp >> 5) + (lane >> 4)) << a.lb) + at);
    uint64_t d0 = 0, d1 = 0;
    const uint8_t* const kc = a.codes[0] + ((cell << a.lb) + at) * (a.dp >> 1) + lane;
    if (is_v) {
      const uint64_t* const vc = (const uint64_t*)(a.codes[1] + ((cell << lp) * a.dp + (at >> 4) * a.dp + 2 * lane) * 8);
      d0 = vc[0];
      d1 = vc[1];
    }
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      if (!(rows >> u & 1)) continue;
      const int o = __builtin_amdgcn_readlane(off, u);
      const uint32_t byte = is_v ? (uint32_t)(d0 >> (4 * o) & 15) | (uint32_t)(d1 >> (4 * o) & 15) << 4 : kc[o * (a.dp >> 1)];
      const half2v v = numbers<0>(byte) * scale_twice<0>(sc[o]);
      const T f[2] = {(T)(float)v[0], (T)(float)v[1]};
      uint32_t bits;
      __builtin_memcpy(&bits, f, 4);
      *(uint32_t*)(out + u * step) = bits;
    }
  }
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
  const int64_t per_row = 2 * p.kv_heads;
  const int64_t span = p.tokens * per_row / 8192;
  a.span = (int)(span < 1 ? 1 : span < 48 ? span : 48);
  const int64_t blocks = ((p.tokens + a.span - 1) / a.span * per_row + 3) / 4;
  if (blocks >= (1ll << 31)) return hipErrorInvalidValue;
  const auto fn = p.dtype == DT_BF16 ? kv4_append<__bf16> : kv4_append<_Float16>;
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4CacheProblem& p, hipStream_t stream) {
  CArgs a = cache_args(p);
  a.out[0] = (char*)p.k_out;
  a.out[1] = (char*)p.v_out;
  const int64_t blocks = ((p.tokens + 15) / 16 * 2 * p.kv_heads + 3) / 4;
  if (blocks >= (1ll << 31)) return hipErrorInvalidValue;
  const auto fn = p.dtype == DT_BF16 ? kv4_read<__bf16> : kv4_read<_Float16>;
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace hxmi
