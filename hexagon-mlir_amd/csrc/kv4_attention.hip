// Attention over the 4-bit key/value cache (numbers and layout: kv4.h), causal over
// ragged requests, grouped heads: row i of a request with n rows and L tokens
// in the cache sees keys j <= L - n + i,
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - max).
//
// A workgroup of four waves owns a tile of 16 rows (token, head of the group) of
// one key/value head and, where there are few such tiles, one of `nsplit`
// shares of the keys.  The waves take every fourth group of 64 keys; numbers go
// from memory straight to registers, and what the cache holds is exact in fp16
// (number * scale, two instructions for two values), so both products take it
// as it is:
//   * scores as D[key][row] = K . Q^T (16x16x32 MFMAs).  The dims of a step may
//     come in any order, so a lane takes 16 (of 64) or 32 (of 128) dims of a key
//     that lie together, under one scale.  Row m of tile t is key 16 (m / 4) + 4 t +
//     m % 4 of the group (four keys in a row an access), and a lane's 16 scores
//     (row l % 16, g = l / 16) are keys 16 g .. 16 g + 15 in order, one page's;
//   * those 16 weights are the B operand of P.V as they are.  A lane's V numbers
//     are two dims of those 16 tokens, tiles 2 c and 2 c + 1 of 32 dims (row m is
//     dim 2 m or 2 m + 1), so that a lane ends with eight dims that lie together;
//   * q in bf16 is brought to fp16 under a power of two a row: multiples of 2^-38
//     of its largest element;
//   * weights are relative to 2^m, m from 7 to 15 below the running maximum, in
//     11 bits or multiples of 2^-31 of the row's largest (fp16 below 2^-14);
//     scores, maxima, sums and O are fp32.  Scales that are part of V and K, and
//     not of the weights, keep that one maximum valid whatever they are.
// One token a request: 64 requests of 4096 to 8192 tokens, 32 heads over 8 of 128
// dims, 94-100 us (422 MB at 4.2-4.5 TB/s; a copy reaches 4.98).  It is bound by the vector
// ALUs as much as by memory: 500 instructions a wave and group, 256 of them the
// conversion; with every V number from one block (half the bytes) it is only 10 %
// faster.  Two groups in flight a wave, non-temporal loads, three shares a
// tile and equal shares of fewer keys were no faster.  One token of 131072 keys 41 us, 1900
// tokens of one user 7.1-7.5 (latency; launch, two rounds of loads, joins).
#include "kv4.h"
#include "kv_attention_impl.h"

namespace hxmi {
namespace {

using namespace kv4;

struct KArgs : TileArgs {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t sbytes;  // of a block's scales of one head
};

// Weights are 2^(score - m): m stays until a score is more than kHigh above it,
// then follows to kLow below the largest.
constexpr float kLow = 7.f, kHigh = 15.f;
// From this magnitude of m on, a score's product with c is rounded before m is
// subtracted: what fp32 leaves of m is steps of 1/8 and more, and the unrounded
// product's distance from it would be a factor on the weights, 2^4096 at scores of 2^36.
constexpr float kFar = 0x1p20f;
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) >= kFar && m != -INFINITY; }

// a * b, rounded (never part of an fma).
__device__ __forceinline__ float times(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// What the products of K and a row of q (times 2^ex) are to be multiplied by.  They are
// below 2^40 and, where not 0, above 2^-45: from 2^-126 down they are all alike, and
// from 2^80 up any two lie further apart than weights reach, so that c can stop there. In
// between it is neither 0 nor infinite, and a masked key's -inf stays one, 0 stays 0.
__device__ __forceinline__ float score_scale(float c, int ex) {
  return fminf(fmaxf(__builtin_ldexpf(c, -ex), 0x1p-126f), 0x1p80f);
}

// Eight numbers times their scales (pairs) as one MFMA operand.
template <typename F>
__device__ __forceinline__ half8v operand(uint32_t w, F&& scale) {
  const half2v a = numbers<0>(w) * scale(0), b = numbers<1>(w) * scale(1), c = numbers<2>(w) * scale(2),
               d = numbers<3>(w) * scale(3);
  return half8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// l + the sum of eight weights, as P.V takes them (two an instruction), those below
// fp16's normal range with the bits that they keep there.
__device__ __forceinline__ float sum_of(const half8v& p, float l) {
  const half2v one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
  for (int e = 0; e < 8; e += 2) l = __builtin_amdgcn_fdot2(half2v{p[e], p[e + 1]}, one, l, false);
  return l;
}
// Scales of eight values in a row (words w0 and w1), pair by pair.
struct Pairs {
  half2v p[4];
  __device__ __forceinline__ Pairs(uint32_t w0, uint32_t w1)
      : p{scale_pair<0>(w0), scale_pair<1>(w0), scale_pair<0>(w1), scale_pair<1>(w1)} {}
};
// Bytes of word x (of four) that belong to the first n of 16.
__device__ __forceinline__ uint32_t first_bytes(int n, int x) {
  const int c = min(max(n - 4 * x, 0), 4);
  return c == 4 ? ~0u : (1u << (8 * c)) - 1;
}

// Bytes of a word of scales past the largest, as 255: fp16 holds no six of them, or
// not even one, so a product may be infinite (kv4_append writes none).
__device__ __forceinline__ uint32_t past_largest(uint32_t w) {
  // the byte's upper bit set, and its lower seven at least 99: that and 29 reach the upper bit
  const uint32_t b = ((w & 0x7f7f7f7fu) + (0x7f - (kMostScale & 0x7f)) * 0x01010101u) & w & 0x80808080u;
  return (b >> 7) * 255u;
}

// What a wave knows of its 16 rows: O and the sum of the weights (this lane's part).
template <int DT>
struct Partial {
  static constexpr int N = DT * 4 + 2;  // floats a lane
  float4v o[DT];
  float m, l;

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = float4v{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }
  // Every float becomes f(its index, it).
  template <typename F>
  __device__ __forceinline__ void each(F&& f) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[t][i] = f(t * 4 + i, o[t][i]);
    m = f(DT * 4, m);
    l = f(DT * 4 + 1, l);
  }
  template <int M>
  __device__ __forceinline__ void add(const Partial (&p)[M]) {
    float top = m;
#pragma unroll
    for (int j = 0; j < M; ++j) top = fmaxf(top, p[j].m);
    const float f = rel_exp2(m, top);
    m = top;
    l *= f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] *= f;
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const float g = rel_exp2(p[j].m, top);
      l += p[j].l * g;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] += p[j].o[t][i] * g;
    }
  }
};

// DC: 64-dim pieces of a row; WHOLE: the head dim is 64 * DC.
template <typename T, int DC, bool WHOLE>
__global__ __launch_bounds__(256, 2) void kv4_attention(KArgs a) {
  constexpr int DT = DC * 4, G = DC * 2, RT = 16, NV = Partial<DT>::N, KD = 16 * DC;  // KD: dims of a lane's keys
  constexpr bool BF16 = !std::is_same_v<T, _Float16>;
  __shared__ __attribute__((aligned(16))) float joined[3 * NV * 64];
  __shared__ int last_split;

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lg = lane >> 4;

  const Share part = share_of(a);
  const int split = part.split, nsplit = part.count, item = part.item;
  const int kvh = item / a.tiles;
  Rows tile;
  if (!rows_of<RT>(a, item - kvh * a.tiles, tile)) return;
  const int r = tile.r, first = tile.first, n = tile.n, row0 = tile.row0, len = tile.len;
  const int64_t nrows = tile.count;

  // This lane's row (past the last one: the last one's q, not stored)
  const int64_t row = (int64_t)row0 + lr, rowq = min(row, nrows - 1);
  const int token = (int)(rowq / a.group), head = kvh * a.group + (int)(rowq - (int64_t)token * a.group);
  const int last = (int)min((int64_t)len - n + token, (int64_t)len - 1);  // the last key it sees
  half8v qf[2 * DC];
  float c;
  {
    const T* q = (const T*)a.q + (int64_t)(first + token) * a.ldq + (int64_t)head * a.hq;
    T raw[2 * DC][8];
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * DC; ++s) {
      const int d = lg * KD + s * 8;
      int4v v{};
      if (WHOLE || d < a.d) v = *(const int4u*)(q + d);
      __builtin_memcpy(raw[s], &v, 16);
      if constexpr (BF16) top = largest(raw[s], top);
    }
    const int ex = BF16 ? exponent_of(row_max(top)) : 0;
    c = score_scale(a.c, ex);
#pragma unroll
    for (int s = 0; s < 2 * DC; ++s) qf[s] = q_operand(raw[s], ex);
  }

  // keys this tile / all of its rows see
  const int i1 = (int)min((int64_t)n - 1, ((int64_t)row0 + RT - 1) / a.group);
  const int kend = max(0, min(len, len - n + i1 + 1));
  const int kfull = max(0, min(len, len - n + row0 / a.group + 1));
  const int groups = (kend + 63) >> 6, share = (groups + nsplit - 1) / nsplit;
  const int g1 = min(groups, (split + 1) * share);

  Partial<DT> acc;
  acc.clear();
  bool far = false;  // some row's m is

  const uint32_t kbyte = twice_byte(lr & 3);  // (of the words of scales, those of this lane's keys)
  const int ck = lr >> 2;  // 16-key piece of a group that this lane's K rows lie in (V's and the scores': lg)
  const int* const table = a.table + (int64_t)r * a.ldt;
  const int64_t hb = (int64_t)kvh * a.bytes, kv_bytes = (int64_t)a.kv_heads * a.bytes;
  const int pm = (1 << a.lb) - 1;  // 16-key pieces of a page, less one
  // The block of 16-key piece `piece`, -1 where there is none or a bad one.
  auto page = [&](int piece) {
    const int p = piece >> a.lb;
    const int b = p < a.width && piece * 16 < kend ? table[p] : -1;
    return (unsigned)b < (unsigned)a.blocks ? b : -1;
  };
  uint32_t kr[4][2 * DC];
  int4v ksw{}, vr[G], vsw[G];
  bool there;
  // (a piece that is not there reads block 0's numbers, which its mask leaves out)
  auto load_k = [&](int g, int b) {
    const int64_t blk = max(b, 0);
    const int at = ((4 * g + ck) & pm) * 16;
    const uint8_t* p = a.k + blk * kv_bytes + hb + (int64_t)(at + (lr & 3)) * (a.dp >> 1) + lg * (KD / 2);
    const bool in = WHOLE || lg * KD < a.dp;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if constexpr (DC == 1) {
        const uint2 v = in ? *(const uint2*)(p + 4 * t * (a.dp >> 1)) : uint2{};
        kr[t][0] = v.x;
        kr[t][1] = v.y;
      } else {
        const uint4 v = in ? *(const uint4*)(p + 4 * t * (a.dp >> 1)) : uint4{};
        kr[t][0] = v.x;
        kr[t][1] = v.y;
        kr[t][2] = v.z;
        kr[t][3] = v.w;
      }
    }
    if (in) ksw = *(const int4v*)(a.ks + (blk * a.kv_heads + kvh) * a.sbytes + ((int64_t)(lg * KD / 32) << (a.lb + 4)) + at);
  };
  auto load_v = [&](int g, int b) {
    const int64_t blk = max(b, 0);
    const int piece = (4 * g + lg) & pm;
    const uint8_t* p = a.v + blk * kv_bytes + hb + ((int64_t)piece * a.dp + 2 * lr) * 8;
    const uint8_t* s = a.vs + (blk * a.kv_heads + kvh) * a.sbytes + piece * 16;
#pragma unroll
    for (int x = 0; x < G; ++x) {
      const bool in = WHOLE || x * 32 < a.dp;
      vr[x] = in ? *(const int4v*)(p + x * 256) : int4v{};
      vsw[x] = in ? *(const int4v*)(s + ((int64_t)x << (a.lb + 4))) : int4v{};
    }
    there = b >= 0;
  };

  int g = split * share + w, bk2 = -1, bv2 = -1;
  if (g < g1) {
    const int bk = page(4 * g + ck), bv = page(4 * g + lg);
    load_k(g, bk);
    load_v(g, bv);
    if (g + 4 < g1) {
      bk2 = page(4 * (g + 4) + ck);
      bv2 = page(4 * (g + 4) + lg);
    }
  }
  for (; g < g1; g += 4) {
    // scores
    float4v s[4];
    static_for<4>([&](auto t) {
      const half2v sc = scale_twice((uint32_t)ksw[int(t)], kbyte);
#pragma unroll
      for (int x = 0; x < 2 * DC; ++x)
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand(kr[t][x], [&](int) { return sc; }), qf[x],
                                                      x == 0 ? float4v{0.f, 0.f, 0.f, 0.f} : s[t], 0, 0, 0);
    });
    const bool more = g + 4 < g1;
    const bool there0 = there;
    if (more) load_k(g + 4, bk2);
    // softmax
    const bool whole = g * 64 + 64 <= kfull && __all(there0);  // (wave-uniform)
    float mx = -INFINITY;
    if (!whole) {
      const int left = there0 ? last - (g * 64 + lg * 16) : -1;  // keys of this lane up to this one are seen
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][i] = 4 * t + i > left ? -INFINITY : s[t][i];
      // A weight of 0 has to leave nothing behind whatever the scale is: those of
      // keys past all rows' are 0, and so are others that may make an infinite
      // product, which make the rows that see them NaN by their sum.
      const int held = there0 ? kend - (g * 64 + lg * 16) : 0;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t mask = first_bytes(held, y);
        uint32_t bad = 0;
#pragma unroll
        for (int x = 0; x < G; ++x) {
          const uint32_t b = past_largest((uint32_t)vsw[x][y]) & mask;
          vsw[x][y] &= (int)(mask & ~b);
          bad |= b;
        }
        if (bad & first_bytes(left + 1, y)) acc.l = NAN;
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[t][i]);
    mx = row_max(mx) * c;  // (c > 0)
    if (__any(mx > acc.m + kHigh)) {
      const float now = mx > acc.m + kHigh ? mx - kLow : acc.m, f = rel_exp2(acc.m, now);
      acc.m = now;
      acc.l *= f;
#pragma unroll
      for (int t = 0; t < DT; ++t) acc.o[t] *= f;
      far = __any(is_far(now));
    }
    const float off = acc.m == -INFINITY ? 0.f : -acc.m;
    float cw = c;
    if (far) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][i] = times(s[t][i], c);
      cw = 1.f;
    }
    half8v p[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[2 * u + (j >> 2)][j & 3], cw, off));
        acc.l += e;
        p[u][j] = (_Float16)e;
      }
    }
    // values
#pragma unroll
    for (int x = 0; x < G; ++x) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const Pairs sc((uint32_t)vsw[x][2 * u], (uint32_t)vsw[x][2 * u + 1]);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          acc.o[2 * x + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              operand((uint32_t)vr[x][2 * e + u], [&](int i) { return sc.p[i]; }), p[u], acc.o[2 * x + e], 0, 0, 0);
      }
    }
    if (more) {
      load_v(g + 4, bv2);
      if (g + 8 < g1) {
        bk2 = page(4 * (g + 8) + ck);
        bv2 = page(4 * (g + 8) + lg);
      }
    }
  }

  // Join the waves' parts: waves 1..3 through LDS into wave 0.
  auto join = [&]() {
    __syncthreads();
    if (w > 0) acc.each([&](int i, float v) { return joined[((w - 1) * NV + i) * 64 + lane] = v; });
    __syncthreads();
    if (w > 0) return;
    Partial<DT> other[3];
#pragma unroll
    for (int o = 0; o < 3; ++o) other[o].each([&](int i, float) { return joined[(o * NV + i) * 64 + lane]; });
    acc.add(other);
  };
  join();

  if (nsplit > 1) {
    // Every share stores its part (system-coherent stores, visible to every
    // XCD once vmcnt drains) and arrives on the tile's counter; the last one
    // joins them.
    constexpr int kCoherent = 17;  // sc0 | sc1
    constexpr int PART = NV * 64 * 4;
    const __amdgpu_buffer_rsrc_t rP =
        make_rsrc(a.ws + kWsCounterBytes + (int64_t)(item - a.full) * nsplit * PART, (uint32_t)(nsplit * PART));
    if (w == 0) {
      acc.each([&](int i, float v) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rP, (uint32_t)(split * PART + (i * 64 + lane) * 4), 0,
                                              kCoherent);
        return v;
      });
      wait_vmcnt0();
      if (lane == 0) {
        unsigned long long* cnt = (unsigned long long*)a.ws + (item - a.full);  // < kWsMaxTiles (the host's check)
        const unsigned long long before =
            __hip_atomic_fetch_add(cnt, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_split = before + 1 == (unsigned long long)nsplit;
        if (last_split) __hip_atomic_store(cnt, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    __syncthreads();
    if (!last_split) return;
    acc.clear();
    for (int sp = w; sp < nsplit; sp += 4) {  // (in this order whichever came last)
      Partial<DT> other[1];
      other[0].each([&](int i, float) {
        return __uint_as_float(
            __builtin_amdgcn_raw_buffer_load_b32(rP, (uint32_t)(sp * PART + (i * 64 + lane) * 4), 0, kCoherent));
      });
      acc.add(other);
    }
    join();
  }
  if (w > 0) return;

  // O: lane holds row l % 16, dims 32 x + 8 (l / 16) + 0..7
  const float l = row_reduce(acc.l, [](float y, float z) { return y + z; });
  const float f = l == 0.f ? 0.f : 1.f / l;
  if (row >= nrows) return;
  T* const o = (T*)a.o + (int64_t)(first + token) * a.ldo + (int64_t)head * a.ho;
#pragma unroll
  for (int x = 0; x < G; ++x) {
    const int d = x * 32 + lg * 8;
    if (!WHOLE && d >= a.d) continue;
    T o8[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o8[j] = (T)(acc.o[2 * x + (j & 1)][j >> 1] * f);
    int4v bits;
    __builtin_memcpy(&bits, o8, 16);
    *(int4u*)(o + d) = bits;
  }
}

// ---- rows in the hundreds ----------------------------------------------------------
//
// A workgroup of four waves owns 128 rows (32 a wave) and takes 64 keys at a
// time through two LDS stages: its threads bring the numbers to fp16 on the way
// in, once for 128 rows (the kernel above: for 16), under the score MFMAs, and
// those of the next stage but one are in flight meanwhile.  Scores are
// D[key][row] of 32x32x16 MFMAs; row m of a 32-key block reads key 16 (m / 16) +
// 8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4, so that a lane's eight weights of 16 keys
// are eight in order, the B operand of P.V.  2350 rows x 32 heads over 8000 keys of 128
// dims: 253 us (780 TFLOP/s; 397 by the kernel above), 64 dims over 4 heads 223 us. The
// vector ALUs bound it: softmax (an exponential is two slots, a sum of weights half
// a one: both as v_dot2), then conversion.
// D: LDS rows of K (64 or 128 dims).
template <typename T, int D, bool WHOLE>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void kv4_attention_tiles(KArgs a) {
  constexpr bool BF16 = !std::is_same_v<T, _Float16>;
  constexpr int DS = D / 16, DT = D / 32, RB = 2 * D;
  constexpr int KB = 64 * RB, STAGE = KB + D * 128;
  constexpr int KW = D / 32, VD = D / 64;  // words of K, dims of V (of 16 keys) a thread converts a stage
  constexpr int NV = DT * 16 + 2;
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  __shared__ uint32_t unheld[2][4];  // of a stage's pieces: keys with a value that is no number, a bit each
  __shared__ int last_split;

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 31, h = lane >> 5;
  const Share part = share_of(a);
  const int split = part.split, nsplit = part.count, item = part.item;
  const int kvh = item / a.tiles;
  Rows tile;
  if (!rows_of<128>(a, a.tiles - 1 - (item - kvh * a.tiles), tile)) return;  // (the last rows see the most keys)
  const int n = tile.n, len = tile.len;

  // This lane's row (past the last one: the last one's q, not stored)
  const int64_t row = (int64_t)tile.row0 + w * 32 + lr, rowq = min(row, tile.count - 1);
  const int token = (int)(rowq / a.group), head = kvh * a.group + (int)(rowq - (int64_t)token * a.group);
  const int last = (int)min((int64_t)len - n + token, (int64_t)len - 1);  // the last key it sees
  half8v qf[DS];
  float c;
  {
    const T* q = (const T*)a.q + (int64_t)(tile.first + token) * a.ldq + (int64_t)head * a.hq;
    T raw[DS][8];
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      const int d = s * 16 + h * 8;
      int4v v{};
      if (WHOLE || d < a.d) v = *(const int4u*)(q + d);
      __builtin_memcpy(raw[s], &v, 16);
      if constexpr (BF16) top = largest(raw[s], top);
    }
    int ex = 0;
    if constexpr (BF16) {
      const auto t2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      ex = exponent_of(fmaxf(__uint_as_float(t2[0]), __uint_as_float(t2[1])));
    }
    c = score_scale(a.c, ex);
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[s] = q_operand(raw[s], ex);
  }

  // keys that some / all rows of the workgroup, and all rows of the wave, see
  const int i1 = (int)min((int64_t)n - 1, ((int64_t)tile.row0 + 127) / a.group);
  const int kend = max(0, min(len, len - n + i1 + 1));
  const int kall = max(0, min(len, len - n + tile.row0 / a.group + 1));
  const int wrow = tile.row0 + w * 32;
  const int kfull = wrow < tile.count ? max(0, min(len, len - n + wrow / a.group + 1)) : 0;
  const int stages = (kend + 63) >> 6, share = (stages + nsplit - 1) / nsplit;
  const int c0 = split * share, c1 = min(stages, c0 + share);

  const int* const table = a.table + (int64_t)tile.r * a.ldt;
  const int64_t hb = (int64_t)kvh * a.bytes, kv_bytes = (int64_t)a.kv_heads * a.bytes;
  const int pm = (1 << a.lb) - 1;
  // Lane l's page of a stage: that of its 16-key piece l % 4, -1 where there is none or a bad one.
  auto page = [&](int st) {
    const int piece = 4 * st + (lane & 3), p = piece >> a.lb;
    const int b = p < a.width && piece * 16 < kend ? table[p] : -1;
    return (unsigned)b < (unsigned)a.blocks ? b : -1;
  };

  // Thread t's part of a stage: K, key t / 4 (one of the wave's 16), dims 8 KW (t %
  // 4) on, under one scale; V, the wave's 16 keys of dims VD (t % 64) on.
  const int t = threadIdx.x, kd = (lane & 3) * 8 * KW, vd = lane * VD;
  uint32_t kc[KW], vc[2 * VD], ksw = 0;
  int4v vsw{};
  // The numbers and scales of a stage with pages `pg` (a page that is not there: block 0's, left out below).
  auto load = [&](int st, int pg) {
    const int b = __builtin_amdgcn_readlane(pg, w), at = ((4 * st + w) & pm) * 16;
    const int64_t blk = max(b, 0), sb = (blk * a.kv_heads + kvh) * a.sbytes + at;
    const uint8_t* const kp = a.k + blk * kv_bytes + hb + (int64_t)(at + (lane >> 2)) * (a.dp >> 1) + (kd >> 1);
    const uint8_t* const vp = a.v + blk * kv_bytes + hb + ((int64_t)(at >> 4) * a.dp + vd) * 8;
    const bool kin = WHOLE || kd < a.dp, vin = WHOLE || vd < a.dp;
    if constexpr (D == 64) {
      const uint2 k2 = kin ? *(const uint2*)kp : uint2{}, v2 = vin ? *(const uint2*)vp : uint2{};
      kc[0] = k2.x;
      kc[1] = k2.y;
      vc[0] = v2.x;
      vc[1] = v2.y;
    } else {
      const uint4 k4 = kin ? *(const uint4*)kp : uint4{}, v4 = vin ? *(const uint4*)vp : uint4{};
      __builtin_memcpy(kc, &k4, 16);
      __builtin_memcpy(vc, &v4, 16);
    }
    if (kin) ksw = a.ks[sb + ((int64_t)(kd >> 5) << (a.lb + 4)) + (lane >> 2)];
    vsw = vin ? *(const int4v*)(a.vs + sb + ((int64_t)(vd >> 5) << (a.lb + 4))) : int4v{};
    return pg;
  };
  // A weight of 0 has to leave nothing behind whatever a scale is: in a stage that
  // not every row sees whole, scales of keys past all rows' are 0, and so are others
  // that may make an infinite product, which make the rows that see them NaN by their sum.
  auto clear = [&](int st, int pg) {
    const int b = __builtin_amdgcn_readlane(pg, w);
    if (b >= 0 && st * 64 + 64 <= kall) return;
    const int held = b >= 0 ? kend - (st * 64 + 16 * w) : 0;
    uint32_t any = 0;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const uint32_t mask = first_bytes(held, y), bad = past_largest((uint32_t)vsw[y]) & mask;
      vsw[y] &= (int)(mask & ~bad);
      any |= (bad & 1) << (4 * y) | (bad >> 7 & 2) << (4 * y) | (bad >> 14 & 4) << (4 * y) | (bad >> 21 & 8) << (4 * y);
    }
    if (__any(any)) {
      for (int o = 32; o >= 1; o >>= 1) any |= (uint32_t)__shfl_xor((int)any, o, 64);
    }
    if (lane == 0) unheld[st & 1][w] = any;
  };
  // 16-byte chunks of LDS rows are XOR-swizzled: the rows that one read takes
  // 16 bytes of (16 lanes at a time) fall on different banks.
  auto k_at = [](int key, int chunk) { return key * RB + ((chunk ^ (key / (256 / RB) & (RB / 16 - 1))) << 4); };
  auto v_at = [](int d, int chunk) { return KB + d * 128 + ((chunk ^ (d >> 1 & 7)) << 4); };
  // (the swizzle is an XOR of chunk bits: another chunk of a row lies at the row's chunk 0 with those bits flipped)
  const int k_store = k_at(t >> 2, (lane & 3) * KW), v_store = v_at(vd, 2 * w);
  // Unit j of DS: eight numbers, of K or of V.
  auto store = [&](char* base, auto j_) {
    constexpr int j = j_;
    if constexpr (j < KW) {
      const half2v sc = scale_twice<0>(ksw);
      *(half8v*)(base + (k_store ^ (j << 4))) = operand(kc[j], [&](int) { return sc; });
    } else {
      constexpr int u = (j - KW) / VD, e = (j - KW) % VD;  // (both dims under the same scales)
      const Pairs sc((uint32_t)vsw[2 * u], (uint32_t)vsw[2 * u + 1]);
      *(half8v*)(base + (v_store ^ (u << 4)) + e * 128) = operand(vc[2 * e + u], [&](int i) { return sc.p[i]; });
    }
  };
  static_assert(KW + 2 * VD == DS, "a unit a step of the scores");

  float16v o[DT];
  float m = -INFINITY, l = 0.f;
  bool far = false;  // some row's m is
#pragma unroll
  for (int x = 0; x < DT; ++x) o[x] = float16v{};

  const int key = 16 * (lr >> 4) + 8 * (lr >> 2 & 1) + 4 * (lr >> 3 & 1) + (lr & 3);
  const int k_read = k_at(key, h), v_read = v_at(lr, h);
  int pg = -1, after = -1;  // pages of the stage after next, and of the one loaded
  // Stage st (pages `here`) in `base`, while `other` takes the next one (pages `next`).
  auto compute = [&](int st, const char* base, char* other, int here, int next) {
    const uint64_t there = __ballot(here >= 0);
    const bool all = st * 64 + 64 <= kfull && there == ~0ull;
    // Fragments are read a step ahead of their MFMAs; the scheduling barriers
    // keep the compiler from reading them all first.
    float16v s[2];
    half8v kf[2][2], vf[2][DT];
    auto read_k = [&](int x) {
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) kf[x & 1][nb] = *(const half8v*)(base + (k_read ^ (x << 5)) + nb * 32 * RB);
    };
    auto read_v = [&](int x) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vf[x & 1][dt] = *(const half8v*)(base + (v_read ^ (x << 5)) + dt * 32 * 128);
    };
    if (st + 1 < c1) clear(st + 1, next);
    read_k(0);
    static_for<DS>([&](auto x) {
      if (x + 1 < DS) read_k(x + 1);
      else read_v(0);
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
        s[nb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[x & 1][nb], qf[x], x == 0 ? float16v{} : s[nb], 0, 0, 0);
      // (conversion passes under the score MFMAs, which need few vector
      // instructions; past the last stage old numbers go where nobody reads)
      store(other, x);
      __builtin_amdgcn_sched_barrier(0);
    });
    // (the numbers' registers are free)
    if (st + 2 < c1) after = load(st + 2, pg);
    if (st + 3 < c1) pg = page(st + 3);
    // a lane's eight keys of a piece up to this one are seen
    auto left_of = [&](int x) { return there >> x & 1 ? last - (st * 64 + x * 16 + 8 * h) : -1; };
    if (!all) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int left = left_of(x);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[x >> 1][8 * (x & 1) + e] = e > left ? -INFINITY : s[x >> 1][8 * (x & 1) + e];
      }
    }
    if (st * 64 + 64 > kall) {
      uint32_t bad = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (there >> x & 1) bad |= unheld[st & 1][x] >> (8 * h) & ((1u << min(max(left_of(x) + 1, 0), 8)) - 1);
      l = bad ? NAN : l;
    }
    float mx = s[0][0];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[x][i]);
    const auto m2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    mx = fmaxf(__uint_as_float(m2[0]), __uint_as_float(m2[1])) * c;  // (c > 0)
    if (__any(mx > m + kHigh)) {
      const float now = mx > m + kHigh ? mx - kLow : m, f = rel_exp2(m, now);
      m = now;
      l *= f;
#pragma unroll
      for (int x = 0; x < DT; ++x) o[x] *= f;
      far = __any(is_far(now));
    }
    const float off = m == -INFINITY ? 0.f : -m;
    float cw = c;
    if (far) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[x][i] = times(s[x][i], c);
      cw = 1.f;
    }
    // the weights of 16 keys while the MFMAs of the 16 before run
    auto weights = [&](int x) {
      half8v p;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        p[e] = (_Float16)__builtin_amdgcn_exp2f(fmaf(s[x >> 1][8 * (x & 1) + e], cw, off));
      l = sum_of(p, l);
      return p;
    };
    half8v p = weights(0);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      half8v then = p;
      if (x < 3) {
        read_v(x + 1);
        then = weights(x + 1);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[x & 1][dt], p, o[dt], 0, 0, 0);
      p = then;
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (c0 < c1) {
    // Ahead of the stage computed: the next one's numbers on their way into LDS,
    // those of the one after, pages of the one after that.
    int now = load(c0, page(c0)), next = -1;
    clear(c0, now);
    static_for<DS>([&](auto x) { store(lds, x); });
    if (c0 + 1 < c1) next = load(c0 + 1, page(c0 + 1));
    if (c0 + 2 < c1) pg = page(c0 + 2);
    auto step = [&](int st, char* base, char* other) {
      __syncthreads();  // stage st is written, and nobody reads the other one
      compute(st, base, other, now, next);
      now = next;
      next = after;
    };
    // (LDS addresses that differ by constants)
    for (int st = c0; st < c1; st += 2) {
      step(st, lds, lds + STAGE);
      if (st + 1 < c1) step(st + 1, lds + STAGE, lds);
    }
  }

  // A wave's floats: o, m, l; a tile's shares joined as in the kernel above.
  auto each = [&](auto&& f) {
#pragma unroll
    for (int x = 0; x < DT; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) f(x * 16 + i, o[x][i]);
    f(DT * 16, m);
    f(DT * 16 + 1, l);
  };
  if (nsplit > 1) {
    constexpr int kCoherent = 17;  // sc0 | sc1
    constexpr int PART = 4 * NV * 64 * 4;
    const __amdgpu_buffer_rsrc_t rP =
        make_rsrc(a.ws + kWsCounterBytes + (int64_t)(item - a.full) * nsplit * PART, (uint32_t)(nsplit * PART));
    each([&](int i, float v) {
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rP, (uint32_t)(split * PART + ((w * NV + i) * 64 + lane) * 4),
                                            0, kCoherent);
    });
    wait_vmcnt0();
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long* cnt = (unsigned long long*)a.ws + (item - a.full);  // < kWsMaxTiles (the host's check)
      const unsigned long long before = __hip_atomic_fetch_add(cnt, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last_split = before + 1 == (unsigned long long)nsplit;
      if (last_split) __hip_atomic_store(cnt, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last_split) return;
    auto held = [&](int sp, int i) {
      return __uint_as_float(
          __builtin_amdgcn_raw_buffer_load_b32(rP, (uint32_t)(sp * PART + ((w * NV + i) * 64 + lane) * 4), 0, kCoherent));
    };
    m = -INFINITY;
#pragma unroll 4
    for (int sp = 0; sp < nsplit; ++sp) m = fmaxf(m, held(sp, DT * 16));
    l = 0.f;
#pragma unroll
    for (int x = 0; x < DT; ++x) o[x] = float16v{};
    for (int sp = 0; sp < nsplit; ++sp) {  // (in this order whichever came last)
      const float f = rel_exp2(held(sp, DT * 16), m);
      l += f * held(sp, DT * 16 + 1);
#pragma unroll
      for (int x = 0; x < DT; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[x][i] += f * held(sp, x * 16 + i);
    }
  }

  // O: lane holds row l % 32, dims 32 x + 8 g + 4 h + 0..3
  const auto l2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
  const float whole = __uint_as_float(l2[0]) + __uint_as_float(l2[1]), f = whole == 0.f ? 0.f : 1.f / whole;
  if (row >= tile.count) return;
  T* const out = (T*)a.o + (int64_t)(tile.first + token) * a.ldo + (int64_t)head * a.ho;
#pragma unroll
  for (int x = 0; x < DT; ++x)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = x * 32 + 8 * g + 4 * h;
      if (!WHOLE && d >= a.d) continue;
      T o4[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o4[j] = (T)(o[x][4 * g + j] * f);
      int2v bits;
      __builtin_memcpy(&bits, o4, 8);
      *(int2u*)(out + d) = bits;
    }
}

// The card takes four workgroups a CU of the kernel for 16 rows at up to 64 dims (the
// 8-bit one is planned for two): 64 requests of 8192 tokens over 4 heads 35.0 us in
// two shares a tile, 31.5 in four.  Fewer tiles have their keys shared out as far
// as it pays either way (64 tiles of 4000 keys: 10.0 us in eight, 11.4 in sixteen; 170
// of drafts over 1500 keys: 11.0 in three, 11.4 in six).  The line between them, 128
// tiles, lies between those two, which are all that was measured around it; from there a
// share has at least 512 keys (plan_of), below it 256.
KvPlan plan4_of(const KvAttnSizes& p) {
  const int64_t group = p.heads / p.kv_heads;
  const int64_t tiles = p.cu ? p.tokens * group / 16 + p.requests : p.requests * ((group + 15) / 16);
  return plan_of(p, p.d <= 64 && tiles * p.kv_heads >= 128 ? 1024 : 512);
}
int64_t part_bytes(const KvAttnSizes& p, const KvPlan& k) {  // of a tile's share
  const int64_t dt = p.d <= 64 ? 4 : 8;
  return k.rt == 16 ? (dt * 4 + 2) * 64 * 4 : 4 * (dt * 8 + 2) * 64 * 4;
}

template <typename T>
hipError_t launch_t(int64_t d, int rt, dim3 grid, const KArgs& a, hipStream_t stream) {
  const bool small = d <= 64, whole = d == 64 || d == 128;
  const auto fn = rt == 16 ? (small ? whole ? kv4_attention<T, 1, true> : kv4_attention<T, 1, false>
                                    : whole ? kv4_attention<T, 2, true> : kv4_attention<T, 2, false>)
                           : (small ? whole ? kv4_attention_tiles<T, 64, true> : kv4_attention_tiles<T, 64, false>
                                    : whole ? kv4_attention_tiles<T, 128, true> : kv4_attention_tiles<T, 128, false>);
  hipLaunchKernelGGL(fn, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

int64_t kv4_attention_workspace_bytes(const Kv4AttnProblem& p) {
  const KvPlan k = plan4_of(p);
  return k.nsplit > 1 ? kWsCounterBytes + (k.tiles * p.kv_heads - k.full) * k.nsplit * part_bytes(p, k) : 0;
}

hipError_t launch_kv4_attention(const Kv4AttnProblem& p, hipStream_t stream) {
  KvPlan k = plan4_of(p);
  const int64_t items = k.tiles * p.kv_heads;
  if (k.nsplit > 1 && (!p.ws || p.ws_bytes < kv4_attention_workspace_bytes(p))) {
    k.nsplit = 1;
    k.full = items;
  }
  const int64_t grid = k.full + (items - k.full) * k.nsplit;
  static_assert(1024 <= kWsMaxTiles, "a counter for every shared tile");
  if (grid >= (1ll << 31)) return hipErrorInvalidValue;
  KArgs a{};
  a.k = p.k_codes;
  a.v = p.v_codes;
  a.ks = p.k_scale;
  a.vs = p.v_scale;
  a.dp = (int)((p.d + 31) / 32 * 32);
  a.bytes = p.block * a.dp / 2;
  a.sbytes = p.block * a.dp / 32;
  tile_args(p, k, a);
  const dim3 blocks((unsigned)grid);
  return p.dtype == DT_BF16 ? launch_t<__bf16>(p.d, k.rt, blocks, a, stream) : launch_t<_Float16>(p.d, k.rt, blocks, a, stream);
}

}  // namespace hxmi
