// Attention over the 8-bit key/value cache (layout: kvcache.hip), causal over
// ragged requests, grouped heads: row i of a request with n rows and L tokens
// in the cache sees keys j <= L - n + i,
//   o = sum_j p_j vc_j vs_j / sum_j p_j,  p_j = exp(scale * ks_j (q . kc_j) - max).
//
// A workgroup of four waves owns a tile of rows (token, head of the group) of
// one key/value head and, where there are few such tiles, one of `nsplit`
// shares of the keys.  Two kernels: this one for 16 rows,
// kv_attention_tiles below for 128.  Here the waves take every fourth group of
// 64 keys and codes go from memory straight to registers in the layout of the
// MFMA operands, so nothing passes through LDS until the waves' partial results
// are joined:
//   * scores as D[key][row] = Kc . Q^T (16x16x32 MFMAs).  A lane's K codes
//     are 16 bytes of one token; the head dims of a step may come in any
//     order, so they feed two steps as they lie.  Tile t's row 4 g + i is key
//     16 g + 4 t + i of the group, so the 16 scores of a lane (row l % 16,
//     g = l / 16) are keys 16 g .. 16 g + 15 in order: one page's, with one
//     K and one V scale a lane;
//   * those 16 weights are the B operand of P.V as they are, and 16 bytes of
//     V (16 tokens of one head dim) the A operand: D[dim][row];
//   * codes become fp16 exactly (conversion below).  q in bf16 is brought to
//     fp16 under a power of two a row: multiples of 2^-38 of its largest element;
//   * the K scale multiplies the score.  The V scale multiplies the weight
//     before its rounding to fp16, relative to 2^m, m following the running
//     maximum of score + log2(vs) from 7 to 15 below it: the largest weight P.V
//     sees lies in [2^7, 2^15] whatever the ratio of the scales.  The sum of the
//     p_j is that of the fp32 weights over their V scale, relative to 2^m as
//     well: one maximum does for both while the V scales leave what counts in
//     fp32's range (near_one).  A wave (in the kernel below, a workgroup) that
//     meets any other, or scores in the thousands (kFar), takes its keys again
//     with the sum relative to a maximum of its own (Frame).
//     Weights from 2^-21 of the row's largest on round to 11 bits, smaller ones
//     to multiples of 2^-31 of it (fp16 below 2^-14), so that the others keep
//     their part beside one key far above them; scores, maxima, sums and O are
//     fp32.
// One token a request is bound by the codes' bytes: 64 requests of 8192 tokens,
// 32 heads over 8 of 128 dims, 157 us (814 MB, 5.2 TB/s); one of 131072 tokens
// 63 us (268 MB, 4.3 TB/s; 55 where the call before has left part of them in the
// last-level cache).  Short ones are bound by latency: 1900 tokens of one user
// 7.2 us, over a table as wide as that (plan_of).  Keys taken again cost their
// time again: scales far apart all over, 64 x 8192 183 -> 364 us and prompt chunks
// 362 -> 832 (random codes throughout).
#include "kv_attention_impl.h"

namespace hxmi {
namespace {

struct KArgs : TileArgs {
  const int8_t* k;
  const int8_t* v;
  const float* ks;
  const float* vs;
};

// Four codes as two pairs of fp16: 0x6400 | u is 1024 + u, u = code + 128.
__device__ __forceinline__ void codes_f16(int w, half2v& a, half2v& b) {
  const uint32_t u = (uint32_t)w ^ 0x80808080u;
  const half2v off = {(_Float16)-1152.f, (_Float16)-1152.f};
  a = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
  b = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
}
// Eight codes as one MFMA operand.
__device__ __forceinline__ half8v operand(int w0, int w1) {
  half2v p[4];
  codes_f16(w0, p[0], p[1]);
  codes_f16(w1, p[2], p[3]);
  return half8v{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}

// x + lv, -inf where lv is (whatever x is).
__device__ __forceinline__ float left_out(float x, float lv) { return lv == -INFINITY ? -INFINITY : x + lv; }

// A page's V scale as the weights take it: its logarithm, and its inverse for
// the sum.  A page that is not there, or whose keys are all masked, has
// logarithm -inf.  A page of zeros (scale 0) counts in the sum alone: with sums
// of their own (apart) it has logarithm -inf too, otherwise it takes 2^-64, so
// that whatever its codes are they are lost beside any page that is near_one.
__device__ __forceinline__ void value_scale(float vs, bool apart, float& lv, float& rv) {
  vs = vs == 0.f && !apart ? 0x1p-64f : vs;
  lv = __builtin_amdgcn_logf(vs);
  rv = __builtin_amdgcn_rcpf(vs);
}
// Whether the sum can be taken from a page's weighted scores, 2^(score + log2(vs)
// - m): m is at most 10 above the largest score then, so that the weighted
// scores of keys of zeros 2^45 below that are still normal numbers, and at most
// 64 + 15 below it.
__device__ __forceinline__ bool near_one(float vs) {  // 0, or from 2^-30 to 2^10
  const uint32_t b = __float_as_uint(vs), lo = (127 - 30) << 23, hi = (127 + 10) << 23;
  return b - lo <= hi - lo || b == 0;
}

// A running maximum of this magnitude or more has no bits left for log2(vs) - m
// beside a weight's 11 (2^-13 at this one; at 2^27 it is off by powers of two
// that fp16 does not hold): such rows take their keys again with sums of their
// own too, where scores are rounded and subtracted before log2(vs) comes to them.
constexpr float kFar = 4096.f;

// a * b, rounded (never part of an fma).
__device__ __forceinline__ float times(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// What a row's numbers are relative to: the sum l of its p_j to 2^m, O to
// 2^(m + d).  d is 0 and m kLow to kHigh below the running maximum of score +
// log2(vs), or, with sums of their own, m is the largest score and d that far
// below the running maximum of score - m + log2(vs): -inf where nothing has been
// added to O.  (kLow 0 and kHigh 8 would leave the upper half of fp16's range
// unused: a key 24 bits above all others cost these a third of their part.)
constexpr float kLow = 7.f, kHigh = 15.f;
struct Frame {
  float m, d;

  // The largest score is now at least `top`: what l is to be multiplied by.
  __device__ __forceinline__ float raise(float top) {
    const float now = fmaxf(m, top), f = rel_exp2(m, now);
    d = m == -INFINITY ? -INFINITY : d + (m - now);
    m = now;
    return f;
  }
  // The maximum of score - m + log2(vs) is now at least `cand`: what O is to be multiplied by.
  __device__ __forceinline__ float raise_o(float cand) {
    const float now = cand > d + kHigh ? cand - kLow : d, f = rel_exp2(d, now);
    d = now;
    return f;
  }
  // Relative to a larger m.
  __device__ __forceinline__ Frame from(float now) const {
    const float to = m == -INFINITY ? -INFINITY : m - now;
    return Frame{to, d + to};
  }
  // What O is to be multiplied by at the end (l: the whole sum, 0 if no key was seen).
  __device__ __forceinline__ float over(float l) const { return l == 0.f ? 0.f : __builtin_amdgcn_exp2f(d) / l; }
};

// Frames joined into the first: what l and O of each are to be multiplied by.
template <int N>
__device__ __forceinline__ void join_frames(Frame (&at)[N], float (&fl)[N], float (&fo)[N]) {
  float m = at[0].m, d = -INFINITY;
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, at[i].m);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    at[i] = at[i].from(m);
    fl[i] = __builtin_amdgcn_exp2f(at[i].m);
    d = fmaxf(d, at[i].d);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) fo[i] = rel_exp2(at[i].d, d);
  at[0] = Frame{m, d};
}

// What a wave knows of its 16 rows: O and the sum of the p_j (this lane's part).
template <int DT>
struct Partial {
  static constexpr int N = DT * 4 + 3;  // floats a lane
  float4v o[DT];
  Frame at;
  float l;

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = float4v{0.f, 0.f, 0.f, 0.f};
    at = Frame{-INFINITY, 0.f};
    l = 0.f;
  }
  // Every float becomes f(its index, it).
  template <typename F>
  __device__ __forceinline__ void each(F&& f) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[t][i] = f(t * 4 + i, o[t][i]);
    at.m = f(DT * 4, at.m);
    at.d = f(DT * 4 + 1, at.d);
    l = f(DT * 4 + 2, l);
  }
  template <int N>
  __device__ __forceinline__ void add(const Partial (&p)[N]) {
    Frame f[N + 1] = {at};
#pragma unroll
    for (int j = 0; j < N; ++j) f[j + 1] = p[j].at;
    float fl[N + 1], fo[N + 1];
    join_frames(f, fl, fo);
    at = f[0];
    l *= fl[0];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] *= fo[0];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      l += p[j].l * fl[j + 1];
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] += p[j].o[t][i] * fo[j + 1];
    }
  }
};

// DC: 64-dim pieces of a row; WHOLE: the head dim is 64 * DC.  (Waves a SIMD: as the
// first pass over the keys allows; the second one's registers would take one.)
template <typename T, int DC, bool WHOLE>
__global__ __launch_bounds__(256, DC == 1 ? 4 : 2) void kv_attention(KArgs a) {
  constexpr int DT = DC * 4, RT = 16, NV = Partial<DT>::N;
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
  float c = a.c;
  {
    const T* q = (const T*)a.q + (int64_t)(first + token) * a.ldq + (int64_t)head * a.hq;
    T raw[2 * DC][8];
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * DC; ++s) {
      const int d = (s >> 1) * 64 + lg * 16 + (s & 1) * 8;
      int4v v{};
      if (WHOLE || d < a.d) v = *(const int4u*)(q + d);
      __builtin_memcpy(raw[s], &v, 16);
      if constexpr (BF16) top = largest(raw[s], top);
    }
    const int ex = BF16 ? exponent_of(row_max(top)) : 0;
    if constexpr (BF16) c = __builtin_ldexpf(a.c, -ex);
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
  bool odd = false;  // a page's scale was not near_one, or a maximum far from 0 (a lane's)

  const int ck = (lane >> 2) & 3;  // 16-key piece of a group that this lane's K rows lie in (V's and the scores': lg)
  const int* const table = a.table + (int64_t)r * a.ldt;
  const int64_t hb = (int64_t)kvh * a.bytes, kv_bytes = (int64_t)a.kv_heads * a.bytes;
  const int pm = (1 << a.lb) - 1;  // 16-key pieces of a page, less one
  // The block of 16-key piece `piece`, -1 where there is none or a bad one.
  auto page = [&](int piece) {
    const int p = piece >> a.lb;
    const int b = p < a.width && piece * 16 < kend ? table[p] : -1;
    return (unsigned)b < (unsigned)a.blocks ? b : -1;
  };
  int4v kr[4][DC], vr[DT];
  float ks, vs;
  bool there;
  // (a piece that is not there reads block 0's codes, which its mask leaves out)
  auto load_k = [&](int g, int b) {
    const int piece = 4 * g + ck;
    const int8_t* p = a.k + max(b, 0) * kv_bytes + hb + ((int64_t)((piece & pm) * 16 + (lane & 3)) * a.dp + lg * 16);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int x = 0; x < DC; ++x) {
        const bool in = WHOLE || x * 64 + lg * 16 < a.dp;
        kr[t][x] = in ? *(const int4v*)(p + (int64_t)(4 * t) * a.dp + x * 64) : int4v{};
      }
  };
  auto load_v = [&](int g, int b) {
    const int piece = 4 * g + lg;
    const int8_t* p = a.v + max(b, 0) * kv_bytes + hb + ((int64_t)(piece & pm) * a.dp + lr) * 16;
#pragma unroll
    for (int t = 0; t < DT; ++t)
      vr[t] = WHOLE || t * 16 < a.dp ? *(const int4v*)(p + t * 256) : int4v{};
    there = b >= 0;
    ks = there ? a.ks[(int64_t)b * a.kv_heads + kvh] : 0.f;
    vs = there ? a.vs[(int64_t)b * a.kv_heads + kvh] : 0.f;
  };

  // The wave's keys; APART: with sums of their own, and loads as they are needed.
  auto pass = [&](auto APART_) {
    constexpr bool APART = decltype(APART_)::value;
    acc.clear();
    int g = split * share + w;
    int bk2 = -1, bv2 = -1;
    if (!APART && g < g1) {
      const int bk = page(4 * g + ck), bv = page(4 * g + lg);
      load_k(g, bk);
      load_v(g, bv);
      if (g + 4 < g1) {
        bk2 = page(4 * (g + 4) + ck);
        bv2 = page(4 * (g + 4) + lg);
      }
    }
    for (; g < g1; g += 4) {
      if constexpr (APART) {
        const int bk = page(4 * g + ck), bv = page(4 * g + lg);
        load_k(g, bk);
        load_v(g, bv);
      }
      // scores
      float4v s[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int x = 0; x < DC; ++x)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand(kr[t][x][2 * u], kr[t][x][2 * u + 1]), qf[2 * x + u],
                                                          x == 0 && u == 0 ? float4v{0.f, 0.f, 0.f, 0.f} : s[t], 0, 0, 0);
      }
      const bool more = !APART && g + 4 < g1;
      const float ks0 = ks, vs0 = vs;
      const bool there0 = there;
      if (more) load_k(g + 4, bk2);
      // softmax
      const bool whole = g * 64 + 64 <= kfull && __all(there0);  // (wave-uniform)
      float lv, rv;
      value_scale(vs0, APART, lv, rv);
      half8v p[2];
      const float cs = c * ks0;
      float mx = -INFINITY;
      if (whole && !APART) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[t][i]);
        mx *= cs;  // (cs >= 0)
        odd |= !near_one(vs0);
      } else {
        // the scores times cs, masked ones -inf
        const int left = there0 ? last - (g * 64 + lg * 16) : -1;  // keys of this lane up to this one are seen
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[t][i] = 4 * t + i > left ? -INFINITY : times(s[t][i], cs);
            mx = fmaxf(mx, s[t][i]);
          }
        // (a page whose every key is masked takes no part, whatever its scale)
        if (left < 0) lv = -INFINITY;
        odd |= left >= 0 && !near_one(vs0);
      }
      float ref, f = 1.f;  // a weight is relative to 2^ref
      bool up = true;
      if constexpr (APART) {
        acc.l *= acc.at.raise(row_max(mx));
        const float m = acc.at.m == -INFINITY ? 0.f : acc.at.m;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[t][i] -= m;
            acc.l += __builtin_amdgcn_exp2f(s[t][i]);
          }
        f = acc.at.raise_o(row_max(left_out(mx - m, lv)));
        ref = acc.at.d;
      } else {
        const float mxv = row_max(left_out(mx, lv));
        up = __any(mxv > acc.at.m + kHigh);
        if (up) {
          odd |= mxv > acc.at.m + kHigh && fabsf(mxv) >= kFar;
          const float now = mxv > acc.at.m + kHigh ? mxv - kLow : acc.at.m;
          f = rel_exp2(acc.at.m, now);
          acc.l *= f;
          acc.at.m = now;
        }
        ref = acc.at.m;
      }
      if (up) {
#pragma unroll
        for (int t = 0; t < DT; ++t) acc.o[t] *= f;
      }
      const float off = lv == -INFINITY ? -INFINITY : lv - (ref == -INFINITY ? 0.f : ref);
      const float cw = whole && !APART ? cs : 1.f;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[t][i], cw, off));
          sum += e;
          p[t >> 1][(t & 1) * 4 + i] = (_Float16)e;
        }
      if (!APART) acc.l += lv == -INFINITY ? 0.f : sum * rv;
      // values
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          acc.o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand(vr[t][2 * u], vr[t][2 * u + 1]), p[u], acc.o[t], 0, 0, 0);
      if (more) {
        load_v(g + 4, bv2);
        if (g + 8 < g1) {
          bk2 = page(4 * (g + 8) + ck);
          bv2 = page(4 * (g + 8) + lg);
        }
      }
    }
  };
  pass(std::false_type{});
  if (__any(odd)) pass(std::true_type{});

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

  // O: lane holds row l % 16, dims 16 t + 4 (l / 16) + 0..3
  const float l = row_reduce(acc.l, [](float y, float z) { return y + z; });
  const float f = acc.at.over(l);
  if (row >= nrows) return;
  T* const o = (T*)a.o + (int64_t)(first + token) * a.ldo + (int64_t)head * a.ho;
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    const int d = t * 16 + lg * 4;
    if (!WHOLE && d >= a.d) continue;
    T o4[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o4[j] = (T)(acc.o[t][j] * f);
    int2v bits;
    __builtin_memcpy(&bits, o4, 8);
    *(int2u*)(o + d) = bits;
  }
}

// ---- rows in the hundreds ----------------------------------------------------------
//
// A workgroup of four waves owns 128 rows (32 a wave) and takes 64 keys at a
// time through two LDS stages: its threads convert the codes to fp16 on the way
// in, so a code is converted once for 128 rows (the kernel above: for 16), and codes of the next stage but one are in flight meanwhile.  2350 rows x
// 32 heads over 8000 keys: 271 us (727 TFLOP/s), 507 by the kernel above; bound
// by the vector ALUs (softmax, then conversion) of two waves a SIMD.  Eight waves
// of 256 rows convert half as often and were slower (289 us, 279 of four at that
// time): one workgroup a CU has nothing to run while it waits at its barriers.
// Scores are D[key][row] of 32x32x16 MFMAs; row m of a 32-key block
// reads key 16 (m / 16) + 8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4, so that a
// lane's eight weights of 16 keys are eight in order, the B operand of P.V.  The
// 16 keys are one piece of a page: K and V scales are wave-uniform.
// D: LDS rows of K (64 or 128 dims; with 64, two waves a SIMD were 8 % slower than three).
template <typename T, int D, bool WHOLE>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void kv_attention_tiles(KArgs a) {
  constexpr bool BF16 = !std::is_same_v<T, _Float16>;
  constexpr int DS = D / 16, DT = D / 32, RB = 2 * D;
  constexpr int KB = 64 * RB, STAGE = KB + D * 128;
  constexpr int PIECES = 64 * D / 16 / 256;  // 16-byte pieces of K (and of V) a thread converts a stage
  constexpr int NV = DT * 16 + 3;
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  __shared__ int last_split, odd;  // odd: a page's scale was not near_one, or a maximum far from 0

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
  float c = a.c;
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
      c = __builtin_ldexpf(a.c, -ex);
    }
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[s] = q_operand(raw[s], ex);
  }

  // keys that some / all rows of the workgroup, and all rows of the wave, see
  const int i1 = (int)min((int64_t)n - 1, ((int64_t)tile.row0 + 127) / a.group);
  const int kend = max(0, min(len, len - n + i1 + 1));
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

  // Thread t's pieces of a stage: K, key t / 4, bytes 16 (t % 4 + 4 i); V, 16
  // keys (the wave's) of dims t % 64 + 64 i.  Wave w's keys are 16 w .. 16 w + 15.
  const int t = threadIdx.x;
  int4v kc[PIECES], vc[PIECES];
  struct Scales {  // of a lane's piece
    int b;
    float k, v;
  };
  // The codes and scales of a stage with pages `pg` (a page that is not there: block 0's, left out below).
  auto load = [&](int st, int pg) {
    const int piece = 4 * st + w, b = max(__builtin_amdgcn_readlane(pg, w), 0);
    const int8_t* const kp = a.k + b * kv_bytes + hb + ((int64_t)((piece & pm) * 16 + (lane >> 2)) * a.dp + (lane & 3) * 16);
    const int8_t* const vp = a.v + b * kv_bytes + hb + ((int64_t)(piece & pm) * a.dp + lane) * 16;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      kc[i] = WHOLE || (lane & 3) * 16 + 64 * i < a.dp ? *(const int4v*)(kp + 64 * i) : int4v{};
      vc[i] = WHOLE || lane + 64 * i < a.dp ? *(const int4v*)(vp + 1024 * i) : int4v{};
    }
    const int64_t at = (int64_t)max(pg, 0) * a.kv_heads + kvh;
    return Scales{pg, a.ks[at], a.vs[at]};
  };
  // 16-byte chunks of LDS rows are XOR-swizzled: the rows that one read takes
  // 16 bytes of (16 lanes at a time) fall on different banks.
  auto k_at = [](int key, int chunk) { return key * RB + ((chunk ^ (key / (256 / RB) & (RB / 16 - 1))) << 4); };
  auto v_at = [](int d, int chunk) { return KB + d * 128 + ((chunk ^ (d >> 1 & 7)) << 4); };
  // (the swizzle is an XOR of chunk bits: chunk 2 i + u of a row lies at the row's chunk 0 with those bits flipped)
  const int k_store = k_at(t >> 2, (t & 3) * 2), v_store = v_at(lane, 2 * w);
  // Unit j of 4 * PIECES = DS: half a piece, eight codes.
  auto store = [&](char* base, int j) {
    const int i = j >> 2, u = j & 1;
    if (j & 2) *(half8v*)(base + (v_store ^ (u << 4)) + 64 * i * 128) = operand(vc[i][2 * u], vc[i][2 * u + 1]);
    else *(half8v*)(base + (k_store ^ ((8 * i + u) << 4))) = operand(kc[i][2 * u], kc[i][2 * u + 1]);
  };
  static_assert(4 * PIECES == DS, "a unit a step of the scores");

  float16v o[DT];
  Frame at;
  float l;
  bool bad = false;  // (a lane's)

  const int key = 16 * (lr >> 4) + 8 * (lr >> 2 & 1) + 4 * (lr >> 3 & 1) + (lr & 3);
  const int k_read = k_at(key, h), v_read = v_at(lr, h);
  Scales after{};
  int pg = -1;
  // Stage st in `base`, while `other` takes the next one.
  auto compute = [&](auto APART_, int st, const char* base, char* other, const Scales& sc) {
    constexpr bool APART = decltype(APART_)::value;
    // each lane's piece, then the four as scalars
    float lane_lv, lane_rv;
    value_scale(sc.v, APART, lane_lv, lane_rv);
    if (sc.b < 0) lane_lv = -INFINITY;
    const float lane_ks = sc.b < 0 ? 0.f : sc.k;
    const uint64_t there = __ballot(sc.b >= 0);
    if (!APART) bad |= sc.b >= 0 && !near_one(sc.v);
    const bool all = !APART && st * 64 + 64 <= kfull && there == ~0ull;
    float ks[4], lv[4], rv[4];
    auto lane_of = [](float v, int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i)); };
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      ks[x] = lane_of(lane_ks, x);
      lv[x] = lane_of(lane_lv, x);
      rv[x] = lane_of(lane_rv, x);
    }
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
    read_k(0);
#pragma unroll
    for (int x = 0; x < DS; ++x) {
      if (x + 1 < DS) read_k(x + 1);
      else read_v(0);
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
        s[nb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[x & 1][nb], qf[x], x == 0 ? float16v{} : s[nb], 0, 0, 0);
      // (conversion passes under the score MFMAs, which need few vector
      // instructions; past the last stage old codes go where nobody reads)
      store(other, x);
      __builtin_amdgcn_sched_barrier(0);
    }
    // (the codes' registers are free)
    if (st + 2 < c1) after = load(st + 2, pg);
    if (st + 3 < c1) pg = page(st + 3);
    // the largest weighted score of the keys that are seen: the first `left` + 1
    // of a lane's eight of a piece (all of a piece: more than that)
    int left[4];
    float mx = -INFINITY;
    if (all) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        left[x] = 8;
        float m = s[x >> 1][8 * (x & 1)];
#pragma unroll
        for (int e = 1; e < 8; ++e) m = fmaxf(m, s[x >> 1][8 * (x & 1) + e]);
        mx = fmaxf(mx, fmaf(m, c * ks[x], lv[x]));
      }
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        left[x] = there >> x & 1 ? last - (st * 64 + x * 16 + 8 * h) : -1;
        float m = -INFINITY;
        if constexpr (APART) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = e > left[x] ? -INFINITY : times(s[x >> 1][8 * (x & 1) + e], c * ks[x]);
            s[x >> 1][8 * (x & 1) + e] = v;
            mx = fmaxf(mx, v);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) m = fmaxf(m, e > left[x] ? -INFINITY : s[x >> 1][8 * (x & 1) + e]);
          mx = fmaxf(mx, left[x] < 0 ? -INFINITY : fmaf(m, c * ks[x], lv[x]));
        }
      }
    }
    auto both = [](float v) {  // the maximum of the two lanes of a row
      const auto v2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      return fmaxf(__uint_as_float(v2[0]), __uint_as_float(v2[1]));
    };
    mx = both(mx);
    float ref, f = 1.f;  // a weight is relative to 2^ref
    bool up = true;
    if constexpr (APART) {
      l *= at.raise(mx);
      const float m = at.m == -INFINITY ? 0.f : at.m;
      float cand = -INFINITY;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float most = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = s[x >> 1][8 * (x & 1) + e] - m;
          s[x >> 1][8 * (x & 1) + e] = v;
          most = fmaxf(most, v);
          l += __builtin_amdgcn_exp2f(v);
        }
        cand = fmaxf(cand, left[x] < 0 ? -INFINITY : left_out(most, lv[x]));
      }
      f = at.raise_o(both(cand));
      ref = at.d;
    } else {
      up = __any(mx > at.m + kHigh);
      if (up) {
        bad |= mx > at.m + kHigh && fabsf(mx) >= kFar;
        const float now = mx > at.m + kHigh ? mx - kLow : at.m;
        f = rel_exp2(at.m, now);
        l *= f;
        at.m = now;
      }
      ref = at.m;
    }
    if (up) {
#pragma unroll
      for (int x = 0; x < DT; ++x) o[x] *= f;
    }
    ref = ref == -INFINITY ? 0.f : ref;
    // the weights of 16 keys while the MFMAs of the 16 before run
    auto weights = [&](int x) {
      const float off = lv[x] - ref, cs = APART ? 1.f : c * ks[x];
      float v[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __builtin_amdgcn_exp2f(fmaf(s[x >> 1][8 * (x & 1) + e], cs, off));
      if (!all) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e > left[x] ? 0.f : v[e];
      }
      half8v p;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum += v[e];
        p[e] = (_Float16)v[e];
      }
      if (!APART) l += sum == 0.f ? 0.f : sum * rv[x];  // (rv is of no use where nothing is seen)
      return p;
    };
    half8v p = weights(0);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      half8v after = p;
      if (x < 3) {
        read_v(x + 1);
        after = weights(x + 1);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[x & 1][dt], p, o[dt], 0, 0, 0);
      p = after;
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  auto pass = [&](auto APART) {
    at = Frame{-INFINITY, 0.f};
    l = 0.f;
#pragma unroll
    for (int x = 0; x < DT; ++x) o[x] = float16v{};
    if (c0 >= c1) return;
    // Ahead of the stage computed: the next one's codes on their way into LDS,
    // codes and scales of the one after, pages of the one after that.
    Scales now = load(c0, page(c0)), next{};
#pragma unroll
    for (int x = 0; x < DS; ++x) store(lds, x);
    if (c0 + 1 < c1) next = load(c0 + 1, page(c0 + 1));
    if (c0 + 2 < c1) pg = page(c0 + 2);
    auto step = [&](int st, char* base, char* other) {
      __syncthreads();  // stage st is written, and nobody reads the other one
      compute(APART, st, base, other, now);
      now = next;
      next = after;
    };
    for (int st = c0; st < c1; st += 2) {  // (LDS addresses that differ by constants)
      step(st, lds, lds + STAGE);
      if (st + 1 < c1) step(st + 1, lds + STAGE, lds);
    }
  };
  if (t == 0) odd = 0;
  pass(std::false_type{});
  __syncthreads();  // (nobody reads a stage any more)
  if (bad) odd = 1;
  __syncthreads();
  if (odd) pass(std::true_type{});

  // A wave's floats: o, its frame, l; a tile's shares joined as in the kernel above.
  auto each = [&](auto&& f) {
#pragma unroll
    for (int x = 0; x < DT; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) f(x * 16 + i, [&](float v) { o[x][i] = v; }, o[x][i]);
    f(DT * 16, [&](float v) { at.m = v; }, at.m);
    f(DT * 16 + 1, [&](float v) { at.d = v; }, at.d);
    f(DT * 16 + 2, [&](float v) { l = v; }, l);
  };
  if (nsplit > 1) {
    constexpr int kCoherent = 17;  // sc0 | sc1
    constexpr int PART = 4 * NV * 64 * 4;
    const __amdgpu_buffer_rsrc_t rP =
        make_rsrc(a.ws + kWsCounterBytes + (int64_t)(item - a.full) * nsplit * PART, (uint32_t)(nsplit * PART));
    each([&](int i, auto&&, float v) {
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
    auto frame = [&](int sp) { return Frame{held(sp, DT * 16), held(sp, DT * 16 + 1)}; };
    at = Frame{-INFINITY, 0.f};
#pragma unroll 4
    for (int sp = 0; sp < nsplit; ++sp) {
      Frame two[2] = {at, frame(sp)};
      float fl[2], fo[2];
      join_frames(two, fl, fo);
      at = two[0];
    }
    l = 0.f;
#pragma unroll
    for (int x = 0; x < DT; ++x) o[x] = float16v{};
    for (int sp = 0; sp < nsplit; ++sp) {  // (in this order whichever came last)
      const Frame to = frame(sp).from(at.m);
      const float f = rel_exp2(to.d, at.d);
      l += __builtin_amdgcn_exp2f(to.m) * held(sp, DT * 16 + 2);
#pragma unroll
      for (int x = 0; x < DT; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[x][i] += f * held(sp, x * 16 + i);
    }
  }

  // O: lane holds row l % 32, dims 32 x + 8 g + 4 h + 0..3
  const auto l2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
  const float whole = __uint_as_float(l2[0]) + __uint_as_float(l2[1]);
  const float f = at.over(whole);
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

int64_t part_bytes(const KvAttnProblem& p, const KvPlan& k) {  // of a tile's share
  const int64_t dt = p.d <= 64 ? 4 : 8;
  return k.rt == 16 ? (dt * 4 + 3) * 64 * 4 : 4 * (dt * 8 + 3) * 64 * 4;
}

template <typename T>
hipError_t launch_t(int64_t d, int rt, dim3 grid, const KArgs& a, hipStream_t stream) {
  const bool small = d <= 64, whole = d == 64 || d == 128;
  const auto fn = rt == 16 ? (small ? whole ? kv_attention<T, 1, true> : kv_attention<T, 1, false>
                                    : whole ? kv_attention<T, 2, true> : kv_attention<T, 2, false>)
                           : (small ? whole ? kv_attention_tiles<T, 64, true> : kv_attention_tiles<T, 64, false>
                                    : whole ? kv_attention_tiles<T, 128, true> : kv_attention_tiles<T, 128, false>);
  hipLaunchKernelGGL(fn, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

int64_t kv_attention_workspace_bytes(const KvAttnProblem& p) {
  const KvPlan k = plan_of(p);
  return k.nsplit > 1 ? kWsCounterBytes + (k.tiles * p.kv_heads - k.full) * k.nsplit * part_bytes(p, k) : 0;
}

hipError_t launch_kv_attention(const KvAttnProblem& p, hipStream_t stream) {
  KvPlan k = plan_of(p);
  const int64_t items = k.tiles * p.kv_heads;
  if (k.nsplit > 1 && (!p.ws || p.ws_bytes < kv_attention_workspace_bytes(p))) {
    k.nsplit = 1;
    k.full = items;
  }
  const int64_t grid = k.full + (items - k.full) * k.nsplit;
  static_assert(512 <= kWsMaxTiles, "a counter for every shared tile");
  if (grid >= (1ll << 31)) return hipErrorInvalidValue;
  KArgs a{};
  a.k = p.k_codes;
  a.v = p.v_codes;
  a.ks = p.k_scale;
  a.vs = p.v_scale;
  a.dp = (int)((p.d + 15) / 16 * 16);
  a.bytes = p.block * a.dp;
  tile_args(p, k, a);
  const dim3 blocks((unsigned)grid);
  return p.dtype == DT_BF16 ? launch_t<__bf16>(p.d, k.rt, blocks, a, stream) : launch_t<_Float16>(p.d, k.rt, blocks, a, stream);
}

}  // namespace hxmi
