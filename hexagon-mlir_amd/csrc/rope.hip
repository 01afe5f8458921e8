// Queries and keys at their positions: each head of a token normalised (where a
// weight is given) and its pairs of dimensions turned,
//   y = x * rsqrt(mean(x^2) + eps) * w
//   (a, b) -> s (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq
// rounded once.  Pair i is dims i and i + R/2 of the first R ("halves") or 2 i
// and 2 i + 1; with several axes (time, height, width) pair i takes the
// position of its own axis.
//
// A pair's angle goes round once in 2 pi / inv_freq tokens, so positions in the
// hundred thousands leave fp32 nothing of the fraction that counts: position *
// (inv_freq / 2 pi) is taken in 64 bits and its whole turns dropped (at inv_freq 1 off
// by 2^-32 radians at position 2^20, 2^-21 at 2^31); cosine and sine are polynomials
// in 32 bits over an eighth of a turn either way.
//
// A workgroup takes a few tokens: a thread computes each pair's cosine and
// sine into LDS, once for all heads, then groups of lanes take heads, a lane the
// same eight pairs (16 values) of every one, the next head's in flight meanwhile.
// Memory bounds it: 16384 tokens of 40 heads of 128 dims with norms 74 us (336 MB at 4.5
// TB/s; 98 without the head ahead); one token of 36 heads of 64 2.9 us, a launch
// and three dependent loads.
#include "hxmi_common.h"
#include "hxmi_internal.h"

namespace hxmi {
namespace {

typedef int int4u __attribute__((ext_vector_type(4), aligned(2)));  // (rows start anywhere)
typedef int int4f __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kMaxPairs = 256;  // of a workgroup's tokens

struct RArgs {
  const char* x[2];  // q, k
  char* y[2];
  const char* w[2];  // or null
  int64_t ld[2], hs[2], ldo[2], hso[2];
  const void* pos;
  const double* freq;
  const int* axis;
  int64_t ldp, tokens;
  int heads, all, d, pairs, axes;  // heads of q, of both
  int tb;                          // tokens of a workgroup
  int pos64, w32;
  float eps, scale, inv_d;
};

// Cosine and sine of 2 pi `turns`.
__device__ __forceinline__ float2 cos_sin(double turns) {
  const double x = 4.0 * (turns - __builtin_rint(turns)), n = __builtin_rint(x);  // quarters
  const float r = (float)((x - n) * 1.57079632679489661923), z = r * r;
  // Taylor to r^9 and r^10: what is left out is below 2^-29 at pi / 4
  float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(s, z, 8.3333333e-3f);
  s = fmaf(s, z, -1.6666667e-1f);
  s = fmaf(s * z, r, r);
  float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(c, z, -1.3888889e-3f);
  c = fmaf(c, z, 4.1666667e-2f);
  c = fmaf(c, z, -0.5f);
  c = fmaf(c, z, 1.f);
  const int q = (int)n & 3;  // (a NaN stays one through r)
  const float cq = q & 1 ? s : c, sq = q & 1 ? c : s;
  return make_float2(q == 1 || q == 2 ? -cq : cq, q & 2 ? -sq : sq);
}

template <typename T>
__device__ __forceinline__ void floats(const int4v& raw, float (&f)[8]) {
  T t[8];
  __builtin_memcpy(t, &raw, 16);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (float)t[e];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  T t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = (T)f[e];
  int4v raw;
  __builtin_memcpy(&raw, t, 16);
  *(int4u*)p = raw;
}

// How a lane's values lie in a head.
enum Form {
  kWhole,  // eight pairs of halves, or eight values past them: R a multiple of 16
  kSplit,  // eight values of halves, their partners loaded one by one: any R
  kNext,   // four pairs of neighbours
};

// 2^log lanes a head.
template <typename T, int FORM, bool NORM>
__global__ __launch_bounds__(256) void qk_rope(RArgs a, int log) {
  __shared__ __attribute__((aligned(16))) float cs[kMaxPairs], sn[kMaxPairs];
  const int64_t t0 = (int64_t)blockIdx.x * a.tb;
  const int nt = (int)min((int64_t)a.tb, a.tokens - t0), pairs = a.pairs;
  const int u = threadIdx.x & ((1 << log) - 1), slot = threadIdx.x >> log, slots = 256 >> log;
  const int half = pairs, rot = 2 * pairs;
  // the lane's values: d0 on, and (kWhole) their partners d1 on
  const int whole = pairs >> 3;
  const bool turned = FORM == kWhole ? u < whole : u * 8 < rot;
  const int d0 = FORM == kWhole ? (turned ? u * 8 : rot + (u - whole) * 8) : u * 8;
  const bool in = d0 < a.d;
  constexpr int NV = FORM == kWhole ? 16 : 8;
  float wq[NV], wk[NV];

  // Head i of the workgroup's: its pieces, loaded a head ahead (what is in flight
  // belongs to no head that is written meanwhile, in place or not).
  struct Head {
    int t, h;  // h: k's heads after q's
  };
  auto after = [&](Head n) {
    n.h += slots;
    while (n.h >= a.all) {
      n.h -= a.all;
      ++n.t;
    }
    return n;
  };
  auto row = [&](const Head& n) {
    const int is_k = n.h >= a.heads;
    return (const T*)a.x[is_k] + (t0 + n.t) * a.ld[is_k] + (n.h - (is_k ? a.heads : 0)) * a.hs[is_k];
  };
  int4v v_raw{}, w_raw{};
  auto load = [&](const T* x) {
    if (in) v_raw = *(const int4u*)(x + d0);
    if (FORM == kWhole && turned) w_raw = *(const int4u*)(x + half + d0);
  };
  Head now = after(Head{0, slot - slots});
  if (now.t < nt) load(row(now));
  for (int i = threadIdx.x; i < nt * pairs; i += 256) {
    const int t = i / pairs, p = i - t * pairs;
    const int ax = a.axis ? min(max(a.axis[p], 0), a.axes - 1) : 0;
    const int64_t at = ax * a.ldp + t0 + t;
    const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int*)a.pos)[at];
    const float2 v = cos_sin(pos * (a.freq[p] * 0.15915494309189533577));
    cs[i] = v.x * a.scale;
    sn[i] = v.y * a.scale;
  }
  __syncthreads();

  if constexpr (NORM) {
    auto eight = [&](const char* w, int d, float* f) {
      float t[8];
      if (a.w32) {
        const int4v lo = *(const int4f*)(w + 4 * d), hi = *(const int4f*)(w + 4 * d + 16);
        __builtin_memcpy(t, &lo, 16);
        __builtin_memcpy(t + 4, &hi, 16);
      } else {
        floats<T>(*(const int4u*)(w + 2 * d), t);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = t[e];
    };
    auto weights = [&](const char* w, float (&f)[NV]) {
#pragma unroll
      for (int e = 0; e < NV; ++e) f[e] = 1.f;
      if (w && in) eight(w, d0, f);
      if (FORM == kWhole && w && turned) eight(w, half + d0, f + NV - 8);
    };
    weights(a.w[0], wq);
    weights(a.w[1], wk);
  }

  for (Head next; now.t < nt; now = next) {  // (a head's lanes stay together)
    const int is_k = now.h >= a.heads;
    T* const y = (T*)a.y[is_k] + (t0 + now.t) * a.ldo[is_k] + (now.h - (is_k ? a.heads : 0)) * a.hso[is_k];
    const float *const c = cs + now.t * pairs, *const s = sn + now.t * pairs;
    float v[8] = {}, w[8] = {};
    if (in) floats<T>(v_raw, v);
    if (FORM == kWhole && turned) floats<T>(w_raw, w);
    next = after(now);
    if (next.t < nt) load(row(next));
    if constexpr (FORM == kSplit) {
      const T* const x = row(now);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        w[e] = d < half ? (float)x[d + half] : d < rot ? (float)x[d - half] : 0.f;
      }
    }
    if constexpr (NORM) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum = fmaf(v[e], v[e], sum);
        if constexpr (FORM == kWhole) sum = fmaf(w[e], w[e], sum);
      }
      for (int o = 1; o < 1 << log; o <<= 1) sum += __shfl_xor(sum, o, 64);
      const bool has = a.w[is_k] != nullptr;
      const float f = has ? __builtin_amdgcn_rsqf(fmaf(sum, a.inv_d, a.eps)) : 1.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] *= f * (is_k ? wk[e] : wq[e]);
        if constexpr (FORM == kWhole) w[e] *= f * (is_k ? wk[8 + e] : wq[8 + e]);
        if constexpr (FORM == kSplit) {
          const int d = d0 + e, dp = d < half ? d + half : d < rot ? d - half : d;
          const char* const wt = a.w[is_k];
          if (has && in) w[e] *= f * (a.w32 ? ((const float*)wt)[dp] : (float)((const T*)wt)[dp]);
        }
      }
    }
    if constexpr (FORM == kWhole) {
      if (turned) {
        float o[8];
#pragma unroll
        for (int x = 0; x < 8; x += 4) {
          const float4v ce = *(const float4v*)(c + d0 + x), se = *(const float4v*)(s + d0 + x);  // (pairs: a multiple of 8)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = v[x + j], r = w[x + j];
            v[x + j] = p * ce[j] - r * se[j];
            o[x + j] = r * ce[j] + p * se[j];
          }
        }
        store8(y + half + d0, o);
      }
    } else if constexpr (FORM == kSplit) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        if (d < half) v[e] = v[e] * c[d] - w[e] * s[d];
        else if (d < rot) v[e] = v[e] * c[d - half] + w[e] * s[d - half];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const int p = (d0 + e) >> 1;
        if (p < pairs) {
          const float x0 = v[e], x1 = v[e + 1];
          v[e] = x0 * c[p] - x1 * s[p];
          v[e + 1] = x1 * c[p] + x0 * s[p];
        }
      }
    }
    if (in) store8(y + d0, v);
  }
}

template <typename T, int FORM>
auto pick(bool norm) {
  return norm ? qk_rope<T, FORM, true> : qk_rope<T, FORM, false>;
}
template <typename T>
auto pick(int form, bool norm) {
  return form == kWhole ? pick<T, kWhole>(norm) : form == kSplit ? pick<T, kSplit>(norm) : pick<T, kNext>(norm);
}

}  // namespace

hipError_t launch_qk_rope(const RopeProblem& p, hipStream_t stream) {
  RArgs a{};
  a.x[0] = (const char*)p.q;
  a.x[1] = (const char*)p.k;
  a.y[0] = (char*)p.q_out;
  a.y[1] = (char*)p.k_out;
  a.w[0] = (const char*)p.q_weight;
  a.w[1] = (const char*)p.k_weight;
  const int64_t strides[4][2] = {{p.ldq, p.ldk}, {p.hsq, p.hsk}, {p.ldqo, p.ldko}, {p.hsqo, p.hsko}};
  for (int i = 0; i < 2; ++i) {
    a.ld[i] = strides[0][i];
    a.hs[i] = strides[1][i];
    a.ldo[i] = strides[2][i];
    a.hso[i] = strides[3][i];
  }
  a.pos = p.positions;
  a.freq = p.inv_freq;
  a.axis = p.axis;
  a.ldp = p.ldp;
  a.tokens = p.tokens;
  a.heads = (int)p.heads;
  a.all = (int)(p.heads + p.kv_heads);
  a.d = (int)p.d;
  a.pairs = (int)(p.rotary / 2);
  a.axes = (int)p.axes;
  a.pos64 = p.pos64;
  a.w32 = p.w32;
  a.eps = p.eps;
  a.inv_d = 1.f / (float)p.d;
  a.scale = p.scale;
  const int form = p.interleaved ? kNext : p.rotary % 16 == 0 ? kWhole : kSplit;
  const int units = form == kWhole ? (int)(p.rotary / 16 + (p.d - p.rotary) / 8) : (int)(p.d / 8);
  int log = 0;
  while (1 << log < units) ++log;  // (up to 32 lanes: 256 dims)
  // a thread an angle where there are tokens enough for every CU
  a.tb = a.pairs ? kMaxPairs / a.pairs : 8;
  while (a.tb > 1 && (p.tokens + a.tb - 1) / a.tb < 1024) a.tb /= 2;
  a.tb = a.tb > 8 ? 8 : a.tb;
  const int64_t blocks = (p.tokens + a.tb - 1) / a.tb;
  if (blocks >= (1ll << 31)) return hipErrorInvalidValue;
  const bool norm = p.q_weight || p.k_weight;
  const auto fn = p.dtype == DT_BF16 ? pick<__bf16>(form, norm) : pick<_Float16>(form, norm);
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), 0, stream, a, log);
  return hipGetLastError();
}

}  // namespace hxmi
