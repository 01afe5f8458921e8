// A token a row from logits: temperature, top-k, top-p, min-p and the
// inverse of the kept tokens' distribution at a given u, in index order.
//
//   w_i = exp((x_i - max x) / T)
//   top-k   the k largest (of equal ones the lowest indices)
//   top-p   in descending order (of equal ones the lowest index first) while
//           the weight of the tokens before is < p * (weight of the top k)
//   min-p   w_i >= min_p
//   token   the lowest kept i whose running weight exceeds u * (kept weight)
//
// Weights are integers, round(w * 2^shift) with room for the whole row's sum
// in 62 bits (44 fraction bits at a vocabulary of 2^18): integer sums do not
// depend on their order, so neither does the token, and every comparison above
// is exact in them (p * sum and u * sum as 128-bit products).  w comes from a
// 64-bit evaluation good to 2^-48, a few 2^-45 of the largest weight in all.
// fp32 sums would put about one row in a hundred of a flat distribution on
// another token.
//
// One workgroup a row.  top-k and top-p are thresholds on the logits: a radix
// descent over order-preserving integer keys (8 bits a pass; 16-bit logits
// have 16-bit keys, fp32 ones 32) gives the key of the last token kept and
// how many of its equals stay.  The pass's histogram has a column for each
// lane: no two lanes of a wave meet in one counter however the logits
// cluster.  The last passes sum the kept weights by pieces of 512 tokens,
// then look inside one piece.  Bound by the passes over a row in L2 (2-3 us
// each at 151936 16-bit logits) and the 64-bit weights.
#include "hxmi_common.h"
#include "hxmi_internal.h"

namespace hxmi {
namespace {

typedef int int4u2 __attribute__((ext_vector_type(4), aligned(2)));
typedef int int4u4 __attribute__((ext_vector_type(4), aligned(4)));

struct SArgs {
  const char* x;
  const float* u;
  const float* temperature;  // a row's own, or null: t
  const int* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* token;
  int64_t ldx;
  int vocab, shift;
  float t, p, m;
  int k;
};

constexpr int NT = 1024, NW = NT / 64, PIECE = 512;
constexpr int kMaxPieces = kSampleMaxVocab / PIECE;

// Keys that order as the logits do, equal for -0 and 0.
template <typename T>
struct Key;
template <>
struct Key<_Float16> {
  static constexpr int bits = 16;
  static __device__ __forceinline__ uint32_t of(_Float16 v) {
    const uint32_t b = __builtin_bit_cast(unsigned short, (_Float16)(v + (_Float16)0.f));
    return b & 0x8000u ? 0xffffu & ~b : b | 0x8000u;
  }
};
template <>
struct Key<__bf16> {
  static constexpr int bits = 16;
  static __device__ __forceinline__ uint32_t of(__bf16 v) {
    uint32_t b = __builtin_bit_cast(unsigned short, v);
    b = b == 0x8000u ? 0 : b;
    return b & 0x8000u ? 0xffffu & ~b : b | 0x8000u;
  }
};
template <>
struct Key<float> {
  static constexpr int bits = 32;
  static __device__ __forceinline__ uint32_t of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
};

// 2^(j / 32)
struct Exp2Table {
  double v[32];
};
__device__ __forceinline__ double exp2_poly(double r) {
  // 2^r = e^(r ln 2) for |r| <= 1/64, Taylor to degree 6: the next term is below 2^-58
  const double z = r * 0.69314718055994530942;
  double p = 1.0 / 720;
  p = __builtin_fma(p, z, 1.0 / 120);
  p = __builtin_fma(p, z, 1.0 / 24);
  p = __builtin_fma(p, z, 1.0 / 6);
  p = __builtin_fma(p, z, 0.5);
  p = __builtin_fma(p, z, 1.0);
  return __builtin_fma(p, z, 1.0);
}
// w * 2^shift for y = log2 w <= 0 (0 far below).
__device__ __forceinline__ double weight(double y, int shift, const double* table) {
  y = y > -1000.0 ? y : -1000.0;
  const double k = __builtin_rint(y * 32.0);
  const int j = (int)k;
  return __builtin_ldexp(table[j & 31] * exp2_poly(__builtin_fma(k, -1.0 / 32, y)), (j >> 5) + shift);
}
__device__ __forceinline__ uint64_t to_fixed(double w) { return (uint64_t)__builtin_rint(w); }

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__shfl((int)(v >> 32), lane, 64) << 32) | (uint32_t)__shfl((int)v, lane, 64);
}
__device__ __forceinline__ uint64_t scan64(uint64_t v) {  // inclusive, over the wave
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t t = __shfl_up((unsigned long long)v, o, 64);
    if (lane >= o) v += t;
  }
  return v;
}
// floor(f * 2^64) of f in [0, 1)
__device__ __forceinline__ uint64_t fraction64(float f) {
  return (uint64_t)((double)f * 0x1p32) << 32 |
         (uint64_t)(((double)f * 0x1p32 - __builtin_floor((double)f * 0x1p32)) * 0x1p32);
}

struct Shared {
  union {
    unsigned long long mass[256][64];
    uint32_t count[256][64];
    struct {
      unsigned long long sum[kMaxPieces];  // kept weight of a piece, less its equals of the last key
      uint32_t ties[kMaxPieces];
    } piece;
  };
  double table[32];
  unsigned long long part[NW];
  uint32_t upart[NW];
  uint32_t key;
  unsigned long long above;
};

// The eight logits of piece-lane i (8 i .. 8 i + 7); `n` of them exist.
template <typename T>
__device__ __forceinline__ int load8(const T* x, int i, int vocab, T (&v)[8]) {
  const int at = i * 8, n = vocab - at;
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) {
      const int4v r = *(const int4u2*)(x + at);
      __builtin_memcpy(v, &r, 16);
    } else {
      const int4v r0 = *(const int4u4*)(x + at), r1 = *(const int4u4*)(x + at + 4);
      __builtin_memcpy(v, &r0, 16);
      __builtin_memcpy(v + 4, &r1, 16);
    }
    return 8;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < n ? x[at + e] : (T)0.f;
  return n < 0 ? 0 : n;
}

template <typename T>
__global__ __launch_bounds__(NT) void sample_rows(SArgs a) {
  __shared__ __attribute__((aligned(16))) Shared sh;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const T* const x = (const T*)a.x + row * a.ldx;
  const int lanes = (a.vocab + 7) >> 3;  // groups of eight logits
  constexpr int KB = Key<T>::bits;

  if (threadIdx.x < 32) sh.table[threadIdx.x] = exp2((double)threadIdx.x / 32);

  // the largest logit and its first index
  uint32_t top = 0, first = 0;
  bool bad = false;
  for (int i = threadIdx.x; i < lanes; i += NT) {
    T v[8];
    const int n = load8(x, i, a.vocab, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= n) continue;
      const uint32_t key = Key<T>::of(v[e]);
      bad |= v[e] != v[e];
      if (key > top) {  // (a lane's indices grow)
        top = key;
        first = i * 8 + e;
      }
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint32_t k2 = __shfl_xor((int)top, o, 64), f2 = __shfl_xor((int)first, o, 64);
    if (k2 > top || (k2 == top && f2 < first)) {
      top = k2;
      first = f2;
    }
  }
  bad = __any(bad);
  if (lane == 0) {
    sh.part[w] = ((unsigned long long)top << 32) | first;
    sh.upart[w] = bad;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const uint32_t k2 = (uint32_t)(sh.part[i] >> 32), f2 = (uint32_t)sh.part[i];
    bad |= sh.upart[i] != 0;
    if (k2 > top || (k2 == top && f2 < first)) {
      top = k2;
      first = f2;
    }
  }
  const float xmax = (float)x[first];
  const float t = a.temperature ? a.temperature[row] : a.t;
  if (bad || xmax == -INFINITY || !(t > 0.f)) {
    if (threadIdx.x == 0) a.token[row] = bad || xmax == -INFINITY ? -1 : (int64_t)first;
    return;
  }
  const double rate = 1.44269504088896340736 / (double)t;
  // (the largest logit's weight is 1 also where it is infinite)
  auto weight_of = [&](float v) {
    return v == xmax ? __builtin_ldexp(1.0, a.shift) : weight(((double)v - (double)xmax) * rate, a.shift, sh.table);
  };

  // Descends to the key at which the counts (or weights) from the largest key
  // down first reach `goal`; `above`: what lies over that key.
  auto descend = [&](auto COUNT_, uint64_t goal, uint64_t& above) {
    constexpr bool COUNT = decltype(COUNT_)::value;
    uint32_t prefix = 0;
    above = 0;
    for (int b = KB - 8; b >= 0; b -= 8) {
      __syncthreads();
      for (int i = threadIdx.x; i < 256 * 64; i += NT) {
        if constexpr (COUNT) ((uint32_t*)sh.count)[i] = 0;
        else ((unsigned long long*)sh.mass)[i] = 0;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < lanes; i += NT) {
        T v[8];
        const int n = load8(x, i, a.vocab, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t key = Key<T>::of(v[e]);
          if (e < n && (b + 8 >= KB || key >> (b + 8) == prefix)) {
            if constexpr (COUNT) atomicAdd(&sh.count[(key >> b) & 255][lane], 1u);
            else atomicAdd(&sh.mass[(key >> b) & 255][lane], (unsigned long long)to_fixed(weight_of((float)v[e])));
          }
        }
      }
      __syncthreads();
      // Each wave sums 16 digits' columns; then wave 0 looks for the digit.
      for (int d = w * 16; d < w * 16 + 16; ++d) {
        uint64_t s;
        if constexpr (COUNT) s = sh.count[d][lane];
        else s = sh.mass[d][lane];
        s = scan64(s);
        if (lane == 63) {  // (column 0 of the digit's row: only this wave reads it)
          if constexpr (COUNT) sh.count[d][0] = (uint32_t)s;
          else sh.mass[d][0] = s;
        }
      }
      __syncthreads();
      if (w == 0) {
        uint64_t own[4], sum = 0;  // digits 255 - 4 lane .. 252 - 4 lane
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (COUNT) own[j] = sh.count[255 - 4 * lane - j][0];
          else own[j] = sh.mass[255 - 4 * lane - j][0];
          sum += own[j];
        }
        const uint64_t incl = scan64(sum);
        const uint64_t reach = __ballot(above + incl >= goal);
        const int at = __ffsll((unsigned long long)reach) - 1;  // (some lane: the whole reaches the goal)
        if (lane == at) {
          uint64_t over = above + incl - sum;
          int j = 0;
          for (; j < 3 && over + own[j] < goal; ++j) over += own[j];
          sh.key = (prefix << 8) | (uint32_t)(255 - 4 * lane - j);
          sh.above = over;
        }
      }
      __syncthreads();
      prefix = sh.key;
      above = sh.above;
    }
    return prefix;
  };

  // Kept: keys over `tau`, and the first `equal` tokens whose key is tau.
  uint32_t tau = 0;
  uint32_t equal = 0xffffffffu;
  const int k = a.top_k ? a.top_k[row] : a.k;
  if (k > 0 && k < a.vocab) {
    uint64_t above;
    tau = descend(std::true_type{}, (uint64_t)k, above);
    equal = (uint32_t)((uint64_t)k - above);
  }
  auto value_of = [&](uint32_t key) -> float {
    if constexpr (KB == 32) return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
    else return (float)__builtin_bit_cast(T, (unsigned short)(key & 0x8000u ? key & 0x7fffu : ~key));
  };

  // Sum over the workgroup of what each piece keeps; fills the pieces' sums
  // and equals of tau.
  const int pieces = (lanes + 63) >> 6;
  const float mp = a.min_p ? a.min_p[row] : a.m;
  auto pieces_of = [&](double least) {
    __syncthreads();
    for (int c = w; c < pieces; c += NW) {
      T v[8];
      const int n = load8(x, c * 64 + lane, a.vocab, v);
      uint64_t sum = 0;
      uint32_t ties = 0;
      bool over = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t key = Key<T>::of(v[e]);
        over |= e < n && key > tau;
        ties += e < n && key == tau;
      }
      if (__any(over)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (e < n && Key<T>::of(v[e]) > tau) {
            const double wd = weight_of((float)v[e]);
            sum += wd >= least ? to_fixed(wd) : 0;
          }
        }
        sum = scan64(sum);
      }
      if (__any(ties != 0)) ties = (uint32_t)scan64(ties);
      if (lane == 63) {
        sh.piece.sum[c] = sum;
        sh.piece.ties[c] = ties;
      }
    }
    __syncthreads();
  };
  // Wave 0: sums of the pieces with the first `equal` ties of weight wt.
  auto total_of = [&](uint64_t wt) {
    uint64_t sum = 0, seen = 0;
    for (int c0 = 0; c0 < pieces; c0 += 64) {
      const int c = c0 + lane;
      const uint64_t ties = c < pieces ? sh.piece.ties[c] : 0;
      const uint64_t incl = scan64(ties), before = seen + incl - ties;
      const uint64_t kept = before >= equal ? 0 : min(ties, (uint64_t)equal - before);
      seen = shfl64(seen + incl, 63);
      const uint64_t s = scan64((c < pieces ? sh.piece.sum[c] : 0) + kept * wt);
      sum += shfl64(s, 63);
    }
    return sum;
  };

  const float p = a.top_p ? a.top_p[row] : a.p;
  if (!(p >= 1.f)) {
    pieces_of(0.0);
    if (w == 0) {
      const uint64_t sum = total_of(to_fixed(weight_of(value_of(tau))));
      if (lane == 0) sh.above = sum;
    }
    __syncthreads();
    const uint64_t whole = sh.above;
    const uint64_t f = fraction64(p > 0.f ? p : 0.f);
    uint64_t goal = __umul64hi(f, whole) + (f * whole != 0);  // ceil(p * whole)
    goal = goal > 1 ? goal : 1;
    uint64_t above;
    tau = descend(std::false_type{}, goal, above);
    const uint64_t wt = to_fixed(weight_of(value_of(tau)));
    equal = (uint32_t)min((goal - above + wt - 1) / wt, (uint64_t)0xffffffffu);
    __syncthreads();
  }

  const double one = __builtin_ldexp(1.0, a.shift);
  const double least = mp > 0.f ? (double)fminf(mp, 1.f) * one : 0.0;
  pieces_of(least);
  if (w != 0) return;
  const double wtd = weight_of(value_of(tau));
  const uint64_t wt = wtd >= least ? to_fixed(wtd) : 0;
  const uint64_t whole = total_of(wt);
  float u = a.u[row];
  u = u > 0.f ? (u < 1.f ? u : 0x1.fffffep-1f) : 0.f;
  const uint64_t goal = __umul64hi(fraction64(u), whole);  // floor(u * whole) < whole

  // the piece, then the token in it, whose running weight first exceeds the goal
  uint64_t sum = 0, seen = 0;
  int at = 0;
  for (int c0 = 0; c0 < pieces; c0 += 64) {
    const int c = c0 + lane;
    const uint64_t ties = c < pieces ? sh.piece.ties[c] : 0;
    const uint64_t incl = scan64(ties), before = seen + incl - ties;
    const uint64_t kept = before >= equal ? 0 : min(ties, (uint64_t)equal - before);
    const uint64_t own = (c < pieces ? sh.piece.sum[c] : 0) + kept * wt, s = sum + scan64(own);
    const uint64_t reach = __ballot(s > goal);
    if (reach) {
      const int l = __ffsll((unsigned long long)reach) - 1;
      at = c0 + l;
      sum = shfl64(s - own, l);
      seen = shfl64(before, l);
      break;
    }
    sum = shfl64(s, 63);
    seen = shfl64(seen + incl, 63);
  }
  T v[8];
  const int n = load8(x, at * 64 + lane, a.vocab, v);
  uint32_t ties = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) ties += e < n && Key<T>::of(v[e]) == tau;
  uint64_t before = seen + scan64(ties) - ties, own[8], mine = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t key = Key<T>::of(v[e]);
    own[e] = 0;
    if (e < n && key > tau) {
      const double wd = weight_of((float)v[e]);
      own[e] = wd >= least ? to_fixed(wd) : 0;
    } else if (e < n && key == tau) {
      own[e] = before < equal ? wt : 0;
      ++before;
    }
    mine += own[e];
  }
  const uint64_t s = sum + scan64(mine);
  const uint64_t reach = __ballot(s > goal);
  if (lane == __ffsll((unsigned long long)reach) - 1) {
    uint64_t run = s - mine;
    int e = 0;
    for (; e < 7; ++e) {
      run += own[e];
      if (run > goal) break;
    }
    a.token[row] = (int64_t)(at * 64 + lane) * 8 + e;
  }
}

}  // namespace

hipError_t launch_sample(const SampleProblem& p, hipStream_t stream) {
  SArgs a{};
  a.x = (const char*)p.logits;
  a.u = p.u;
  a.temperature = p.temperature;
  a.top_k = p.top_k;
  a.top_p = p.top_p;
  a.min_p = p.min_p;
  a.token = p.tokens;
  a.ldx = p.ldx;
  a.vocab = (int)p.vocab;
  a.shift = 62;
  while ((1ll << (62 - a.shift)) < p.vocab) --a.shift;
  a.t = p.t;
  a.k = p.k;
  a.p = p.p;
  a.m = p.m;
  const auto fn = p.dtype == DT_F16 ? sample_rows<_Float16> : p.dtype == DT_BF16 ? sample_rows<__bf16> : sample_rows<float>;
  hipLaunchKernelGGL(fn, dim3((unsigned)p.rows), dim3(NT), 0, stream, a);
  return hipGetLastError();
}

}  // namespace hxmi
