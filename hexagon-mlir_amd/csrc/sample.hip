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
// in 62 bits (44 fraction bits up to a vocabulary of 2^18): integer sums do not
// depend on their order, so neither does the token, and every comparison above
// is exact in them (p * sum and u * sum as 128-bit products).  w comes from a
// 64-bit evaluation good to 2^-46.  fp32 sums would put about one row in a
// hundred of a flat distribution on another token.
//
// One workgroup a row.  top-k and top-p are thresholds on the logits, kept as
// the key (an integer that orders as the logits do) of the last token kept and
// the number of its equals that stay:
//   * top-k of up to 512: the k-th largest of the threads' own largest logits
//     over the row's first quarter is a bound below the k-th largest of all; one
//     pass puts the tokens from it on (a few thousand) on a list in LDS, and
//     everything else happens there;
//   * 16-bit logits otherwise: the tokens are counted by value in LDS (65536
//     counts of 16 bits, 128 KB) in the pass that finds the largest; both
//     thresholds follow from counts and one weight a value.  Values of masks take
//     no part, and in a second count none whose weight is 0;
//   * fp32 logits otherwise: counted by the upper 16 bits, those of the top k's
//     bins on the list; without top-k the weights are summed in 16384 bins by
//     distance from the largest logit and the list is the threshold's bin;
//   * where a count passes 16 bits (more than 65535 equal values) or a list
//     its room, a radix descent over the row, 8 bits a pass with a column of
//     the histogram for each lane, takes their place.
// Then the kept weights are summed by pieces of 512 tokens (from the list, from
// a table of the weight of every kept value, or evaluated), the piece that
// reaches u * sum is found and the token in it.
//
// What bounds it is one CU's work on its row, not memory (rows of 151936 logits
// in us, at 64 rows and about the same up to 256): bf16 top-p 47 (largest and
// counts 19, threshold 9, table and sums 15; 53 with a pass of its own for the
// largest), every token kept 42 (59 with a weight evaluated for each), fp32
// top-k of 400 56 (two passes of 600 KB and the list), fp32 top-p 107 (a weight
// each into bins, the kept ones again); one row of 32000 with top-k 18.  A radix
// descent over the row for every threshold took 314 us for the first of them,
// 375 for fp32.  Rows are not shared out over workgroups: 64 rows leave 192 CUs
// idle.  (Counts and sums are integers, so shares could be joined in any order.)
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

// Verification of drafted tokens: rows of requests, `u` a row's number for its
// draft, `draw` a request's for the token after the accepted ones.
struct RowState {
  uint32_t state;
  int owner;      // the request that the row was judged for, -1: none
  int64_t token;  // drawn (state kDrawn)
  uint64_t whole, least;
  uint32_t tau, top, from;
  int ties_end;  // equals of tau before this token are kept
  float t;
};
enum : uint32_t { kDrawn, kAccepted, kToDraw };
struct VArgs : SArgs {
  const int64_t* drafts;
  const float* draw;
  const int* cu;  // null: `per` rows a request
  const char* q;  // the draft's probabilities, or null: the drafted token is certain
  int64_t ldq, rows;
  RowState* state;
  uint64_t* sums;               // [requests, pieces]: what is left of a stopping row's weight
  unsigned long long* arrived;  // [requests] shares that are done: 0 before and after
  int* counts;
  int requests, per, q_type, shares;
};

constexpr int NT = 1024, NW = NT / 64, PIECE = 512;
constexpr int kMaxPieces = kSampleMaxVocab / PIECE;
constexpr int kList = 6144, kFewTop = 512, kTable = 16384, kBins = 16384;
constexpr int kTieBit = 54;  // of a table entry: an equal of the last key (a piece's weights sum to 2^53 at most)

// A logit's key: an unsigned integer that orders as the logits do, equal for
// -0 and 0 (its magnitude's bits under its sign, moved up by half the range).
template <typename T>
struct Key {
  static constexpr int bits = 16;
  static constexpr uint32_t zero = 0x8000, magnitude = 0x7fff;
  static constexpr uint32_t inf = std::is_same_v<T, _Float16> ? 0x7c00 : 0x7f80;
  static __device__ __forceinline__ uint32_t of(T v) {
    const short b = __builtin_bit_cast(short, v), s = b >> 15;
    return (uint32_t)(uint16_t)(short)((b ^ (s & 0x7fff)) - s) ^ zero;
  }
};
template <>
struct Key<float> {
  static constexpr int bits = 32;
  static constexpr uint32_t zero = 0x80000000u, magnitude = 0x7fffffffu, inf = 0x7f800000u;
  static __device__ __forceinline__ uint32_t of(float v) {
    const int b = (int)__float_as_uint(v), s = b >> 31;
    return (uint32_t)((b ^ (s & 0x7fffffff)) - s) ^ zero;
  }
};
template <typename T>
__device__ __forceinline__ float value_of(uint32_t key) {
  const bool neg = key < Key<T>::zero;
  const uint32_t mag = neg ? Key<T>::zero - key : key - Key<T>::zero, b = neg ? mag | Key<T>::zero : mag;
  if constexpr (Key<T>::bits == 32) return __uint_as_float(b);
  else return (float)__builtin_bit_cast(T, (unsigned short)b);
}

// 2^(j / 512), by its Taylor series at compile time.
constexpr int kSteps = 512;
struct Exp2Table {
  double v[kSteps];
};
constexpr Exp2Table exp2_table() {
  Exp2Table t{};
  for (int j = 0; j < kSteps; ++j) {
    const double z = 0.69314718055994530942 * j / kSteps;
    double p = 1.0;
    for (int n = 22; n >= 1; --n) p = 1.0 + p * z / n;
    t.v[j] = p;
  }
  return t;
}
__constant__ const Exp2Table kExp2 = exp2_table();

// The weights of a row: round(2^shift * 2^y), y = (v - max) * log2(e) / T.
struct Weights {
  double rate;    // log2(e) / T, in steps of the table
  double top;     // the largest logit
  float xmax, least;  // values below `least` have weight 0
  int shift;
  const double* table;
  int lone;  // only logits equal to the largest have a weight (in a scalar register)

  __device__ __forceinline__ uint64_t of(float v) const {
    if (lone) return v == xmax ? 1ull << shift : 0;
    // k = round(y), from the low bits of y + 1.5 * 2^52; 2^(r / 512) by its
    // series, |r ln 2 / 512| <= 6.8e-4: the first term left out is below 2^-46
    const double y = ((double)fmaxf(v, least) - top) * rate;
    const double t = y + 0x1.8p52, r = y - (t - 0x1.8p52);
    const int k = __double2loint(t);
    constexpr double z = 0.69314718055994530942 / kSteps;
    double p = __builtin_fma(z * z * z / 6, r, z * z / 2);
    p = __builtin_fma(p, r, z);
    p = __builtin_fma(p, r, 1.0);
    p *= table[k & (kSteps - 1)];
    // times 2^(k / 512 + shift) in its exponent; the sum rounds it (below 2^51)
    const int e = (k >> 9) + shift;
    p = __hiloint2double(__double2hiint(p) + (e << 20), __double2loint(p)) + 0x1p52;
    return (uint64_t)__double_as_longlong(p) & 0xfffffffffffffull;
  }
};

// The weights of a row with the largest key `top` at temperature t.
template <typename T>
__device__ __forceinline__ Weights weights_of(uint32_t top, float t, int shift, const double* table) {
  const float xmax = value_of<T>(top);
  const double rate = 1.44269504088896340736 / (double)fminf(t, 1e28f);  // (an infinite T leaves -inf its weight, 0)
  // `least`, 20 bits below where weights end and rounded down: y stays above -200 bits.
  // Where a float holds nothing between it and the largest logit (T of 1e-9 of
  // that, or 1e28), only the largest have a weight, as where that is infinite.
  const double under = (double)xmax - (shift + 20) / rate;
  float least_x = (float)under;
  const bool lone = xmax == INFINITY || least_x >= xmax;
  if ((double)least_x > under) least_x = value_of<float>(Key<float>::of(least_x) - 1);
  return Weights{rate * kSteps, (double)xmax, xmax, least_x, shift, table, __builtin_amdgcn_readfirstlane(lone)};
}

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__shfl((int)(v >> 32), lane, 64) << 32) | (uint32_t)__shfl((int)v, lane, 64);
}
// floor(f * 2^64) of f in [0, 1)
__device__ __forceinline__ uint64_t fraction64(float f) {
  const double g = (double)f * 0x1p32, hi = __builtin_floor(g);
  return (uint64_t)(uint32_t)hi << 32 | (uint32_t)((g - hi) * 0x1p32);
}

struct Shared {
  union {
    uint32_t count2[32768];            // 16-bit counts of the upper 16 bits of a key, two a word
    unsigned long long bin[kBins];     // weights by the distance from the largest logit
    unsigned long long table[kTable];  // weight of a value by its key
    unsigned long long mass[256][64];  // radix descent: a column a lane
    uint32_t count[256][64];
    struct {
      unsigned long long weight[kList];
      uint32_t key[kList], index[kList];
      uint32_t kept[NW][PIECE];  // (a wave's own)
    } list;
  };
  union {
    struct {
      unsigned long long sum[kMaxPieces];  // kept weight of a piece, less its equals of the last key
      uint32_t ties[kMaxPieces];
    } piece;
    struct {
      unsigned long long weight[NT];  // of 64 values each
      uint32_t count[NT];
    } group;
  };
  double exp2[kSteps];
  unsigned long long digit[256];
  unsigned long long part[NW];
  uint32_t key, listed;
  unsigned long long above;
};

// Eight logits as they lie, and their keys.
template <typename T>
struct Eight {
  int4v r[sizeof(T) / 2];

  __device__ __forceinline__ void load(const T* x) {
    if constexpr (sizeof(T) == 2) {
      r[0] = *(const int4u2*)x;
    } else {
      r[0] = *(const int4u4*)x;
      r[1] = *(const int4u4*)(x + 4);
    }
  }
  __device__ __forceinline__ void keys(uint32_t (&key)[8]) const {
    if constexpr (sizeof(T) == 2) {
      typedef short short2v __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // two at a time
        const int bits = r[0][e];
        const short2v b = __builtin_bit_cast(short2v, bits), s = b >> 15;
        const uint32_t k2 = __builtin_bit_cast(uint32_t, (short2v)((b ^ (s & (short)0x7fff)) - s)) ^ 0x80008000u;
        key[2 * e] = k2 & 0xffffu;
        key[2 * e + 1] = k2 >> 16;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) key[e] = Key<T>::of(__uint_as_float((uint32_t)r[e >> 2][e & 3]));
    }
  }
};
// The keys of logits 8 i .. 8 i + 7, 0 (no logit's key, below them all) past the row.
template <typename T>
__device__ __forceinline__ void load_keys(const T* x, int i, int vocab, uint32_t (&key)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) key[e] = i * 8 + e < vocab ? Key<T>::of(x[i * 8 + e]) : 0;
}

// f(keys of logits 8 i .. 8 i + 7, j) for i = i0 + step * j, j < U: the loads
// all ahead of the first use where the whole wave's are inside the row.
template <int U, typename T, typename F>
__device__ __forceinline__ void load_groups(const T* x, int i0, int step, int vocab, F&& f) {
  if (__all((i0 + step * (U - 1)) * 8 + 8 <= vocab)) {
    Eight<T> raw[U];
#pragma unroll
    for (int j = 0; j < U; ++j) raw[j].load(x + (i0 + step * j) * 8);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      uint32_t key[8];
      raw[j].keys(key);
      f(key, j);
    }
  } else {
    for (int j = 0; j < U; ++j) {
      uint32_t key[8];
      load_keys(x, i0 + step * j, vocab, key);
      f(key, j);
    }
  }
}

// f(key, index) for the logits of a row (and for a few keys 0, which none has).
template <int U, typename T, typename F>
__device__ __forceinline__ void each_key(const T* x, int vocab, F&& f) {
  const int lanes = (vocab + 7) >> 3, wave0 = threadIdx.x & ~63;
  for (int i0 = wave0; i0 < lanes; i0 += NT * U)  // (a wave stays together)
    load_groups<U>(x, i0 + (threadIdx.x & 63), NT, vocab, [&](const uint32_t (&key)[8], int j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f(key[e], (i0 + (int)(threadIdx.x & 63) + j * NT) * 8 + e);
    });
}

// Inclusive sum over the workgroup's threads and (in `total`) the whole.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, Shared& sh, uint64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  v = scan64(v);
  __syncthreads();
  if (lane == 63) sh.part[w] = v;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const uint64_t t = sh.part[i];
    before += i < w ? t : 0;
    total += t;
  }
  return before + v;
}
__device__ __forceinline__ uint64_t block_sum(uint64_t v, Shared& sh) {
  uint64_t total;
  block_scan(v, sh, total);
  return total;
}

// Element i of a row of the draft's probabilities; NaN and negative ones count as 0.
__device__ __forceinline__ float prob_of(const char* q, int type, int64_t i) {
  const float f = type == SAMPLE_F32 ? ((const float*)q)[i]
                  : type == DT_BF16  ? (float)((const __bf16*)q)[i]
                                     : (float)((const _Float16*)q)[i];
  return fmaxf(f, 0.f);
}
// floor(f * whole) for a probability f.
__device__ __forceinline__ uint64_t share_of(float f, double whole) {
  return (uint64_t)fmin((double)f * whole, 0x1p62);
}
__device__ __forceinline__ float unit(float u) { return u > 0.f ? (u < 1.f ? u : 0x1.fffffep-1f) : 0.f; }

// The rows [first, end) of request r.
__device__ __forceinline__ void rows_of(const VArgs& a, int r, int64_t& first, int64_t& end) {
  first = a.cu ? min(max((int64_t)a.cu[r], (int64_t)0), a.rows) : (int64_t)r * a.per;
  end = a.cu ? min(max((int64_t)a.cu[r + 1], first), a.rows) : first + a.per;
}

// A row to its token; or (VERIFY, A = VArgs) a row to whether its drafted token is
// accepted, and if not what is drawn in its place, as far as the row's own
// weights say: with a draft's probabilities verify_rows draws it.
template <typename T, typename A>
__global__ __launch_bounds__(NT) void sample_rows(A a) {
  constexpr bool VERIFY = std::is_same_v<A, VArgs>;
  __shared__ __attribute__((aligned(16))) Shared sh;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  int64_t owner = row;  // index of the row's settings
  bool final = true;  // VERIFY: its request's last row, which has no draft
  if constexpr (VERIFY) {
    int lo = 0;
    if (a.cu) {
      for (int hi = a.requests; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= row) lo = mid;
        else hi = mid;
      }
    } else {
      lo = (int)(row / a.per);
    }
    int64_t first, end;
    rows_of(a, lo, first, end);
    if (threadIdx.x == 0) a.token[row] = -1;  // (verify_rows: accepted and drawn ones)
    if (row < first || row >= end) {  // of no request (or, where bounds do not ascend, one that the search passes by)
      if (threadIdx.x == 0) a.state[row] = RowState{.state = kDrawn, .owner = -1, .token = -1};
      return;
    }
    owner = lo;
    final = row + 1 == end;
  }
  const T* const x = (const T*)a.x + row * a.ldx;
  const int vocab = a.vocab;
  constexpr int KB = Key<T>::bits;

  if (threadIdx.x < kSteps) sh.exp2[threadIdx.x] = kExp2.v[threadIdx.x];

  int k = a.top_k ? a.top_k[owner] : a.k;
  float p = a.top_p ? a.top_p[owner] : a.p, mp = a.min_p ? a.min_p[owner] : a.m;
  float t = a.temperature ? a.temperature[owner] : a.t;
  if (!(t > 0.f)) {  // the first of the largest
    t = 1.f;
    k = 1;
    p = 1.f;
    mp = 0.f;
  }
  bool need_k = k > 0 && k < vocab, need_p = !(p >= 1.f);

  // Largest and smallest key: NaNs have keys over inf's or under -inf's.
  uint32_t top = 0, low = 0xffffffffu;
  auto extremes = [&]() {  // of the workgroup from the threads'
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
      low = min(low, (uint32_t)__shfl_xor((int)low, o, 64));
    }
    if (lane == 0) sh.part[w] = ((unsigned long long)top << 32) | low;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      top = max(top, (uint32_t)(sh.part[i] >> 32));
      low = min(low, (uint32_t)sh.part[i]);
    }
  };
  // The key, from `hi` down, at which the weights of the workgroup's entries
  // over it and its own first reach the goal, with `above` over hi; to within
  // 2^slack.  each(f) calls f(key, weight) for a thread's entries.  Eight bits
  // of the distance from lo (which the goal is reached at) a round.
  auto radix = [&](uint32_t lo, uint32_t hi, int slack, uint64_t goal, uint64_t& above, auto&& each) {
    const int bits = 32 - __builtin_clz((hi - lo) | 1);
    for (int b = max(bits - 8, 0);; b = max(b - 8, 0)) {
      __syncthreads();
      if (threadIdx.x < 256) sh.digit[threadIdx.x] = 0;
      __syncthreads();
      each([&](uint32_t key, uint64_t weight) {
        if (key >= lo && key <= hi) atomicAdd(&sh.digit[(key - lo) >> b], (unsigned long long)weight);
      });
      __syncthreads();
      uint64_t own[4], sum = 0;  // (every wave the same)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += own[j] = sh.digit[255 - 4 * lane - j];
      const uint64_t incl = above + scan64(sum);
      const int at = __ffsll((unsigned long long)__ballot(incl >= goal)) - 1;
      uint64_t over = incl - sum;
      int j = 0;
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (j == i && over + own[i] < goal) {
          over += own[i];
          ++j;
        }
      const uint32_t digit = __builtin_amdgcn_readlane(255 - 4 * lane - j, at);
      above = shfl64(over, at);
      lo += digit << b;
      hi = min(hi, lo + ((1u << b) - 1));
      if (b <= slack) return lo;
    }
  };

  // Appends the tokens of a wave that `take` says to the list: one atomic for
  // all (a row whose every logit is the same puts all of them here).
  auto put = [&](bool take, uint32_t key, int i) {
    const uint64_t m = __ballot(take);
    if (!m) return;
    uint32_t at = 0;
    if (lane == __ffsll((unsigned long long)m) - 1) at = atomicAdd(&sh.listed, (uint32_t)__popcll(m));
    at = __builtin_amdgcn_readlane(at, __ffsll((unsigned long long)m) - 1) +
         __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
    if (take && at < kList) {
      sh.list.key[at] = key;
      sh.list.index[at] = i;
    }
  };
  uint32_t bound = 1;   // no less than k keys are as large
  uint32_t listed = 0;  // tokens on the list, all that the top k can hold among them; 0: no list
  if (need_k && k <= kFewTop) {
    uint32_t own = 0;
    each_key<4>(x, min(vocab, (vocab / 4 + 8 * NT - 1) & ~(8 * NT - 1)), [&](uint32_t key, int) { own = max(own, key); });
    // (any bound below the k-th largest does; a thread without a token has key 0)
    uint64_t above = 0;
    bound = max(radix(0, KB == 16 ? 0xffffu : 0xffffffffu, KB == 16 ? 0 : 16, k, above, [&](auto&& f) { f(own, 1); }), 1u);
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    each_key<4>(x, vocab, [&](uint32_t key, int i) {
      low = min(low, key - 1);  // (0, no key, goes past every other)
      put(key >= bound, key, i);
    });
    __syncthreads();
    listed = sh.listed;
    if (listed > kList) listed = 0;
    for (uint32_t i = threadIdx.x; i < listed; i += NT) top = max(top, sh.list.key[i]);
  }
  constexpr uint32_t kInf = Key<T>::zero + Key<T>::inf, kMinusInf = Key<T>::zero - Key<T>::inf;
  // Counts the tokens with keys from `least` on by their upper 16 bits:
  // `in_bins` of them by this thread.
  uint32_t in_bins = 0;
  auto count_pass = [&](uint32_t least) {
    __syncthreads();
    int4v* const z = (int4v*)sh.count2;
    for (int i = threadIdx.x; i < 32768 / 4; i += NT) z[i] = int4v{};
    __syncthreads();
    in_bins = 0;
    each_key<4>(x, vocab, [&](uint32_t key, int) {
      top = max(top, key);
      low = min(low, key - 1);
      if (key < least) return;
      const uint32_t bin = key >> (KB - 16);
      atomicAdd(&sh.count2[bin >> 1], 1u + (bin & 1) * 0xffffu);
      ++in_bins;
    });
  };
  // 16-bit logits: counted in the pass that finds the largest, all but -inf and
  // the lowest finite value (masks, which could be more than a count holds).
  constexpr uint32_t kMasks = kMinusInf + 2;
  const bool early = KB == 16 && !listed && (need_k || need_p);
  if (early) count_pass(kMasks);
  else if (!listed) each_key<8>(x, vocab, [&](uint32_t key, int) {
      top = max(top, key);
      low = min(low, key - 1);
    });
  extremes();
  if (top > kInf || low + 1 < kMinusInf || top == kMinusInf) {
    if (threadIdx.x == 0) {
      if constexpr (VERIFY) a.state[row] = RowState{.state = kDrawn, .owner = (int)owner, .token = -1};
      else a.token[row] = -1;
    }
    return;
  }
  const Weights weights = weights_of<T>(top, t, a.shift, sh.exp2);
  const float xmax = weights.xmax;
  const double rate = 1.44269504088896340736 / (double)fminf(t, 1e28f);
  auto key_from = [&](double v) {  // the key from which logits are at least v (of a NaN: all)
    const float f = (float)v;
    if constexpr (KB == 32) return f != f ? 1u : max(1u, Key<float>::of(f));
    else {
      // (rounded to 16 bits: down to a value, or up to one that v's side of it is all below)
      const T h = (T)f;
      return f != f ? 1u : max(1u, Key<T>::of(h));
    }
  };
  // Logits with keys below `cut` have a weight that rounds to 0: they change no
  // sum, and whether the top k holds some of them changes nothing.  (Any value
  // under the rounding of a bound is under the bound.)
  const uint32_t cut = min(top, key_from((double)xmax - (a.shift + 3) / rate * 1.000001));
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
      each_key<1>(x, vocab, [&](uint32_t key, int) {
        if (key < cut || (b + 8 < KB && key >> (b + 8) != prefix)) return;
        if constexpr (COUNT) atomicAdd(&sh.count[(key >> b) & 255][lane], 1u);
        else atomicAdd(&sh.mass[(key >> b) & 255][lane], (unsigned long long)weights.of(value_of<T>(key)));
      });
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

  // ---- counts by the upper 16 bits ------------------------------------------------
  // Thread t owns the 64 bins from 64 * (1023 - t) on: threads in order go
  // from the largest keys down.
  const uint32_t bin0 = 64u * (NT - 1 - threadIdx.x);
  auto count_of = [&](uint32_t bin) -> uint32_t { return sh.count2[bin >> 1] >> (16 * (bin & 1)) & 0xffffu; };
  // Counts the tokens with a weight (`counted` in all; where the masks have none,
  // the early counts do); false if a count passed 16 bits.
  uint64_t counted = 0, count_incl = 0, count_own = 0;
  auto count_keys = [&](bool again) {
    if (again) count_pass(cut);
    counted = block_sum(in_bins, sh);
    count_own = 0;
    for (int j = 0; j < 32; ++j) {
      const uint32_t two = sh.count2[(bin0 >> 1) + ((j + threadIdx.x) & 31)];  // (banks apart)
      count_own += (two & 0xffffu) + (two >> 16);
    }
    uint64_t held;
    count_incl = block_scan(count_own, sh, held);
    return held == counted;  // (a carry loses 65535 of 65536)
  };
  // The bin, from the largest down, at which per-thread sums (`incl`
  // inclusive, `own`, of weight_of_bin over a thread's bins) reach the goal;
  // `above`: what lies over it.
  auto find_bin = [&](uint64_t incl, uint64_t own, uint64_t goal, uint64_t& above, auto&& weight_of_bin) {
    __syncthreads();
    if (incl >= goal && incl - own < goal) {  // (one thread)
      sh.key = bin0;
      sh.above = incl - own;
    }
    __syncthreads();
    const uint32_t base = sh.key;
    const uint64_t over = sh.above;
    const uint32_t bin = base + 63 - lane;
    const uint64_t mine = weight_of_bin(bin), s = over + scan64(mine);  // (every wave the same)
    const int at = __ffsll((unsigned long long)__ballot(s >= goal)) - 1;
    above = shfl64(s - mine, at);
    return base + 63 - (uint32_t)at;
  };

  // Kept: keys over `tau`, and the first `equal` tokens whose key is tau.
  uint32_t tau = 0, equal = 0;
  const uint64_t pf = fraction64(p > 0.f ? fminf(p, 0x1.fffffep-1f) : 0.f);
  auto goal_of = [&](uint64_t whole) {  // ceil(p * whole), at least 1
    const uint64_t g = __umul64hi(pf, whole) + (pf * whole != 0);
    return g > 1 ? g : 1;
  };
  // How many equals of tau make up what `above` leaves to the goal (which
  // tau's weight reaches, so it is not 0).
  auto equals_of = [&](uint64_t goal, uint64_t above) {
    const uint64_t wt = weights.of(value_of<T>(tau));
    return (uint32_t)min((goal - above + wt - 1) / wt, (uint64_t)0xffffffffu);
  };

  // List of the tokens whose key `in` takes: their number (over kList: not all are there).
  auto make_list = [&](auto&& in) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    each_key<4>(x, vocab, [&](uint32_t key, int i) {
      put(key >= cut && in(key), key, i);
    });
    __syncthreads();
    return sh.listed;
  };
  auto list_weights = [&](uint32_t n) {
    for (uint32_t i = threadIdx.x; i < n; i += NT) sh.list.weight[i] = weights.of(value_of<T>(sh.list.key[i]));
  };  // (each thread reads its own entries)
  // A thread's entries of a list of n tokens.
  auto list_keys = [&](uint32_t n) {
    return [&, n](auto&& f) {
      for (uint32_t i = threadIdx.x; i < n; i += NT) f(sh.list.key[i], 1);
    };
  };
  auto list_masses = [&](uint32_t n) {
    return [&, n](auto&& f) {
      for (uint32_t i = threadIdx.x; i < n; i += NT) f(sh.list.key[i], sh.list.weight[i]);
    };
  };
  // Both thresholds from a list of n tokens that holds the top k, keys from lo on.
  auto list_thresholds = [&](uint32_t n, uint32_t lo) {
    uint64_t above = 0;
    tau = radix(lo, top, 0, k, above, list_keys(n));
    equal = (uint32_t)(k - above);
    list_weights(n);
    if (need_p) {
      uint64_t own = 0;
      list_masses(n)([&](uint32_t key, uint64_t wf) { own += key > tau ? wf : 0; });
      const uint64_t goal = goal_of(block_sum(own, sh) + equal * weights.of(value_of<T>(tau)));
      above = 0;
      tau = radix(tau, top, 0, goal, above, list_masses(n));
      equal = equals_of(goal, above);
    }
    need_k = need_p = false;
  };

  const double m = mp > 0.f ? (double)fminf(mp, 1.f) : 0.0;
  const uint64_t least = (uint64_t)__builtin_rint(__builtin_ldexp(m, a.shift));
  // (logits below `from` are below min_p or have weight 0)
  const uint32_t from = m > 0.0 ? max(cut, min(top, key_from((double)xmax + (log2(m) * 1.000001 - 1e-5) / rate))) : cut;
  // What each piece keeps: the weights (of at least `least`) of its keys over
  // `last` and from `from` on, and the number of its equals of `last`; or, with
  // LIST, tokens with keys from `low` to `last` go onto the list.  Where there
  // is a bound, the wave first gathers those keys: 64 at a time then take one
  // evaluation.
  const int pieces = (vocab + PIECE - 1) / PIECE;
  auto sum_pieces = [&](auto LIST_, uint64_t least, uint32_t from, uint32_t last, uint32_t low) {
    constexpr bool LIST = decltype(LIST_)::value;
    __syncthreads();
    if (LIST && threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    constexpr int U = 4;
    uint32_t* const kept = sh.list.kept[w];
    const uint32_t over = max(last, from - 1);
    const bool dense = last == 0 && from == cut;  // (few are left out)
    for (int c0 = w; c0 < pieces; c0 += NW * U)
      load_groups<U>(x, c0 * 64 + lane, NW * 64, vocab, [&](const uint32_t (&key)[8], int j) {
        const int c = c0 + j * NW;
        if (c >= pieces) return;
        int some = 0, ties = 0;
        uint64_t sum = 0;
        if (!LIST && dense) {
          uint64_t wf[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) wf[e] = weights.of(value_of<T>(key[e]));
#pragma unroll
          for (int e = 0; e < 8; ++e) sum += key[e] > over && wf[e] >= least ? wf[e] : 0;
          some = PIECE;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint64_t m = __ballot(key[e] > over);
            if (key[e] > over)
              kept[some + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0))] = key[e];
            some += __popcll(m);
            if constexpr (LIST) put(key[e] >= low && key[e] <= last, key[e], (c * 64 + lane) * 8 + e);
            else ties += __popcll(__ballot(key[e] == last));
          }
          for (int i = lane; i < some; i += 128) {  // (two evaluations side by side)
            const uint64_t w0 = weights.of(value_of<T>(kept[i])), w1 = weights.of(value_of<T>(kept[min(i + 64, some - 1)]));
            sum += w0 >= least ? w0 : 0;
            sum += i + 64 < some && w1 >= least ? w1 : 0;
          }
        }
        if (some) sum = scan64(sum);
        if (lane == 63) {
          sh.piece.sum[c] = sum;
          sh.piece.ties[c] = (uint32_t)ties;
        }
      });
    __syncthreads();
  };
  // Adds what is kept of a list of n tokens to its pieces.
  auto add_list = [&](uint32_t n) {
    for (uint32_t i = threadIdx.x; i < n; i += NT) {
      const uint32_t key = sh.list.key[i], c = sh.list.index[i] / PIECE;
      if (key > tau && sh.list.weight[i] >= least) atomicAdd(&sh.piece.sum[c], sh.list.weight[i]);
      if (key == tau) atomicAdd(&sh.piece.ties[c], 1u);
    }
    __syncthreads();
  };
  bool summed = false;  // the pieces are

  if (listed) {
    list_thresholds(listed, bound);
  } else if constexpr (KB == 16) {
    if ((need_k || need_p) && ((early && cut >= kMasks && count_keys(false)) || count_keys(true))) {
      if (need_k && (uint64_t)k < counted) {
        uint64_t above;
        tau = find_bin(count_incl, count_own, (uint64_t)k, above, [&](uint32_t bin) -> uint64_t { return count_of(bin); });
        equal = (uint32_t)(k - above);
      }
      if (need_p) {
        auto masses = [&](uint32_t bin) -> uint64_t {
          const uint32_t c = bin > tau ? count_of(bin) : bin == tau ? min(count_of(bin), equal) : 0;
          return c ? c * weights.of(value_of<T>(bin)) : 0;
        };
        // each wave takes every 16th group of 64 bins, those that hold something
        sh.group.count[threadIdx.x] = (uint32_t)count_own;
        __syncthreads();
        const uint32_t some = sh.group.count[lane * NW + w];
        if (some == 0) sh.group.weight[lane * NW + w] = 0;
        for (uint64_t left = __ballot(some != 0); left; left &= left - 1) {
          const int g = (__ffsll((unsigned long long)left) - 1) * NW + w;
          const uint64_t sum = scan64(masses(64u * (NT - 1 - g) + lane));
          if (lane == 63) sh.group.weight[g] = sum;
        }
        __syncthreads();
        const uint64_t own = sh.group.weight[threadIdx.x];
        uint64_t whole, above;
        const uint64_t incl = block_scan(own, sh, whole), goal = goal_of(whole);
        tau = find_bin(incl, own, goal, above, masses);
        equal = equals_of(goal, above);
      }
      need_k = need_p = false;
    } else if (need_k && (uint64_t)k >= counted) {
      need_k = false;
    }
  } else {
    if (need_k) {
      const bool ok = count_keys(true);
      if ((uint64_t)k >= counted) {
        need_k = false;
      } else if (ok) {
        uint64_t above;
        const uint32_t bin =
            find_bin(count_incl, count_own, (uint64_t)k, above, [&](uint32_t b) -> uint64_t { return count_of(b); });
        if (above + count_of(bin) <= kList) {
          listed = make_list([&](uint32_t key) { return key >> 16 >= bin; });
          list_thresholds(listed, bin << 16);
        }
      }
    }
    if (!need_k && need_p) {
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += NT) sh.bin[i] = 0;
      __syncthreads();
      // Bins of equal width from the largest logit down to where weights end
      // (by the keys' upper bits, most tokens would share a hundred bins).
      const float per_bin = fminf((float)((kBins - 1) * rate / (a.shift + 3)), 0x1.fffffep127f), cut_x = value_of<T>(cut);
      auto bin_of = [&](float v) {  // (v <= xmax, which may be infinite)
        return v == xmax ? 0u : (uint32_t)fminf((xmax - v) * per_bin, (float)(kBins - 1));
      };
      const int lanes = (vocab + 7) >> 3;
      auto values = [&](int i, float (&v)[8]) {  // of logits 8 i .. 8 i + 7, -inf past the row
        if (__all(i * 8 + 8 <= vocab)) {
          Eight<T> raw;
          raw.load(x + i * 8);
          __builtin_memcpy(v, raw.r, sizeof(v));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = i * 8 + e < vocab ? (float)x[i * 8 + e] : -INFINITY;
        }
      };
      float now[8], next[8];
      values((int)threadIdx.x, now);
      for (int i0 = w * 64; i0 < lanes; i0 += NT) {
        values(i0 + lane + NT, next);
        uint64_t wf[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) wf[e] = weights.of(now[e]);  // (side by side)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (now[e] >= cut_x) atomicAdd(&sh.bin[bin_of(now[e])], (unsigned long long)wf[e]);
          now[e] = next[e];
        }
      }
      __syncthreads();
      uint64_t own = 0, whole;
      const uint32_t b0 = kBins / NT * threadIdx.x;
      for (int j = 0; j < kBins / NT; ++j) own += sh.bin[b0 + ((j + threadIdx.x) & (kBins / NT - 1))];
      const uint64_t incl = block_scan(own, sh, whole), goal = goal_of(whole);
      __syncthreads();
      if (incl >= goal && incl - own < goal) {  // (one thread)
        uint64_t over = incl - own;
        int j = 0;
        for (; j < kBins / NT - 1 && over + sh.bin[b0 + j] < goal; ++j) over += sh.bin[b0 + j];
        sh.key = b0 + j;
        sh.above = over;
      }
      __syncthreads();
      const uint32_t bin = sh.key;
      const uint64_t above = sh.above;
      // Its keys: one pass lists them and sums the pieces of all above.
      auto first_key = [&](uint32_t bin) {  // the lowest key in the bins up to it
        uint32_t lo = cut, hi = top;
        while (lo < hi) {
          const uint32_t mid = lo + ((hi - lo) >> 1);
          if (bin_of(value_of<T>(mid)) <= bin) hi = mid;
          else lo = mid + 1;
        }
        return lo;
      };
      const uint32_t lo = first_key(bin), hi = bin ? first_key(bin - 1) - 1 : top;
      sum_pieces(std::true_type{}, least, from, hi, lo);
      const uint32_t n = sh.listed;
      if (n <= kList) {
        list_weights(n);
        uint64_t over = above;
        tau = radix(lo, hi, 0, goal, over, list_masses(n));
        equal = equals_of(goal, over);
        add_list(n);
        need_p = false;
        summed = true;
      }
    }
  }
  if (need_k) {
    uint64_t above;
    tau = descend(std::true_type{}, (uint64_t)k, above);
    equal = (uint32_t)((uint64_t)k - above);
  }

  // A wave over the pieces, each lane a run of `per`: its pieces' kept weight
  // `own` (equals of tau at wt each), the equals before its run.
  const int per = (pieces + 63) >> 6;
  auto lane_pieces = [&](uint64_t wt, uint64_t& before) {
    uint64_t ties = 0, own = 0;
    for (int c = lane * per; c < min(lane * per + per, pieces); ++c) {
      ties += sh.piece.ties[c];
      own += sh.piece.sum[c];
    }
    before = scan64(ties) - ties;
    return own + (before >= equal ? 0 : min(ties, (uint64_t)equal - before)) * wt;
  };

  if (need_p) {
    sum_pieces(std::false_type{}, 0, cut, tau, 0);
    uint64_t before, above;
    const uint64_t whole = shfl64(scan64(lane_pieces(weights.of(value_of<T>(tau)), before)), 63);  // (every wave the same)
    const uint64_t goal = goal_of(whole);
    tau = descend(std::false_type{}, goal, above);
    equal = equals_of(goal, above);
  }

  const uint32_t base = max(tau, from) - 1;
  // 16-bit logits of both signs can have more keys than a table holds: then
  // those next to zero, where the fewest logits are, are a gap in it.
  uint32_t gap0 = top + 1, gap = 0;
  if (KB == 16 && top - base >= kTable) {
    const uint32_t half = (top - base - kTable + 2) / 2;
    if (half <= top - min(top, Key<T>::zero) && half < Key<T>::zero - min(Key<T>::zero, base)) {
      gap0 = Key<T>::zero - half;
      gap = 2 * half;
    }
  }
  if (summed) {
  } else if (listed) {
    __syncthreads();
    for (int i = threadIdx.x; i < pieces; i += NT) {
      sh.piece.sum[i] = 0;
      sh.piece.ties[i] = 0;
    }
    __syncthreads();
    add_list(listed);
  } else if (KB == 16 && top - base - gap < kTable) {
    // every kept value's weight by its key: an addition a token (and an
    // evaluation in the gap)
    __syncthreads();
    for (uint32_t i = threadIdx.x; i <= top - base - gap; i += NT) {
      const uint32_t key = base + i + (base + i >= gap0 ? gap : 0);
      const uint64_t wf = i ? weights.of(value_of<T>(key)) : 0;
      sh.table[i] = key == tau ? 1ull << kTieBit : wf >= least ? wf : 0;
    }
    if (threadIdx.x == 0) sh.table[0] = 0;
    __syncthreads();
    constexpr int U = 4;
    auto add_up = [&](auto GAP_) {
      for (int c0 = w; c0 < pieces; c0 += NW * U)
        load_groups<U>(x, c0 * 64 + lane, NW * 64, vocab, [&](const uint32_t (&key)[8], int j) {
          const int c = c0 + j * NW;
          if (c >= pieces) return;
          uint64_t sum = 0;
          if constexpr (decltype(GAP_)::value) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t k = max(key[e], base);
              if (k - gap0 < gap) {
                const uint64_t wf = weights.of(value_of<T>(k));
                sum += k == tau ? 1ull << kTieBit : wf >= least ? wf : 0;
              } else {
                sum += sh.table[k - base - (k >= gap0 ? gap : 0)];
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += sh.table[max(key[e], base) - base];
          }
          sum = scan64(sum);
          if (lane == 63) {
            sh.piece.sum[c] = sum & ((1ull << kTieBit) - 1);
            sh.piece.ties[c] = (uint32_t)(sum >> kTieBit);
          }
        });
    };
    if (gap) add_up(std::true_type{});
    else add_up(std::false_type{});
    __syncthreads();
  } else {
    sum_pieces(std::false_type{}, least, from, tau, 0);
  }
  if (w != 0) return;
  const uint64_t wt_all = weights.of(value_of<T>(tau)), wt = wt_all >= least ? wt_all : 0;
  uint64_t before;
  uint64_t run = lane_pieces(wt, before), incl = scan64(run), whole = shfl64(incl, 63);
  int64_t out = -1;    // the drafted token where that takes no part any more
  uint64_t w_out = 0;  // its weight
  float u = 0.f;
  if constexpr (VERIFY) {
    const int64_t d = final ? -1 : a.drafts[row];
    const bool in = d >= 0 && d < vocab;
    uint64_t wd = 0;
    if (in) {
      const uint32_t kd = Key<T>::of(x[d]);
      if (kd > tau && kd >= from) {
        const uint64_t wf = weights.of(value_of<T>(kd));
        wd = wf >= least ? wf : 0;
      } else if (kd == tau && wt) {
        // its place among tau's equals
        const int c = (int)(d / PIECE);
        uint64_t ties = 0;
        for (int i = lane; i < c; i += 64) ties += sh.piece.ties[i];
        uint32_t key[8];
        load_keys(x, c * 64 + lane, vocab, key);
#pragma unroll
        for (int e = 0; e < 8; ++e) ties += key[e] == tau && (c * 64 + lane) * 8 + e < d;
        wd = shfl64(scan64(ties), 63) < equal ? wt : 0;
      }
    }
    const float qd = !in ? 0.f : a.q ? prob_of(a.q + row * a.ldq * (a.q_type == SAMPLE_F32 ? 4 : 2), a.q_type, d) : 1.f;
    const bool accepted = (double)wd > (double)unit(a.u[row]) * qd * (double)whole;
    if (accepted || (a.q && !final)) {
      int ties_end = vocab;  // of tau's equals, those before this token are kept
      if (!accepted && equal > 0) {
        uint64_t seen = 0;  // (a wave over the pieces, 64 at a time, to the one that holds the first that is not)
        for (int c0 = 0; c0 < pieces; c0 += 64) {
          const uint64_t ties = c0 + lane < pieces ? sh.piece.ties[c0 + lane] : 0, incl = seen + scan64(ties);
          const uint64_t past = __ballot(incl > equal);
          if (!past) {
            seen = shfl64(incl, 63);
            continue;
          }
          const int l = __ffsll((unsigned long long)past) - 1, c = c0 + l;
          seen = shfl64(incl - ties, l);
          uint32_t key[8];
          load_keys(x, c * 64 + lane, vocab, key);
          uint64_t mine = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) mine += key[e] == tau;
          uint64_t at = seen + scan64(mine) - mine;
          int first = vocab;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (key[e] != tau) continue;
            if (at >= equal && first == vocab) first = (c * 64 + lane) * 8 + e;
            ++at;
          }
#pragma unroll
          for (int o = 32; o >= 1; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
          ties_end = first;
          break;
        }
      }
      if (lane == 0)
        a.state[row] = RowState{accepted ? kAccepted : kToDraw, (int)owner, -1, whole, least, tau, top, from, ties_end, t};
      return;
    }
    if (in && !a.q && !final) {
      out = d;
      w_out = wd;
    }
    u = unit(a.draw[owner]);
  } else {
    u = unit(a.u[row]);
  }
  const int out_piece = out >= 0 ? (int)(out / PIECE) : -1;
  if (out_piece >= 0) {
    const uint64_t less = out_piece / per == lane ? w_out : 0;
    run -= less;
    incl -= out_piece / per <= lane ? w_out : 0;
    whole -= w_out;
  }
  const uint64_t goal = __umul64hi(fraction64(u), whole);  // floor(u * whole) < whole

  // the lane's run, the piece, then the token whose running weight first exceeds the goal
  const int l = __ffsll((unsigned long long)__ballot(incl > goal)) - 1;
  uint64_t sum = shfl64(incl - run, l);
  before = shfl64(before, l);
  int at = l * per;
  for (;; ++at) {  // (every lane the same)
    const uint64_t ties = sh.piece.ties[at];
    uint64_t own = sh.piece.sum[at] + (before >= equal ? 0 : min(ties, (uint64_t)equal - before)) * wt;
    if (at == out_piece) own -= w_out;
    if (sum + own > goal || at + 1 >= min((l + 1) * per, pieces)) break;
    sum += own;
    before += ties;
  }
  uint32_t key[8];
  load_keys(x, at * 64 + lane, vocab, key);
  uint32_t ties = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) ties += key[e] == tau;
  before += scan64(ties) - ties;
  uint64_t own[8], mine = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    own[e] = 0;
    if (key[e] > tau && key[e] >= from) {
      const uint64_t wf = weights.of(value_of<T>(key[e]));
      own[e] = wf >= least ? wf : 0;
    } else if (key[e] == tau) {
      own[e] = before < equal ? wt : 0;
      ++before;
    }
    if (VERIFY && (at * 64 + lane) * 8 + e == out) own[e] = 0;
    mine += own[e];
  }
  const uint64_t s = sum + scan64(mine);
  const uint64_t reach = __ballot(s > goal);
  if (lane == __ffsll((unsigned long long)reach) - 1) {
    uint64_t so_far = s - mine;
    int e = 0;
    for (; e < 7; ++e) {
      so_far += own[e];
      if (so_far > goal) break;
    }
    const int64_t token = (int64_t)(at * 64 + lane) * 8 + e;
    if constexpr (VERIFY) a.state[row] = RowState{.state = kDrawn, .owner = (int)owner, .token = token};
    else a.token[row] = token;
  }
}

// ---- verification of drafted tokens ------------------------------------------------
//
//   p_i    a row's kept weights over their sum, as above
//   accept token d of a row (not its request's last) if p_d > u * q_d
//   the first row that is not accepted draws a token from max(p - q, 0), or, with
//   no probabilities of the draft, from p without d; the request's last row from p
//
// sample_rows says for every row whether its token is accepted and draws from
// what needs the row's own weights alone; this kernel, a workgroup a request,
// finds the row that stops it and, given q, goes over that row again: the kept
// weights less floor(q * sum), integers as they are, by pieces of 512 tokens,
// then the token in the piece that reaches draw * sum.
// A request's pieces go to a.shares workgroups of four waves, which store their
// sums; the last to arrive draws.  Each finds the stopping row for itself.  64
// requests over 151936 tokens, top-p: 18 us in 19 shares (22 in ten, 48 by one
// workgroup of sixteen waves), after 64 us of sample_rows (190 rows, a CU each).
constexpr int VW = 4;
template <typename T, typename Q>
__global__ __launch_bounds__(64 * VW) void verify_rows(VArgs a) {
  struct Local {
    uint32_t key[VW][PIECE];
    float q[VW][PIECE];
    double exp2[kSteps];
    unsigned long long sum[kMaxPieces];
    int last;
  };
  __shared__ Local sh;
  for (int i = threadIdx.x; i < kSteps; i += 64 * VW) sh.exp2[i] = kExp2.v[i];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, vocab = a.vocab;
  const int r = (int)(blockIdx.x / a.shares), share = (int)(blockIdx.x - (uint32_t)r * a.shares);
  int64_t first, end;
  rows_of(a, r, first, end);
  // A row that was judged for another request, or for none, stops this one, and
  // its token is left to that one: every row's state was written by this call, the
  // thresholds of the one that is drawn from for this request, and no row has two writers.
  int64_t stop = end;
  for (int64_t i0 = first; i0 < end && stop == end; i0 += 64) {  // (every wave the same)
    const RowState& s = a.state[min(i0 + lane, end - 1)];
    const uint64_t m = __ballot(i0 + lane < end && (s.state != kAccepted || s.owner != r));
    if (m) stop = i0 + __ffsll((unsigned long long)m) - 1;
  }
  if (share == 0) {
    for (int64_t i = first + threadIdx.x; i < stop; i += 64 * VW) a.token[i] = a.drafts[i];
    if (threadIdx.x == 0) a.counts[r] = stop < end ? (int)(stop - first + 1) : 0;
  }
  if (stop >= end) return;  // (without rows)
  const RowState st = a.state[stop];
  if (st.owner != r) return;
  if (st.state == kDrawn) {  // (without q every row that does not accept)
    if (share == 0 && threadIdx.x == 0) a.token[stop] = st.token;
    return;
  }
  __syncthreads();

  const T* const x = (const T*)a.x + stop * a.ldx;
  const Q* const q = (const Q*)a.q + stop * a.ldq;
  const Weights weights = weights_of<T>(st.top, st.t, a.shift, sh.exp2);
  const int pieces = (vocab + PIECE - 1) / PIECE;
  // what is left of a kept token's weight
  const double whole = (double)st.whole;
  auto left_of = [&](uint32_t key, float prob, bool with_q) {
    const uint64_t wf = weights.of(value_of<T>(key)), take = with_q ? share_of(prob, whole) : 0;
    return wf >= st.least && wf > take ? wf - take : 0;
  };
  auto kept = [&](uint32_t key, int i) {
    return key >= st.from && (key > st.tau || (key == st.tau && i < st.ties_end));
  };
  struct Raw {  // eight logits and probabilities as they lie
    Eight<T> x;
    Eight<Q> q;
  };
  auto load = [&](int i, Raw& raw) {
    if (i * 8 + 8 <= vocab) {
      raw.x.load(x + i * 8);
      raw.q.load(q + i * 8);
    }
  };
  auto values = [&](int i, const Raw& raw, uint32_t (&key)[8], float (&prob)[8]) {
    if (__all(i * 8 + 8 <= vocab)) {
      raw.x.keys(key);
      Q p[8];
      __builtin_memcpy(p, raw.q.r, sizeof(p));
#pragma unroll
      for (int e = 0; e < 8; ++e) prob[e] = fmaxf((float)p[e], 0.f);
    } else {
      load_keys(x, i, vocab, key);
#pragma unroll
      for (int e = 0; e < 8; ++e) prob[e] = i * 8 + e < vocab ? fmaxf((float)q[i * 8 + e], 0.f) : 0.f;
    }
  };
  constexpr int kCoherent = 17;  // sc0 | sc1
  const __amdgpu_buffer_rsrc_t sums = make_rsrc(a.sums + (int64_t)r * pieces, (uint32_t)(pieces * 8));
  // the sums of pieces c0 to c1
  auto sum_up = [&](int c0, int c1, bool with_q) {
    Raw next;
    load((c0 + w) * 64 + lane, next);
    for (int c = c0 + w; c < c1; c += VW) {
      uint32_t key[8];
      float prob[8];
      values(c * 64 + lane, next, key, prob);
      if (c + VW < c1) load((c + VW) * 64 + lane, next);
      int some = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // the kept ones together: 64 of them take one evaluation
        const bool k = kept(key[e], (c * 64 + lane) * 8 + e);
        const uint64_t m = __ballot(k);
        const int at = some + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        if (k) {
          sh.key[w][at] = key[e];
          sh.q[w][at] = prob[e];
        }
        some += __popcll(m);
      }
      uint64_t sum = 0;
      for (int i = lane; i < some; i += 64) sum += left_of(sh.key[w][i], sh.q[w][i], with_q);
      if (some) sum = scan64(sum);
      if (lane == 63) {
        const int2v both = {(int)(uint32_t)sum, (int)(sum >> 32)};
        __builtin_amdgcn_raw_buffer_store_b64(both, sums, (uint32_t)c * 8, 0, kCoherent);
      }
    }
    wait_vmcnt0();  // (what this wave stored is there for every XCD)
    __syncthreads();
  };
  const int per_share = (pieces + a.shares - 1) / a.shares;
  sum_up(min(share * per_share, pieces), min((share + 1) * per_share, pieces), true);
  if (a.shares > 1) {
    if (threadIdx.x == 0) {
      unsigned long long* const cnt = a.arrived + r;  // (at most kWsMaxTiles requests are shared out)
      const unsigned long long before = __hip_atomic_fetch_add(cnt, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      sh.last = before + 1 == (unsigned long long)a.shares;
      if (sh.last) __hip_atomic_store(cnt, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!sh.last) return;
  }
  const int per = (pieces + 63) >> 6;
  bool with_q = true;
  uint64_t whole_left = 0, incl = 0, run = 0;
  for (;;) {
    for (int c = threadIdx.x; c < pieces; c += 64 * VW) {
      const int2v both = __builtin_amdgcn_raw_buffer_load_b64(sums, (uint32_t)c * 8, 0, kCoherent);
      sh.sum[c] = (uint64_t)(uint32_t)both[1] << 32 | (uint32_t)both[0];
    }
    __syncthreads();
    run = 0;  // (every wave the same)
    for (int c = lane * per; c < min(lane * per + per, pieces); ++c) run += sh.sum[c];
    incl = scan64(run);
    whole_left = shfl64(incl, 63);
    if (whole_left || !with_q) break;
    with_q = false;  // (nothing left: the draft's distribution covers the target's; from p then)
    __syncthreads();
    sum_up(0, pieces, false);
  }
  if (w != 0) return;
  const uint64_t goal = __umul64hi(fraction64(unit(a.draw[r])), whole_left);
  const int l = __ffsll((unsigned long long)__ballot(incl > goal)) - 1;
  uint64_t sum = shfl64(incl - run, l);
  int at = l * per;
  for (;; ++at) {  // (every lane the same)
    if (sum + sh.sum[at] > goal || at + 1 >= min((l + 1) * per, pieces)) break;
    sum += sh.sum[at];
  }
  Raw raw;
  uint32_t key[8];
  float prob[8];
  load(at * 64 + lane, raw);
  values(at * 64 + lane, raw, key, prob);
  uint64_t own[8], mine = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    own[e] = kept(key[e], (at * 64 + lane) * 8 + e) ? left_of(key[e], prob[e], with_q) : 0;
    mine += own[e];
  }
  const uint64_t s = sum + scan64(mine);
  const uint64_t reach = __ballot(s > goal);
  if (lane == __ffsll((unsigned long long)reach) - 1) {
    uint64_t so_far = s - mine;
    int e = 0;
    for (; e < 7; ++e) {
      so_far += own[e];
      if (so_far > goal) break;
    }
    a.token[stop] = (int64_t)(at * 64 + lane) * 8 + e;
  }
}

}  // namespace

static void settings(const SampleProblem& p, SArgs& a) {
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
  a.shift = a.shift < 44 ? a.shift : 44;
  a.t = p.t;
  a.k = p.k;
  a.p = p.p;
  a.m = p.m;
}

hipError_t launch_sample(const SampleProblem& p, hipStream_t stream) {
  SArgs a{};
  settings(p, a);
  const auto fn = p.dtype == DT_F16    ? sample_rows<_Float16, SArgs>
                  : p.dtype == DT_BF16 ? sample_rows<__bf16, SArgs>
                                       : sample_rows<float, SArgs>;
  hipLaunchKernelGGL(fn, dim3((unsigned)p.rows), dim3(NT), 0, stream, a);
  return hipGetLastError();
}

static int64_t sums_bytes(int64_t requests, int64_t vocab) { return requests * ((vocab + PIECE - 1) / PIECE) * 8; }
int64_t verify_workspace_bytes(int64_t rows, int64_t requests, int64_t vocab) {
  return kWsCounterBytes + sums_bytes(requests, vocab) + rows * (int64_t)sizeof(RowState);
}

template <typename T>
static hipError_t launch_verify_t(const VerifyProblem& p, const VArgs& a, hipStream_t stream) {
  if (p.rows) hipLaunchKernelGGL((sample_rows<T, VArgs>), dim3((unsigned)p.rows), dim3(NT), 0, stream, a);
  const auto fn = p.q_type == SAMPLE_F32 ? verify_rows<T, float>
                  : p.q_type == DT_BF16  ? verify_rows<T, __bf16>
                                         : verify_rows<T, _Float16>;
  if (p.requests) hipLaunchKernelGGL(fn, dim3((unsigned)(p.requests * a.shares)), dim3(64 * VW), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_verify(const VerifyProblem& p, hipStream_t stream) {
  VArgs a{};
  settings(p, a);
  a.drafts = p.drafts;
  a.draw = p.draw;
  a.cu = p.cu;
  a.q = (const char*)p.q;
  a.ldq = p.ldq;
  a.rows = p.rows;
  a.arrived = (unsigned long long*)p.ws;
  a.sums = (uint64_t*)((char*)p.ws + kWsCounterBytes);
  a.state = (RowState*)((char*)a.sums + sums_bytes(p.requests, p.vocab));
  // four pieces a wave, while every CU has no more than eight of these workgroups
  const int64_t pieces = (p.vocab + PIECE - 1) / PIECE, most = p.requests <= kWsMaxTiles ? 2048 / (p.requests ? p.requests : 1) : 1;
  int64_t shares = p.q ? (pieces + 4 * VW - 1) / (4 * VW) : 1;
  shares = shares < most ? shares : most;
  a.shares = (int)(shares < 1 ? 1 : shares);  // (no rows, no vocabulary: counts are still to be written)
  a.counts = p.counts;
  a.requests = (int)p.requests;
  a.per = p.requests ? (int)(p.rows / p.requests) : 0;
  a.q_type = p.q_type;
  return p.dtype == DT_F16    ? launch_verify_t<_Float16>(p, a, stream)
         : p.dtype == DT_BF16 ? launch_verify_t<__bf16>(p, a, stream)
                              : launch_verify_t<float>(p, a, stream);
}

}  // namespace hxmi
