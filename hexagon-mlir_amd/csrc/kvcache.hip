// The 8-bit key/value cache: block tables and slot maps from request lengths
// (kv_plan), rows of keys and values into it (kv_append) and back (kv_read).
//
// Layout (block of B tokens, Dp = head dim rounded up to 16):
//   K codes [blocks][heads][B][Dp]        rows as they came: K.Q^T's operand
//   V codes [blocks][heads][B/16][Dp][16] 16 tokens of one dimension together:
//                                         the operand of P.V's MFMAs as it lies
//   scales  [blocks][heads]               value = code * scale, one each for K and V
// A scale has 11 significant bits (kept in fp32).  Then code * scale and
// 127 * scale are exact in 32 bits, and a quotient of a 16-bit value (or of
// code * old scale) by a scale is either a tie of two codes or at least
// 2^-19 (relative) away from one, so that 32-bit arithmetic finds the code
// that the exact quotient rounds to (round_code).
#include "hxmi_common.h"
#include "hxmi_internal.h"

namespace hxmi {
namespace {

typedef int int4u __attribute__((ext_vector_type(4), aligned(2)));  // (rows start anywhere)

// ---- kv_plan -------------------------------------------------------------------

struct PArgs {
  const int* lens;
  const int* added;
  int* table;
  int* stack;
  const int* count;
  int64_t* slots;
  int* positions;
  int* cu;
  int* lens_out;
  int* count_out;
  int requests, width, capacity, tokens, lb;  // lb: log2 of the block size
  int64_t ldt;
};

// Inclusive sum over the workgroup's threads; `total` receives the whole sum.
template <int NT>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* part, int64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t t = __shfl_up(v, o, 64);
    if (lane >= o) v += t;
  }
  __syncthreads();
  if (lane == 63) part[w] = v;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    const int64_t t = part[i];
    if (i < w) before += t;
    total += t;
  }
  return before + v;
}

// Every workgroup takes the sums over all requests (at most kPlanRequests,
// a few KB of lengths out of L2), then its waves take a request each: no
// workgroup waits for another and one launch does.  What bounds it is that
// chain: load, sums, look-ups, stores.
template <int NT>
__global__ __launch_bounds__(NT) void kv_plan(PArgs a) {
  extern __shared__ int shared[];  // cu [requests + 1], first block taken (-1: not admitted), first released
  __shared__ int64_t part[NT / 64];
  int* const cu = shared;
  int* const first = cu + a.requests + 1;
  int* const freed = first + a.requests;
  const int64_t bs1 = (1ll << a.lb) - 1, limit = (int64_t)a.width << a.lb;
  auto held = [&](int r) { return min(max((int64_t)a.lens[r], (int64_t)0), limit); };

  int64_t back_all = 0;
  for (int r0 = 0; r0 < a.requests; r0 += NT) {
    const int r = r0 + threadIdx.x;
    const bool in = r < a.requests;
    const int64_t back = in && a.added[r] < 0 ? (held(r) + bs1) >> a.lb : 0;
    int64_t total;
    const int64_t incl = block_scan<NT>(back, part, total);
    if (in) freed[r] = (int)(back_all + incl - back);
    back_all += total;
  }
  const int64_t had = min(max((int64_t)*a.count, (int64_t)0), (int64_t)a.capacity), avail = had + back_all;
  int64_t rows = 0, wanted = 0, taken = 0;
  for (int r0 = 0; r0 < a.requests; r0 += NT) {
    const int r = r0 + threadIdx.x;
    const bool in = r < a.requests;
    const int64_t add = in ? max(a.added[r], 0) : 0, len = in ? held(r) : 0;
    int64_t total;
    const int64_t end = rows + block_scan<NT>(add, part, total);
    rows += total;
    const int64_t have = (len + bs1) >> a.lb, need = ((len + add + bs1) >> a.lb) - have;
    const bool fits = add > 0 && have + need <= a.width && end <= a.tokens;
    const int64_t want = fits ? need : 0, incl = wanted + block_scan<NT>(want, part, total);
    wanted += total;
    const bool admitted = fits && (want == 0 || incl <= avail);
    int64_t unused = block_scan<NT>(admitted ? want : 0, part, total);
    (void)unused;
    taken += total;
    if (in) {
      cu[r] = (int)min(end - add, (int64_t)INT32_MAX);
      // (the admitted ones that want blocks come first among those that want any)
      first[r] = admitted ? (int)(incl - want) : -1;
      if (blockIdx.x == 0) {
        a.cu[r] = cu[r];
        a.lens_out[r] = a.added[r] < 0 ? 0 : (int)(admitted ? len + add : len);
      }
    }
  }
  const int all = (int)min(rows, (int64_t)INT32_MAX);
  const int64_t left = min(avail - taken, (int64_t)a.capacity);
  if (threadIdx.x == 0) {
    cu[a.requests] = all;
    if (blockIdx.x == 0) {
      a.cu[a.requests] = all;
      *a.count_out = (int)left;
    }
  }
  __syncthreads();

  // The block that comes i-th off the stack: one of the held ones, or one
  // that a request of this step has released (still in its table row).
  auto block = [&](int64_t i) {
    const int64_t p = avail - 1 - i;
    if (p < had) return a.stack[p];
    const int q = (int)(p - had);
    int lo = 0, hi = a.requests;  // the last request with freed <= q that has released any
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (freed[mid] <= q) lo = mid;
      else hi = mid;
    }
    return a.table[lo * a.ldt + (q - freed[lo])];
  };

  const int lane = threadIdx.x & 63, waves = NT / 64 * gridDim.x;
  for (int r = blockIdx.x * (NT / 64) + (threadIdx.x >> 6); r < a.requests; r += waves) {
    const int64_t len = held(r), have = (len + bs1) >> a.lb;
    int* const row = a.table + r * a.ldt;
    const int add = a.added[r];
    if (add < 0) {
      for (int64_t i = lane; i < have; i += 64) {
        const int64_t p = had + freed[r] + i;
        if (p < left) a.stack[p] = row[i];
      }
      continue;
    }
    const int64_t at = first[r];
    const int64_t c0 = cu[r], c1 = cu[r + 1];  // (at most 2^31 - 1: sums with them need 64 bits)
    if (at < 0) {
      for (int64_t t = c0 + lane; t < min(c1, (int64_t)a.tokens); t += 64) {
        a.slots[t] = -1;
        a.positions[t] = 0;
      }
      continue;
    }
    const int64_t need = ((len + add + bs1) >> a.lb) - have;
    for (int64_t j = lane; j < need; j += 64) row[have + j] = block(at + j);
    for (int64_t t = c0 + lane; t < c1; t += 64) {
      const int64_t p = len + t - c0, b = p >> a.lb;
      const int64_t id = b < have ? row[b] : block(at + b - have);
      a.slots[t] = id < 0 ? -1 : (id << a.lb) + (p & bs1);
      a.positions[t] = (int)p;
    }
  }
  for (int64_t t = (int64_t)all + blockIdx.x * NT + threadIdx.x; t < a.tokens; t += (int64_t)NT * gridDim.x) {
    a.slots[t] = -1;
    a.positions[t] = 0;
  }
}

// ---- codes and scales ------------------------------------------------------------

// The smallest number of 11 significant bits that is at least amax / 127 (at
// least 2^-100: smaller values are held as zero codes), 0 for 0 and NaN where
// a value is not finite.
__device__ __forceinline__ float block_scale(float amax) {
  if (!(amax < INFINITY)) return __uint_as_float(0x7fc00000u);
  uint32_t b = __float_as_uint(amax / 127.f) & ~0x1fffu;
  if (__uint_as_float(b) * 127.f < amax) b += 0x2000u;
  return amax > 0.f ? fmaxf(__uint_as_float(b), 0x1p-100f) : 0.f;
}

// The integer that y's exact value rounds to (half to even), y being off by
// at most 2^-22 of it: three bits fewer take a tie back to the tie (ties have
// 9 significant bits), and anything else stays on its side.  NaN gives 0.
__device__ __forceinline__ int round_code(float y) {
  return (int)rintf(__uint_as_float((__float_as_uint(y) + 4u) & ~7u));
}

template <typename T>
struct Bits16;
template <>
struct Bits16<_Float16> {
  static constexpr uint32_t inf = 0x7c00;
};
template <>
struct Bits16<__bf16> {
  static constexpr uint32_t inf = 0x7f80;
};

// ---- kv_append -------------------------------------------------------------------

struct CArgs {
  const char* x[2];   // rows of k and of v
  int8_t* codes[2];   // cache: K, V
  float* scale[2];
  const int64_t* slots;
  char* out[2];       // kv_read
  int64_t ld[2], hs[2];  // row and head strides of x, elements
  int64_t tokens, cells;  // cells: blocks * block size
  int heads, d, dp, lb, span;
  int64_t bytes;  // of a block's codes of one head
};

// A wave writes one run (rows of the call that go to consecutive slots of one
// block) of one head of K or V: the largest magnitude of its rows, the
// block's scale, the block's earlier codes again if the scale has grown, its
// own codes.  A run is found by its first row: the row before it does not go
// to the slot before.  Latency bounds it at one token a request (three
// dependent loads: slot, scale and row, codes), the loads and stores at a
// prompt's length.
template <typename T>
__global__ __launch_bounds__(256) void kv_append(CArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int hv = (int)(item % (2 * a.heads)), h = hv >> 1, is_v = hv & 1;
  const int64_t t0 = item / (2 * a.heads) * a.span, t1 = min(t0 + a.span, a.tokens);
  const int bs = 1 << a.lb;
  for (int64_t t = t0; t < t1; ++t) {
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.cells) continue;
    const int off = (int)(slot & (bs - 1));
    if (off > 0 && t > 0 && a.slots[t - 1] == slot - 1) continue;
    int n = 0;  // rows of the run
    for (;;) {
      const int64_t u = t + n + lane;
      const bool in = n + lane < bs - off && u < a.tokens && a.slots[u] == slot + n + lane;
      const uint64_t miss = __ballot(!in);
      if (miss) {
        n += __ffsll((unsigned long long)miss) - 1;
        break;
      }
      n += 64;
    }
    const T* const x = (const T*)a.x[is_v] + t * a.ld[is_v] + h * a.hs[is_v];
    const int64_t ld = a.ld[is_v];
    const int64_t blk = slot >> a.lb;
    int8_t* const codes = a.codes[is_v] + (blk * a.heads + h) * a.bytes;
    float* const scale = a.scale[is_v] + blk * a.heads + h;

    const int per = a.d >> 3;  // 16-byte pieces of a row
    uint32_t top = 0;
    for (int i = lane; i < n * per; i += 64) {
      const int row = i / per, c = i - row * per;
      const int4v raw = *(const int4u*)(x + row * ld + c * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t b = (uint32_t)raw[e] & 0x7fff7fffu;
        top = max(top, max(b & 0xffffu, b >> 16));
      }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    const float amax = top >= Bits16<T>::inf ? INFINITY : (float)__builtin_bit_cast(T, (unsigned short)top);

    const float old = off == 0 ? 0.f : *scale;
    float now = old;
    if (amax > 127.f * old) {
      now = block_scale(amax);
      if (n < bs) {  // the codes that are there, at the new scale (a block that starts anew has none)
        const float ratio = old / now;
        for (int64_t i = lane * 16; i < a.bytes; i += 1024) {
          int4v w{};
          if (old != 0.f) {
            w = *(int4v*)(codes + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t o4 = 0;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                o4 |= ((uint32_t)round_code((float)(int8_t)((uint32_t)w[e] >> (8 * j)) * ratio) & 0xffu) << (8 * j);
              w[e] = (int)o4;
            }
          }
          *(int4v*)(codes + i) = w;
        }
        wait_vmcnt0();  // (the run's own codes go over some of them)
      }
    }
    if (lane == 0) *scale = now;
    const float inv = 1.f / now;
    // (a zero block: 0 * inf is NaN, code 0)

    if (!is_v) {
      const int pp = a.dp >> 3;
      for (int i = lane; i < n * pp; i += 64) {
        const int row = i / pp, c = i - row * pp;
        uint32_t o2[2] = {0, 0};
        if (c < per) {
          const int4v raw = *(const int4u*)(x + row * ld + c * 8);
          T f[8];
          __builtin_memcpy(f, &raw, 16);
#pragma unroll
          for (int e = 0; e < 8; ++e) o2[e >> 2] |= ((uint32_t)round_code((float)f[e] * inv) & 0xffu) << (8 * (e & 3));
        }
        *(uint2*)(codes + (int64_t)(off + row) * a.dp + c * 8) = make_uint2(o2[0], o2[1]);
      }
    } else {
      for (int c = off >> 4; c <= (off + n - 1) >> 4; ++c) {
        const int k0 = max(off, c * 16), k1 = min(off + n, c * 16 + 16);
        for (int d = lane; d < a.dp; d += 64) {
          int8_t* const dst = codes + ((int64_t)c * a.dp + d) * 16;
          if (k1 - k0 == 16) {
            uint32_t o4[4] = {0, 0, 0, 0};
            if (d < a.d) {
#pragma unroll
              for (int e = 0; e < 16; ++e)
                o4[e >> 2] |= ((uint32_t)round_code((float)x[(int64_t)(k0 + e - off) * ld + d] * inv) & 0xffu)
                              << (8 * (e & 3));
            }
            *(int4v*)dst = int4v{(int)o4[0], (int)o4[1], (int)o4[2], (int)o4[3]};
          } else {
            for (int k = k0; k < k1; ++k)
              dst[k & 15] = d < a.d ? (int8_t)round_code((float)x[(int64_t)(k - off) * ld + d] * inv) : (int8_t)0;
          }
        }
      }
    }
  }
}

// ---- kv_read ---------------------------------------------------------------------

// Eight values of a row a lane; outputs [tokens, heads, d], zeros for a slot
// outside the cache, values past the type's range at its end.
template <typename T>
__global__ __launch_bounds__(256) void kv_read(CArgs a) {
  const int per = a.d >> 3;
  const int64_t all = a.tokens * a.heads * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int c = (int)(i % per);
    const int64_t th = i / per;
    const int h = (int)(th % a.heads);
    const int64_t t = th / a.heads, slot = a.slots[t];
    const bool in = slot >= 0 && slot < a.cells;
    T f[2][8] = {};
    if (in) {
      const int64_t blk = slot >> a.lb;
      const int off = (int)(slot & ((1 << a.lb) - 1));
      const int8_t* const kc = a.codes[0] + (blk * a.heads + h) * a.bytes + (int64_t)off * a.dp + c * 8;
      const int8_t* const vc =
          a.codes[1] + (blk * a.heads + h) * a.bytes + ((int64_t)(off >> 4) * a.dp + c * 8) * 16 + (off & 15);
      const float ks = a.scale[0][blk * a.heads + h], vs = a.scale[1][blk * a.heads + h];
      const float top = std::is_same_v<T, _Float16> ? 65504.f : 0x1.fep+127f;
      const uint2 kw = *(const uint2*)kc;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float k = (float)(int8_t)((e < 4 ? kw.x : kw.y) >> (8 * (e & 3))) * ks, v = (float)vc[16 * e] * vs;
        f[0][e] = (T)(k != k ? k : fminf(fmaxf(k, -top), top));
        f[1][e] = (T)(v != v ? v : fminf(fmaxf(v, -top), top));
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) __builtin_memcpy(a.out[s] + i * 16, f[s], 16);
  }
}

}  // namespace

hipError_t launch_kv_plan(const KvPlanProblem& p, hipStream_t stream) {
  constexpr int NT = 1024;
  PArgs a{p.lens, p.added, p.table, p.stack, p.count, p.slots, p.positions, p.cu, p.lens_out, p.count_out,
          (int)p.requests, (int)p.width, (int)p.capacity, (int)p.tokens, p.log2_block, p.ldt};
  const int64_t lds = (3 * p.requests + 1) * 4;
  const int64_t work = p.requests > p.tokens / 256 ? p.requests : p.tokens / 256;
  const int64_t wgs = (work + NT / 64 - 1) / (NT / 64);
  hipLaunchKernelGGL(kv_plan<NT>, dim3((unsigned)(wgs < 1 ? 1 : wgs < 128 ? wgs : 128)), dim3(NT), (unsigned)lds, stream,
                     a);
  return hipGetLastError();
}

static CArgs cache_args(const KvCacheProblem& p) {
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
  a.dp = (int)((p.d + 15) / 16 * 16);
  a.lb = p.log2_block;
  a.bytes = (int64_t)a.dp << a.lb;
  return a;
}

hipError_t launch_kv_append(const KvCacheProblem& p, hipStream_t stream) {
  CArgs a = cache_args(p);
  a.x[0] = (const char*)p.k;
  a.x[1] = (const char*)p.v;
  a.ld[0] = p.ldk;
  a.ld[1] = p.ldv;
  a.hs[0] = p.hsk;
  a.hs[1] = p.hsv;
  // a wave looks for runs in `span` rows: one while that leaves at most 8192
  // waves, more (up to a block's) for long prompts, whose rows mostly begin none
  const int64_t per_row = 2 * p.kv_heads;
  int64_t span = p.tokens * per_row / 8192;
  const int64_t bs = 1ll << p.log2_block;
  a.span = (int)(span < 1 ? 1 : span < bs ? span : bs);
  const int64_t blocks = ((p.tokens + a.span - 1) / a.span * per_row + 3) / 4;
  if (blocks >= (1ll << 31)) return hipErrorInvalidValue;
  const auto fn = p.dtype == DT_BF16 ? kv_append<__bf16> : kv_append<_Float16>;
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_kv_read(const KvCacheProblem& p, hipStream_t stream) {
  CArgs a = cache_args(p);
  a.out[0] = (char*)p.k_out;
  a.out[1] = (char*)p.v_out;
  const int64_t n = p.tokens * p.kv_heads * (p.d / 8), blocks = (n + 255) / 256;
  const auto fn = p.dtype == DT_BF16 ? kv_read<__bf16> : kv_read<_Float16>;
  hipLaunchKernelGGL(fn, dim3((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace hxmi
