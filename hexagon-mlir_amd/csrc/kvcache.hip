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

// Inclusive sums of two numbers over the workgroup's threads in thread order,
// and their totals.
template <int NT>
__device__ __forceinline__ void block_scan2(int64_t& a, int64_t& b, int64_t (*part)[NT / 64], int64_t& total_a,
                                            int64_t& total_b) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  a = (int64_t)scan64((uint64_t)a);
  b = (int64_t)scan64((uint64_t)b);
  __syncthreads();
  if (lane == 63) {
    part[0][w] = a;
    part[1][w] = b;
  }
  __syncthreads();
  total_a = total_b = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    const int64_t ta = part[0][i], tb = part[1][i];
    a += i < w ? ta : 0;
    b += i < w ? tb : 0;
    total_a += ta;
    total_b += tb;
  }
}

// Every workgroup takes the sums over all requests (at most kPlanRequests,
// a few KB of lengths out of L2), then its waves take a request each: no
// workgroup waits for another and one launch does.  What bounds it is that
// chain: load, sums, look-ups, stores.  A request's page numbers are looked up
// 64 at a time, a lane each, before the slots that lie in them.
// 16 requests: 10.1 us with shuffled sums and lengths read again, 3.9 us;
// 1024 requests, 16384 rows: 18 us with a look-up a row, 8.3 us.
template <int NT>
__global__ __launch_bounds__(NT) void kv_plan(PArgs a) {
  __shared__ int cu[kPlanRequests + 1], first[kPlanRequests];  // rows; first block taken (-1: not admitted)
  __shared__ int freed[kPlanRequests];                         // first block released
  __shared__ int lens[kPlanRequests], added[kPlanRequests];
  __shared__ int64_t part[2][NT / 64];
  __shared__ unsigned long long taken;
  const int64_t bs1 = (1ll << a.lb) - 1, limit = (int64_t)a.width << a.lb;
  const int lane = threadIdx.x & 63;

  if (threadIdx.x == 0) taken = 0;
  const int64_t had = min(max((int64_t)*a.count, (int64_t)0), (int64_t)a.capacity);
  int64_t back_all = 0, rows = 0;
  for (int r0 = 0; r0 < a.requests; r0 += NT) {
    const int r = r0 + threadIdx.x;
    const bool in = r < a.requests;
    const int add = in ? a.added[r] : 0;
    const int64_t len = in ? min(max((int64_t)a.lens[r], (int64_t)0), limit) : 0;
    const int64_t back = add < 0 ? (len + bs1) >> a.lb : 0, more = max(add, 0);
    int64_t back_to = back, rows_to = more, back_total, rows_total;
    block_scan2<NT>(back_to, rows_to, part, back_total, rows_total);
    if (in) {
      lens[r] = (int)len;
      added[r] = add;
      freed[r] = (int)(back_all + back_to - back);
      cu[r] = (int)min(rows + rows_to - more, (int64_t)INT32_MAX);
    }
    back_all += back_total;
    rows += rows_total;
  }
  const int64_t avail = had + back_all;
  const int all = (int)min(rows, (int64_t)INT32_MAX);
  if (threadIdx.x == 0) cu[a.requests] = all;
  __syncthreads();
  int64_t wanted = 0;
  for (int r0 = 0; r0 < a.requests; r0 += NT) {
    const int r = r0 + threadIdx.x;
    const bool in = r < a.requests;
    const int64_t len = in ? lens[r] : 0, add = in ? max(added[r], 0) : 0, have = (len + bs1) >> a.lb;
    const int64_t need = ((len + add + bs1) >> a.lb) - have;
    // (a row count that passed 2^31 passes any `tokens`)
    const bool fits = add > 0 && have + need <= a.width && cu[in ? r : 0] + add <= a.tokens;
    const int64_t want = fits ? need : 0;
    int64_t to = want, unused = 0, total, none;
    block_scan2<NT>(to, unused, part, total, none);
    to += wanted;
    wanted += total;
    const bool admitted = fits && (want == 0 || to <= avail);
    // (the admitted ones that want blocks come first among those that want any)
    if (admitted && want > 0) atomicMax(&taken, (unsigned long long)to);
    if (in) {
      first[r] = admitted ? (int)(to - want) : -1;
      if (blockIdx.x == 0) {
        a.cu[r] = cu[r];
        a.lens_out[r] = added[r] < 0 ? 0 : (int)(admitted ? len + add : len);
      }
    }
  }
  __syncthreads();
  const int64_t left = min(avail - (int64_t)taken, (int64_t)a.capacity);
  if (threadIdx.x == 0 && blockIdx.x == 0) {
    a.cu[a.requests] = all;
    *a.count_out = (int)left;
  }

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

  const int waves = NT / 64 * gridDim.x;
  for (int r = blockIdx.x * (NT / 64) + (threadIdx.x >> 6); r < a.requests; r += waves) {
    const int64_t len = lens[r], have = (len + bs1) >> a.lb;
    int* const row = a.table + r * a.ldt;
    const int add = added[r];
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
    const int64_t end = len + add, p1 = (end + bs1) >> a.lb;
    for (int64_t p0 = len >> a.lb; p0 < p1; p0 += 64) {  // pages that take rows, 64 at a time
      const int64_t page = p0 + lane;
      int id = -1;
      if (page < p1) {
        if (page < have) {
          id = row[page];
        } else {
          id = block(at + page - have);
          row[page] = id;
        }
      }
      const int64_t q0 = max(len, p0 << a.lb), q1 = min(end, (p0 + 64) << a.lb);
      for (int64_t q = q0; q < q1; q += 64) {  // (the wave together: lanes read each other's pages)
        const int64_t pos = q + lane;
        const int64_t b = __shfl(id, (int)((pos >> a.lb) - p0) & 63, 64);
        if (pos < q1) {
          a.slots[c0 + pos - len] = b < 0 ? -1 : (b << a.lb) + (pos & bs1);
          a.positions[c0 + pos - len] = (int)pos;
        }
      }
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
// to the slot before.  Latency bounds it at one token a request (slot, scale and
// row, and where the scale grows the codes, there and back): 128 requests, 8 x
// 128 bf16, 12.6 us into blocks not touched before (about a fifth of the scales grow),
// 5 us once they have.  A prompt's rows are loaded twice, for the largest value
// and for the codes (V two bytes at a time): 6853 of 4 x 64 fp16 14 us.
template <typename T>
__global__ __launch_bounds__(256) void kv_append(CArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int hv = (int)(item % (2 * a.heads)), h = hv >> 1, is_v = hv & 1;
  const int64_t t0 = item / (2 * a.heads) * a.span;  // (a.span <= 64)
  const int bs = 1 << a.lb;
  // Rows that begin a run, among this wave's span: a slot in the cache that
  // does not follow the row before in its block.
  int64_t slot_l = -1;
  bool begins = false;
  if (t0 + lane < a.tokens) {
    slot_l = a.slots[t0 + lane];
    const int64_t before = t0 + lane > 0 ? a.slots[t0 + lane - 1] : -1;
    begins = slot_l >= 0 && slot_l < a.cells && ((slot_l & (bs - 1)) == 0 || before != slot_l - 1);
  }
  for (uint64_t runs = __ballot(begins && lane < a.span); runs; runs &= runs - 1) {
    const int l = __ffsll((unsigned long long)runs) - 1;
    const int64_t t = t0 + l;
    const int64_t slot = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)slot_l, l) |
                         (int64_t)__builtin_amdgcn_readlane((int)(slot_l >> 32), l) << 32;
    const int off = (int)(slot & (bs - 1));
    // its rows: up to the end of its block, as far as the slots follow each other
    int n = 0;
    {
      const uint64_t miss = ~(__ballot(slot_l == slot + (lane - l)) >> l);  // (lane l's own bit is 0)
      n = l == 0 ? (miss ? __ffsll((unsigned long long)miss) - 1 : 64) : min(__ffsll((unsigned long long)miss) - 1, 64 - l);
      if (n == 64 - l)
        for (;;) {
          const int64_t u = t + n + lane;
          const bool in = n + lane < bs - off && u < a.tokens && a.slots[u] == slot + n + lane;
          const uint64_t out = __ballot(!in);
          if (out) {
            n += __ffsll((unsigned long long)out) - 1;
            break;
          }
          n += 64;
        }
      n = min(n, bs - off);
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

// Outputs [tokens, heads, d], zeros for a slot outside the cache, values past
// the type's range at its end.  A wave takes 16 rows of a head of K or of V, two
// dims a lane, piece of 16 tokens by piece: those of a piece take their V codes
// from one 32-byte load a lane (4500 rows of 8 x 128: 13.5 us with a load a byte,
// 13.7 us with K and V by one wave, 11.0 us).
template <typename T>
__global__ __launch_bounds__(256) void kv_read(CArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int hv = (int)(item % (2 * a.heads)), h = hv >> 1, is_v = hv & 1;
  const int64_t t0 = item / (2 * a.heads) * 16;
  const float top = std::is_same_v<T, _Float16> ? 65504.f : 0x1.fep+127f;
  const bool mine = lane < a.d >> 1;
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
    const int64_t at = (piece >> lp) * a.heads + h, c = piece & ((1 << lp) - 1);
    const int off = (int)slot & 15;  // (lane u: row u's token)
    int4v v0{}, v1{};
    uint16_t two[16] = {};  // two codes of each row
    if (is_v) {
      if (mine) {
        const int8_t* const vc = a.codes[1] + at * a.bytes + (c * a.dp + 2 * lane) * 16;
        v0 = *(const int4v*)vc;
        v1 = *(const int4v*)(vc + 16);
      }
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const int o = __builtin_amdgcn_readlane(off, u), w = o >> 2, b = (o & 3) * 8;
        const int x = w & 2 ? (w & 1 ? v0[3] : v0[2]) : (w & 1 ? v0[1] : v0[0]);
        const int y = w & 2 ? (w & 1 ? v1[3] : v1[2]) : (w & 1 ? v1[1] : v1[0]);
        two[u] = (uint16_t)((x >> b & 0xff) | (y >> b & 0xff) << 8);
      }
    } else if (mine) {
      const int8_t* const kc = a.codes[0] + at * a.bytes + c * 16 * a.dp + 2 * lane;
#pragma unroll
      for (int u = 0; u < 16; ++u) two[u] = *(const uint16_t*)(kc + __builtin_amdgcn_readlane(off, u) * a.dp);
    }
    const float scale = a.scale[is_v][at];
    const bool inside = scale * 127.f <= top;  // (false for NaN)
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      if (!(rows >> u & 1)) continue;
      float x = (float)(int8_t)two[u] * scale, y = (float)(int8_t)(two[u] >> 8) * scale;
      if (!inside) {
        x = x != x ? x : fminf(fmaxf(x, -top), top);
        y = y != y ? y : fminf(fmaxf(y, -top), top);
      }
      const T f[2] = {(T)x, (T)y};
      uint32_t bits;
      __builtin_memcpy(&bits, f, 4);
      if (mine) *(uint32_t*)(out + u * step) = bits;
    }
  }
}

}  // namespace

hipError_t launch_kv_plan(const KvPlanProblem& p, hipStream_t stream) {
  const PArgs a{p.lens, p.added, p.table, p.stack, p.count, p.slots, p.positions, p.cu, p.lens_out, p.count_out,
                (int)p.requests, (int)p.width, (int)p.capacity, (int)p.tokens, p.log2_block, p.ldt};
  // a wave a request, or 256 rows; few requests: the fewer waves the sums pass over
  const int64_t work = p.requests > p.tokens / 256 ? p.requests : p.tokens / 256;
  const int nt = work <= 64 ? 256 : 1024;
  const int64_t wgs = (work + nt / 64 - 1) / (nt / 64);
  const dim3 grid((unsigned)(wgs < 1 ? 1 : wgs < 128 ? wgs : 128));
  if (nt == 256) hipLaunchKernelGGL(kv_plan<256>, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(kv_plan<1024>, grid, dim3(1024), 0, stream, a);
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
  // waves, more (up to 64) for long prompts, whose rows mostly begin none
  const int64_t per_row = 2 * p.kv_heads;
  int64_t span = p.tokens * per_row / 8192;
  a.span = (int)(span < 1 ? 1 : span < 64 ? span : 64);
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
  const int64_t blocks = ((p.tokens + 15) / 16 * 2 * p.kv_heads + 3) / 4;
  if (blocks >= (1ll << 31)) return hipErrorInvalidValue;
  const auto fn = p.dtype == DT_BF16 ? kv_read<__bf16> : kv_read<_Float16>;
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace hxmi
