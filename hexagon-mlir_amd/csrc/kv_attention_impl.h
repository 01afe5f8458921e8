// What both attention kernels over a key/value cache share (kv_attention.hip: 8
// bits, kv4_attention.hip: 4): tiles of a request's rows, shares of their keys,
// queries as MFMA operands.
#pragma once

#include "hxmi_common.h"
#include "hxmi_internal.h"

namespace hxmi {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
typedef int int4u __attribute__((ext_vector_type(4), aligned(2)));
typedef int int2u __attribute__((ext_vector_type(2), aligned(2)));

// A call's queries, requests and tiles.
struct TileArgs {
  const char* q;
  const int* table;
  const int* lens;
  const int* cu;  // null: one row a request
  char* o;
  char* ws;
  int64_t ldq, hq, ldo, ho, ldt;
  int64_t bytes;  // of a block's codes of one head
  int requests, tokens, kv_heads, group, d, dp, lb, blocks, width;
  int tiles;         // of a key/value head
  int full, nsplit;  // the first `full` tiles of all heads run whole, the others in nsplit shares of their keys
  float c;  // scale * log2(e)
};

// Combine the four lanes that hold a row (l, l + 16, l + 32, l + 48).
template <typename Op>
__device__ __forceinline__ float row_reduce(float v, Op op) {
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(r32[0]), __uint_as_float(r32[1]));
}
__device__ __forceinline__ float row_max(float v) {
  return row_reduce(v, [](float x, float y) { return fmaxf(x, y); });
}

// 2^(x - top), 0 where x is -inf (so is top where nothing has been seen).
__device__ __forceinline__ float rel_exp2(float x, float top) {
  return x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x - top);
}

// The request and rows of a tile of RT rows.  With cu, request r's tiles begin
// at number floor(cu[r] * group / RT) + r: never more than RT rows a tile, and
// no sums over the requests before it.  Numbers in between have no rows.
struct Rows {
  int r, first, n, row0, len;
  int64_t count;
};
template <int RT>
__device__ __forceinline__ bool rows_of(const TileArgs& a, int tile, Rows& t) {
  if (a.cu) {
    int lo = 0, hi = a.requests;
    auto start = [&](int i) { return (int64_t)min(max(a.cu[i], 0), a.tokens) * a.group / RT + i; };
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start(mid) <= tile) lo = mid;
      else hi = mid;
    }
    t.r = lo;
    t.first = min(max(a.cu[lo], 0), a.tokens);
    t.n = min(max(a.cu[lo + 1], t.first), a.tokens) - t.first;
    t.row0 = (int)min((tile - start(lo)) * RT, (int64_t)INT32_MAX);
  } else {
    const int per = (a.group + RT - 1) / RT;
    t.r = t.first = tile / per;
    t.n = 1;
    t.row0 = (tile - t.r * per) * RT;
  }
  t.count = (int64_t)t.n * a.group;
  if (t.row0 < 0 || t.row0 >= t.count) return false;
  t.len = (int)min(max((int64_t)a.lens[t.r], (int64_t)0), (int64_t)a.width << (a.lb + 4));
  return true;
}

// A workgroup's tile (of all heads) and share of its keys.
struct Share {
  int item, split, count;
};
// Workgroups go round-robin over the 8 XCDs; each XCD takes a contiguous run of
// numbers, so the tiles that read the same keys read them through one L2.
__device__ __forceinline__ int xcd_run(int id, int total) {
  const int per = total >> 3, rem = total & 7, xcd = id & 7;
  return xcd * per + (xcd < rem ? xcd : rem) + (id >> 3);
}

__device__ __forceinline__ Share share_of(const TileArgs& a) {
  const int id = blockIdx.x;
  if (id < a.full) return Share{xcd_run(id, a.full), 0, 1};
  const int j = xcd_run(id - a.full, gridDim.x - a.full);
  return Share{a.full + j / a.nsplit, j % a.nsplit, a.nsplit};
}

// Eight elements of q as fp16, and what the scores are to be multiplied by.  q
// in bf16 takes a power of two `ex` that brings the row's largest element to
// [2^14, 2^15): the row's elements become multiples of 2^-24, at most 2^-38 of it.
template <typename T>
__device__ __forceinline__ float largest(const T (&x)[8], float top) {
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf((float)x[e]));
  return top;
}
__device__ __forceinline__ int exponent_of(float top) {
  const int ex = top > 0.f && top < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
  return min(max(ex, -120), 120);
}
template <typename T>
__device__ __forceinline__ half8v q_operand(const T (&x)[8], int ex) {
  half8v h;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    h[e] = std::is_same_v<T, _Float16> ? (_Float16)(float)x[e] : (_Float16)__builtin_ldexpf((float)x[e], ex);
  return h;
}

// Rows of a workgroup, tiles of them and the shares of the keys: from sizes
// alone, so the workspace can be asked for beforehand.
struct KvPlan {
  int rt, nsplit;  // rows of a tile: 16, or 128 (kv_attention_tiles)
  int64_t tiles, full;
};
inline KvPlan plan_of(const KvAttnSizes& p, int64_t slots = 512) {  // slots: workgroups for 16 rows on the card at a time
  KvPlan r;
  const int64_t group = p.heads / p.kv_heads;
  const int64_t rows = (p.cu ? (p.tokens + p.requests - 1) / p.requests : 1) * group;  // of a request, on average
  // Tiles of 128 rows where a request has about as many and every CU would get
  // one of 16 (us, 16 / 128 rows a tile, contexts of 4000 tokens; dims of 128, 8
  // key/value heads, 37 requests: 80 rows 186 / 188, 112 rows 250 / 167; dims of
  // 64, 4 heads, 48 requests: 192 rows 107 / 140, 256 rows 139 / 117; one request,
  // 128 dims: 256 rows 28 / 30, 1024 rows 56 / 43).  Tiles of 32 rows were slower
  // than 16 up to 100 rows and never the fastest.  The average is over requests
  // that have no rows or one as well, so a call that mixes decoding requests and
  // a prompt's chunk runs both on tiles that suit one of them: over 8192 keys,
  // 63 rows and a chunk of 2048 722 us in one call, 180 + 283 in two; 256 rows and
  // a chunk of 512 928 us, 711 + 110 in two.
  const bool wide = rows > (p.d > 64 ? 96 : 255) && p.tokens * p.heads >= 4096;
  r.rt = wide ? 128 : 16;
  const int64_t rt = r.rt;
  r.tiles = p.cu ? p.tokens * group / rt + p.requests : p.requests * ((group + rt - 1) / rt);
  // The card takes 512 workgroups at a time, two a CU.  Whole rounds of them
  // run unshared; the tiles that are left share their keys out until they make
  // one more round, at least 256 keys to a share (a group of 64 for each wave), or
  // 512 in 128-row tiles (eight stages) and where the card takes more than 512
  // workgroups.  575 tiles of 128 rows x 8000 keys, before later
  // steps: 391 us unshared, 292 with all of them in two shares, 281 with the last
  // 63 in eight.  The table's width stands for the lengths, which only the GPU
  // knows: shares past a request's keys are joined for nothing (one user of 1900
  // tokens: 7.5 us with a table of 30 pages, 10.6 with 128, 24 with 512 or more).
  const int64_t items = r.tiles * p.kv_heads, least = wide || slots > 512 ? 512 : 256, most = (p.width * p.block + least - 1) / least;
  if (wide) slots = 512;
  const int64_t left = items % slots;
  int64_t n = left ? slots / left : 1;
  n = n < most ? n : most;
  r.nsplit = (int)(n < 1 ? 1 : n < 128 ? n : 128);
  r.full = r.nsplit > 1 ? items - left : items;
  return r;
}

// What a launch takes from its sizes and plan (not the cache's own: dp, bytes).
inline void tile_args(const KvAttnSizes& p, const KvPlan& k, TileArgs& a) {
  a.q = (const char*)p.q;
  a.table = p.table;
  a.lens = p.lens;
  a.cu = p.cu;
  a.o = (char*)p.o;
  a.ws = (char*)p.ws;
  a.ldq = p.ldq;
  a.hq = p.hsq;
  a.ldo = p.ldo;
  a.ho = p.hso;
  a.ldt = p.ldt;
  a.requests = (int)p.requests;
  a.tokens = (int)p.tokens;
  a.kv_heads = (int)p.kv_heads;
  a.group = (int)(p.heads / p.kv_heads);
  a.d = (int)p.d;
  a.lb = __builtin_ctzll((unsigned long long)p.block) - 4;
  a.blocks = (int)p.blocks;
  a.width = (int)p.width;
  a.tiles = (int)k.tiles;
  a.full = (int)k.full;
  a.nsplit = k.nsplit;
  a.c = p.scale * kLog2e;
}

}  // namespace
}  // namespace hxmi
