// Attention over the 8-bit key/value cache (layout: kvcache.hip), causal over
// ragged requests, grouped heads: row i of a request with n rows and L tokens
// in the cache sees keys j <= L - n + i,
//   o = sum_j p_j vc_j vs_j / sum_j p_j,  p_j = exp(scale * ks_j (q . kc_j) - max).
//
// A workgroup of four waves owns 16 * QT rows (token, head of the group) of
// one key/value head and, where there are few such tiles, one of `nsplit`
// shares of the keys; its waves take every fourth group of 64 keys.  Codes go
// from memory straight to registers in the layout of the MFMA operands, so
// nothing passes through LDS until the waves' partial results are joined:
//   * scores as D[key][row] = Kc . Q^T (16x16x32 MFMAs).  A lane's K codes
//     are 16 bytes of one token; the head dims of a step may come in any
//     order, so they feed two steps as they lie.  Tile t's row 4 g + i is key
//     16 g + 4 t + i of the group, so the 16 scores of a lane (row l % 16,
//     g = l / 16) are keys 16 g .. 16 g + 15 in order: one page's, with one
//     K and one V scale a lane;
//   * those 16 weights are the B operand of P.V as they are, and 16 bytes of
//     V (16 tokens of one head dim) the A operand: D[dim][row];
//   * codes become fp16 exactly (conversion below).  q in bf16 is brought to
//     fp16 under a power of two a row, exact for all that counts beside the
//     row's largest element;
//   * the K scale multiplies the score.  The V scale multiplies the weight
//     before its rounding to fp16, relative to 2^mv, the running maximum of
//     score + log2(vs): the weights P.V sees stay in (0, 2^8] whatever the
//     ratio of the scales, and the sum of the p_j stays apart in fp32.
//     Weights round to 11 bits, half a step relative each, like the fp16
//     weights of the fused attention; scores, maxima, sums and O are fp32.
// One token a request is bound by the codes' bytes; rows in the hundreds by
// the vector ALUs (conversion and softmax), which QT tiles of rows share.
#include "hxmi_common.h"
#include "hxmi_internal.h"

namespace hxmi {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
typedef int int4u __attribute__((ext_vector_type(4), aligned(2)));
typedef int int2u __attribute__((ext_vector_type(2), aligned(2)));

struct KArgs {
  const char* q;
  const int8_t* k;
  const int8_t* v;
  const float* ks;
  const float* vs;
  const int* table;
  const int* lens;
  const int* cu;  // null: one row a request
  char* o;
  char* ws;
  int64_t ldq, hq, ldo, ho, ldt;
  int64_t bytes;  // of a block's codes of one head
  int requests, tokens, kv_heads, group, d, dp, lb, blocks, width;
  int tiles, nsplit;
  float c;  // scale * log2(e)
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

// What a wave knows of its QT x 16 rows: O relative to 2^mv, the sum of the
// weights (this lane's part) relative to 2^m.
template <int QT, int DT>
struct Partial {
  static constexpr int N = QT * (DT * 4 + 3);  // floats a lane
  float4v o[QT][DT];
  float m[QT], mv[QT], l[QT];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int a = 0; a < QT; ++a) {
#pragma unroll
      for (int t = 0; t < DT; ++t) o[a][t] = float4v{0.f, 0.f, 0.f, 0.f};
      m[a] = mv[a] = -INFINITY;
      l[a] = 0.f;
    }
  }
  // Every float becomes f(its index, it).
  template <typename F>
  __device__ __forceinline__ void each(F&& f) {
#pragma unroll
    for (int a = 0; a < QT; ++a) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[a][t][i] = f((a * DT + t) * 4 + i, o[a][t][i]);
      m[a] = f(QT * DT * 4 + a, m[a]);
      mv[a] = f(QT * DT * 4 + QT + a, mv[a]);
      l[a] = f(QT * DT * 4 + 2 * QT + a, l[a]);
    }
  }
  __device__ __forceinline__ void add(const Partial& p) {
#pragma unroll
    for (int a = 0; a < QT; ++a) {
      const float mn = fmaxf(m[a], p.m[a]), vn = fmaxf(mv[a], p.mv[a]);
      l[a] = l[a] * rel_exp2(m[a], mn) + p.l[a] * rel_exp2(p.m[a], mn);
      const float x = rel_exp2(mv[a], vn), y = rel_exp2(p.mv[a], vn);
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[a][t][i] = o[a][t][i] * x + p.o[a][t][i] * y;
      m[a] = mn;
      mv[a] = vn;
    }
  }
};

// DC: 64-dim pieces of a row; WHOLE: the head dim is 64 * DC.
template <typename T, int DC, bool WHOLE, int QT>
__global__ __launch_bounds__(256, QT == 1 ? 2 : 1) void kv_attention(KArgs a) {
  constexpr int DT = DC * 4, RT = 16 * QT, NV = Partial<QT, DT>::N;
  constexpr bool BF16 = !std::is_same_v<T, _Float16>;
  __shared__ __attribute__((aligned(16))) float joined[3 * NV * 64];
  __shared__ int last_split;

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lg = lane >> 4;

  // Workgroups go round-robin over the 8 XCDs; each XCD takes a contiguous
  // run of tiles, so those that read the same keys read them through one L2.
  int id = blockIdx.x;
  {
    const int total = gridDim.x, per = total >> 3, rem = total & 7, xcd = id & 7;
    id = xcd * per + (xcd < rem ? xcd : rem) + (id >> 3);
  }
  const int split = id % a.nsplit, item = id / a.nsplit;
  const int kvh = item / a.tiles, tile = item - kvh * a.tiles;

  // The tile's request and rows.  Request r's tiles begin at number
  // floor(cu[r] * group / RT) + r: never more than RT rows a tile, and no sums
  // over the requests before it.  Numbers in between have no rows.
  int r, first, n, row0;
  if (a.cu) {
    int lo = 0, hi = a.requests;
    auto start = [&](int i) {
      return (int64_t)min(max(a.cu[i], 0), a.tokens) * a.group / RT + i;
    };
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start(mid) <= tile) lo = mid;
      else hi = mid;
    }
    r = lo;
    first = min(max(a.cu[r], 0), a.tokens);
    n = min(max(a.cu[r + 1], first), a.tokens) - first;
    row0 = (int)min((tile - start(r)) * RT, (int64_t)INT32_MAX);
  } else {
    const int per = (a.group + RT - 1) / RT;
    r = tile / per;
    first = r;
    n = 1;
    row0 = (tile - r * per) * RT;
  }
  const int64_t nrows = (int64_t)n * a.group;
  if (row0 < 0 || row0 >= nrows) return;
  const int len = (int)min(max((int64_t)a.lens[r], (int64_t)0), (int64_t)a.width << (a.lb + 4));

  // This lane's rows (a row past the last one reads the last one's q)
  int last[QT];  // the last key the row sees
  half8v qf[QT][2 * DC];
  float c[QT];
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const int64_t row = min((int64_t)row0 + x * 16 + lr, nrows - 1);
    const int i = (int)(row / a.group), head = kvh * a.group + (int)(row - (int64_t)i * a.group);
    last[x] = (int)min((int64_t)len - n + i, (int64_t)len - 1);
    const T* q = (const T*)a.q + (int64_t)(first + i) * a.ldq + (int64_t)head * a.hq;
    T raw[2 * DC][8];
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * DC; ++s) {
      const int d = (s >> 1) * 64 + lg * 16 + (s & 1) * 8;
      int4v v{};
      if (WHOLE || d < a.d) v = *(const int4u*)(q + d);
      __builtin_memcpy(raw[s], &v, 16);
      if constexpr (BF16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf((float)raw[s][e]));
      }
    }
    int ex = 0;
    if constexpr (BF16) {
      // the row's largest element comes to [2^14, 2^15): what is below 2^-39
      // of it is lost, far under the fp32 sums
      top = row_max(top);
      ex = top > 0.f && top < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
      ex = min(max(ex, -120), 120);
    }
    c[x] = BF16 ? __builtin_ldexpf(a.c, -ex) : a.c;
#pragma unroll
    for (int s = 0; s < 2 * DC; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        qf[x][s][e] = BF16 ? (_Float16)__builtin_ldexpf((float)raw[s][e], ex) : (_Float16)(float)raw[s][e];
  }

  // keys this tile / all of its rows see
  const int i1 = (int)min((int64_t)n - 1, ((int64_t)row0 + RT - 1) / a.group);
  const int kend = max(0, min(len, len - n + i1 + 1));
  const int kfull = max(0, min(len, len - n + row0 / a.group + 1));
  const int groups = (kend + 63) >> 6, share = (groups + a.nsplit - 1) / a.nsplit;
  const int g1 = min(groups, (split + 1) * share);

  Partial<QT, DT> acc;
  acc.clear();

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

  int g = split * share + w;
  int bk = -1, bv = -1, bk2 = -1, bv2 = -1;
  if (g < g1) {
    bk = page(4 * g + ck);
    bv = page(4 * g + lg);
    load_k(g, bk);
    load_v(g, bv);
    if (g + 4 < g1) {
      bk2 = page(4 * (g + 4) + ck);
      bv2 = page(4 * (g + 4) + lg);
    }
  }
  for (; g < g1; g += 4) {
    // scores
    float4v s[QT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int x = 0; x < DC; ++x)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const half8v kf = operand(kr[t][x][2 * u], kr[t][x][2 * u + 1]);
#pragma unroll
          for (int y = 0; y < QT; ++y)
            s[y][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                kf, qf[y][2 * x + u], x == 0 && u == 0 ? float4v{0.f, 0.f, 0.f, 0.f} : s[y][t], 0, 0, 0);
        }
    }
    const bool more = g + 4 < g1;
    const float ks0 = ks, vs0 = vs;
    const bool there0 = there;
    if (more) load_k(g + 4, bk2);
    // softmax
    const bool whole = g * 64 + 64 <= kfull && __all(there0);  // (wave-uniform)
    const float lv = __builtin_amdgcn_logf(vs0);
    half8v p[QT][2];
#pragma unroll
    for (int y = 0; y < QT; ++y) {
      const float cs = c[y] * ks0;
      const int left = there0 ? last[y] - (g * 64 + lg * 16) : -1;  // keys of this lane up to this one are seen
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[y][t][i] *= cs;
          if (!whole && 4 * t + i > left) s[y][t][i] = -INFINITY;
          mx = fmaxf(mx, s[y][t][i]);
        }
      const float lane_max = mx;
      const float mxv = row_max(mx == -INFINITY ? -INFINITY : mx + lv);
      mx = row_max(mx);
      const bool upd = mx > acc.m[y] + 8.f || mxv > acc.mv[y] + 8.f;
      if (__any(upd)) {
        const float mn = upd ? fmaxf(acc.m[y], mx) : acc.m[y], vn = upd ? fmaxf(acc.mv[y], mxv) : acc.mv[y];
        acc.l[y] *= rel_exp2(acc.m[y], mn);
        const float f = rel_exp2(acc.mv[y], vn);
#pragma unroll
        for (int t = 0; t < DT; ++t) acc.o[y][t] *= f;
        acc.m[y] = mn;
        acc.mv[y] = vn;
      }
      const float m_use = acc.m[y] == -INFINITY ? 0.f : acc.m[y];
      const float v_use = acc.mv[y] == -INFINITY ? 0.f : acc.mv[y];
      // (a page whose every key is masked takes no part, whatever its scale;
      // the bound keeps 0 * f at 0 for scales 2^120 apart)
      float f = lane_max == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lv + m_use - v_use);
      f = f > 0x1p120f ? 0x1p120f : f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(s[y][t][i] - m_use);
          acc.l[y] += e;
          p[y][t >> 1][(t & 1) * 4 + i] = (_Float16)(e * f);
        }
    }
    // values
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const half8v vf = operand(vr[t][2 * u], vr[t][2 * u + 1]);
#pragma unroll
        for (int y = 0; y < QT; ++y)
          acc.o[y][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p[y][u], acc.o[y][t], 0, 0, 0);
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
#pragma unroll
    for (int o = 0; o < 3; ++o) {
      Partial<QT, DT> other;
      other.each([&](int i, float) { return joined[(o * NV + i) * 64 + lane]; });
      acc.add(other);
    }
  };
  join();

  if (a.nsplit > 1) {
    // Every share stores its part (system-coherent stores, visible to every
    // XCD once vmcnt drains) and arrives on the tile's counter; the last one
    // joins them.
    constexpr int kCoherent = 17;  // sc0 | sc1
    constexpr int PART = NV * 64 * 4;
    const __amdgpu_buffer_rsrc_t rP =
        make_rsrc(a.ws + kWsCounterBytes + (int64_t)item * a.nsplit * PART, (uint32_t)(a.nsplit * PART));
    if (w == 0) {
      acc.each([&](int i, float v) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rP, (uint32_t)(split * PART + (i * 64 + lane) * 4), 0,
                                              kCoherent);
        return v;
      });
      wait_vmcnt0();
      if (lane == 0) {
        unsigned long long* cnt = (unsigned long long*)a.ws + item;  // < kWsMaxTiles (the host's check)
        const unsigned long long before =
            __hip_atomic_fetch_add(cnt, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_split = before + 1 == (unsigned long long)a.nsplit;
        if (last_split) __hip_atomic_store(cnt, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    __syncthreads();
    if (!last_split) return;
    acc.clear();
    for (int sp = w; sp < a.nsplit; sp += 4) {  // (in this order whichever came last)
      Partial<QT, DT> other;
      other.each([&](int i, float) {
        return __uint_as_float(
            __builtin_amdgcn_raw_buffer_load_b32(rP, (uint32_t)(sp * PART + (i * 64 + lane) * 4), 0, kCoherent));
      });
      acc.add(other);
    }
    join();
  }
  if (w > 0) return;

  // O: lane holds row l % 16, dims 16 t + 4 (l / 16) + 0..3
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const int64_t row = (int64_t)row0 + x * 16 + lr;
    const float l = row_reduce(acc.l[x], [](float y, float z) { return y + z; });
    // no key seen: zeros
    const float f = l == 0.f || acc.mv[x] == -INFINITY ? (l == l ? 0.f : l)
                                                       : __builtin_amdgcn_exp2f(acc.mv[x] - acc.m[x]) / l;
    if (row >= nrows) continue;
    const int i = (int)(row / a.group), head = kvh * a.group + (int)(row - (int64_t)i * a.group);
    T* const o = (T*)a.o + (int64_t)(first + i) * a.ldo + (int64_t)head * a.ho;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const int d = t * 16 + lg * 4;
      if (!WHOLE && d >= a.d) continue;
      T o4[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o4[j] = (T)(acc.o[x][t][j] * f);
      int2v bits;
      __builtin_memcpy(&bits, o4, 8);
      *(int2u*)(o + d) = bits;
    }
  }
}

// Row tiles a workgroup takes (QT), their number and the shares of the keys:
// from sizes alone, so the workspace can be asked for beforehand.
struct KvPlan {
  int qt, nsplit;
  int64_t tiles;
};
KvPlan plan_of(const KvAttnProblem& p) {
  KvPlan r;
  const int64_t group = p.heads / p.kv_heads;
  const int64_t rows = (p.cu ? (p.tokens + p.requests - 1) / p.requests : 1) * group;  // of a request, on average
  r.qt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int64_t rt = 16 * r.qt;
  r.tiles = p.cu ? p.tokens * group / rt + p.requests : p.requests * ((group + rt - 1) / rt);
  // Shares until 512 workgroups (two a CU) are there, of at least one group
  // of 64 keys a wave.
  const int64_t items = r.tiles * p.kv_heads, most = (p.width * p.block + 255) / 256;
  int64_t n = items >= 512 ? 1 : (512 + items - 1) / items;
  n = n < most ? n : most;
  r.nsplit = (int)(n < 1 ? 1 : n < 128 ? n : 128);
  return r;
}

int64_t part_bytes(const KvAttnProblem& p, int qt) {
  const int64_t dt = p.d <= 64 ? 4 : 8;
  return qt * (dt * 4 + 3) * 64 * 4;
}

template <typename T, int DC, bool WHOLE>
hipError_t launch_qt(int qt, dim3 grid, const KArgs& a, hipStream_t stream) {
  const auto fn = qt == 1   ? kv_attention<T, DC, WHOLE, 1>
                  : qt == 2 ? kv_attention<T, DC, WHOLE, 2>
                            : kv_attention<T, DC, WHOLE, 4>;
  hipLaunchKernelGGL(fn, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_t(int64_t d, int qt, dim3 grid, const KArgs& a, hipStream_t stream) {
  if (d == 64) return launch_qt<T, 1, true>(qt, grid, a, stream);
  if (d == 128) return launch_qt<T, 2, true>(qt, grid, a, stream);
  return d < 64 ? launch_qt<T, 1, false>(qt, grid, a, stream) : launch_qt<T, 2, false>(qt, grid, a, stream);
}

}  // namespace

int64_t kv_attention_workspace_bytes(const KvAttnProblem& p) {
  const KvPlan k = plan_of(p);
  return k.nsplit > 1 ? kWsCounterBytes + k.tiles * p.kv_heads * k.nsplit * part_bytes(p, k.qt) : 0;
}

hipError_t launch_kv_attention(const KvAttnProblem& p, hipStream_t stream) {
  KvPlan k = plan_of(p);
  const int64_t items = k.tiles * p.kv_heads;
  if (k.nsplit > 1 && (!p.ws || p.ws_bytes < kv_attention_workspace_bytes(p) || items > kWsMaxTiles)) k.nsplit = 1;
  if (items * k.nsplit >= (1ll << 31)) return hipErrorInvalidValue;
  KArgs a{};
  a.q = (const char*)p.q;
  a.k = p.k_codes;
  a.v = p.v_codes;
  a.ks = p.k_scale;
  a.vs = p.v_scale;
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
  a.dp = (int)((p.d + 15) / 16 * 16);
  a.bytes = p.block * a.dp;
  a.requests = (int)p.requests;
  a.tokens = (int)p.tokens;
  a.kv_heads = (int)p.kv_heads;
  a.group = (int)(p.heads / p.kv_heads);
  a.d = (int)p.d;
  a.lb = __builtin_ctzll((unsigned long long)p.block) - 4;
  a.blocks = (int)p.blocks;
  a.width = (int)p.width;
  a.tiles = (int)k.tiles;
  a.nsplit = k.nsplit;
  a.c = p.scale * kLog2e;
  const dim3 grid((unsigned)(items * k.nsplit));
  return p.dtype == DT_BF16 ? launch_t<__bf16>(p.d, k.qt, grid, a, stream) : launch_t<_Float16>(p.d, k.qt, grid, a, stream);
}

}  // namespace hxmi
