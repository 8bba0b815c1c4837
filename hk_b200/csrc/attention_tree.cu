// Attention of drafted token trees over the paged cache.  A request has `context` rows in the cache and, behind them, one row for
// each of its `count` drafted tokens, in the order of the step's rows; the drafted token i sees every row of the context (or those
// inside its window) and the drafted rows whose bits are set in its row of `ancestors` (its ancestors and itself, for a tree).
//
//   out[t, h, :] = sum_j p_j v_j,   p = softmax over the visible j of cap(scale q[t, h] . k_j)   (+ a sink in the denominator)
//
// A row that sees nothing gives zeros.  All rows of a request and of a group's heads (row = token * group + head of the group) share
// the keys and values of their key head, so the floor is one read of those: 4 T H hd flops against 4 G hd bytes a key stays below
// what the tensor cores do in that time for T H / G up to about 250 rows.
//
// Work is cut on the device.  A unit is (request, tile of rows, key head) with its key tiles; all units' tiles, side by side, are
// dealt to the CTAs of one wave in equal contiguous shares.  So whatever the lengths are, every CTA reads as much as the others,
// and only a unit that a border falls into leaves partial results (at most two a CTA), which `tree_combine_kernel` merges in order.
// Nothing depends on the host but bounds on the sizes: a launch can be captured and replayed over other contexts.
//
// What the device arrays say is checked where it is read: a request whose slot, rows or lengths lie outside the arrays is skipped,
// and a page outside the pool is not read.
#include <cuda.h>
#include <math_constants.h>

#include <mutex>

#include "common.cuh"

namespace {

struct TreeReq {
  int slot, first, count, context;
};

struct TreeArgs {
  const void *q, *k, *v;
  void* out;
  const int* block_table;
  const TreeReq* requests;
  const uint32_t* ancestors;
  const int* positions;
  const float* sinks;      // one score per query head (natural units), or null: 0
  float *part_o, *part_ml;
  int* status;
  long long num_pages;
  int n, n_requests, most_tokens, words, table_rows, table_stride, page_tokens, H, G, hd, window, sink, rows_cap;
  float scale, softcap;    // scale on q . k; softcap c (0: none)
};

// A request as the kernels take it: with nothing to do (count 0) where its numbers lie outside the arrays.
__device__ __forceinline__ TreeReq load_request(const TreeArgs& a, int r) {
  const int4 x = __ldg(reinterpret_cast<const int4*>(a.requests) + r);
  TreeReq q = {x.x, x.y, x.z, x.w};
  const bool fits = q.slot >= 0 && q.slot < a.table_rows && q.first >= 0 && q.count > 0 && q.count <= a.most_tokens && q.count <= 32 * a.words &&
                    q.first <= a.n - q.count && q.context >= 0 &&
                    (long long)q.context + q.count <= (long long)a.table_stride * a.page_tokens;
  if (!fits) q.count = 0;
  return q;
}

// the first key that any row of a request may see: drafted tokens stand at positions from `context` on
__device__ __forceinline__ int first_key(const TreeArgs& a, const TreeReq& q) {
  return a.window > 0 ? max(0, q.context - a.window + 1) : 0;
}

// What one row (a drafted token) sees.
struct TreeRow {
  const uint32_t* bits;
  const int* places;       // positions of the request's drafted tokens (with a window)
  int context, count, lo, beyond;     // beyond: a key at a position up to here has left the window
};

__device__ __forceinline__ TreeRow tree_row(const TreeArgs& a, const TreeReq& q, int token, bool valid) {
  TreeRow w;
  const int t = q.first + (valid ? token : 0);
  w.bits = a.ancestors + (size_t)t * a.words;
  w.places = a.window > 0 ? a.positions + q.first : nullptr;
  w.context = valid ? q.context : 0;
  w.count = valid ? q.count : 0;
  w.beyond = a.window > 0 ? (int)max((long long)a.positions[t] - a.window, -1LL) : -1;
  w.lo = w.beyond + 1;
  return w;
}

// bit i: key j0 + i is visible
__device__ __forceinline__ uint32_t visible32(const TreeRow& w, int j0) {
  uint32_t see = 0;
  const int b = w.context - j0, a = w.lo - j0;
  if (b > 0 && a < 32) {
    see = b >= 32 ? 0xffffffffu : (1u << b) - 1u;
    if (a > 0) see &= 0xffffffffu << a;
  }
  const int t0 = j0 - w.context;           // place in the tree of key j0
  if (t0 > -32 && t0 < w.count) {
    auto word = [&](int i) -> uint32_t {
      if (i < 0 || 32 * i >= w.count) return 0u;
      const int n = w.count - 32 * i;
      return __ldg(w.bits + i) & (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
    };
    const int i = t0 >> 5;                 // rounds down
    uint32_t tree = __funnelshift_r(word(i), word(i + 1), (uint32_t)(t0 & 31));
    if (w.places) {
      for (uint32_t left = tree; left; left &= left - 1) {
        const int bit = __ffs(left) - 1;
        if (__ldg(w.places + t0 + bit) <= w.beyond) tree &= ~(1u << bit);
      }
    }
    see |= tree;
  }
  return see;
}

// cap c and scale as the tensor-core and float32 kernels use them, in the base-2 domain: c log2(e) tanh(s / c)
__device__ __forceinline__ float log2_score(float raw, float scale_log2, float cap_log2, float cap_in2) {
  if (cap_log2 > 0.f) {
    // C - 2 C / (e^(2z) + 1), z = score / c: saturates the right way at both ends, absolute error of the tanh about 2e-7
    float t, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(raw * cap_in2));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t + 1.0f));
    return fmaf(-2.0f * cap_log2, r, cap_log2);
  }
  return raw * scale_log2;
}

// ---- the shares of the CTAs ----------------------------------------------------------------------------------------------

// The units of a request: tiles of ROWS rows times key heads, each of `tiles` key tiles of KEYS from tile `t_first` on.
template <int ROWS, int KEYS>
__device__ __forceinline__ void unit_shape(const TreeArgs& a, const TreeReq& q, int& t_first, int& tiles, int& units) {
  t_first = first_key(a, q) / KEYS;
  tiles = q.count > 0 ? (q.context + q.count + KEYS - 1) / KEYS - t_first : 0;
  units = q.count > 0 ? (q.count * (a.H / a.G) + ROWS - 1) / ROWS * a.G : 0;
}

template <int ROWS, int KEYS>
__device__ __forceinline__ long long tiles_of(const TreeArgs& a, int r) {
  if (r >= a.n_requests) return 0;
  int t_first, tiles, units;
  unit_shape<ROWS, KEYS>(a, load_request(a, r), t_first, tiles, units);
  return (long long)tiles * units;
}

__device__ __forceinline__ long long warp_sum64(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// By a whole warp: the tiles of all requests, and of those before request `upto`.
template <int ROWS, int KEYS>
__device__ __forceinline__ void count_tiles(const TreeArgs& a, int upto, long long& before, long long& total) {
  const int lane = threadIdx.x & 31;
  long long b = 0, t = 0;
  for (int r = lane; r < a.n_requests; r += 32) {
    const long long n = tiles_of<ROWS, KEYS>(a, r);
    t += n;
    if (r < upto) b += n;
  }
  before = warp_sum64(b);
  total = warp_sum64(t);
}

// Where a CTA is in its share.
struct Walk {
  int r, unit, tile;
  long long left;
};

// By a whole warp: the start of share `cta` of `ctas`.
template <int ROWS, int KEYS>
__device__ __forceinline__ Walk share_start(const TreeArgs& a, int cta, int ctas) {
  const int lane = threadIdx.x & 31;
  long long none, total;
  count_tiles<ROWS, KEYS>(a, 0, none, total);
  const long long from = total * cta / ctas, to = total * (cta + 1) / ctas;
  Walk w = {a.n_requests, 0, 0, to - from};
  long long base = 0;
  if (to > from) {
    for (int r0 = 0; r0 < a.n_requests; r0 += 32) {
      const long long n = tiles_of<ROWS, KEYS>(a, r0 + lane);
      long long sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const unsigned here = __ballot_sync(0xffffffffu, base + sum > from);
      if (here) {
        const int src = __ffs(here) - 1;
        const long long start = base + __shfl_sync(0xffffffffu, sum - n, src);
        w.r = r0 + src;
        int t_first, tiles, units;
        unit_shape<ROWS, KEYS>(a, load_request(a, w.r), t_first, tiles, units);
        w.unit = (int)((from - start) / tiles);
        w.tile = (int)((from - start) % tiles);
        break;
      }
      base += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  return w;
}

// A unit, or the part of one that falls into a share.
struct Segment {
  TreeReq q;
  int g, row0, rows;       // key head; first row of the tile in the request, rows of the tile
  int t0, n;               // first key tile, key tiles
  bool whole, begins;      // all of the unit's tiles; its first among them
};

template <int ROWS, int KEYS>
__device__ __forceinline__ bool next_segment(const TreeArgs& a, Walk& w, Segment& s) {
  if (w.left <= 0) return false;
  int t_first, tiles, units;
  for (;; ++w.r, w.unit = 0, w.tile = 0) {
    if (w.r >= a.n_requests) return false;
    s.q = load_request(a, w.r);
    unit_shape<ROWS, KEYS>(a, s.q, t_first, tiles, units);
    if (w.unit < units) break;
  }
  s.g = w.unit % a.G;
  s.row0 = w.unit / a.G * ROWS;
  s.rows = min(ROWS, s.q.count * (a.H / a.G) - s.row0);
  s.t0 = t_first + w.tile;
  s.n = (int)min((long long)(tiles - w.tile), w.left);
  s.whole = s.n == tiles;
  s.begins = w.tile == 0;
  w.left -= s.n;
  w.tile += s.n;
  if (w.tile == tiles) {
    w.tile = 0;
    ++w.unit;
  }
  return true;
}

// Where a segment's partial result goes: a share's first segment may begin inside a unit (2 cta), its last may end inside the unit
// that it began (2 cta + 1).
__device__ __forceinline__ size_t part_slot(int cta, bool begins) { return 2 * (size_t)cta + (begins ? 1 : 0); }

// A warp a row (token, query head): the partial results of the shares that its unit is cut into, in order.
constexpr int CW = 4;      // warps
template <typename T, int ROWS, int KEYS>
__global__ void __launch_bounds__(CW * 32) tree_combine_kernel(const TreeArgs a, int ctas) {
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.y, group = a.H / a.G;
  const TreeReq q = load_request(a, r);
  if (q.count == 0) return;
  long long before, total;
  count_tiles<ROWS, KEYS>(a, r, before, total);
  int t_first, tiles, units;
  unit_shape<ROWS, KEYS>(a, q, t_first, tiles, units);
  for (int i = blockIdx.x * CW + warp; i < q.count * a.H; i += gridDim.x * CW) {
    const int token = i / a.H, head = i % a.H, g = head / group, row = token * group + head % group;
    const long long start = before + (long long)(row / ROWS * a.G + g) * tiles;
    const int c0 = (int)(((start + 1) * ctas - 1) / total), c1 = (int)(((start + tiles) * ctas - 1) / total);
    if (c0 == c1) continue;                              // whole in one share: written there
    float m = -CUDART_INF_F, l = 0.f, acc[8];            // up to 256 dims
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    for (int c = c0; c <= c1; ++c) {
      const size_t at = part_slot(c, c == c0) * a.rows_cap + row % ROWS;
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + at);
      const float mn = fmaxf(m, ml.x), safe = mn == -CUDART_INF_F ? 0.f : mn;
      const float f0 = exp2f(m - safe), f1 = exp2f(ml.x - safe);
      l = l * f0 + ml.y * f1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = lane + 32 * e;
        if (d < a.hd) acc[e] = acc[e] * f0 + __ldcg(a.part_o + at * a.hd + d) * f1;
      }
      m = mn;
    }
    if (a.sink) l += exp2f((a.sinks ? a.sinks[head] * 1.4426950408889634f : 0.f) - m);
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    T* out = reinterpret_cast<T*>(a.out) + ((size_t)(q.first + token) * a.H + head) * a.hd;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = lane + 32 * e;
      if (d < a.hd) out[d] = from_f32<T>(acc[e] * inv);
    }
  }
}

template <typename T, int ROWS, int KEYS>
int launch_combine(const TreeArgs& a, int ctas, cudaStream_t s) {
  const long long rows = (long long)a.most_tokens * a.H;
  const long long blocks = (rows + CW - 1) / CW;
  return hk_launch_pdl(tree_combine_kernel<T, ROWS, KEYS>, dim3((unsigned)(blocks < 4096 ? blocks : 4096), (unsigned)a.n_requests), dim3(CW * 32), 0, s,
                       a, ctas);
}

// ---- any size: a block a (token, query head) -------------------------------------------------------------------------------
// Four warps take the keys in turn with a running maximum and sum each; the four are merged in order.  For head sizes and pages
// that the kernels below do not take.
constexpr int GW = 4;
template <typename T>
__global__ void __launch_bounds__(GW * 32) tree_generic_kernel(const TreeArgs a) {
  __shared__ float acc_s[GW][256], m_s[GW], l_s[GW];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.x % a.H, token = blockIdx.x / a.H % a.most_tokens, r = blockIdx.x / a.H / a.most_tokens;
  const TreeReq q = load_request(a, r);
  if (token >= q.count) return;
  const TreeRow w = tree_row(a, q, token, true);
  const int g = head / (a.H / a.G), hd = a.hd;
  const int* bt = a.block_table + (size_t)q.slot * a.table_stride;
  const T* qp = reinterpret_cast<const T*>(a.q) + ((size_t)(q.first + token) * a.H + head) * hd;
  float qr[8], acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    qr[i] = d < hd ? to_f32<T>(qp[d]) : 0.f;
    acc[i] = 0.f;
  }
  float m = -CUDART_INF_F, l = 0.f;
  const int end = q.context + q.count;
  for (int j0 = first_key(a, q) / 32 * 32 + 32 * warp; j0 < end; j0 += 32 * GW) {
    for (uint32_t see = visible32(w, j0); see; see &= see - 1) {
      const int j = j0 + __ffs(see) - 1;
      const int page = bt[j / a.page_tokens];
      if (page < 0 || page >= a.num_pages) continue;
      const size_t at = (((size_t)page * a.G + g) * a.page_tokens + j % a.page_tokens) * hd;
      const T *kp = reinterpret_cast<const T*>(a.k) + at, *vp = reinterpret_cast<const T*>(a.v) + at;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < hd) s = fmaf(qr[i], to_f32<T>(kp[d]), s);
      }
      s = warp_sum(s) * a.scale;
      if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
      const float mn = fmaxf(m, s), safe = mn == -CUDART_INF_F ? 0.f : mn;
      const float corr = expf(m - safe), p = expf(s - safe);
      l = l * corr + p;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < hd) acc[i] = fmaf(p, to_f32<T>(vp[d]), acc[i] * corr);
      }
      m = mn;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) acc_s[warp][lane + 32 * i] = acc[i];
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
  __syncthreads();
  const float sink_score = a.sink && a.sinks ? a.sinks[head] : 0.f;
  float top = a.sink ? sink_score : -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < GW; ++i) top = fmaxf(top, m_s[i]);
  const float safe = top == -CUDART_INF_F ? 0.f : top;
  float f[GW], total = a.sink ? expf(sink_score - safe) : 0.f;
#pragma unroll
  for (int i = 0; i < GW; ++i) {
    f[i] = expf(m_s[i] - safe);
    total += l_s[i] * f[i];
  }
  const float inv = total > 0.f || total != total ? 1.0f / total : 0.f;
  T* out = reinterpret_cast<T*>(a.out) + ((size_t)(q.first + token) * a.H + head) * hd;
  for (int d = threadIdx.x; d < hd; d += GW * 32) {
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < GW; ++i) y = fmaf(acc_s[i][d], f[i], y);
    out[d] = from_f32<T>(y * inv);
  }
}

template <typename T>
int launch_generic(const TreeArgs& a, cudaStream_t s) {
  const long long blocks = (long long)a.n_requests * a.most_tokens * a.H;
  if (blocks > 0x7fffffffLL) return HK_ERR_UNSUPPORTED;
  return hk_launch(tree_generic_kernel<T>, dim3((unsigned)blocks), dim3(GW * 32), 0, s, a);
}

}  // namespace

// q, out [n, H, hd]; k, v [num_pages, G, page_tokens, hd]; block_table int32 [table_rows, table_stride]; requests int32
// [n_requests, 4] = (slot, first row of q, drafted tokens, rows in the cache before them); ancestors [n, words] 32-bit words: bit j
// of a token's row: it sees the drafted token j of its request; positions int32 [n] (read with a window only): drafted tokens stand
// at their request's `context` or behind it.  Only rows of q that belong to a request are computed.  scale on q . k, softcap c (0:
// none), window w (0: none): a key at position x is seen from position p if x > p - w; sink, sinks: one more term of the
// denominator.  most_tokens, n_requests: bounds of the grid.  `kernel` 0: any size up to heads of 256.
HK_API int hk_tree_attention(const void* q, const void* k, const void* v, void* out, int dtype, const int* block_table, int table_rows,
                             int table_stride, const int* requests, int n_requests, int most_tokens, const void* ancestors, int words,
                             const int* positions, int n, long long num_pages, int page_tokens, int H, int G, int hd, int window,
                             float scale, float softcap, int sink, const float* sinks, int kernel, int ctas, float* part_o,
                             float* part_ml, int rows_cap, int* status, void* stream) {
  if (n <= 0 || n_requests <= 0 || most_tokens <= 0) return 0;
  if (H < 1 || G < 1 || H % G != 0 || hd < 1 || hd > 256 || page_tokens < 1 || table_rows < 1 || table_stride < 1 || words < 1 ||
      n_requests > 65535 || num_pages < 1 || softcap < 0.f || !(scale > 0.f) || (dtype != HK_F32 && dtype != HK_BF16) ||
      (((uintptr_t)requests) & 15) != 0)
    return HK_ERR_UNSUPPORTED;
  TreeArgs a;
  a.q = q; a.k = k; a.v = v; a.out = out;
  a.block_table = block_table;
  a.requests = reinterpret_cast<const TreeReq*>(requests);
  a.ancestors = static_cast<const uint32_t*>(ancestors);
  a.positions = positions;
  a.sinks = sink ? sinks : nullptr;
  a.part_o = part_o; a.part_ml = part_ml; a.status = status;
  a.num_pages = num_pages;
  a.n = n; a.n_requests = n_requests; a.most_tokens = most_tokens; a.words = words;
  a.table_rows = table_rows; a.table_stride = table_stride; a.page_tokens = page_tokens;
  a.H = H; a.G = G; a.hd = hd; a.window = window > 0 ? window : 0; a.sink = sink; a.rows_cap = rows_cap;
  a.scale = scale; a.softcap = softcap;
  cudaStream_t s = (cudaStream_t)stream;
  if (kernel == 0) return dtype == HK_F32 ? launch_generic<float>(a, s) : launch_generic<bf16>(a, s);
  return HK_ERR_UNSUPPORTED;
}
