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
// dealt to the CTAs of one wave in equal contiguous shares (a unit counts LEAD tiles more: what starting one costs).  So whatever the
// lengths are, every CTA works as long as the others, and only a unit that a border falls into leaves partial results (at most two a
// CTA), which `tree_combine_kernel` merges in order.
// Nothing depends on the host but bounds on the sizes: a launch can be captured and replayed over other contexts.
//
// Measured (32 heads over 8 key heads of 128, captured and replayed): 16 tokens behind 2,000 rows 16.6 us, all of it the start and end of
// the two kernels (8.5 MB); 8 requests of 32 tokens, ragged up to 8,000 rows, 41 us (122 MB, 3.0 TB/s); 32 requests of 64 tokens behind up to
// 8,192 rows 184 us (680 MB, 3.7 TB/s, 625 TFLOP/s); 64 tokens behind 131,001 rows 144 us (954 TFLOP/s); the last two at the power cap,
// called again and again for a second, 209 to 217 and 164 to 172.  The generic kernel took 391, 4,463, 47,593 and 76,055.
//
// What the device arrays say is checked where it is read: a request whose slot, rows or lengths lie outside the arrays or the bounds is
// skipped, and the keys of a page that is not in the pool are not seen.
#include <cuda.h>
#include <math_constants.h>

#include <mutex>

#include "common.cuh"

namespace {

struct TreeReq {
  int slot, first, count, context;
};

}  // namespace

// What a call says, in one piece: the host's language takes longer to hand over thirty numbers than to pack them.
struct TreeCall {
  const void *q, *k, *v;
  void* out;
  const int *block_table, *requests;
  const void* ancestors;
  const int* positions;
  const float* sinks;
  long long num_pages;
  int dtype, table_rows, table_stride, n_requests, most_tokens, most_keys, words, n, page_tokens, H, G, hd, window, sink;
  float scale, softcap;
};
static_assert(sizeof(TreeCall) == 10 * 8 + 16 * 4, "packed without gaps");

namespace {

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
  int n, n_requests, most_tokens, most_keys, words, table_rows, table_stride, page_tokens, H, G, hd, window, sink, rows_cap, group;
  uint32_t group_inverse;  // 2^32 / group, rounded up (a group of 1: 0)
  float scale, softcap;    // scale on q . k; softcap c (0: none)
};

// Row `i` of a request (token * group + head of the group, at most 256 tokens): its token.  A division by a variable takes a hundred and
// more clocks, of which the start of a short kernel has none to spare.  Exact while
// i * group < 2^32: groups of up to 4,095 heads.
__device__ __forceinline__ int token_of(const TreeArgs& a, int i) { return a.group == 1 ? i : (int)__umulhi((uint32_t)i, a.group_inverse); }

// A request as the kernels take it: with nothing to do (count 0) where its numbers lie outside the arrays.
__device__ __forceinline__ TreeReq load_request(const TreeArgs& a, int r) {
  const int4 x = __ldg(reinterpret_cast<const int4*>(a.requests) + r);
  TreeReq q = {x.x, x.y, x.z, x.w};
  const bool fits = q.slot >= 0 && q.slot < a.table_rows && q.first >= 0 && q.count > 0 && q.count <= a.most_tokens && q.count <= 32 * a.words &&
                    q.first <= a.n - q.count && q.context >= 0 &&
                    q.context <= a.most_keys - q.count;
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

// cap c and scale as the tensor-core kernel uses them, in the base-2 domain: c log2(e) tanh(s / c)
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

// How a kernel cuts: rows and keys of a tile, and what starting a unit costs in tiles.  All counts fit 32 bits (the launch sees to it).
template <int R, int K, int L>
struct Cut {
  static constexpr int ROWS = R, KEYS = K, LEAD = L;
};

// The units of a request: tiles of ROWS rows times key heads, each of `tiles` key tiles from tile `t_first` on.
template <typename C>
__device__ __forceinline__ void unit_shape(const TreeArgs& a, const TreeReq& q, int& t_first, int& tiles, int& units) {
  t_first = first_key(a, q) / C::KEYS;
  tiles = q.count > 0 ? (q.context + q.count + C::KEYS - 1) / C::KEYS - t_first : 0;
  units = q.count > 0 ? (q.count * a.group + C::ROWS - 1) / C::ROWS * a.G : 0;
}

template <typename C>
__device__ __forceinline__ uint32_t size_of(const TreeArgs& a, const TreeReq& q) {
  int t_first, tiles, units;
  unit_shape<C>(a, q, t_first, tiles, units);
  return (uint32_t)(tiles + C::LEAD) * units;
}
__device__ __forceinline__ TreeReq request_or_none(const TreeArgs& a, int r) { return r < a.n_requests ? load_request(a, r) : TreeReq{0, 0, 0, 0}; }

__device__ __forceinline__ uint32_t warp_sum32(uint32_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Where a CTA is in its share: a request (`q`, as it was loaded), a unit of it and the place in that, LEAD before its first tile.
struct Walk {
  int r, unit, place, left;
  TreeReq q;
};
struct Share {
  Walk w;
  uint32_t from, total, each, wide;   // the share's first place among all; all of them: `wide` shares of each + 1, then shares of `each`
};
__device__ __forceinline__ uint32_t share_from(const Share& s, uint32_t share) { return s.each * share + min(share, s.wide); }
__device__ __forceinline__ int share_of(const Share& s, uint32_t place) {
  const uint32_t edge = s.wide * (s.each + 1);
  return (int)(place < edge ? place / (s.each + 1) : s.wide + (place - edge) / s.each);
}

// By a whole warp: the start of share `cta` of `ctas`.
template <typename C>
__device__ __forceinline__ Share share_start(const TreeArgs& a, uint32_t cta, uint32_t ctas) {
  const int lane = threadIdx.x & 31;
  Share share = {{a.n_requests, 0, 0, 0, {0, 0, 0, 0}}, 0, 0, 0, 0};
  TreeReq q = request_or_none(a, lane);
  uint32_t total = size_of<C>(a, q);
#pragma unroll 1
  for (int r = lane + 32; r < a.n_requests; r += 32) total += size_of<C>(a, load_request(a, r));
  share.total = total = warp_sum32(total);
  ctas = min(ctas, total);                       // no empty share between two of one unit
  if (cta >= ctas) return share;
  share.each = total / ctas;
  share.wide = total - share.each * ctas;
  share.from = share_from(share, cta);
  share.w.left = (int)(share.each + (cta < share.wide ? 1 : 0));
  uint32_t base = 0;
#pragma unroll 1
  for (int r0 = 0; r0 < a.n_requests; r0 += 32) {
    if (r0 > 0) q = request_or_none(a, r0 + lane);
    const uint32_t n = size_of<C>(a, q);
    uint32_t sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const unsigned here = __ballot_sync(0xffffffffu, base + sum > share.from);
    if (here) {
      const int src = __ffs(here) - 1;
      const uint32_t in = share.from - base - __shfl_sync(0xffffffffu, sum - n, src);
      share.w.r = r0 + src;
      share.w.q = {__shfl_sync(0xffffffffu, q.slot, src), __shfl_sync(0xffffffffu, q.first, src), __shfl_sync(0xffffffffu, q.count, src),
                   __shfl_sync(0xffffffffu, q.context, src)};
      int t_first, tiles, units;
      unit_shape<C>(a, share.w.q, t_first, tiles, units);
      share.w.unit = (int)(in < (uint32_t)(tiles + C::LEAD) ? 0 : in / (uint32_t)(tiles + C::LEAD));
      share.w.place = (int)in - share.w.unit * (tiles + C::LEAD);
      break;
    }
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  return share;
}

// A unit, or the part of one that falls into a share.
struct Segment {
  TreeReq q;
  int g, row0, rows;       // key head; first row of the tile in the request, rows of the tile
  int t0, n;               // first key tile, key tiles
  bool whole, begins;      // all of the unit's tiles; its first among them
};

template <typename C>
__device__ __forceinline__ bool next_segment(const TreeArgs& a, Walk& w, Segment& s) {
  int t_first, tiles, units;
#pragma unroll 1
  while (w.left > 0 && w.r < a.n_requests) {
    unit_shape<C>(a, w.q, t_first, tiles, units);
    if (w.unit >= units) {
      w.q = request_or_none(a, ++w.r);
      w.unit = w.place = 0;
      continue;
    }
    s.q = w.q;
    const int at = w.unit < a.G ? 0 : w.unit / a.G, begin = max(w.place - C::LEAD, 0), take = min(tiles + C::LEAD - w.place, w.left);
    s.g = w.unit - at * a.G;
    s.row0 = at * C::ROWS;
    s.rows = min(C::ROWS, s.q.count * a.group - s.row0);
    s.t0 = t_first + begin;
    s.n = w.place + take - C::LEAD - begin;
    s.whole = s.n == tiles;
    s.begins = begin == 0;
    w.left -= take;
    w.place += take;
    if (w.place == tiles + C::LEAD) {
      w.place = 0;
      ++w.unit;
    }
    if (s.n > 0) return true;
  }
  return false;
}

// Where a segment's partial result goes: a share's first segment may begin inside a unit (2 cta), its last may end inside the unit
// that it began (2 cta + 1).
__device__ __forceinline__ size_t part_slot(int cta, bool begins) { return 2 * (size_t)cta + (begins ? 1 : 0); }

// The exponentials' domain: base 2 for bfloat16, natural in float32 (a score times log2(e) would be rounded once more).
template <typename T>
__device__ __forceinline__ float power(float x) {
  return sizeof(T) == 4 ? expf(x) : exp2f(x);
}

// Partial sums lie [slot][dim / 4][row][4]: neighbouring rows, which neighbouring threads hold, side by side.
__device__ __forceinline__ float* part_place(const TreeArgs& a, size_t slot, int row, int dim, int hd) {
  return a.part_o + ((slot * (hd / 4) + dim / 4) * a.rows_cap + row) * 4;
}

// The partial results of a unit that lies in several shares, merged in order.  A block takes the border between two shares, if it is
// the first inside its unit, 32 of the unit's rows and 32 dims: a thread a row and eight dims.  It starts beside the kernel that leaves
// the parts (which lets it only behind its own wait, so what that one reads is there) and waits with its unit found.
constexpr int CW = 4;
template <typename T, int HD, typename C>
__global__ void __launch_bounds__(CW * 32) tree_combine_kernel(const TreeArgs a, int ctas) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x + 1;
  const Share share = share_start<C>(a, c, ctas);
  const Walk w = share.w;
  const uint32_t first = share.from - w.place + C::LEAD;                // the place of the unit's first tile
  const int row = blockIdx.y * 32 + lane, dim = blockIdx.z * 32 + warp * 8;
  int t_first = 0, tiles = 0, units = 0, row0 = 0, rows = 0, g = 0;
  TreeReq q = {0, 0, 0, 0};
  if (w.left > 0 && w.place > C::LEAD && share_from(share, c - 1) <= first) {
    q = w.q;
    unit_shape<C>(a, q, t_first, tiles, units);
    const int at = w.unit < a.G ? 0 : w.unit / a.G;
    g = w.unit - at * a.G;
    row0 = at * C::ROWS;
    rows = min(C::ROWS, q.count * a.group - row0);
  }
  // (the first block waits in any case: this kernel must not be through before the one that it waits for)
  if (row >= rows && blockIdx.x + blockIdx.y + blockIdx.z > 0) return;
  const int parts = rows > 0 ? share_of(share, first + tiles - 1) - c + 2 : 0;        // shares c - 1, c, ...
  const int token = token_of(a, row0 + row), head = g * a.group + row0 + row - token * a.group;
  pdl_wait();
  if (row >= rows) return;
  // parts on their way at once: in float32 there are more (1,500 rows: 24.5 us with 12, 26.7 with 8); in bfloat16 there are more rows, and
  // blocks of more registers leave some waiting (8 ragged requests: 40.9 us with 8, 43.4 with 12)
  constexpr int DEEP = sizeof(T) == 4 ? 12 : 8;
  float m = -CUDART_INF_F, l = 0.f, acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  // slot 2 (c - 1) + 1, then every second one from 2 c on
  const float2* ml_at = reinterpret_cast<const float2*>(a.part_ml) + part_slot(c - 1, true) * a.rows_cap + row;
  const float* o_at = part_place(a, part_slot(c - 1, true), row, dim, HD);
  const int ml_step = 2 * a.rows_cap, o_step = 2 * HD * a.rows_cap, o_next = 4 * a.rows_cap;
  for (int p0 = 0; p0 < parts; p0 += DEEP) {
    float2 ml[DEEP];
    float4 u[DEEP], v[DEEP];
#pragma unroll
    for (int i = 0; i < DEEP; ++i) {
      ml[i] = make_float2(-CUDART_INF_F, 0.f);
      u[i] = v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p0 + i < parts) {
        ml[i] = __ldcg(ml_at);
        u[i] = __ldcg(reinterpret_cast<const float4*>(o_at));
        v[i] = __ldcg(reinterpret_cast<const float4*>(o_at + o_next));
      }
      ml_at += p0 + i == 0 ? a.rows_cap : ml_step;
      o_at += p0 + i == 0 ? HD * a.rows_cap : o_step;
    }
    float mn = m;
#pragma unroll
    for (int i = 0; i < DEEP; ++i) mn = fmaxf(mn, ml[i].x);
    const float safe = mn == -CUDART_INF_F ? 0.f : mn, old = power<T>(m - safe);
    l *= old;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= old;
    m = mn;
#pragma unroll
    for (int i = 0; i < DEEP; ++i) {
      const float f = power<T>(ml[i].x - safe);      // a part that there is not: 0
      l = fmaf(ml[i].y, f, l);
      acc[0] = fmaf(u[i].x, f, acc[0]), acc[1] = fmaf(u[i].y, f, acc[1]), acc[2] = fmaf(u[i].z, f, acc[2]), acc[3] = fmaf(u[i].w, f, acc[3]);
      acc[4] = fmaf(v[i].x, f, acc[4]), acc[5] = fmaf(v[i].y, f, acc[5]), acc[6] = fmaf(v[i].z, f, acc[6]), acc[7] = fmaf(v[i].w, f, acc[7]);
    }
  }
  float factor = 1.0f;
  if (a.sink) {
    const float score = (a.sinks ? a.sinks[head] : 0.f) * (sizeof(T) == 4 ? 1.0f : 1.4426950408889634f), top = fmaxf(m, score);
    factor = m == -CUDART_INF_F ? 0.f : power<T>(m - top);
    l = l * factor + power<T>(score - top);
  }
  const float inv = l > 0.f || l != l ? factor / l : 0.f;
  T* out = reinterpret_cast<T*>(a.out) + ((size_t)(q.first + token) * a.H + head) * HD + dim;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(out) = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<float4*>(out + 4) = make_float4(acc[4] * inv, acc[5] * inv, acc[6] * inv, acc[7] * inv);
  } else {
    uint32_t pk[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __nv_bfloat162 y = __floats2bfloat162_rn(acc[2 * e] * inv, acc[2 * e + 1] * inv);
      pk[e] = *reinterpret_cast<const uint32_t*>(&y);
    }
    *reinterpret_cast<uint4*>(out) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
  }
}

// Whether all places fit 32 bits.
template <typename C>
bool cut_fits(const TreeArgs& a) {
  const unsigned long long units = ((unsigned long long)a.most_tokens * a.group + C::ROWS - 1) / C::ROWS * a.G;
  return units * a.n_requests < (1ull << 31) / ((unsigned long long)a.most_keys / C::KEYS + 2 + C::LEAD);
}

template <typename T, int HD, typename C>
int launch_combine(const TreeArgs& a, int ctas, cudaStream_t s) {
  if (ctas < 2) return 0;
  return hk_launch_pdl(tree_combine_kernel<T, HD, C>, dim3((unsigned)(ctas - 1), (unsigned)((a.rows_cap + 31) / 32), HD / 32), dim3(CW * 32), 0, s,
                       a, ctas);
}

// ---- any size: a block a (token, query head) -------------------------------------------------------------------------------
// Four warps take the keys in turn with a running maximum and sum each; the four are merged in order.  For head sizes and pages
// that the kernels below do not take.  Bound by reading every key and value once a query head and token instead of once a tile of them.
constexpr int GW = 4;
template <typename T>
__global__ void __launch_bounds__(GW * 32) tree_generic_kernel(const TreeArgs a) {
  __shared__ float acc_s[GW][256], m_s[GW], l_s[GW];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.x % a.H, token = blockIdx.x / a.H % a.most_tokens, r = blockIdx.x / a.H / a.most_tokens;
  const TreeReq q = load_request(a, r);
  if (token >= q.count) return;
  const TreeRow w = tree_row(a, q, token, true);
  const int g = head / a.group, hd = a.hd;
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

// ---- bfloat16 on the tensor cores ---------------------------------------------------------------------------------------------
// A tile has up to 256 rows.  Two groups of eight softmax warps, a lane for each that issues its products and two warps that
// load K and V by TMA work on it side by side: with more than 128 rows each group has half of them and every key tile serves both; with up to 128 rows
// both groups have the same rows and take the key tiles in turn, and their sums meet in tensor memory at the end.  A group's first four
// warps take the first 64 keys of a tile, a thread a row, and the others the last 64: so there are four streams of scores -> probabilities
// -> product with V, and while the tensor core works for one the exponentials of the others run.  Tensor memory (512 columns): per stream
// 64 columns of scores, which the probabilities overwrite (bfloat16, 32 columns), per group HD of sums.  A stream's next scores are issued
// behind its product with V; products of one thread run in order, so they overwrite P only once it was read.  (One lane for both groups was
// what the kernel waited for: a product takes it some 40 clocks to issue, and a tile of 256 rows is 48 of them.)
//
// With two row tiles the two lanes issue a stream's product with V and its next scores in turns.  Side by side, both groups' products end
// at the same time, then their exponentials run at the same time, and each unit waits for the other (151 us for 143 below); in turns the
// four streams keep a quarter apart.  With one row tile (every lane's next keys come when they come) that waits for more than it saves.
//
// Bound by a stream's own way around, some 3,500 clocks a tile: 170 until the first scores are in registers, 1,200 of exponentials (512
// alone), 300 until the tensor core's lane has seen them and has its turn, 900 for the products and their announcement, of which shared
// memory's bandwidth takes 640 (a product of 64 keys reads 128 rows of Q: 6 KB in 32 clocks' work).  The exponentials' unit is active 58 %
// of that, shared memory 73 %.
// Probabilities are rounded to bfloat16 for the product with V, as the tensor core takes both operands in one type; their sum is of the
// unrounded ones.  That is an error of up to 2^-8 of each term beside the 2^-8 of the result's own rounding: 0.0024 of the result's norm
// against 0.0017 of a result that is rounded once (rows of independent values: each rounding is 0.0017).  Two products, with the rounding's
// remainder in the second, would take it away for half as many products again.
//
// Dropped (64 tokens behind 131,001 rows, 144 us): scores of 128 keys at once, two streams, 153; an eighth, a quarter and a third of the
// exponentials by a polynomial 145, 146 and 147; the turn passed on behind the product with V 145; tiles asked into L2 ahead 148.
constexpr int TC_ROWS = 128, TC_KEYS = 128, TC_SOFTMAX = 512, TC_THREADS = TC_SOFTMAX + 128;
typedef Cut<2 * TC_ROWS, TC_KEYS, 4> TcCut;
constexpr float MUCH = 16777216.0f, TOO_MUCH = 1152921504606846976.0f;      // 2^24, 2^60
constexpr long long WAIT_CLOCKS = 1ll << 25;   // some 17 ms, far beyond any legitimate wait

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"      // sleeps until the phase comes, or some 100 us
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(100000u) : "memory");
  return ok != 0;
}
// Waits for the phase of this parity, a bounded time; false (and the flag set) if it did not come or another gave up.  (Without sleeps
// between the tries: the tensor core's answers come in less than one.)  Behind the flag lies the pulse of the warps that take lost rows
// again, which takes as long as it takes: while it beats, time does not run.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  long long start = clock64();
  int beat = abort_flag[1];
  while (!*abort_flag && clock64() - start < WAIT_CLOCKS) {
    if (mbar_try_wait(bar, parity)) return true;
    const int now = abort_flag[1];
    if (now != beat) {
      beat = now;
      start = clock64();
    }
  }
  *abort_flag = 1;
  return false;
}
// The same for what is still on its way when the kernel gives up.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
  const long long start = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - start < WAIT_CLOCKS) {
  }
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory matrix descriptors, 128-byte swizzle, version 1 (sm_100); 8-row groups lie 1024 bytes apart.
// K-major ([row][64 elements = 128 bytes]): leading offset unused.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// MN-major ([k row][64 elements of the MN dimension]): the next 64 MN elements `lbo` bytes further (leading).
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
// The same with the A operand in tensor memory (128 lanes = rows, 8 columns of two bf16 each per 16 k).
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// x0, x1 times a plus b, and x0, x1 plus y0, y1: two float32 numbers an instruction, rounded as one by one
__device__ __forceinline__ void fma_two(float& x0, float& x1, float a, float b) {
  asm("{\n\t.reg .b64 x, f, s;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 f, {%2, %2};\n\tmov.b64 s, {%3, %3};\n\tfma.rn.f32x2 x, x, f, s;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}" : "+f"(x0), "+f"(x1) : "f"(a), "f"(b));
}
__device__ __forceinline__ void add_two(float& x0, float& x1, float y0, float y1) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x0), "+f"(x1) : "f"(y0), "f"(y1));
}
__device__ __forceinline__ float ex2(float x) {      // 2^x, one instruction; 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// Barrier 1 among the softmax threads; whether any of them says so.
__device__ __forceinline__ bool softmax_any(bool said) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 512, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any) : "r"(said ? 1u : 0u) : "memory");
  return any != 0;
}
// byte offset of (row r, 16-byte chunk c along the row) in a [halves][128 rows][128 bytes] swizzled tile
__device__ __forceinline__ uint32_t swz(int r, int c) { return (uint32_t)((c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

template <int HD>
struct TcSmem {
  static constexpr int STAGES = HD == 64 ? 4 : 2;      // of K, and of V
  alignas(1024) uint8_t q[2][TC_ROWS * HD * 2];
  alignas(1024) uint8_t k[STAGES][TC_KEYS * HD * 2];
  alignas(1024) uint8_t v[STAGES][TC_KEYS * HD * 2];
  alignas(8) uint64_t q_full, k_full[STAGES], v_full[STAGES], k_empty[STAGES], v_empty[STAGES], s_full[2][2], p_full[2][2], o_done[2], drained[2], pair[2][4], turn[2];
  float first[2][2][2][TC_ROWS], asked[8][2][2][TC_ROWS];   // [tile % 2][group][half of the keys][row]: a first tile's largest score;
                                                            // [tile % 8]..: the reference asked for
  float2 ml[2][2][TC_ROWS];   // the reference and the sum
  Walk start;                 // the share behind its first segment
  Segment lead;               // its first segment, if it has any
  int led;
  Segment segment[3];         // the softmax warps' segments: the last one (until its results are out), the one in hand, the next one
  int any[3];
  uint32_t tmem_base;
  int abort_flag, pulse;      // (side by side: mbar_wait)
  int gone;                   // a page of the share is not in the pool
};

// One row once more, by one warp in 32 bits over the keys of a segment that it sees.  For a row whose sums came out NaN or Inf: the
// tensor core's product takes whole tiles of values, and a probability of zero does not keep out a NaN or Inf among those that the row
// does not see; or one tile's scores ran too far ahead of the reference; or a page of the share is not in the pool.
struct RowKeys {
  const bf16* q;
  const int* bt;
  TreeRow w;
  volatile int* pulse;
  float scale_log2;
  int j, end;
};
__device__ __forceinline__ RowKeys row_keys(const TreeArgs& a, const Segment& s, int row, volatile int* pulse) {
  const int token = token_of(a, s.row0 + row), head = s.g * a.group + s.row0 + row - token * a.group;
  RowKeys k;
  k.pulse = pulse;
  k.w = tree_row(a, s.q, token, true);
  k.q = reinterpret_cast<const bf16*>(a.q) + ((size_t)(s.q.first + token) * a.H + head) * a.hd;
  k.bt = a.block_table + (size_t)s.q.slot * a.table_stride;
  k.scale_log2 = a.scale * 1.4426950408889634f;
  k.j = s.t0 * TC_KEYS;
  k.end = min((s.t0 + s.n) * TC_KEYS, s.q.context + s.q.count);
  return k;
}
// This lane's key of the next 32: its score and the place of its row in the pages, or -1 where the row does not see it.
__device__ __forceinline__ long long next_key(const TreeArgs& a, const Segment& s, RowKeys& k, float cap_log2, float cap_in2, float& score) {
  const uint32_t see = visible32(k.w, k.j);
  const int j = k.j + (int)(threadIdx.x & 31);
  k.j += 32;
  if ((threadIdx.x & 31) == 0) *k.pulse = (int)clock64();
  if (!((see >> (threadIdx.x & 31)) & 1u)) return -1;
  const int page = k.bt[j / a.page_tokens];
  if (page < 0 || page >= a.num_pages) return -1;
  const long long at = (((long long)page * a.G + s.g) * a.page_tokens + j % a.page_tokens) * a.hd;
  const uint4 *key = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.k) + at), *query = reinterpret_cast<const uint4*>(k.q);
  float x = 0.f;
  for (int d = 0; d < a.hd / 8; ++d) {
    const uint4 u = query[d], v = key[d];
    const uint32_t us[4] = {u.x, u.y, u.z, u.w}, vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x = fmaf(__uint_as_float(us[e] << 16), __uint_as_float(vs[e] << 16), x);
      x = fmaf(__uint_as_float(us[e] & 0xffff0000u), __uint_as_float(vs[e] & 0xffff0000u), x);
    }
  }
  score = log2_score(x, k.scale_log2, cap_log2, cap_in2);
  return at;
}
// The row's largest score m and the sum l of exp2(score - m).
__device__ __noinline__ void tree_row_top(const TreeArgs& a, const Segment& s, int row, float cap_log2, float cap_in2, float& m, float& l, volatile int* pulse) {
  float score, top = -CUDART_INF_F, sum = 0.f;
  for (RowKeys k = row_keys(a, s, row, pulse); k.j < k.end;)
    if (next_key(a, s, k, cap_log2, cap_in2, score) >= 0) top = fmaxf(top, score);
  top = warp_max(top);
  const float safe = top == -CUDART_INF_F ? 0.f : top;
  for (RowKeys k = row_keys(a, s, row, pulse); k.j < k.end;)
    if (next_key(a, s, k, cap_log2, cap_in2, score) >= 0) sum += exp2f(score - safe);
  m = top;
  l = warp_sum(sum);
}
// A dim a lane of the row's sums against the reference m.
__device__ __noinline__ float tree_row_again(const TreeArgs& a, const Segment& s, int row, int dim, float m, float cap_log2, float cap_in2, volatile int* pulse) {
  const float safe = m == -CUDART_INF_F ? 0.f : m;
  float acc = 0.f, score = 0.f;
  for (RowKeys k = row_keys(a, s, row, pulse); k.j < k.end;) {
    const long long at = next_key(a, s, k, cap_log2, cap_in2, score);
    const float p = exp2f(score - safe);
    for (uint32_t left = __ballot_sync(0xffffffffu, at >= 0); left; left &= left - 1) {
      const int i = __ffs(left) - 1;
      const float f = __shfl_sync(0xffffffffu, p, i);
      acc = fmaf(f, __bfloat162float(reinterpret_cast<const bf16*>(a.v)[__shfl_sync(0xffffffffu, at, i) + dim]), acc);
    }
  }
  return acc;
}

// CAP: with a soft cap on the scores (an instance of its own: its code would be in the way of every call)
template <int HD, bool CAP>
__global__ void __launch_bounds__(TC_THREADS, 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TreeArgs a, float cap_log2, float cap_in2) {
  constexpr int STAGES = TcSmem<HD>::STAGES, CPR = HD / 8, KSTEPS = HD / 16, HALVES = HD / 64;
  constexpr int MMA_WARP = TC_SOFTMAX / 32, LOAD_WARP = MMA_WARP + 2;
  constexpr uint32_t TMEM_COLS = 512, SP_COL[2] = {0, 128}, O_COL[2] = {256, 256 + HD};
  // fp32 accumulators, bf16 operands; N at bit 17 (>> 3), M at bit 24 (>> 4); bit 16: B is MN-major
  constexpr uint32_t IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TC_KEYS >> 4) << 17) | ((uint32_t)(TC_ROWS >> 4) << 24);
  constexpr uint32_t IDESC_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(TC_ROWS >> 4) << 24);

  extern __shared__ uint8_t smem_raw[];
  TcSmem<HD>& sm = *reinterpret_cast<TcSmem<HD>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  volatile int* abort_flag = &sm.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 32) {
    mbar_init(&sm.q_full, TC_SOFTMAX / 32);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.k_empty[i], 2);
      mbar_init(&sm.v_empty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      for (int j = 0; j < 2; ++j) {
        mbar_init(&sm.s_full[i][j], 2);
        mbar_init(&sm.p_full[i][j], TC_SOFTMAX / 128);
      }
      mbar_init(&sm.o_done[i], 1);
      mbar_init(&sm.drained[i], 1);
      mbar_init(&sm.turn[i], 1);
      for (int j = 0; j < 4; ++j) mbar_init(&sm.pair[i][j], 2);
    }
    sm.abort_flag = sm.pulse = sm.gone = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();             // not before the wait: tree_combine_kernel reads the requests ahead of its own
  if (warp == 0) {
    Walk w = share_start<TcCut>(a, blockIdx.x, gridDim.x).w;
    Segment s;
    const bool any = next_segment<TcCut>(a, w, s);
    if (lane == 0) {
      sm.start = w;
      sm.lead = sm.segment[0] = s;
      sm.led = any;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  Walk w = sm.start;
  Segment s = sm.lead;
  bool more = sm.led != 0;

  if (warp >= LOAD_WARP) {
    // ================================================================= loads (a lane per box of a page's keys and half of the head)
    const int box_rows = a.page_tokens < TC_KEYS ? a.page_tokens : TC_KEYS, boxes = TC_KEYS / box_rows, per_page = a.page_tokens <= TC_KEYS ? 1 : a.page_tokens / TC_KEYS;
    const int box_shift = __ffs(box_rows) - 1, box = lane & (boxes - 1), h = lane >> (__ffs(boxes) - 1);      // powers of two, boxes up to 16
    // A warp for K and one for V: a stream's next scores want K tiles before the V tiles are free that one warp would have to send for first.
    const bool is_v = warp != LOAD_WARP;
    uint64_t *full = is_v ? sm.v_full : sm.k_full, *empty = is_v ? sm.v_empty : sm.k_empty;
    const uint32_t stages = smem_u32(is_v ? sm.v[0] : sm.k[0]) + (uint32_t)(box * box_rows + h * TC_KEYS) * 128u;
    const CUtensorMap* map = is_v ? &map_v : &map_k;
    int n = 0;                    // tiles sent for so far
    bool alive = true;
    for (; alive && more; more = next_segment<TcCut>(a, w, s)) {
      const int* bt = a.block_table + (size_t)s.q.slot * a.table_stride;
      const int first = first_key(a, s.q) >> box_shift, last = (s.q.context + s.q.count - 1) >> box_shift;
      // Box b of the request: its page, and from that its first row of the pages, seen as one matrix.  A box that holds no key of the
      // request is the one of its nearest key, so that nothing but cache rows ever lies in a stage: an old NaN pattern there would not
      // be kept out of the sums by a probability of zero.
      auto box_of = [&](int b) { return min(max(b, first), last); };
      auto page_of = [&](int b) { return bt[per_page == 1 ? box_of(b) : box_of(b) / per_page]; };
      auto row_of = [&](int b, int page) {
        return page >= 0 && page < a.num_pages ? (page * a.G + s.g) * a.page_tokens + (per_page == 1 ? 0 : box_of(b) % per_page * box_rows) : 0;
      };
      // 32 boxes at a time, a lane each; the next 32 are on their way meanwhile
      int at = s.t0 * boxes + lane;
      // Keys of a page that is not there are found too late for the scores' masks: rows of the pool lie in their place, and the softmax
      // threads take every row once more without them, from here on for all of the share (this is no usual call).  The arrival for the
      // tile's keys publishes the flag.
      auto tell = [&](int page) {
        if (__any_sync(0xffffffffu, page < 0 || page >= a.num_pages) && lane == 0) *static_cast<volatile int*>(&sm.gone) = 1;
      };
      int page = page_of(at);
      int row = row_of(at, page);
      tell(page);
      page = page_of(at + 32);
      int sent = 0;
      for (int i = 0; i < s.n && alive; ++i, ++n) {
        if (sent == 32) {
          at += 32;
          row = row_of(at, page);
          tell(page);
          page = page_of(at + 32);
          sent = 0;
        }
        const int mine = __shfl_sync(0xffffffffu, row, sent + box), st = n % STAGES;
        sent += boxes;
        const uint32_t parity = (uint32_t)(((n / STAGES) & 1) ^ 1);      // a fresh barrier lets the first fill through
        int go = 1;
        if (lane == 0) {
          go = mbar_wait(&empty[st], parity, abort_flag) ? 1 : 0;
          if (go) mbar_expect_tx(&full[st], TC_KEYS * HD * 2);
        }
        alive = __shfl_sync(0xffffffffu, go, 0) != 0;
        if (alive && h < HALVES) tma_load_3d(stages + (uint32_t)(st * TC_KEYS * HD * 2), map, &full[st], 0, mine, h);
      }
    }
    if (*abort_flag && lane == 0) {          // the copies that are still on their way
      for (int i = max(0, n - STAGES); i < n; ++i) mbar_drain(&full[i % STAGES], (uint32_t)((i / STAGES) & 1));
    }
  } else if (warp >= MMA_WARP) {
    // ================================================================= products (one lane a group)
    const uint32_t x = __shfl_sync(0xffffffffu, (uint32_t)(warp - MMA_WARP), 0);
    if (elect_one()) {
      bool ok = true, issued = false;
      uint32_t tiles_done = 0, steps = 0, seg = 0, turns = x ^ 1;      // (the first turn is the first group's)
      const uint32_t sp = tmem + x * SP_COL[1], oc = tmem + O_COL[0] + x * HD;
      const uint64_t dq0 = desc_k_major(smem_u32(sm.q[0])), dk0 = desc_k_major(smem_u32(sm.k[0])), dv0 = desc_mn_major(smem_u32(sm.v[0]), TC_KEYS * 128);
      constexpr uint32_t STAGE16 = TC_KEYS * HD * 2 >> 4, HALF16 = TC_KEYS / 2 * 128 >> 4;      // descriptors count in 16 bytes
      for (; ok && more; more = ok && next_segment<TcCut>(a, w, s)) {
        const bool two = s.rows > TC_ROWS;
        const int jobs = two ? s.n : (s.n + 1 - (int)x) / 2;
        if (!mbar_wait(&sm.q_full, seg & 1u, abort_flag)) { ok = false; break; }
        ++seg;
        const uint64_t dq = dq0 + (two && x ? TC_ROWS * HD * 2 >> 4 : 0);
        // Step t of the group: tile t of the unit with two row tiles, else tile 2 t + x.  A tile is free when both groups are through with
        // it, or where only one takes it, when that one is.
        auto issue_s = [&](int h, uint32_t n) -> bool {
          const uint32_t st = n % STAGES;
          if (h == 0 && !mbar_wait(&sm.k_full[st], (n / STAGES) & 1u, abort_flag)) return false;
          tc_fence_after();
          const uint64_t dk = dk0 + st * STAGE16 + (uint32_t)h * HALF16;
#pragma unroll
          for (int kk = 0; kk < KSTEPS; ++kk)
            umma(sp + (uint32_t)(h * (TC_KEYS / 2)), dq + ((kk >> 2) * (TC_ROWS * 128 >> 4) + (kk & 3) * 2), dk + ((kk >> 2) * (TC_KEYS * 128 >> 4) + (kk & 3) * 2),
                 IDESC_S, kk ? 1u : 0u);
          issued = true;
          umma_commit(&sm.s_full[x][h]);
          mbar_arrive(&sm.s_full[x][h]);          // what this thread has seen of the softmax threads' announcements, in order with the scores
          if (h == 1) {
            umma_commit(&sm.k_empty[st]);
            if (!two) mbar_arrive(&sm.k_empty[st]);
          }
          return true;
        };
        uint32_t n = tiles_done + (two ? 0 : x);
        if (jobs > 0) ok = issue_s(0, n) && issue_s(1, n);
        for (int t = 0; t < jobs && ok; ++t) {
          const uint32_t st = n % STAGES, next = n + (two ? 1 : 2);
          const uint64_t dv = dv0 + st * STAGE16;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!ok) break;
            if (!mbar_wait(&sm.p_full[x][h], (steps + t) & 1u, abort_flag) ||
                (h == 0 && !mbar_wait(&sm.v_full[st], (n / STAGES) & 1u, abort_flag)) ||
                (two && !mbar_wait(&sm.turn[x], turns++ & 1u, abort_flag))) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < TC_KEYS / 32; ++kk)
              umma_ts(oc, sp + (uint32_t)(h * (TC_KEYS / 2) + kk * 8), dv + (uint32_t)h * HALF16 + kk * (2048 >> 4), IDESC_O, (t > 0 || h > 0 || kk > 0) ? 1u : 0u);
            if (h == 1) {
              umma_commit(&sm.v_empty[st]);
              if (!two) mbar_arrive(&sm.v_empty[st]);
            }
            if (t + 1 < jobs) ok = issue_s(h, next);       // behind this stream's product with V: it overwrites the P that it reads
            else if (h == 1) umma_commit(&sm.o_done[x]);
            if (two) mbar_arrive(&sm.turn[x ^ 1]);
          }
          n = next;
        }
        tiles_done += s.n;
        steps += jobs;
      }
      if (!ok && issued) {                             // the products that are still under way
        umma_commit(&sm.drained[x]);
        mbar_drain(&sm.drained[x], 0);
      }
    }
  } else {
    // ================================================================= softmax (two groups of 256 threads, two a row)
    // Warps w and w + 4 of a group read the same lanes of tensor memory (32 * (w & 3) ..): the first the lower half of a tile's keys, the
    // second the upper.
    const int x = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3, r = quarter * 32 + lane;      // r: row of the tile = lane of tensor memory
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    constexpr int HK = TC_KEYS / 2, EC = 16;        // keys a thread; dims of the sums that a thread finishes at once
    const float scale_log2 = a.scale * 1.4426950408889634f;
    const float sl = CAP ? 1.0f : scale_log2;       // capped scores are in the exponent's domain already
    const uint32_t sp = lane_addr + (x ? SP_COL[1] : SP_COL[0]), oc = lane_addr + (x ? O_COL[1] : O_COL[0]);
    uint32_t jobs_done = 0, met = 0, o_done[2] = {0, 0};
    bool ok = true;
    // Q: the threads of a row share it out; rows past the unit are zeros
    auto send_q = [&](const Segment& u) {
      const bool two = u.rows > TC_ROWS;
      const int row = two ? x * TC_ROWS + r : r, i = u.row0 + (row < u.rows ? row : 0), token = token_of(a, i);
      const bf16* src = reinterpret_cast<const bf16*>(a.q) + ((size_t)(u.q.first + token) * a.H + u.g * a.group + i - token * a.group) * HD;
      const uint32_t qs = smem_u32(sm.q[two ? x : 0]);
      const int c_from = two ? half * (CPR / 2) : (2 * x + half) * (CPR / 4), c_to = c_from + (two ? CPR / 2 : CPR / 4);
#pragma unroll 4
      for (int c = c_from; c < c_to; ++c) cp_async16(qs + swz(r, c), src + c * 8, row < u.rows);
      cp_async_commit();
    };
    // (the segment stays in shared memory, and the next one is found by one thread: registers are what these threads are short of, and
    // what they would spill comes back late)
    if (more) send_q(sm.segment[0]);
    for (int at = 0, next = 1; ok && more; at = next, next = next == 2 ? 0 : next + 1) {
      const Segment& s = sm.segment[at];
      if (threadIdx.x == 0) sm.any[next] = next_segment<TcCut>(a, w, sm.segment[next]);
      const bool two = s.rows > TC_ROWS;
      const int row = two ? x * TC_ROWS + r : r;
      const bool valid = row < s.rows, busy = row - lane < s.rows;        // busy: any row of the warp is one
      const int t0 = s.t0, context = s.q.context;
      const int token = valid ? token_of(a, s.row0 + row) : 0;
      const int lo = valid ? tree_row(a, s.q, token, true).lo : 0;
      cp_async_wait<0>();
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full);
      const int jobs = two ? s.n : (s.n + 1 - x) / 2;
      float m = -CUDART_INF_F, l0 = 0.f, l1 = 0.f;
      for (int n = 0; n < jobs; ++n, ++jobs_done) {
        // what can be done while the scores are on their way
        const int j0 = (t0 + (two ? n : 2 * n + x)) * TC_KEYS + half * HK;
        const bool part = j0 < lo || j0 + HK > context;
        uint32_t see[2] = {0xffffffffu, 0xffffffffu}, su[32];
        if (part) {
          const TreeRow tr = tree_row(a, s.q, token, valid);
          see[0] = visible32(tr, j0);
          see[1] = visible32(tr, j0 + 32);
        }
        // m is alike in a row's two threads, and so are the branches that they take
        const bool fresh = __any_sync(0xffffffffu, valid && m == -CUDART_INF_F);
        float asked = m;
        // what the two asked for three tiles ago: the tensor core's thread had seen both announce it before it issued the last tile's scores
        if (n >= 3) asked = fmaxf(sm.asked[(n - 3) & 7][x][0][r], sm.asked[(n - 3) & 7][x][1][r]);
        const bool moves = __any_sync(0xffffffffu, asked > m);
        if (!__all_sync(0xffffffffu, mbar_wait(&sm.s_full[x][half], jobs_done & 1u, abort_flag))) { ok = false; break; }
        if (!busy) {
          if (lane == 0) mbar_arrive(&sm.p_full[x][half]);
          continue;
        }
        tc_fence_after();
        // 32 of the thread's scores, capped and in the exponent's domain but for the factor sl, -inf where they do not count
        auto load = [&](int c) {
          tmem_ld32(sp + (uint32_t)(half * HK + 32 * c), su);
          tmem_ld_wait();
          if (CAP) {
#pragma unroll
            for (int i = 0; i < 32; ++i) su[i] = __float_as_uint(log2_score(__uint_as_float(su[i]), 1.0f, cap_log2, cap_in2));
          }
          if (part) {
#pragma unroll
            for (int i = 0; i < 32; ++i) su[i] = ((c ? see[1] : see[0]) >> i) & 1u ? su[i] : 0xff800000u;
          }
        };
        if (fresh) {
          float top = -CUDART_INF_F;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            load(c);
            float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
            for (int i = 0; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(su[i]));
            top = fmaxf(top, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          }
          sm.first[n & 1][x][half][r] = top * sl;
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.pair[x][quarter]);
          if (!__all_sync(0xffffffffu, mbar_wait(&sm.pair[x][quarter], met & 1u, abort_flag))) { ok = false; break; }
          ++met;
          if (m == -CUDART_INF_F) m = ceilf(fmaxf(sm.first[n & 1][x][0][r], sm.first[n & 1][x][1][r]));
        } else if (moves) {
          // O may be touched: this half's product with V of the last tile is complete, since these scores are, and the other half's is
          // once its scores are; the next ones wait for the two warps, which meet when both have done their part of the dims
          bool fine = mbar_wait(&sm.s_full[x][half ^ 1], jobs_done & 1u, abort_flag);
          tc_fence_after();
          const float corr = asked > m ? exp2f(m - asked) : 1.0f;
          l0 *= corr;
          l1 *= corr;
#pragma unroll 1
          for (int c0 = half * (HD / 2); c0 < (half + 1) * (HD / 2); c0 += 16) {
            uint32_t o[16];
            tmem_ld16(oc + (uint32_t)c0, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tmem_st16(oc + (uint32_t)c0, o);
          }
          m = fmaxf(m, asked);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.pair[x][quarter]);
          fine = mbar_wait(&sm.pair[x][quarter], met & 1u, abort_flag) && fine;
          tc_fence_after();
          if (!__all_sync(0xffffffffu, fine)) { ok = false; break; }
          ++met;
        }
        const float shift = m == -CUDART_INF_F ? 0.f : -m, l_before = l0 + l1;
        // a half's P lies in the columns of its own scores that are read already (a loop: a short call waits for its instructions)
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          load(c);
          uint32_t pw[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float p0 = __uint_as_float(su[2 * e]), p1 = __uint_as_float(su[2 * e + 1]);
            fma_two(p0, p1, sl, shift);
            p0 = ex2(p0);
            p1 = ex2(p1);
            add_two(l0, l1, p0, p1);
            const __nv_bfloat162 pk = __floats2bfloat162_rn(p0, p1);
            pw[e] = *reinterpret_cast<const uint32_t*>(&pk);
          }
          tmem_st16(sp + (uint32_t)(half * HK + 16 * c), pw);
        }
        const float more_l = l0 + l1 - l_before;
        float ask = m;
        if (!(more_l <= MUCH)) {
          ask = m + ceilf(log2f(more_l));
          if (!(more_l <= TOO_MUCH)) {
            l0 = CUDART_NAN_F;
            ask = m;
          }
        }
        sm.asked[n & 7][x][half][r] = ask;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[x][half]);
      }
      // the sums of both groups: a row's two threads (four where the groups share their rows) take a part of its dims each
      const bool second = two || s.n > 1;              // the second group had a tile at all
      for (int y = 0; y < 2 && ok; ++y) {
        if (y == 1 && !second) break;
        if (!__all_sync(0xffffffffu, mbar_wait(&sm.o_done[y], o_done[y] & 1u, abort_flag))) ok = false;
        else ++o_done[y];
      }
      // (a thread has seen what was told before its own tiles came; a row's sums meet, and one that is lost makes all of them)
      sm.ml[x][half][r] = make_float2(m, *static_cast<volatile int*>(&sm.gone) ? CUDART_NAN_F : l0 + l1);
      tc_fence_before();
      ok = !softmax_any(!ok);
      if (!ok) break;
      tc_fence_after();
      more = sm.any[next] != 0;
      if (more) send_q(sm.segment[next]);              // both groups' scores are through: Q is free
      if (busy) {
        float f[2] = {1.0f, 1.0f}, l;
        if (two) {
          l = sm.ml[x][0][r].y + sm.ml[x][1][r].y;
        } else {
          const float2 u = sm.ml[0][0][r], v = sm.ml[1][0][r];
          m = fmaxf(u.x, v.x);
          const float safe = m == -CUDART_INF_F ? 0.f : m;
          f[0] = exp2f(u.x - safe);
          f[1] = exp2f(v.x - safe);
          l = (u.y + sm.ml[0][1][r].y) * f[0] + (v.y + sm.ml[1][1][r].y) * f[1];
        }
        const int head = s.g * a.group + (valid ? s.row0 + row - token * a.group : 0);
        const size_t slot = part_slot(blockIdx.x, s.begins);
        // one over a row's denominator, the sink's term in it
        auto finish = [&](float top, float sum, int of_head) {
          float f = 1.0f;
          if (a.sink) {
            const float score = (a.sinks ? a.sinks[of_head] : 0.f) * 1.4426950408889634f, high = fmaxf(top, score);
            f = top == -CUDART_INF_F ? 0.f : exp2f(top - high);
            sum = sum * f + exp2f(score - high);
          }
          return sum > 0.f || sum != sum ? f / sum : 0.f;
        };
        float inv = 1.0f;
        if (s.whole) inv = finish(m, l, head);
        else if (valid && half == 0 && (two || x == 0)) *(reinterpret_cast<float2*>(a.part_ml) + slot * a.rows_cap + row) = make_float2(m, l);
        bf16* op = reinterpret_cast<bf16*>(a.out) + ((size_t)(s.q.first + token) * a.H + head) * HD;
        float odd = 0.f;                               // NaN where a sum is NaN or Inf
        const int c_from = two ? half * (HD / 2) : (2 * x + half) * (HD / 4), c_to = c_from + (two ? HD / 2 : HD / 4);
        for (int c0 = c_from; c0 < c_to; c0 += EC) {
          uint32_t o[EC], o2[EC];
          tmem_ld16((two ? oc : lane_addr + O_COL[0]) + (uint32_t)c0, o);
          if (!two && second) tmem_ld16(lane_addr + O_COL[1] + (uint32_t)c0, o2);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < EC; ++i) {
            float y = __uint_as_float(o[i]) * f[0];
            if (!two && second) y = fmaf(__uint_as_float(o2[i]), f[1], y);
            odd = fmaf(y, 0.f, odd);
            o[i] = __float_as_uint(y * inv);
          }
          if (valid && s.whole) {
#pragma unroll
            for (int i = 0; i < EC; i += 8) {
              uint32_t pk[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 y = __floats2bfloat162_rn(__uint_as_float(o[i + 2 * e]), __uint_as_float(o[i + 2 * e + 1]));
                pk[e] = *reinterpret_cast<const uint32_t*>(&y);
              }
              *reinterpret_cast<uint4*>(op + c0 + i) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
          } else if (valid) {
#pragma unroll
            for (int i = 0; i < EC; i += 4)
              *reinterpret_cast<uint4*>(part_place(a, slot, row, c0 + i, HD)) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        if (!(l <= CUDART_MAX_NORMAL_F)) odd = CUDART_NAN_F;         // alike in all threads of a row
        for (unsigned again = __ballot_sync(0xffffffffu, valid && odd != 0.f); again; again &= again - 1) {
          const Segment unit = s;
          __syncwarp();
          const int from = __ffs(again) - 1, odd_row = row - lane + from;
          float m_row = __shfl_sync(0xffffffffu, m, from), l_row = __shfl_sync(0xffffffffu, l, from), inv_row = __shfl_sync(0xffffffffu, inv, from);
          bf16* op_row = reinterpret_cast<bf16*>(__shfl_sync(0xffffffffu, (unsigned long long)op, from));
          const int head_row = __shfl_sync(0xffffffffu, head, from);
          if (!(l_row <= CUDART_MAX_NORMAL_F)) {        // the reference and the sum as well
            tree_row_top(a, unit, odd_row, cap_log2, cap_in2, m_row, l_row, &sm.pulse);
            if (s.whole) inv_row = finish(m_row, l_row, head_row);
            else if (lane == 0 && half == 0 && (two || x == 0)) *(reinterpret_cast<float2*>(a.part_ml) + slot * a.rows_cap + odd_row) = make_float2(m_row, l_row);
          }
          for (int c0 = c_from; c0 < c_to; c0 += 32) {
            const int dim = c0 + lane;
            const float y = tree_row_again(a, unit, odd_row, min(dim, HD - 1), m_row, cap_log2, cap_in2, &sm.pulse);
            if (dim < c_to) {
              if (s.whole) op_row[dim] = __float2bfloat16_rn(y * inv_row);
              else part_place(a, slot, odd_row, dim, HD)[dim & 3] = y;
            }
          }
        }
      }
      tc_fence_before();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && sm.abort_flag) atomicExch(a.status, 4);
  if (warp == MMA_WARP) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) == cudaSuccess && qr == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// The cache pages of one layer, a bf16 matrix [rows, hd], seen as [64 columns, rows, hd / 64 halves]; a box takes 64 columns x
// box_rows rows of one half and lands as [row][128 bytes] with the 128-byte swizzle.
bool make_page_map(CUtensorMap* map, const void* ptr, unsigned long long rows, int hd, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {64u, (cuuint64_t)rows, (cuuint64_t)(hd / 64)};
  cuuint64_t strides[2] = {(cuuint64_t)hd * 2, 128u};
  cuuint32_t box[3] = {64u, (cuuint32_t)box_rows, 1u};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD>
int launch_tc(const TreeArgs& a, int ctas, cudaStream_t s) {
  const int pt = a.page_tokens;
  if (!((pt % 8 == 0 && TC_KEYS % pt == 0) || pt % TC_KEYS == 0) || a.status == nullptr) return HK_ERR_UNSUPPORTED;
  if ((((uintptr_t)a.k | (uintptr_t)a.v) & 127) != 0) return HK_ERR_UNSUPPORTED;
  const unsigned long long rows = (unsigned long long)a.num_pages * a.G * pt;
  if (rows > 0x7fffffffull || a.rows_cap < (a.most_tokens * a.group < 2 * TC_ROWS ? a.most_tokens * a.group : 2 * TC_ROWS)) return HK_ERR_UNSUPPORTED;
  CUtensorMap mk, mv;
  const int box_rows = pt < TC_KEYS ? pt : TC_KEYS;
  if (!make_page_map(&mk, a.k, rows, HD, box_rows) || !make_page_map(&mv, a.v, rows, HD, box_rows)) return HK_ERR_UNSUPPORTED;
  const size_t smem = sizeof(TcSmem<HD>) + 1024;
  if (!cut_fits<TcCut>(a)) return HK_ERR_UNSUPPORTED;
  // a soft cap c in the base-2 domain: C = c log2(e), and 2 log2(e) scale / c, which takes a raw product to 2 z log2(e), z = score / c
  const float cap_log2 = a.softcap > 0.f ? a.softcap * 1.4426950408889634f : 0.f, cap_in2 = a.softcap > 0.f ? 2.8853900817779268f * a.scale / a.softcap : 0.f;
  const dim3 grid((unsigned)ctas), block(TC_THREADS);
  int e = a.softcap > 0.f ? hk_allow_smem<tree_tc_kernel<HD, true>>(smem) : hk_allow_smem<tree_tc_kernel<HD, false>>(smem);
  if (!e) e = a.softcap > 0.f ? hk_launch_pdl(tree_tc_kernel<HD, true>, grid, block, smem, s, mk, mv, a, cap_log2, cap_in2)
                              : hk_launch_pdl(tree_tc_kernel<HD, false>, grid, block, smem, s, mk, mv, a, cap_log2, cap_in2);
  if (e) return e;
  return launch_combine<bf16, HD, TcCut>(a, ctas, s);
}

// ---- float32 ------------------------------------------------------------------------------------------------------------------
// A tile has 32 rows, keys come 32 at a time through shared memory, and scores and sums are register tiles of multiply-adds over
// 16-byte loads (4 x 2 scores a thread along the head's dims, 4 rows x HD / 16 dims of sums).  The next tile's keys arrive while this
// one's probabilities are made, the next values while the next scores are.  Bound by the shared-memory reads beside the multiply-adds, by
// start and end and by shares of whole tiles: 2 requests of 15 tokens behind 1,500 rows (16 heads over 8 of 128) 24.5 us (the generic
// kernel 334), 19 MB and 0.27 GFLOP, 3.7 us at the multiply-adds' peak.  In tiles of 64 keys, two CTAs a SM, that takes 30.8 us, behind
// 3,000 rows 41.0 for 31.1, 8 requests of 64 tokens behind up to 4,000 197 for 191, but 2 behind 20 rows 14.4 for 16.4.
constexpr int F32_ROWS = 32, F32_KEYS = 32, F32_THREADS = 128, F32_LDP = F32_KEYS + 4;
typedef Cut<F32_ROWS, F32_KEYS, 1> F32Cut;

template <int HD>
struct F32Smem {
  static constexpr int LD = HD + 4;
  float q[F32_ROWS * LD], k[F32_KEYS * LD], v[F32_KEYS * LD], p[F32_ROWS * F32_LDP];
  float corr[F32_ROWS], inv[F32_ROWS];
  float2 ml[F32_ROWS];
  uint32_t see[F32_ROWS][F32_KEYS / 32];
  long long at[2][F32_KEYS];      // [parity of the tile]: where a key's row lies in the pages, -1 where there is none
  uint32_t there[2];              // and the keys that have one
  Walk start;
};

template <int HD>
__global__ void __launch_bounds__(F32_THREADS, 4) tree_f32_kernel(const TreeArgs a) {
  constexpr int LD = F32Smem<HD>::LD, C4 = HD / 4, B = HD / 64, RI = F32_ROWS / 8, WORDS = F32_KEYS / 32, KJ = F32_KEYS / 16;
  extern __shared__ __align__(16) uint8_t f32_raw[];
  F32Smem<HD>& sm = *reinterpret_cast<F32Smem<HD>*>(f32_raw);
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, group = a.group;
  const float* qp = reinterpret_cast<const float*>(a.q);
  pdl_wait();
  pdl_launch_dependents();             // not before the wait: tree_combine_kernel reads the requests ahead of its own
  if (tid < 32) {
    const Walk w = share_start<F32Cut>(a, blockIdx.x, gridDim.x).w;
    if (tid == 0) sm.start = w;
  }
  __syncthreads();
  Walk w = sm.start;
  Segment s;
  while (next_segment<F32Cut>(a, w, s)) {
    const int* bt = a.block_table + (size_t)s.q.slot * a.table_stride;
    const int end = s.q.context + s.q.count;
    // where the keys of a tile lie: found once for keys and values, by a warp that nothing else waits for
    static_assert(F32_KEYS == 32 && WORDS * F32_ROWS == 32, "a lane a key; the rows' masks by the first warp");
    auto find = [&](int tile, int r) {
      const int j = (s.t0 + tile) * F32_KEYS + r, page = j < end ? bt[j / a.page_tokens] : -1;
      sm.at[tile & 1][r] = page >= 0 && page < a.num_pages ? (((long long)page * a.G + s.g) * a.page_tokens + j % a.page_tokens) * HD : -1;
      const uint32_t there = __ballot_sync(0xffffffffu, page >= 0 && page < a.num_pages);
      if (r == 0) sm.there[tile & 1] = there;
    };
    // a tile's keys or values, what does not exist as zeros
    auto fetch = [&](const void* pages, float* dst, int tile) {
#pragma unroll 8
      for (int e = tid; e < F32_KEYS * C4; e += F32_THREADS) {
        const int r = e / C4, d = e % C4 * 4;
        const long long at = sm.at[tile & 1][r];
        cp_async16(smem_u32(dst + r * LD + d), reinterpret_cast<const float*>(pages) + (at >= 0 ? at + d : 0), at >= 0);
      }
      cp_async_commit();
    };
    if (tid < F32_KEYS) find(0, tid);
    __syncthreads();
    fetch(a.k, sm.k, 0);
    fetch(a.v, sm.v, 0);
    for (int e = tid; e < F32_ROWS * C4; e += F32_THREADS) {
      const int r = e / C4, d = e % C4 * 4, i = s.row0 + r;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      const int token = token_of(a, i);
      if (r < s.rows) x = *reinterpret_cast<const float4*>(qp + ((size_t)(s.q.first + token) * a.H + s.g * group + i - token * group) * HD + d);
      *reinterpret_cast<float4*>(sm.q + r * LD + d) = make_float4(x.x * a.scale, x.y * a.scale, x.z * a.scale, x.w * a.scale);
    }
    const float cap = a.softcap, inv_cap = cap > 0.f ? 1.0f / cap : 0.f;
    const TreeRow tr = tree_row(a, s.q, token_of(a, s.row0 + tid / WORDS), tid < WORDS * F32_ROWS && tid / WORDS < s.rows);     // of row tid / WORDS
    // the softmax's state of row tid / 4, alike in its four threads
    const int sr = tid >> 2, sc = (tid & 3) * 4 * KJ;
    float m = -CUDART_INF_F, l = 0.f;
    float4 acc[RI][B];
#pragma unroll
    for (int i = 0; i < RI; ++i)
#pragma unroll
      for (int b = 0; b < B; ++b) acc[i][b] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int t = 0; t < s.n; ++t) {
      const int j0 = (s.t0 + t) * F32_KEYS;
      bool part = false;
      if (tid < WORDS * F32_ROWS) {
        const uint32_t see = visible32(tr, j0 + 32 * (tid % WORDS)) & sm.there[t & 1];
        sm.see[tid / WORDS][tid % WORDS] = see;
        part = tid / WORDS < s.rows && see != 0xffffffffu;
      } else if (t + 1 < s.n && tid - WORDS * F32_ROWS < F32_KEYS) {
        find(t + 1, tid - WORDS * F32_ROWS);
      }
      cp_async_wait<1>();          // the keys
      part = __syncthreads_or(part);
      float x[RI][KJ];
#pragma unroll
      for (int i = 0; i < RI; ++i)
#pragma unroll
        for (int j = 0; j < KJ; ++j) x[i][j] = 0.f;
#pragma unroll 2
      for (int d = 0; d < HD; d += 4) {
        float4 u[RI], v[KJ];
#pragma unroll
        for (int i = 0; i < RI; ++i) u[i] = *reinterpret_cast<const float4*>(sm.q + (ty + 8 * i) * LD + d);
#pragma unroll
        for (int j = 0; j < KJ; ++j) v[j] = *reinterpret_cast<const float4*>(sm.k + (tx + 16 * j) * LD + d);
#pragma unroll
        for (int i = 0; i < RI; ++i)
#pragma unroll
          for (int j = 0; j < KJ; ++j) x[i][j] = fmaf(u[i].w, v[j].w, fmaf(u[i].z, v[j].z, fmaf(u[i].y, v[j].y, fmaf(u[i].x, v[j].x, x[i][j]))));
      }
#pragma unroll
      for (int i = 0; i < RI; ++i) {
        const int r = ty + 8 * i;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const int key = tx + 16 * j;
          float y = x[i][j];
          if (cap > 0.f) y = cap * tanhf(y * inv_cap);
          sm.p[r * F32_LDP + key] = (sm.see[r][key >> 5] >> (key & 31)) & 1u ? y : -CUDART_INF_F;
        }
      }
      __syncthreads();
      if (t + 1 < s.n) fetch(a.k, sm.k, t + 1);
      else cp_async_commit();
      {
        float* row = sm.p + sr * F32_LDP + sc;
        float4 y[KJ];
        float top = -CUDART_INF_F;
#pragma unroll
        for (int e = 0; e < KJ; ++e) {
          y[e] = *reinterpret_cast<const float4*>(row + 4 * e);
          top = fmaxf(top, fmaxf(fmaxf(y[e].x, y[e].y), fmaxf(y[e].z, y[e].w)));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mn = fmaxf(m, top), safe = mn == -CUDART_INF_F ? 0.f : mn;
        const float corr = expf(m - safe);                          // m = -inf: 0
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < KJ; ++e) {
          y[e] = make_float4(expf(y[e].x - safe), expf(y[e].y - safe), expf(y[e].z - safe), expf(y[e].w - safe));
          sum += (y[e].x + y[e].y) + (y[e].z + y[e].w);
          *reinterpret_cast<float4*>(row + 4 * e) = y[e];
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        l = fmaf(l, corr, sum);
        m = mn;
        if ((tid & 3) == 0) sm.corr[sr] = corr;
      }
      cp_async_wait<1>();          // the values
      bool apart = false;          // NaN or Inf among values that some row does not see
      if (part) {
        float odd = 0.f;           // NaN if one of the pieces that this thread fetched holds any
#pragma unroll 4
        for (int e = tid; e < F32_KEYS * C4; e += F32_THREADS) {
          const float4 y = *reinterpret_cast<const float4*>(sm.v + e / C4 * LD + e % C4 * 4);
          odd = fmaf(y.x, 0.f, fmaf(y.y, 0.f, fmaf(y.z, 0.f, fmaf(y.w, 0.f, odd))));
        }
        apart = __syncthreads_or(odd != 0.f);
      } else {
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < RI; ++i) {
        const float c = sm.corr[ty + 8 * i];
#pragma unroll
        for (int b = 0; b < B; ++b) acc[i][b] = make_float4(acc[i][b].x * c, acc[i][b].y * c, acc[i][b].z * c, acc[i][b].w * c);
      }
      if (!apart) {
#pragma unroll 2
        for (int c = 0; c < F32_KEYS; c += 4) {
          float4 p[RI];
#pragma unroll
          for (int i = 0; i < RI; ++i) p[i] = *reinterpret_cast<const float4*>(sm.p + (ty + 8 * i) * F32_LDP + c);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int b = 0; b < B; ++b) {
              const float4 v = *reinterpret_cast<const float4*>(sm.v + (c + e) * LD + 64 * b + 4 * tx);
#pragma unroll
              for (int i = 0; i < RI; ++i) {
                const float f = e == 0 ? p[i].x : e == 1 ? p[i].y : e == 2 ? p[i].z : p[i].w;
                acc[i][b] = make_float4(fmaf(f, v.x, acc[i][b].x), fmaf(f, v.y, acc[i][b].y), fmaf(f, v.z, acc[i][b].z), fmaf(f, v.w, acc[i][b].w));
              }
            }
        }
      } else {
#pragma unroll
        for (int i = 0; i < RI; ++i) {
          const int r = ty + 8 * i;
          for (int word = 0; word < WORDS; ++word)
            for (uint32_t left = sm.see[r][word]; left; left &= left - 1) {
              const int c = 32 * word + __ffs(left) - 1;
              const float f = sm.p[r * F32_LDP + c];
#pragma unroll
              for (int b = 0; b < B; ++b) {
                const float4 v = *reinterpret_cast<const float4*>(sm.v + c * LD + 64 * b + 4 * tx);
                acc[i][b] = make_float4(fmaf(f, v.x, acc[i][b].x), fmaf(f, v.y, acc[i][b].y), fmaf(f, v.z, acc[i][b].z), fmaf(f, v.w, acc[i][b].w));
              }
            }
        }
      }
      __syncthreads();
      if (t + 1 < s.n) fetch(a.v, sm.v, t + 1);
      else cp_async_commit();
    }
    cp_async_wait<0>();
    if ((tid & 3) == 0) {
      float inv = 1.0f, total = l;
      if (s.whole) {
        if (a.sink && sr < s.rows) {
          const float score = a.sinks ? a.sinks[s.g * group + s.row0 + sr - token_of(a, s.row0 + sr) * group] : 0.f, top = fmaxf(m, score);
          inv = m == -CUDART_INF_F ? 0.f : expf(m - top);
          total = l * inv + expf(score - top);
        }
        inv = total > 0.f || total != total ? inv / total : 0.f;
      }
      sm.inv[sr] = inv;
      sm.ml[sr] = make_float2(m, l);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      const int r = ty + 8 * i, at = s.row0 + r;
      if (r >= s.rows) continue;
      const float inv = sm.inv[r];
      const size_t slot = part_slot(blockIdx.x, s.begins);
      const int token = token_of(a, at);
      float* out = reinterpret_cast<float*>(a.out) + ((size_t)(s.q.first + token) * a.H + s.g * group + at - token * group) * HD;
#pragma unroll
      for (int b = 0; b < B; ++b)
        *reinterpret_cast<float4*>(s.whole ? out + 64 * b + 4 * tx : part_place(a, slot, r, 64 * b + 4 * tx, HD)) =
            make_float4(acc[i][b].x * inv, acc[i][b].y * inv, acc[i][b].z * inv, acc[i][b].w * inv);
      if (!s.whole && tx == 0) *(reinterpret_cast<float2*>(a.part_ml) + slot * a.rows_cap + r) = sm.ml[r];
    }
    __syncthreads();
  }
}

template <int HD>
int launch_f32(const TreeArgs& a, int ctas, cudaStream_t s) {
  if (a.rows_cap < (a.most_tokens * a.group < F32_ROWS ? a.most_tokens * a.group : F32_ROWS)) return HK_ERR_UNSUPPORTED;
  if (!cut_fits<F32Cut>(a)) return HK_ERR_UNSUPPORTED;
  if (int e = hk_allow_smem<tree_f32_kernel<HD>>(sizeof(F32Smem<HD>))) return e;
  if (int e = hk_launch_pdl(tree_f32_kernel<HD>, dim3((unsigned)ctas), dim3(F32_THREADS), sizeof(F32Smem<HD>), s, a)) return e;
  return launch_combine<float, HD, F32Cut>(a, ctas, s);
}

}  // namespace

// q, out [n, H, hd]; k, v [num_pages, G, page_tokens, hd]; block_table int32 [table_rows, table_stride]; requests int32
// [n_requests, 4] = (slot, first row of q, drafted tokens, rows in the cache before them); ancestors [n, words] 32-bit words: bit j
// of a token's row: it sees the drafted token j of its request; positions int32 [n] (read with a window only): drafted tokens stand
// at their request's `context` or behind it.  Only rows of q that belong to a request are computed.  scale on q . k, softcap c (0:
// none), window w (0: none): a key at position x is seen from position p if x > p - w; sink, sinks: one more term of the
// denominator.  most_tokens, most_keys: a request with more drafted
// tokens, or more rows with them, is left out.  `kernel` 0: any size up to heads of 256.  `kernel` 1: heads of 64 and
// 128, in bfloat16 on the tensor cores (cache pages that are whole boxes of a 128-key tile: multiples of 8 that divide 128, and
// multiples of 128), in float32 with multiply-adds; `ctas` shares, part_o float [2 ctas, hd / 4, rows_cap, 4] and part_ml [2 ctas,
// rows_cap, 2] for what they leave, rows_cap at least the rows of a tile (256, in float32 32; or most_tokens * H / G where that is less); `status` is set to 4 if a bounded wait ran out.
HK_API int hk_tree_attention(const TreeCall* call, int kernel, int ctas, float* part_o, float* part_ml, int rows_cap, int* status, void* stream) {
  const TreeCall& c = *call;
  if (c.n <= 0 || c.n_requests <= 0 || c.most_tokens <= 0) return 0;
  if (c.most_keys < 1 || c.most_keys > (long long)c.table_stride * c.page_tokens || c.most_tokens > 256) return HK_ERR_UNSUPPORTED;
  if (c.H < 1 || c.G < 1 || c.H % c.G != 0 || c.hd < 1 || c.hd > 256 || c.page_tokens < 1 || c.table_rows < 1 || c.table_stride < 1 || c.words < 1 ||
      c.n_requests > 65535 || c.num_pages < 1 || c.softcap < 0.f || !(c.scale > 0.f) || (c.dtype != HK_F32 && c.dtype != HK_BF16) ||
      (((uintptr_t)c.requests) & 15) != 0)
    return HK_ERR_UNSUPPORTED;
  TreeArgs a;
  a.q = c.q; a.k = c.k; a.v = c.v; a.out = c.out;
  a.block_table = c.block_table;
  a.requests = reinterpret_cast<const TreeReq*>(c.requests);
  a.ancestors = static_cast<const uint32_t*>(c.ancestors);
  a.positions = c.positions;
  a.sinks = c.sink ? c.sinks : nullptr;
  a.part_o = part_o; a.part_ml = part_ml; a.status = status;
  a.num_pages = c.num_pages;
  a.n = c.n; a.n_requests = c.n_requests; a.most_tokens = c.most_tokens; a.most_keys = c.most_keys; a.words = c.words;
  a.table_rows = c.table_rows; a.table_stride = c.table_stride; a.page_tokens = c.page_tokens;
  a.H = c.H; a.G = c.G; a.hd = c.hd; a.window = c.window > 0 ? c.window : 0; a.sink = c.sink; a.rows_cap = rows_cap;
  a.scale = c.scale; a.softcap = c.softcap;
  a.group = c.H / c.G;
  a.group_inverse = a.group == 1 ? 0u : (uint32_t)((0x100000000ull + a.group - 1) / a.group);
  cudaStream_t s = (cudaStream_t)stream;
  if (kernel == 0) return c.dtype == HK_F32 ? launch_generic<float>(a, s) : launch_generic<bf16>(a, s);
  if (kernel != 1 || ctas < 1 || part_o == nullptr || part_ml == nullptr) return HK_ERR_UNSUPPORTED;
  if ((((uintptr_t)c.q | (uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.out | (uintptr_t)part_o) & 15) != 0 || (((uintptr_t)part_ml) & 7) != 0) return HK_ERR_UNSUPPORTED;
  if ((c.hd != 64 && c.hd != 128) || a.group > 4095) return HK_ERR_UNSUPPORTED;
  if (c.dtype == HK_F32) return c.hd == 128 ? launch_f32<128>(a, ctas, s) : launch_f32<64>(a, ctas, s);
  return c.hd == 128 ? launch_tc<128>(a, ctas, s) : launch_tc<64>(a, ctas, s);
}
