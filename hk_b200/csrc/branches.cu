// Several continuations of one request: blocks of a cache copied in all layers at once (pages of forked requests, states that
// surviving beams pass on), the accepted rows of a drafted tree moved up side by side, and the choice over beams and vocabulary.
//
// What the device arrays say is checked where it is read: a copy or a row whose page, slot or place lies outside the arrays is left
// out.
#include <math_constants.h>

#include "common.cuh"

// Every kernel here lets the next one start only behind its own wait: so no more than two calls' kernels are under way at once, and none
// runs beside one that is to be through before the kernel before it.  What a kernel before may have written in part of a 32-byte sector
// (blocks and rows of odd sizes, parts of a choice) is read past L1: it is read once, so L1 gives nothing, and whatever an SM's L1 took in
// for that kernel, while this one had started, does not count.

namespace {

// ---- blocks of a cache --------------------------------------------------------------------------------------------------
// A block is `pieces` runs of `piece` bytes; of each run the first min(rows * row, piece) bytes are copied.
struct BlockArray {
  long long address, blocks, pieces, piece, row;
};

constexpr int COPY_THREADS = 128, COPY_DEEP = 8;      // threads; vectors that a thread has on their way at once

template <typename V>
__device__ __forceinline__ void copy_part(uint8_t* to, const uint8_t* from, long long pieces, long long piece, long long used) {
  const long long per = used / (long long)sizeof(V), all = pieces * per;
  for (long long i0 = (long long)blockIdx.x * COPY_THREADS * COPY_DEEP + threadIdx.x; i0 < all; i0 += (long long)gridDim.x * COPY_THREADS * COPY_DEEP) {
    V v[COPY_DEEP];
    long long at[COPY_DEEP];
#pragma unroll
    for (int k = 0; k < COPY_DEEP; ++k) {
      const long long i = i0 + k * COPY_THREADS;
      at[k] = -1;
      if (i < all) {
        const long long p = pieces == 1 ? 0 : (long long)((unsigned long long)i / (unsigned long long)per);
        at[k] = p * piece + (i - p * per) * (long long)sizeof(V);
        v[k] = __ldcg(reinterpret_cast<const V*>(from + at[k]));
      }
    }
#pragma unroll
    for (int k = 0; k < COPY_DEEP; ++k)
      if (at[k] >= 0) *reinterpret_cast<V*>(to + at[k]) = v[k];
  }
}

// Bound by DRAM: 7 pages of 128 KB in 72 arrays (67 MB, read and written) 13.7 us with the launch, 4.9 TB/s; 19 states of 1 MB in 36
// arrays 167, 8.6 TB/s (part of it in L2).  Blocks of 256 threads (half as many a SM, for the registers): 15.6 and 170; four vectors a
// thread on their way: 14.0 and 166; 2 states 22.9, 24.9 and 23.3.
__global__ void __launch_bounds__(COPY_THREADS, 8)
copy_blocks_kernel(const BlockArray* __restrict__ table, const int* __restrict__ moves) {
  pdl_wait();
  pdl_launch_dependents();
  const BlockArray a = table[blockIdx.z];
  const int from = moves[3 * blockIdx.y], to = moves[3 * blockIdx.y + 1], rows = moves[3 * blockIdx.y + 2];
  if (from < 0 || to < 0 || from >= a.blocks || to >= a.blocks || from == to || rows <= 0) return;
  const long long used = rows >= (a.piece + a.row - 1) / a.row ? a.piece : rows * a.row;
  const uint8_t* src = reinterpret_cast<const uint8_t*>(a.address) + from * a.pieces * a.piece;
  uint8_t* dst = reinterpret_cast<uint8_t*>(a.address) + to * a.pieces * a.piece;
  const unsigned long long all = (unsigned long long)src | (unsigned long long)dst | (unsigned long long)used |
                                 (a.pieces > 1 ? (unsigned long long)a.piece : 0ull);
  if ((all & 15) == 0) copy_part<uint4>(dst, src, a.pieces, a.piece, used);
  else if ((all & 3) == 0) copy_part<uint32_t>(dst, src, a.pieces, a.piece, used);
  else copy_part<uint8_t>(dst, src, a.pieces, a.piece, used);
}

// ---- the accepted rows of a tree --------------------------------------------------------------------------------------------
struct RowArray {
  long long address, heads, row;
  const int* block_table;
};

constexpr int KEEP_THREADS = 128, KEEP_DEEP = 8, KEEP_PATH = 256;

// A thread takes a column (head, 16 bytes of a row) of an array and moves its rows in order: a path climbs, so a row that is written
// (path[i] -> i, i <= path[i]) is none that a later step of the path reads.  `from`, `to`: page, place in the page.
template <typename V>
__device__ __forceinline__ void move_rows(const RowArray& a, const int2* from, const int2* to, int n, int page_tokens, int column) {
  const int per = (int)(a.row / (long long)sizeof(V));
  const long long head_bytes = page_tokens * a.row, page_bytes = a.heads * head_bytes;
  uint8_t* base = reinterpret_cast<uint8_t*>(a.address) + (column / per) * head_bytes + (column % per) * (long long)sizeof(V);
  for (int i0 = 0; i0 < n; i0 += KEEP_DEEP) {
    V v[KEEP_DEEP];
#pragma unroll
    for (int k = 0; k < KEEP_DEEP; ++k)
      if (i0 + k < n) v[k] = __ldcg(reinterpret_cast<const V*>(base + from[i0 + k].x * page_bytes + from[i0 + k].y * a.row));
#pragma unroll
    for (int k = 0; k < KEEP_DEEP; ++k)
      if (i0 + k < n) *reinterpret_cast<V*>(base + to[i0 + k].x * page_bytes + to[i0 + k].y * a.row) = v[k];
  }
}

// A block takes a request and some neighbouring arrays, and finds the pages of its path once for all that share a block table: finding
// them is a chain of three reads, and as long as moving an array's rows.  Bound by the reads' and writes' way through DRAM in pieces of
// a row of a head (256 bytes): 64 requests of up to nine rows in 72 arrays, 42 MB, take 13.4 us one call behind the other, 3.2 TB/s, and
// 15.2 as replays over three caches in turn (over two, which partly stay in L2: 13.5, through L1 14.1; through it in blocks of 256 threads 17.4, of 64 14.4, with
// four reads a thread on their way 16.5, 16 requests 6.2).
__global__ void __launch_bounds__(KEEP_THREADS, 8)
compact_rows_kernel(const RowArray* __restrict__ table, int arrays, int per_block, const int* __restrict__ paths, int width, int table_rows,
                    int table_stride, int page_tokens, long long num_pages) {
  __shared__ int2 from[KEEP_PATH], to[KEEP_PATH];
  __shared__ int count;
  pdl_wait();
  pdl_launch_dependents();
  const int* path = paths + (size_t)blockIdx.x * (width + 2);
  const int slot = path[0], first = path[1], a0 = blockIdx.y * per_block, a1 = min(arrays, a0 + per_block);
  if (slot < 0 || slot >= table_rows || first < 0) return;
  for (int done = 0; done < width; done += KEEP_PATH) {
    const int* found = nullptr;
    for (int i = a0; i < a1;) {
      const int* block_table = table[i].block_table;
      if (block_table != found) {
        __syncthreads();
        if (threadIdx.x < 32) {            // the rows that move, in order
          const int* pages = block_table + (size_t)slot * table_stride;
          auto place = [&](uint32_t row) -> int2 {           // row: below 2^32, two non-negative ints added
            const uint32_t at = row / (uint32_t)page_tokens;
            const int page = at < (uint32_t)table_stride ? pages[at] : -1;
            return make_int2(page < 0 || page >= num_pages ? -1 : page, (int)(row - at * (uint32_t)page_tokens));
          };
          int n = 0;
          for (int i0 = done; i0 < min(width, done + KEEP_PATH); i0 += 32) {
            const int k = i0 + (int)threadIdx.x, row = k < width ? path[2 + k] : -1;
            int2 f = make_int2(-1, 0), t = f;
            if (row > k) {
              f = place((uint32_t)first + (uint32_t)row);
              t = place((uint32_t)first + (uint32_t)k);
            }
            const bool moves = f.x >= 0 && t.x >= 0;
            const unsigned all = __ballot_sync(0xffffffffu, moves);
            if (moves) {
              const int at = n + __popc(all & ((1u << threadIdx.x) - 1u));
              from[at] = f;
              to[at] = t;
            }
            n += __popc(all);
          }
          if (threadIdx.x == 0) count = n;
        }
        __syncthreads();
        found = block_table;
      }
      // the arrays of one kind that follow: their columns side by side
      const RowArray a = table[i];
      int same = 1;
      while (i + same < a1 && table[i + same].block_table == found && table[i + same].heads == a.heads && table[i + same].row == a.row) ++same;
      long long low = 0;
      for (int k = 0; k < same; ++k) low |= table[i + k].address;
      const int wide = ((low | a.row) & 15) == 0 ? 16 : ((low | a.row) & 3) == 0 ? 4 : 1, columns = (int)(a.heads * (a.row / wide)), n = count;
      for (int c = threadIdx.x; c < same * columns; c += KEEP_THREADS) {
        RowArray b = a;
        b.address = table[i + c / columns].address;
        if (wide == 16) move_rows<uint4>(b, from, to, n, page_tokens, c % columns);
        else if (wide == 4) move_rows<uint32_t>(b, from, to, n, page_tokens, c % columns);
        else move_rows<uint8_t>(b, from, to, n, page_tokens, c % columns);
      }
      i += same;
    }
    __syncthreads();
  }
}

// ---- the choice over beams and vocabulary -----------------------------------------------------------------------------------
// score(b, k, v) = scores[b, k] + x_v - log sum_u exp(x_u) over the logits x of beam k; the best `choices` of a prompt's beams and
// tokens, best first, of equal ones the one with the lower k V + v first.  A logit that is not finite counts as -inf, and so does
// every continuation of a beam whose own score is not finite.
//
// One pass over the logits: a CTA takes a part of a row through registers, a tile of 4,096 at a time with the next one on its way, and
// keeps a sum of exponentials a thread against a reference of its own (a tile's sixteen in float32, all beyond that in 64 bits) and the
// largest of each thread's sixteen.  When the part is through, a bar is found that at least `choices` of those reach, and only the few
// sixteens that reach it are read again for the tokens that can be among the part's best.  (Looking for them on the way took a barrier
// a tile and, with some lane over the bar in most tiles, one and a half times the instructions: 42 us for 28.)  A CTA a prompt then joins
// the parts' sums, scores the parts' tokens in 64 bits and ranks them: rounded to float32, scores of some -10 lie 1e-6 apart, and
// neighbours among a million would be equal often enough.  What is left is the error of the exponentials and of their sums by sixteens:
// at most 2^-21 + 2^-24 of a row's sum (5e-7), mostly some 1e-8.
//
// Time: some 15 us of dependent steps (start, bar, read again, sums, rank) and the stream: 4, 8 and 16 prompts of 8 beams over 151,936
// tokens take 20.5, 23.4 and 30.9 us (39 MB more: 7.5 us, 5.2 TB/s), a prompt of 4 beams 12.4, of 128 with 256 choices 159.  (Exponentials
// of differences taken in 32 bits, up to 1.8e-6 off: 28.3 for 16 prompts.  Blocks of 128 threads, eight a SM, or tiles asked into L2 ahead
// were slower.)
constexpr int BT = 256;               // threads
constexpr int BEAM_MOST = 256;        // choices
constexpr int BC = 2048;              // candidates that are ranked side by side; more than that only among equal logits
constexpr int SLOTS = 16;             // maxima that a thread keeps

struct RowPart {
  double sum;                         // of exp(x - top)
  float top, pad;                     // (top: the part's reference, -inf if it holds nothing finite)
};

// A part that the kernel before has left (past L1, see above).
__device__ __forceinline__ RowPart part_of(const RowPart* at) {
  const float4 x = __ldcg(reinterpret_cast<const float4*>(at));
  return {__hiloint2double(__float_as_int(x.y), __float_as_int(x.x)), x.z, x.w};
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// Numbers as integers of the same order, and back.
__device__ __forceinline__ uint32_t in_order(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }

__device__ __forceinline__ uint64_t in_order(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double from_order(uint64_t u) { return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u)); }

// Raises a bar that at least `choices` numbers reach, by halves between it and the largest, until no more than `enough` do (or it is
// found as far as the steps go); reach(to, step) counts how many reach `to`.
template <int STEPS, typename F, typename R>
__device__ __forceinline__ int raise_bar(F& bar, F top, int choices, int enough, R&& reach) {
  int found = reach(bar, 0);
  auto lo = in_order(bar), hi = in_order(top);
  for (int step = 1; step <= STEPS && found > enough && hi - lo > 1; ++step) {
    const auto middle = lo + (hi - lo) / 2;
    const int n = reach(from_order(middle), step);
    if (n >= choices) {
      lo = middle;
      found = n;
    } else {
      hi = middle;
    }
  }
  bar = from_order(lo);
  return found;
}

// (value, index) pairs: more, or as much and further ahead
template <typename F>
__device__ __forceinline__ bool ahead(F x, int i, F y, int j) {
  return x > y || (x == y && i < j);
}

// `mine`: a thread's largest value.  Among the values of the threads, at least `groups` reach `bar`: each of that many groups of
// neighbouring threads holds one.  `top`: the largest of all.
template <int T, typename F>
__device__ __forceinline__ void find_bar(F mine, int groups, F* s_group, F& bar, F& top) {
  const int size = min(T / groups, 32);       // (a warp is at most one group: more of them than asked for)
  for (int o = 1; o < size; o <<= 1) {
    const F other = __shfl_xor_sync(0xffffffffu, mine, o);
    mine = other > mine ? other : mine;
  }
  groups = T / size;
  if (threadIdx.x % size == 0) s_group[threadIdx.x / size] = mine;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  F lo = s_group[lane % groups], hi = lo;
  for (int i = lane; i < groups; i += 32) {
    const F x = s_group[i];
    lo = x < lo ? x : lo;
    hi = x > hi ? x : hi;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const F a = __shfl_xor_sync(0xffffffffu, lo, o), b = __shfl_xor_sync(0xffffffffu, hi, o);
    lo = a < lo ? a : lo;
    hi = b > hi ? b : hi;
  }
  bar = lo;
  top = hi;
}

// The best of all threads' (value, index) that come behind (past, past_index); index -1 if there is none.
template <int T, typename F>
__device__ __forceinline__ void best_of_block(F& x, int& i, F* s_x, int* s_i) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const F y = __shfl_xor_sync(0xffffffffu, x, o);
    const int j = __shfl_xor_sync(0xffffffffu, i, o);
    if (j >= 0 && (i < 0 || ahead(y, j, x, i))) {
      x = y;
      i = j;
    }
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    s_x[threadIdx.x >> 5] = x;
    s_i[threadIdx.x >> 5] = i;
  }
  __syncthreads();
  for (int w = 0; w < T / 32; ++w) {
    const F y = s_x[w];
    const int j = s_i[w];
    if (j >= 0 && (i < 0 || ahead(y, j, x, i))) {
      x = y;
      i = j;
    }
  }
}

constexpr int BE = 16;                // values of a tile a thread

// Two float32 numbers an instruction.
__device__ __forceinline__ uint64_t two(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// A thread's reference: what the exponentials of its sum are held against.  The difference of a logit and the reference is not taken in 32
// bits, since a difference of d is off by up to d 2^-25, which all terms of a sum may share.  Both are split into a whole number and at
// most a half, x log2(e) = n + f, by a product that is not rounded before n comes off; the exponential is 2^(f - the reference's f) with
// the whole numbers' difference added to the bits of its exponent.  So a term is off by the approximation (2 units in the last place) and
// 2^-23, whatever x is, and the reference's own term is 1.  `base` is 0 but for logits of 2^20 and more, which lie so far apart that their
// differences up to 107 are exact.
struct Reference {
  float base, magic, rest, low;         // magic: 1.5 2^23 - n; rest: f; low: what smaller logits (and NaN) count as, e^-80 of the reference
};
constexpr float LOG2E_HIGH = 1.4426950216293335f, LOG2E_LOW = 1.9259629e-8f, WHOLE = 12582912.0f;      // WHOLE: 1.5 2^23
__device__ __forceinline__ Reference reference_of(float ref) {
  const float base = fabsf(ref) < 1048576.0f ? 0.f : ref, x = ref - base, n = fmaf(x, LOG2E_HIGH, WHOLE) - WHOLE;
  return {base, WHOLE - n, fmaf(x, LOG2E_LOW, fmaf(x, LOG2E_HIGH, -n)), x - 80.0f};
}

// The sum of e^(v - reference) over sixteen logits up to 20 above it, added in four steps.  (In two chains of eight, equal terms share the
// chains' roundings.)
__device__ __forceinline__ float tile_sum(float* v, const Reference& of) {
  if (of.base != 0.f)
#pragma unroll
    for (int e = 0; e < BE; ++e) v[e] -= of.base;
  const uint64_t high = two(LOG2E_HIGH, LOG2E_HIGH), less_high = two(-LOG2E_HIGH, -LOG2E_HIGH), less_low = two(-LOG2E_LOW, -LOG2E_LOW),
                 magic = two(of.magic, of.magic), back = two(-of.magic, -of.magic), rest = two(of.rest, of.rest);
  uint64_t sum[BE / 2];
#pragma unroll
  for (int e = 0; e < BE; e += 2) {
    const uint64_t x = two(fmaxf(v[e], of.low), fmaxf(v[e + 1], of.low)), n = fma_two(x, high, magic);      // n: 1.5 2^23 + x's - the reference's
    const uint64_t less_f = add_two(fma_two(x, less_low, fma_two(x, less_high, add_two(n, back))), rest);
    float y0, y1;
    asm("{\n\t.reg .f32 a, b;\n\tmov.b64 {a, b}, %2;\n\tneg.f32 a, a;\n\tneg.f32 b, b;\n\tex2.approx.ftz.f32 %0, a;\n\tex2.approx.ftz.f32 %1, b;\n\t}"
        : "=f"(y0), "=f"(y1) : "l"(less_f));
    sum[e / 2] = two(__uint_as_float(__float_as_uint(y0) + ((uint32_t)n << 23)), __uint_as_float(__float_as_uint(y1) + ((uint32_t)(n >> 32) << 23)));
  }
#pragma unroll
  for (int step = 1; step < BE / 2; step *= 2)
#pragma unroll
    for (int e = 0; e < BE / 2; e += 2 * step) sum[e] = add_two(sum[e], sum[e + step]);
  float a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(sum[0]));
  return a + b;
}

constexpr float LOWEST = -3.402823466e38f;
constexpr int BAR_STEPS = 12;

// The parts of a row are of `length` values (the last of what is left).
__global__ void __launch_bounds__(BT, 4)
beam_rows_kernel(const float* __restrict__ logits, const float* __restrict__ scores, int V, int choices, int groups, int parts, int length,
                 RowPart* __restrict__ part, float* __restrict__ part_x, int* __restrict__ part_i) {
  __shared__ float s_group[BT], s_high[SLOTS][BT], s_x[BC];
  __shared__ int s_i[BC], s_n, s_found[BAR_STEPS + 1];
  __shared__ uint16_t s_pair[BC];
  __shared__ double s_sum[BT / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, row = blockIdx.x / parts, p = blockIdx.x % parts;
  const size_t at = (size_t)row * parts + p;
  if (!finite(scores[row])) {
    if (tid == 0) part[at] = RowPart{0.0, -CUDART_INF_F, 0.f};
    for (int c = tid; c < choices; c += BT) part_x[at * choices + c] = -CUDART_INF_F;
    return;
  }
  const float* x = logits + (size_t)row * V;
  const int begin = p * length, end = min(V, begin + length);
  // A thread's values of a tile: four times four neighbours, or, where a part is short, single ones.  Which it has does not hang on where
  // the row lies (equal rows have equal sums, to the bit); how they are read does.
  const bool fours = length >= 4 * BT, wide = fours && (((uintptr_t)(x + begin)) & 15) == 0;
  auto index = [&](int t, int e, int of) { return begin + t * (BT * BE) + (fours ? (e / 4 * BT + of) * 4 + (e & 3) : e * BT + of); };
  auto load = [&](int t, float* v) {
    if (wide && begin + (t + 1) * (BT * BE) <= end) {
      const float* from = x + begin + t * (BT * BE) + 4 * tid;
#pragma unroll
      for (int e = 0; e < BE; e += 4) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(from + e * BT));
        v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < BE; ++e) v[e] = index(t, e, tid) < end ? __ldg(x + index(t, e, tid)) : -CUDART_INF_F;
  };
  const int tiles = (end - begin + BT * BE - 1) / (BT * BE), per = (tiles + SLOTS - 1) / SLOTS;
  float slot_high = -CUDART_INF_F, mine = -CUDART_INF_F, ref = -CUDART_INF_F;
  Reference reference = {0.f, 0.f, 0.f, 0.f};
  double sum = 0.0;
  int slot = 0, in_slot = 0;
  auto tile = [&](int t, float* v, float* next) {
    if (t + 1 < tiles) load(t + 1, next);
    float high = -CUDART_INF_F;        // (a maximum passes NaN by)
#pragma unroll
    for (int e = 0; e < BE; ++e) high = fmaxf(high, v[e]);
    if (high == CUDART_INF_F) {
      high = -CUDART_INF_F;
#pragma unroll
      for (int e = 0; e < BE; ++e) {
        v[e] = finite(v[e]) ? v[e] : -CUDART_INF_F;
        high = fmaxf(high, v[e]);
      }
    }
    slot_high = fmaxf(slot_high, high);
    if (++in_slot == per || t + 1 == tiles) {
      s_high[slot++][tid] = slot_high;
      mine = fmaxf(mine, slot_high);
      slot_high = -CUDART_INF_F;
      in_slot = 0;
    }
    if (high > ref + 20.0f) {          // also true for the first finite value
      sum *= ref == -CUDART_INF_F ? 0.0 : exp((double)ref - (double)high);
      ref = high;
      reference = reference_of(ref);
    }
    if (ref > -CUDART_INF_F) sum += (double)tile_sum(v, reference);
  };
  float one[BE], other[BE];
  load(0, one);
  for (int t = 0; t < tiles; t += 2) {
    tile(t, one, other);
    if (t + 1 < tiles) tile(t + 1, other, one);
  }
  const int slots = slot;
  if (tid <= BAR_STEPS) s_found[tid] = 0;
  if (tid == 0) s_n = 0;
  float bar, top;
  find_bar<BT>(mine, groups, s_group, bar, top);
  bar = fmaxf(bar, LOWEST);
  double all = ref == top || ref == -CUDART_INF_F ? sum : sum * exp((double)ref - (double)top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  if ((tid & 31) == 0) s_sum[tid >> 5] = all;
  // how many slots reach a bar
  auto reach = [&](float to, int step) {
    int n = 0;
    if (mine >= to)
      for (int k = 0; k < slots; ++k) n += s_high[k][tid] >= to ? 1 : 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((tid & 31) == 0 && n > 0) atomicAdd(&s_found[step], n);
    __syncthreads();
    return s_found[step];
  };
  const int found = raise_bar<BAR_STEPS>(bar, top, choices, choices + choices / 4 + 16, reach);
  if (tid == 0) {
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < BT / 32; ++w) total += s_sum[w];
    part[at] = RowPart{total, top, 0.f};
  }
  int n = BC + 1;
  if (found <= BC) {
    // the slots that reach the bar, and their values that do: four threads a slot
    if (mine >= bar)
      for (int k = 0; k < slots; ++k)
        if (s_high[k][tid] >= bar) s_pair[atomicAdd(&s_n, 1)] = (uint16_t)(k * BT + tid);
    __syncthreads();
    if (tid == 0) s_n = 0;
    __syncthreads();
    for (int c = tid / 4; c < found; c += BT / 4) {
      const int of = s_pair[c] % BT, t0 = s_pair[c] / BT * per;
      for (int t = t0; t < min(tiles, t0 + per); ++t) {
        float y[4];
        int i[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          i[e] = index(t, tid % 4 * 4 + e, of);
          y[e] = i[e] < end ? __ldg(x + i[e]) : -CUDART_INF_F;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (y[e] >= bar && finite(y[e])) {
            const int to = atomicAdd(&s_n, 1);
            if (to < BC) s_x[to] = y[e], s_i[to] = i[e];
          }
      }
    }
    __syncthreads();
    n = s_n;
  }
  if (n <= BC) {
    for (int c = n + tid; c < choices; c += BT) part_x[at * choices + c] = -CUDART_INF_F;
    for (int c = tid; c < n; c += BT) {
      const float mx = s_x[c];
      const int mi = s_i[c];
      int rank = 0;
#pragma unroll 4
      for (int o = 0; o < n; ++o) rank += ahead(s_x[o], s_i[o], mx, mi) ? 1 : 0;
      if (rank < choices) {
        part_x[at * choices + rank] = mx;
        part_i[at * choices + rank] = mi;
      }
    }
    return;
  }
  // very many equal logits: one after the other, from the row itself
  float past = CUDART_INF_F;
  int past_i = -1;
  for (int k = 0; k < choices; ++k) {
    float bx = -CUDART_INF_F;
    int bi = -1;
    for (int i = begin + tid; i < end; i += BT) {
      const float y = x[i];
      if (finite(y) && y >= bar && ahead(past, past_i, y, i) && (bi < 0 || ahead(y, i, bx, bi))) {
        bx = y;
        bi = i;
      }
    }
    best_of_block<BT>(bx, bi, s_x, s_i);
    if (tid == 0) {
      part_x[at * choices + k] = bx;
      part_i[at * choices + k] = bi;
    }
    past = bx;
    past_i = bi;
  }
}

constexpr int CT = 512, CDEEP = 8, CHOICE_STEPS = 24;    // threads of the choice; candidates that a thread has on their way at once

__global__ void __launch_bounds__(CT)
beam_choice_kernel(const float* __restrict__ scores, int K, int V, int choices, int groups, int parts, int ranks, uint32_t ranks_inverse,
                   uint32_t beam_inverse, const RowPart* part,
                   const float* part_x, const int* part_i, float* __restrict__ out_scores,
                   int* __restrict__ out_beams, int* __restrict__ out_tokens) {
  __shared__ double s_group[CT], s_x[BC], s_lift[BEAM_MOST];      // s_lift: a beam's score less the logarithm of its sum
  __shared__ int s_i[BC], s_n, s_taken[BEAM_MOST], s_found[CHOICE_STEPS + 1];
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t row0 = (size_t)b * K;
  // candidate c: the token of rank c % choices of part c / choices of the prompt's rows (-inf where a part has fewer); its flat index
  // is beam * V + token.  The threads hold as many of them as they have registers for, all or the first `ranks` of each part; those are
  // on their way while the rows' sums are joined.
  const int of_beam = parts * choices, all = K * of_beam, held = K * parts * ranks;
  const float* xs = part_x + row0 * of_beam;
  const int* is = part_i + row0 * of_beam;
  const bool kept = ranks == choices;
  float keep_x[CDEEP];
  int keep_i[CDEEP];
#pragma unroll
  for (int j = 0; j < CDEEP; ++j) {
    const int m = threadIdx.x + j * CT, p = ranks == 1 ? m : (int)__umulhi((uint32_t)m, ranks_inverse), c = p * choices + m - p * ranks;
    keep_x[j] = m < held ? __ldcg(xs + c) : -CUDART_INF_F;
    keep_i[j] = m < held ? __ldcg(is + c) : 0;
  }
  for (int k = warp; k < K; k += CT / 32) {
    const RowPart* of = part + (row0 + k) * parts;
    RowPart first = {0.0, -CUDART_INF_F, 0.f};
    if (lane < parts) first = part_of(of + lane);
    float top = first.top;
#pragma unroll 4
    for (int p = lane + 32; p < parts; p += 32) top = fmaxf(top, part_of(of + p).top);
    top = warp_max(top);
    double sum = first.sum > 0.0 ? first.sum * exp((double)first.top - (double)top) : 0.0;
#pragma unroll 4
    for (int p = lane + 32; p < parts; p += 32) {
      const RowPart r = part_of(of + p);
      if (r.sum > 0.0) sum += r.sum * exp((double)r.top - (double)top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_lift[k] = top == -CUDART_INF_F ? -CUDART_INF : (double)scores[row0 + k] - ((double)top + log(sum));
  }
  if (threadIdx.x == 0) s_n = 0;
  if (threadIdx.x <= CHOICE_STEPS) s_found[threadIdx.x] = 0;
  __syncthreads();
  double mine = -CUDART_INF, keep[CDEEP];
#pragma unroll
  for (int j = 0; j < CDEEP; ++j) {
    const uint32_t m = threadIdx.x + j * CT;
    const int k = ranks * parts == 1 ? m : __umulhi(m, beam_inverse);
    keep[j] = keep_x[j] > -CUDART_INF_F ? (double)keep_x[j] + s_lift[k] : -CUDART_INF;
    keep_i[j] += k * V;
    mine = keep[j] > mine ? keep[j] : mine;
  }
  auto each_kept = [&](auto&& take) {
#pragma unroll
    for (int j = 0; j < CDEEP; ++j)
      if (keep[j] > -CUDART_INF) take(keep[j], keep_i[j]);
  };
  auto each = [&](auto&& take) {
    if (kept) return each_kept(take);
    for (int c0 = threadIdx.x; c0 < all; c0 += CT * CDEEP) {
      float x[CDEEP];
#pragma unroll
      for (int j = 0; j < CDEEP; ++j) x[j] = c0 + j * CT < all ? __ldcg(xs + c0 + j * CT) : -CUDART_INF_F;
#pragma unroll
      for (int j = 0; j < CDEEP; ++j)
        if (x[j] > -CUDART_INF_F) {
          const int c = c0 + j * CT, k = c / of_beam;
          take((double)x[j] + s_lift[k], k * V + __ldcg(is + c));
        }
    }
  };
  double bar, top;
  find_bar<CT>(mine, groups, s_group, bar, top);
  auto reach = [&](auto&& each, double to, int step) {
    int n = 0;
    each([&](double x, int) { n += x >= to ? 1 : 0; });
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0 && n > 0) atomicAdd(&s_found[step], n);
    __syncthreads();
    return s_found[step];
  };
  raise_bar<CHOICE_STEPS>(bar, top, choices, choices + choices / 4 + 16, [&](double to, int step) { return reach(each_kept, to, step); });
  auto gather = [&] {
    each([&](double x, int i) {
      if (x < bar) return;
      const int at = atomicAdd(&s_n, 1);
      if (at < BC) {
        s_x[at] = x;
        s_i[at] = i;
      }
    });
    __syncthreads();
    return s_n;
  };
  int n = gather();
  if (n > BC && !kept) {               // a part's further ranks are before the others' first ones: the bar among all
    __syncthreads();
    if (threadIdx.x == 0) s_n = 0;
    if (threadIdx.x <= CHOICE_STEPS) s_found[threadIdx.x] = 0;
    __syncthreads();
    raise_bar<CHOICE_STEPS>(bar, top, choices, BC / 2, [&](double to, int step) { return reach(each, to, step); });
    n = gather();
  }
  auto give = [&](int rank, double x, int i) {
    out_scores[(size_t)b * choices + rank] = (float)x;
    out_beams[(size_t)b * choices + rank] = i / V;
    out_tokens[(size_t)b * choices + rank] = i % V;
    s_taken[rank] = i;
  };
  if (n <= BC) {
    for (int c = threadIdx.x; c < n; c += CT) {
      const double mx = s_x[c];
      const int mi = s_i[c];
      int rank = 0;
      for (int o = 0; o < n; ++o) rank += ahead(s_x[o], s_i[o], mx, mi) ? 1 : 0;
      if (rank < choices) give(rank, mx, mi);
    }
  } else {
    double past = CUDART_INF;
    int past_i = -1;
    for (int k = 0; k < choices; ++k) {
      double bx = -CUDART_INF;
      int bi = -1;
      each([&](double x, int i) {
        if (ahead(past, past_i, x, i) && (bi < 0 || ahead(x, i, bx, bi))) {
          bx = x;
          bi = i;
        }
      });
      best_of_block<CT>(bx, bi, s_x, s_i);
      if (threadIdx.x == 0) give(k, bx, bi);
      past = bx;
      past_i = bi;
    }
  }
  __syncthreads();
  // fewer continuations than choices: those that are left all have the score -inf, the first of them in order
  if (threadIdx.x == 0 && n < choices) {
    int i = 0;
    for (int rank = n; rank < choices; ++i) {
      bool taken = false;
      for (int o = 0; o < n; ++o) taken = taken || s_taken[o] == i;
      if (!taken) {
        out_scores[(size_t)b * choices + rank] = -CUDART_INF_F;
        out_beams[(size_t)b * choices + rank] = i / V;
        out_tokens[(size_t)b * choices + rank] = i % V;
        ++rank;
      }
    }
  }
}

int beam_groups(int choices) {
  int g = 8;
  while (g < choices) g <<= 1;
  return g;
}

// How many parts a row is cut into, a length of 4 values and more: one wave of CTAs (four a SM), and no less than half a tile a part, of
// rows of 16 tiles and more a tile: the stream is shorter with more parts and the choice behind it longer.  In half and in whole tiles, 4
// rows take 12.8 and 15.5 us at 32,000 logits, 12.4 and 15.4 at 50,304, 12.6 and 12.5 at 65,536, 14.1 and 12.7 at 100,352, 15.3 and 13.8 at
// 151,936; 8 rows 12.8 and 15.7, 13.4 and 15.3, 13.5 and 12.6, 15.1 and 13.9, 16.9 and 14.8.  (The other way round of what was measured: 1
// row of 32,000 14.5 and 12.0, 2 of 128,256 and of 151,936 12.9 and 15.0, 13.7 and 15.4.)
void beam_cut(int rows, int V, int* parts, int* length) {
  const int wave = 148 * 4, tile = BT * BE, least = V >= 16 * tile ? tile : tile / 2, most = (V - 1) / least + 1;
  int n = wave / rows;
  n = n < 1 ? 1 : n > most ? most : n;
  *length = ((V + n - 1) / n + 3) & ~3;
  *parts = (V + *length - 1) / *length;
}

}  // namespace

// table [arrays, 5] 64-bit = (address, blocks, pieces a block, bytes a piece, bytes a row); moves int32 [moves, 3] = (from, to,
// rows): in every array, of each piece of block `from` the first rows * bytes a row (at most the piece) go to block `to`.  No block
// is written twice in a call, and none is both read and written.  most_bytes: the most that a block of any array has.
HK_API int hk_copy_blocks(const long long* table, int arrays, const int* moves, int n_moves, long long most_bytes, void* stream) {
  if (arrays <= 0 || n_moves <= 0 || most_bytes <= 0) return 0;
  if (arrays > 65535 || n_moves > 65535) return HK_ERR_UNSUPPORTED;
  const long long part = 16LL * COPY_THREADS * COPY_DEEP, blocks = (most_bytes + part - 1) / part;
  return hk_launch_pdl(copy_blocks_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096), (unsigned)n_moves, (unsigned)arrays), dim3(COPY_THREADS), 0,
                   (cudaStream_t)stream, reinterpret_cast<const BlockArray*>(table), moves);
}

// table [arrays, 4] 64-bit = (address of [num_pages, heads, page_tokens, bytes a row], heads, bytes a row, address of an int32 block
// table [table_rows, table_stride]); paths int32 [requests, 2 + width] = (slot, first row of the tree, kept rows of the tree in
// ascending order, -1 behind the last): kept row i moves to the tree's row i.  No slot appears twice.  heads, row_bytes: the most of
// any array.
HK_API int hk_compact_rows(const long long* table, int arrays, const int* paths, int requests, int width, int table_rows, int table_stride,
                           int page_tokens, int heads, int row_bytes, long long num_pages, void* stream) {
  if (arrays <= 0 || requests <= 0 || width <= 0) return 0;
  if (arrays > 65535 || table_rows < 1 || table_stride < 1 || page_tokens < 1 || heads < 1 || row_bytes < 1 || num_pages < 1)
    return HK_ERR_UNSUPPORTED;
  if ((long long)heads * row_bytes > 0x7fffffffLL / 64) return HK_ERR_UNSUPPORTED;
  // one wave of blocks (eight a SM) where that is up to 8 arrays a block
  int per_block = (int)(((long long)arrays * requests + 148 * 8 - 1) / (148 * 8));
  per_block = per_block < 1 ? 1 : per_block > 8 ? 8 : per_block;
  return hk_launch_pdl(compact_rows_kernel, dim3((unsigned)requests, (unsigned)((arrays + per_block - 1) / per_block)), dim3(KEEP_THREADS), 0,
                   (cudaStream_t)stream, reinterpret_cast<const RowArray*>(table), arrays, per_block, paths, width, table_rows, table_stride, page_tokens,
                   num_pages);
}

// logits float32 [prompts * beams, V], scores float32 [prompts * beams]; out_* [prompts, choices]; scratch (16-byte aligned) of
// max(592, prompts * beams) * (16 + 8 * choices) bytes: rows have no more parts together than that.
HK_API int hk_beam_select(const float* logits, const float* scores, int prompts, int beams, int V, int choices, float* out_scores,
                          int* out_beams, int* out_tokens, void* scratch, long long scratch_bytes, void* stream) {
  if (prompts <= 0) return 0;
  if (beams < 1 || beams > BEAM_MOST || V < 1 || V > (1 << 30) || choices < 1 || choices > BEAM_MOST || (long long)beams * V > 0x7fffffffLL ||
      choices > (long long)beams * V || (long long)prompts * beams > 0x7fffffffLL || (((uintptr_t)scratch) & 15) != 0)
    return HK_ERR_UNSUPPORTED;
  const int rows = prompts * beams, groups = beam_groups(choices);
  int parts, length;
  beam_cut(rows, V, &parts, &length);
  if ((long long)rows * parts > 0x7fffffffLL || (long long)beams * parts * choices > 0x7fffffffLL) return HK_ERR_UNSUPPORTED;
  if (scratch_bytes < (long long)rows * parts * ((long long)sizeof(RowPart) + 8LL * choices)) return HK_ERR_UNSUPPORTED;
  RowPart* part = static_cast<RowPart*>(scratch);
  float* part_x = reinterpret_cast<float*>(part + (size_t)rows * parts);
  int* part_i = reinterpret_cast<int*>(part_x + (size_t)rows * parts * choices);
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid((unsigned)(rows * parts)), block(BT);
  const int e = hk_launch_pdl(beam_rows_kernel, grid, block, 0, s, logits, scores, V, choices, groups, parts, length, part, part_x, part_i);
  if (e) return e;
  // (m / d is the upper half of m times 2^32 / d, rounded up, while m d < 2^32)
  const int most = CT * CDEEP / (beams * parts), ranks = choices < most ? choices : most;
  auto inverse = [](long long d) { return (uint32_t)(d == 1 ? 0 : ((1ll << 32) + d - 1) / d); };
  return hk_launch_pdl(beam_choice_kernel, dim3((unsigned)prompts), dim3(CT), 0, s, scores, beams, V, choices, groups, parts, ranks, inverse(ranks),
                       inverse((long long)ranks * parts), part, part_x, part_i,
                       out_scores, out_beams, out_tokens);
}
