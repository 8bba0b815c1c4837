// Several continuations of one request: blocks of a cache copied in all layers at once (pages of forked requests, states that
// surviving beams pass on), the accepted rows of a drafted tree moved up side by side, and the choice over beams and vocabulary.
//
// What the device arrays say is checked where it is read: a copy or a row whose page, slot or place lies outside the arrays is left
// out.
#include <math_constants.h>

#include "common.cuh"

namespace {

// ---- blocks of a cache --------------------------------------------------------------------------------------------------
// A block is `pieces` runs of `piece` bytes; of each run the first min(rows * row, piece) bytes are copied.
struct BlockArray {
  long long address, blocks, pieces, piece, row;
};

constexpr int COPY_THREADS = 256, COPY_DEEP = 8;      // threads; vectors that a thread has on their way at once

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
        v[k] = *reinterpret_cast<const V*>(from + at[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < COPY_DEEP; ++k)
      if (at[k] >= 0) *reinterpret_cast<V*>(to + at[k]) = v[k];
  }
}

__global__ void __launch_bounds__(COPY_THREADS)
copy_blocks_kernel(const BlockArray* __restrict__ table, const int* __restrict__ moves) {
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

// A thread takes a column (array, request, head, 16 bytes of a row) and moves its rows in order: a path climbs, so a row that is
// written (path[i] -> i, i <= path[i]) is none that a later step of the path reads.
template <typename V>
__device__ __forceinline__ void move_rows(const RowArray& a, const long long* from, const long long* to, int n, long long head_bytes) {
  const int per = (int)(a.row / (long long)sizeof(V));
  for (long long c = (long long)blockIdx.z * KEEP_THREADS + threadIdx.x; c < a.heads * per; c += (long long)gridDim.z * KEEP_THREADS) {
    uint8_t* base = reinterpret_cast<uint8_t*>(a.address) + (c / per) * head_bytes + (c % per) * (long long)sizeof(V);
    for (int i0 = 0; i0 < n; i0 += KEEP_DEEP) {
      V v[KEEP_DEEP];
#pragma unroll
      for (int k = 0; k < KEEP_DEEP; ++k)
        if (i0 + k < n) v[k] = *reinterpret_cast<const V*>(base + from[i0 + k]);
#pragma unroll
      for (int k = 0; k < KEEP_DEEP; ++k)
        if (i0 + k < n) *reinterpret_cast<V*>(base + to[i0 + k]) = v[k];
    }
  }
}

__global__ void __launch_bounds__(KEEP_THREADS)
compact_rows_kernel(const RowArray* __restrict__ table, const int* __restrict__ paths, int width, int table_rows, int table_stride,
                    int page_tokens, long long num_pages) {
  __shared__ long long from[KEEP_PATH], to[KEEP_PATH];
  __shared__ int count;
  const RowArray a = table[blockIdx.y];
  const int* path = paths + (size_t)blockIdx.x * (width + 2);
  const int slot = path[0], first = path[1];
  if (slot < 0 || slot >= table_rows || first < 0) return;
  const long long head_bytes = page_tokens * a.row, page_bytes = a.heads * head_bytes;
  const int* pages = a.block_table + (size_t)slot * table_stride;
  auto place = [&](long long row) -> long long {
    if (row >= (long long)table_stride * page_tokens) return -1;
    const int page = pages[row / page_tokens];
    return page < 0 || page >= num_pages ? -1 : page * page_bytes + (row % page_tokens) * a.row;
  };
  for (int done = 0; done < width; done += KEEP_PATH) {
    if (threadIdx.x < 32) {            // the rows that move, in order
      int n = 0;
      for (int i0 = done; i0 < min(width, done + KEEP_PATH); i0 += 32) {
        const int i = i0 + (int)threadIdx.x, row = i < width ? path[2 + i] : -1;
        long long f = -1, t = -1;
        if (row > i) {
          f = place((long long)first + row);
          t = place((long long)first + i);
        }
        const bool moves = f >= 0 && t >= 0;
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
    const int n = count;
    if (((a.address | a.row) & 15) == 0) move_rows<uint4>(a, from, to, n, head_bytes);
    else if (((a.address | a.row) & 3) == 0) move_rows<uint32_t>(a, from, to, n, head_bytes);
    else move_rows<uint8_t>(a, from, to, n, head_bytes);
    __syncthreads();
  }
}

// ---- the choice over beams and vocabulary -----------------------------------------------------------------------------------
// score(b, k, v) = scores[b, k] + x_v - log sum_u exp(x_u) over the logits x of beam k; the best `choices` of a prompt's beams and
// tokens, best first, of equal ones the one with the lower k V + v first.  A logit that is not finite counts as -inf, and so does
// every continuation of a beam whose own score is not finite.
//
// One pass over the logits: a CTA takes a part of a row into registers, sums its exponentials against its own maximum (32 terms a
// thread in float32, threads and parts in 64 bits) and leaves its best `choices` tokens in order; then a CTA a prompt joins the
// parts' sums, scores the parts' tokens in 64 bits and ranks them.  A 64-bit order: two beams' continuations lie as little as 1e-7
// apart often enough among a million, and which of them comes first must not hang on how a sum was rounded.
constexpr int BT = 256;               // threads
constexpr int BEAM_MOST = 256;        // choices
constexpr int BC = 1024;              // candidates that are ranked side by side; more than that only among equal logits

struct RowPart {
  double sum;                         // of exp(x - top)
  float top;
  int n;                              // tokens left
};

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// (value, index) pairs: more, or as much and further ahead
template <typename F>
__device__ __forceinline__ bool ahead(F x, int i, F y, int j) {
  return x > y || (x == y && i < j);
}

// `mine`: a thread's largest value.  Among the values of the threads, at least `groups` reach `bar`: each of that many groups of
// neighbouring threads holds one.  `top`: the largest of all.
template <typename F>
__device__ __forceinline__ void find_bar(F mine, int groups, F* s_group, F& bar, F& top) {
  const int size = BT / groups;       // 1 to 32 threads
  for (int o = 1; o < size; o <<= 1) {
    const F other = __shfl_xor_sync(0xffffffffu, mine, o);
    mine = other > mine ? other : mine;
  }
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
template <typename F>
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
  for (int w = 0; w < BT / 32; ++w) {
    const F y = s_x[w];
    const int j = s_i[w];
    if (j >= 0 && (i < 0 || ahead(y, j, x, i))) {
      x = y;
      i = j;
    }
  }
}

// E: values a thread
template <int E>
__global__ void __launch_bounds__(BT)
beam_rows_kernel(const float* __restrict__ logits, const float* __restrict__ scores, int V, int choices, int groups, int parts,
                 RowPart* __restrict__ part, float* __restrict__ part_x, int* __restrict__ part_i) {
  __shared__ float s_group[BT], s_x[BC];
  __shared__ int s_i[BC], s_n;
  __shared__ double s_sum[BT / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x / parts, p = blockIdx.x % parts;
  const size_t at = (size_t)row * parts + p;
  if (!finite(scores[row])) {
    if (threadIdx.x == 0) part[at] = RowPart{0.0, -CUDART_INF_F, 0};
    return;
  }
  const float* x = logits + (size_t)row * V;
  const int base = p * (BT * E);
  float v[E];
  const bool wide = (((uintptr_t)x) & 15) == 0;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const int i = base + (e / 4 * BT + (int)threadIdx.x) * 4;
    if (wide && i + 3 < V) {
      const float4 f = __ldcs(reinterpret_cast<const float4*>(x + i));
      v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[e + c] = i + c < V ? __ldcs(x + i + c) : -CUDART_INF_F;
    }
  }
  float mine = -CUDART_INF_F;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (!finite(v[e])) v[e] = -CUDART_INF_F;
    mine = fmaxf(mine, v[e]);
  }
  if (threadIdx.x == 0) s_n = 0;
  float bar, top;
  find_bar(mine, groups, s_group, bar, top);
  const float safe = top == -CUDART_INF_F ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) sum += expf(v[e] - safe);
  double all = sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = all;
  if (mine >= bar && mine > -CUDART_INF_F) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (v[e] >= bar && v[e] > -CUDART_INF_F) {
        const int c = atomicAdd(&s_n, 1);
        if (c < BC) {
          s_x[c] = v[e];
          s_i[c] = base + (e / 4 * BT + (int)threadIdx.x) * 4 + (e & 3);
        }
      }
  }
  __syncthreads();
  const int n = s_n;
  if (threadIdx.x == 0) {
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < BT / 32; ++w) t += s_sum[w];
    part[at] = RowPart{t, top, min(n, choices)};
  }
  if (n <= BC) {
    for (int c = threadIdx.x; c < n; c += BT) {
      const float mx = s_x[c];
      const int mi = s_i[c];
      int rank = 0;
      for (int o = 0; o < n; ++o) rank += ahead(s_x[o], s_i[o], mx, mi) ? 1 : 0;
      if (rank < choices) {
        part_x[at * choices + rank] = mx;
        part_i[at * choices + rank] = mi;
      }
    }
    return;
  }
  // very many equal logits: one after the other
  float past = CUDART_INF_F;
  int past_i = -1;
  for (int k = 0; k < choices; ++k) {
    float bx = -CUDART_INF_F;
    int bi = -1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = base + (e / 4 * BT + (int)threadIdx.x) * 4 + (e & 3);
      if (v[e] > -CUDART_INF_F && ahead(past, past_i, v[e], i) && (bi < 0 || ahead(v[e], i, bx, bi))) {
        bx = v[e];
        bi = i;
      }
    }
    best_of_block(bx, bi, s_x, s_i);
    if (threadIdx.x == 0) {
      part_x[at * choices + k] = bx;
      part_i[at * choices + k] = bi;
    }
    past = bx;
    past_i = bi;
  }
}

__global__ void __launch_bounds__(BT)
beam_choice_kernel(const float* __restrict__ scores, int K, int V, int choices, int groups, int parts, const RowPart* __restrict__ part,
                   const float* __restrict__ part_x, const int* __restrict__ part_i, float* __restrict__ out_scores,
                   int* __restrict__ out_beams, int* __restrict__ out_tokens) {
  __shared__ double s_group[BT], s_x[BC], s_lift[BEAM_MOST];      // s_lift: a beam's score less the logarithm of its sum
  __shared__ int s_i[BC], s_n, s_taken[BEAM_MOST];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t row0 = (size_t)b * K;
  for (int k = warp; k < K; k += BT / 32) {
    float top = -CUDART_INF_F;
    for (int p = lane; p < parts; p += 32) top = fmaxf(top, part[(row0 + k) * parts + p].top);
    top = warp_max(top);
    double sum = 0.0;
    for (int p = lane; p < parts; p += 32) {
      const RowPart r = part[(row0 + k) * parts + p];
      if (r.sum > 0.0) sum += r.sum * exp((double)r.top - (double)top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_lift[k] = top == -CUDART_INF_F ? -CUDART_INF : (double)scores[row0 + k] - ((double)top + log(sum));
  }
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  // candidate c: the token of rank c % choices of part c / choices of the prompt's rows; its flat index is beam * V + token
  const int all = K * parts * choices;
  auto candidate = [&](int c, double& x, int& i) -> bool {
    const int p = c / choices, k = p / parts;
    if (c % choices >= part[row0 * parts + p].n) return false;
    const size_t at = row0 * parts * choices + c;
    x = (double)part_x[at] + s_lift[k];
    i = k * V + part_i[at];
    return true;
  };
  double mine = -CUDART_INF;
  for (int c = threadIdx.x; c < all; c += BT) {
    double x;
    int i;
    if (candidate(c, x, i) && x > mine) mine = x;
  }
  double bar, top;
  find_bar(mine, groups, s_group, bar, top);
  for (int c = threadIdx.x; c < all; c += BT) {
    double x;
    int i;
    if (!candidate(c, x, i) || x < bar) continue;
    const int at = atomicAdd(&s_n, 1);
    if (at < BC) {
      s_x[at] = x;
      s_i[at] = i;
    }
  }
  __syncthreads();
  const int n = s_n;
  auto give = [&](int rank, double x, int i) {
    out_scores[(size_t)b * choices + rank] = (float)x;
    out_beams[(size_t)b * choices + rank] = i / V;
    out_tokens[(size_t)b * choices + rank] = i % V;
    s_taken[rank] = i;
  };
  if (n <= BC) {
    for (int c = threadIdx.x; c < n; c += BT) {
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
      for (int c = threadIdx.x; c < all; c += BT) {
        double x;
        int i;
        if (candidate(c, x, i) && ahead(past, past_i, x, i) && (bi < 0 || ahead(x, i, bx, bi))) {
          bx = x;
          bi = i;
        }
      }
      best_of_block(bx, bi, s_x, s_i);
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

int beam_values(int rows, int V) { return (long long)rows * ((V + BT * 32 - 1) / (BT * 32)) >= 2 * 148 ? 32 : 8; }

}  // namespace

// table [arrays, 5] 64-bit = (address, blocks, pieces a block, bytes a piece, bytes a row); moves int32 [moves, 3] = (from, to,
// rows): in every array, of each piece of block `from` the first rows * bytes a row (at most the piece) go to block `to`.  No block
// is written twice in a call, and none is both read and written.  most_bytes: the most that a block of any array has.
HK_API int hk_copy_blocks(const long long* table, int arrays, const int* moves, int n_moves, long long most_bytes, void* stream) {
  if (arrays <= 0 || n_moves <= 0 || most_bytes <= 0) return 0;
  if (arrays > 65535 || n_moves > 65535) return HK_ERR_UNSUPPORTED;
  const long long part = 16LL * COPY_THREADS * COPY_DEEP, blocks = (most_bytes + part - 1) / part;
  return hk_launch(copy_blocks_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096), (unsigned)n_moves, (unsigned)arrays), dim3(COPY_THREADS), 0,
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
  const long long columns = (long long)heads * ((row_bytes + 15) / 16), blocks = (columns + KEEP_THREADS - 1) / KEEP_THREADS;
  return hk_launch(compact_rows_kernel, dim3((unsigned)requests, (unsigned)arrays, (unsigned)(blocks < 64 ? blocks : 64)), dim3(KEEP_THREADS), 0,
                   (cudaStream_t)stream, reinterpret_cast<const RowArray*>(table), paths, width, table_rows, table_stride, page_tokens, num_pages);
}

static long long beam_parts(int rows, int V) {
  const int e = beam_values(rows, V);
  return (V + BT * e - 1) / (BT * e);
}

// Bytes of scratch (16-byte aligned) that hk_beam_select wants.
HK_API long long hk_beam_select_scratch(int rows, int V, int choices) {
  if (rows <= 0 || V <= 0 || choices <= 0) return 0;
  return (long long)rows * beam_parts(rows, V) * ((long long)sizeof(RowPart) + 8LL * choices);
}

// logits float32 [prompts * beams, V], scores float32 [prompts * beams]; out_* [prompts, choices].
HK_API int hk_beam_select(const float* logits, const float* scores, int prompts, int beams, int V, int choices, float* out_scores,
                          int* out_beams, int* out_tokens, void* scratch, void* stream) {
  if (prompts <= 0) return 0;
  if (beams < 1 || beams > BEAM_MOST || V < 1 || choices < 1 || choices > BEAM_MOST || (long long)beams * V > 0x7fffffffLL ||
      choices > (long long)beams * V || (long long)prompts * beams > 0x7fffffffLL || (((uintptr_t)scratch) & 15) != 0)
    return HK_ERR_UNSUPPORTED;
  const int rows = prompts * beams, parts = (int)beam_parts(rows, V), groups = beam_groups(choices);
  if ((long long)rows * parts > 0x7fffffffLL || (long long)beams * parts * choices > 0x7fffffffLL) return HK_ERR_UNSUPPORTED;
  RowPart* part = static_cast<RowPart*>(scratch);
  float* part_x = reinterpret_cast<float*>(part + (size_t)rows * parts);
  int* part_i = reinterpret_cast<int*>(part_x + (size_t)rows * parts * choices);
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid((unsigned)(rows * parts)), block(BT);
  const int e = beam_values(rows, V) == 32
                    ? hk_launch_pdl(beam_rows_kernel<32>, grid, block, 0, s, logits, scores, V, choices, groups, parts, part, part_x, part_i)
                    : hk_launch_pdl(beam_rows_kernel<8>, grid, block, 0, s, logits, scores, V, choices, groups, parts, part, part_x, part_i);
  if (e) return e;
  return hk_launch_pdl(beam_choice_kernel, dim3((unsigned)prompts), block, 0, s, scores, beams, V, choices, groups, parts, part, part_x, part_i,
                       out_scores, out_beams, out_tokens);
}
