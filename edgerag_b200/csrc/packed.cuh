// What the kernels of attention_packed.cu and attention_packed_tc.cu share: the description of a call, the rows a block owns, and which
// keys each of them sees.
//
// Rows.  The query heads that share a kv head are neighbours, so the rows of one kv head are (token, head in the group) pairs, row r being
// token r / G, head kvh * G + r % G (G = query heads per kv head).  A block owns a run of such rows; every key it fetches serves them all.
//
// Three kinds of calls:
//   kPrompt   keys lie in rows beside the queries, a sequence's rows one behind the other; row i of a sequence sees its keys 0..i
//   kPrefix   keys are the first `prefix_len` of every sequence and lie in the pages `prefix_pages`; a block's rows are of all sequences
//   kOwn      keys are those of one sequence from `prefix_len` on and lie in the sequence's own pages
// In the last two a row sees the keys up to its token's position.
//
// The softmax runs in powers of two: scores are scaled by scale * log2(e).  A call whose keys are cut into pieces leaves a record for each
// (token, head, piece): D floats of sum_j 2^(s_j - m) v_j, and (m, sum_j 2^(s_j - m)); a record whose sum is 0 has no values.
// attention_merge_kernel joins the records of a row.
#pragma once

#include "common.cuh"

namespace erb {

// Keys of a context: the tile that holds the last one (of up to 128) and the one asked for ahead of it end inside an int.
constexpr int kMostKeys = 0x7fffffff - 255;
// Keys of a piece: an int still holds them when they are rounded up to tiles.
constexpr int kMostPieceKeys = 1 << 30;

constexpr int kPrompt = 0, kPrefix = 1, kOwn = 2;

// Codes of the status word beside those of waits: a page that lies outside the pool, sequences that do not lie inside the rows.
constexpr int kBadPage = 9000001, kBadStarts = 9000002;

// Scaled scores (log2 domain) from here on: half a step of a float is a sixteenth at 2^20, and past 2^30 more exponents than a float has, so that a
// weight made from a scaled score and its row's rounded maximum could be infinite, or all of a row's be zero.  A row whose reference maximum lies beyond takes
// its scores' distances to the reference's score before they are scaled: exact for those that matter, and the highest one's weight is 1.
constexpr float kFarScore = 1048576.f;
__device__ __forceinline__ bool far_score(float m) { return fabsf(m) > kFarScore && m > -INFINITY; }

struct PackedArgs {
  const elem_t* q;
  elem_t* out;
  const elem_t *k, *v;             // kPrompt: rows; else the pools [n_pages][nkv][page_size][D]
  long long ld_q, ld_out, ld_k, ld_v;
  int n_pages, page_size;
  const int* tables;               // kOwn: [n_seqs][table_ld]
  int table_ld;
  const int* prefix_pages;
  int prefix_len;
  const int* seq_starts;
  const int* positions;
  int n_seqs, n_tokens, nq, nkv, D;
  float scale_log2;
  float *part_o, *part_ml;         // records: [(token * nq + head) * n_rec + piece]
  int n_rec, rec0, pieces;         // records of a row, the first of this call's pieces, how many pieces it cuts the keys into
  int piece_keys;                  // kOwn: keys of a piece (the last one takes the rest)
  int early;                       // kOwn behind a kernel over the prefix: may run beside it (all that is read was complete when that one began)
  int* status;
};

__device__ __forceinline__ void report(int* status, int code) { atomicCAS(status, 0, code); }

// The sequence and the row tile of block `index` among the tiles of `rows` rows that the sequences give, one after the other; the whole
// warp asks.  seq < 0: there is no such tile.
__device__ __forceinline__ void find_tile(const int* __restrict__ seq_starts, int n_seqs, int G, int rows, int index, int& seq, int& tile) {
  const int lane = threadIdx.x & 31;
  seq = -1;
  tile = 0;
  for (int s0 = 0; s0 < n_seqs; s0 += 32) {
    const int s = s0 + lane;
    const int len = s < n_seqs ? max(0, __ldcg(seq_starts + s + 1) - __ldcg(seq_starts + s)) : 0;
    const int mine = (int)(((long long)len * G + rows - 1) / rows);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int before = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += before;
    }
    const unsigned here = __ballot_sync(0xffffffffu, index >= upto - mine && index < upto);
    if (here) {
      const int who = __ffs(here) - 1;
      seq = s0 + who;
      tile = index - __shfl_sync(0xffffffffu, upto - mine, who);
      return;
    }
    index -= __shfl_sync(0xffffffffu, upto, 31);
  }
}

// The tiles of `rows` rows that the sequences give, those far along their sequences first (they see the most keys): how many there are, and
// the sequence and tile of the index-th.  The whole warp asks; lane l keeps the tiles of sequences l, l + 32, .. apart.
struct TileList {
  const int* starts;
  int n_seqs, G, rows, total, most;
  int first_of_lane, start_of_lane, len_of_lane;              // of sequence `lane`
  __device__ __forceinline__ int tiles(int s) const {
    if (s >= n_seqs) return 0;
    const long long pairs = (long long)max(0, __ldcg(starts + s + 1) - __ldcg(starts + s)) * G;
    return (int)((pairs + rows - 1) / rows);
  }
  __device__ __forceinline__ int of(int s0) const { return s0 == 0 ? first_of_lane : tiles(s0 + (int)(threadIdx.x & 31)); }
  __device__ __forceinline__ TileList(const int* starts, int n_seqs, int G, int rows) : starts(starts), n_seqs(n_seqs), G(G), rows(rows) {
    start_of_lane = n_seqs > 0 ? __ldcg(starts + min((int)(threadIdx.x & 31), n_seqs - 1)) : 0;
    len_of_lane = (int)(threadIdx.x & 31) < n_seqs ? __ldcg(starts + (threadIdx.x & 31) + 1) - start_of_lane : 0;
    first_of_lane = (int)(((long long)max(0, len_of_lane) * G + rows - 1) / rows);
    long long sum = 0;
    most = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += 32) {
      const int n = of(s0);
      sum += __reduce_add_sync(0xffffffffu, n);
      most = max(most, __reduce_max_sync(0xffffffffu, n));
    }
    total = (int)min(sum, (long long)0x3fffffff);
  }
  __device__ __forceinline__ int beyond(int level) const {      // tiles whose number in their sequence is at least `level`
    int sum = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += 32) sum += __reduce_add_sync(0xffffffffu, max(0, of(s0) - level));
    return sum;
  }
  __device__ __forceinline__ void find(int index, int& seq, int& tile) const {
    int low = 0, high = most;                                   // beyond(low) > index >= beyond(high)
    while (high - low > 1) {
      const int mid = (low + high) >> 1;
      if (beyond(mid) > index) low = mid;
      else high = mid;
    }
    tile = low;
    index -= beyond(low + 1);
    seq = -1;
    for (int s0 = 0; s0 < n_seqs; s0 += 32) {
      const unsigned have = __ballot_sync(0xffffffffu, of(s0) > low);
      const int count = __popc(have);
      if (index < count) {
        const int lane = threadIdx.x & 31;
        seq = s0 + __ffs(__ballot_sync(0xffffffffu, (have >> lane & 1) && __popc(have & ((1u << lane) - 1)) == index)) - 1;
        return;
      }
      index -= count;
    }
  }
};

// Where key `key` of this block lies: its row for the head `kvh` (rows of D entries in a pool, of ld entries for kPrompt), or null for a
// page that is none of the pool's (reported).
template <int MODE>
__device__ __forceinline__ void key_rows(const PackedArgs& a, const int* table, long long first_row, int kvh, int key, const elem_t*& k, const elem_t*& v) {
  if (MODE == kPrompt) {
    k = a.k + (first_row + key) * a.ld_k + (long long)kvh * a.D;
    v = a.v + (first_row + key) * a.ld_v + (long long)kvh * a.D;
  } else {
    const int page = table[key / a.page_size];
    if (page < 0 || page >= a.n_pages) {
      report(a.status, kBadPage);
      k = v = nullptr;
      return;
    }
    const long long row = (((long long)page * a.nkv + kvh) * a.page_size + key % a.page_size) * a.D;
    k = a.k + row;
    v = a.v + row;
  }
}

// Joins the n records (at most 128) of a row, in their order; the whole warp, lane l with the entries l + 32 c.  o starts at the row's
// own unnormalised values with maximum m and sum l (l 0: none) and ends as the result.
template <int C>
__device__ __forceinline__ void join_records(const float* part_ml, const float* part_o, int n, int D, float m, float l, float* o) {
  const int lane = threadIdx.x & 31;
  float rm[4], rl[4], x[8][C], top = l != 0.f ? m : -INFINITY;
  auto values = [&](int r0) {                                    // of eight records, on their way at once
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) x[r][c] = r0 + r < n && lane + 32 * c < D ? __ldcg(part_o + (size_t)(r0 + r) * D + lane + 32 * c) : 0.f;
  };
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const int r = lane + 32 * h;
    rm[h] = r < n ? __ldcg(part_ml + 2 * r) : -INFINITY;         // (the pair may lie on any float: one word at a time)
    rl[h] = r < n ? __ldcg(part_ml + 2 * r + 1) : 0.f;
  }
  values(0);
#pragma unroll
  for (int h = 0; h < 4; ++h)
    if (rl[h] != 0.f) top = fmaxf(top, rm[h]);
  top = warp_max(top);
  float sum = 0.f;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    rm[h] = rl[h] != 0.f ? exp2f(rm[h] - top) : 0.f;             // the records' weights
    sum = fmaf(rl[h], rm[h], sum);
  }
  const float mine = l != 0.f ? exp2f(m - top) : 0.f;
  sum = fmaf(l, mine, warp_sum(sum));
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = l != 0.f ? o[c] * mine : 0.f;
  for (int r0 = 0; r0 < n; r0 += 8) {
    if (r0) values(r0);
    const int h = r0 >> 5;
    const float w8 = h == 0 ? rm[0] : h == 1 ? rm[1] : h == 2 ? rm[2] : rm[3], l8 = h == 0 ? rl[0] : h == 1 ? rl[1] : h == 2 ? rl[2] : rl[3];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float w = __shfl_sync(0xffffffffu, w8, (r0 + r) & 31), lr = __shfl_sync(0xffffffffu, l8, (r0 + r) & 31);
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = lr != 0.f ? fmaf(x[r][c], w, o[c]) : o[c];      // (a record without a sum has no values)
    }
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;                // (a row that sees no key: zeros)
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] *= inv;
}

// Joins the records of each (token, head): a warp each.
template <int C>
static __global__ void __launch_bounds__(128)
attention_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, elem_t* __restrict__ out, long long ld_out,
                       const int* __restrict__ seq_starts, int n_seqs, int n_tokens, int nq, int D, int n_rec) {
  chain_wait();
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long long first = seq_starts[0], end = min((long long)seq_starts[n_seqs], (long long)n_tokens);
  if (first < 0 || item < first * nq || item >= end * nq) return;
  float o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = 0.f;
  join_records<C>(part_ml + 2 * item * n_rec, part_o + item * n_rec * D, n_rec, D, 0.f, 0.f, o);
  elem_t* dst = out + (item / nq) * ld_out + (item % nq) * D;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (lane + 32 * c < D) Elem<elem_t>::store(dst + lane + 32 * c, o[c]);
}

static int launch_merge(const PackedArgs& a, cudaStream_t stream, const char* who) {
  const long long blocks = ((long long)a.n_tokens * a.nq + 3) / 4;
  if (blocks > 0x7fffffffLL) return fail(ERB_ERR_UNSUPPORTED, "%s: too many rows", who);
  auto kern = a.D <= 64 ? attention_merge_kernel<2> : a.D <= 128 ? attention_merge_kernel<4> : attention_merge_kernel<8>;
  launch_chained(kern, dim3((unsigned)blocks), dim3(128), 0, stream, (const float*)a.part_o, (const float*)a.part_ml, a.out, a.ld_out, a.seq_starts, a.n_seqs,
                 a.n_tokens, a.nq, a.D, a.n_rec);
  return check_launch(who);
}

}  // namespace erb
