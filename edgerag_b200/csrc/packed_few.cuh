// A request's own keys behind a shared prefix, for few rows (bfloat16, heads of 64 and 128, any page size): mma.sync.m16n8k16 on
// tiles of 16 rows by 16 keys, keys and values fetched by cp.async.  What bounds it is the fetching of keys (tensor pipe 9 % busy, DRAM 28 %, most
// waits on global loads), so the tensor path matters little here; what matters is that many small blocks are resident.
//
//   attention_own_token_kernel   the rows of one token (up to 16 query heads of a kv head) are one tile; the four warps take 16 keys in turn,
//                                each with a ring of its own, and are joined at the end.  A warp asks for its next keys when it is done
//                                with those before (only their page's number is read ahead): the block's other warps and the other blocks
//                                are what a wait is hidden behind.  A request's tokens are done one after the other.
//   attention_own_rows_kernel    64 rows, (token, head) pairs, 16 for each warp; the four warps share the keys, 32 at a time, the next three
//                                times 32 on their way.
//
// 256 requests, 32 query heads on 8 of 128: up to 300 own keys behind 4,007 shared ones 68 us in all; 64 own keys each behind 4,096 63 us, by the
// kernel for many rows 160.
//
// Where the prefix's records are all that is left to join (`final`) the block does that too and writes the result.  It may run while the
// kernel over the prefix does: everything it reads before chain_wait() was complete when that kernel began.
#pragma once

#include "mma_split.cuh"
#include "packed.cuh"
#include "tc_common.cuh"

namespace erb {

constexpr int kFewWarps = 4, kFewThreads = 128, kFewRows = 64;

// Byte offset of 16-byte piece c of row r of a tile with D / 8 pieces a row, so that eight rows' same pieces lie in different banks.
template <int D> __device__ __forceinline__ uint32_t few_at(int r, int c) { return (uint32_t)(r * D * 2 + ((c ^ (r & 7)) << 4)); }

// 16 rows of one warp: rows g = lane / 4 and g + 8, the running maximum (log2 domain), sum and result of each.
template <int D> struct FewRows {
  uint32_t q[D / 16][4];
  float m[2], at[2], l[2], o[D / 8][4];            // at: the score that m is the scaled one of

  __device__ __forceinline__ void start(const elem_t* row0, const elem_t* row1) {         // the two rows' queries, or null
    const int q2 = (threadIdx.x & 3) * 2;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const int c = 16 * k + q2;
      q[k][0] = row0 ? __ldcg(reinterpret_cast<const unsigned*>(row0 + c)) : 0u;
      q[k][1] = row1 ? __ldcg(reinterpret_cast<const unsigned*>(row1 + c)) : 0u;
      q[k][2] = row0 ? __ldcg(reinterpret_cast<const unsigned*>(row0 + c + 8)) : 0u;
      q[k][3] = row1 ? __ldcg(reinterpret_cast<const unsigned*>(row1 + c + 8)) : 0u;
    }
    m[0] = m[1] = at[0] = at[1] = -INFINITY;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int d = 0; d < D / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
  }

  // 16 keys and values in shared memory; row i sees the first vis[i] of them.
  __device__ __forceinline__ void keys(const uint8_t* k_tile, const uint8_t* v_tile, int vis0, int vis1, float scale_log2) {
    const int lane = threadIdx.x & 31, q2 = (lane & 3) * 2;
    float s[2][4] = {};
    {
      const int r = (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;      // lanes 0-7: keys 0-7, dims 0-7; 8-15: dims 8-15; 16-31: keys 8-15
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t b[4];
        ldmatrix4(b, k_tile + few_at<D>(r, 2 * k + c));
        mma16816(s[0], q[k], b[0], b[1]);
        mma16816(s[1], q[k], b[2], b[3]);
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (8 * t + q2 + (e & 1) >= (e < 2 ? vis0 : vis1)) s[t][e] = -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[t][e]);
      }
    uint32_t p[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
    }
    // (the reference maximum moves as in the kernel for many rows: from 2^8 above it on)
    const float n0 = top[0] * scale_log2, n1 = top[1] * scale_log2;
    float b0 = m[0], b1 = m[1];
    if (__any_sync(0xffffffffu, n0 > m[0] + 8.f || n1 > m[1] + 8.f || fabsf(n0) > kFarScore || fabsf(n1) > kFarScore)) {
      const bool move0 = n0 > m[0] + 8.f || (far_score(n0) && top[0] > at[0]), move1 = n1 > m[1] + 8.f || (far_score(n1) && top[1] > at[1]);
      const float a0 = move0 ? fast_exp2(far_score(n0) || far_score(m[0]) ? (at[0] - top[0]) * scale_log2 : m[0] - n0) : 1.f;
      const float a1 = move1 ? fast_exp2(far_score(n1) || far_score(m[1]) ? (at[1] - top[1]) * scale_log2 : m[1] - n1) : 1.f;
      if (move0) { m[0] = n0; at[0] = top[0]; }
      if (move1) { m[1] = n1; at[1] = top[1]; }
      const bool far0 = far_score(m[0]), far1 = far_score(m[1]);
      if (__any_sync(0xffffffffu, far0 || far1)) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][e] -= e < 2 ? (far0 ? at[0] : 0.f) : (far1 ? at[1] : 0.f);
      }
      b0 = far0 ? 0.f : m[0];
      b1 = far1 ? 0.f : m[1];
      l[0] *= a0;
      l[1] *= a1;
#pragma unroll
      for (int d = 0; d < D / 8; ++d) { o[d][0] *= a0; o[d][1] *= a0; o[d][2] *= a1; o[d][3] *= a1; }
    }
    b0 = b0 == -INFINITY ? 0.f : b0;
    b1 = b1 == -INFINITY ? 0.f : b1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float x0 = fast_exp2(fmaf(s[t][0], scale_log2, -b0)), x1 = fast_exp2(fmaf(s[t][1], scale_log2, -b0));
      const float y0 = fast_exp2(fmaf(s[t][2], scale_log2, -b1)), y1 = fast_exp2(fmaf(s[t][3], scale_log2, -b1));
      l[0] += x0 + x1;                                                          // (this lane's keys; the lanes of a row are summed at the end)
      l[1] += y0 + y1;
      const __nv_bfloat162 bx = __floats2bfloat162_rn(x0, x1), by = __floats2bfloat162_rn(y0, y1);
      p[2 * t] = *reinterpret_cast<const uint32_t*>(&bx);
      p[2 * t + 1] = *reinterpret_cast<const uint32_t*>(&by);
    }
    {
      const int r = lane & 15, c = lane >> 4;                                   // lanes 0-15: keys, dims 0-7; 16-31: dims 8-15
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t b[4];
        ldmatrix4t(b, v_tile + few_at<D>(r, 2 * d + c));
        mma16816(o[2 * d], p, b[0], b[1]);
        mma16816(o[2 * d + 1], p, b[2], b[3]);
      }
    }
  }

  __device__ __forceinline__ void sum_lanes() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
  }
};

// The page of key `key`, and with it the key's row in the pools, or -1 where nothing is to be fetched.  The page may be
// asked for before it is known whether the request has the key.  (Rows of a pool are counted in 32 bits: the launch looks.)
__device__ __forceinline__ int few_page(const PackedArgs& a, const int* table, int key) { return __ldcg(table + min(key / a.page_size, a.table_ld - 1)); }
__device__ __forceinline__ int few_row(const PackedArgs& a, int page, int kvh, int key, int hi) {
  if (key >= hi) return -1;
  if (page < 0 || page >= a.n_pages) {
    report(a.status, kBadPage);
    return -1;
  }
  return (page * a.nkv + kvh) * a.page_size + key % a.page_size;
}

// A warp's ask for 16 keys and values; lane r (and r + 16) holds key r's place.
template <int D>
__device__ __forceinline__ void few_fetch(const PackedArgs& a, uint32_t k_tile, uint32_t v_tile, int place) {
  constexpr int PIECES = D / 8, AT_ONCE = 32 / PIECES;
  const int lane = threadIdx.x & 31, c = lane % PIECES;
#pragma unroll
  for (int r0 = 0; r0 < 16; r0 += AT_ONCE) {
    const int r = r0 + lane / PIECES, row = __shfl_sync(0xffffffffu, place, r);
    const bool valid = row >= 0;
    const long long from = (long long)max(row, 0) * D + c * 8;
    cp_async16(k_tile + few_at<D>(r, c), a.k + from, valid);
    cp_async16(v_tile + few_at<D>(r, c), a.v + from, valid);
  }
}

// One row's result: this block's m, l and (unnormalised) o, lane l with the entries l + 32 c, joined with the records of the prefix where
// the block is the last to add to it, else left as a record.
template <int D>
__device__ __forceinline__ void few_result(const PackedArgs& a, int token, int head, int piece, bool final, float m, float l, float* o) {
  constexpr int C = D / 32;
  const int lane = threadIdx.x & 31;
  const size_t row = (size_t)token * a.nq + head;
  if (!final) {
    const size_t record = row * a.n_rec + a.rec0 + piece;
    if (lane == 0) { a.part_ml[2 * record] = m; a.part_ml[2 * record + 1] = l; }
    if (l == 0.f) return;
#pragma unroll
    for (int c = 0; c < C; ++c) a.part_o[record * D + lane + 32 * c] = o[c];
    return;
  }
  join_records<C>(a.part_ml + 2 * row * a.n_rec, a.part_o + row * a.n_rec * D, a.rec0, D, m, l, o);
  elem_t* dst = a.out + (long long)token * a.ld_out + (long long)head * D;
#pragma unroll
  for (int c = 0; c < C; ++c) dst[lane + 32 * c] = __float2bfloat16_rn(o[c]);
}

// Two places, of which one is always empty while a warp multiplies (a place more is a copy under way more); blocks are short (a request's few
// hundred keys), and three of them (heads of 128) or four on a multiprocessor hide more than a deeper ring, for which fewer fit (64 requests of up to
// 1,000 own keys behind 16,384: two places 68 us, three 69, four 75; 256 of up to 300 behind 4,007: 73, 80, 108).
template <int D> struct FewSmem {
  static constexpr int kStages = 2;
  static constexpr uint32_t kTile = 16 * D * 2;                                 // 16 keys or values
  static constexpr uint32_t kRing = kFewWarps * kStages * 2 * kTile, kJoint = kFewWarps * 16 * (D + 2) * 4;
  static constexpr uint32_t kBytes = kRing > kJoint ? kRing : kJoint;           // (the warps' results lie over their rings)
};

template <int D>
__global__ void __launch_bounds__(kFewThreads, D == 64 ? 4 : 3) attention_own_token_kernel(const PackedArgs a, const int early) {
  using S = FewSmem<D>;
  extern __shared__ __align__(128) uint8_t few_smem[];
  if (!early) chain_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.nq / a.nkv, kvh = blockIdx.x, seq = blockIdx.y, piece = blockIdx.z;
  // Asked for at once: the request's rows, its first keys' pages, and the position of its row where every request has one.
  const int* table = a.tables + (size_t)seq * a.table_ld;
  const long long from = (long long)a.prefix_len + (long long)piece * a.piece_keys;
  const int lo = (int)min(from, (long long)INT_MAX - 4096);
  const int page_first = few_page(a, table, lo + 16 * warp + (lane & 15)), position_guess = __ldcg(a.positions + min(seq, a.n_tokens - 1));
  const int t0 = __ldcg(a.seq_starts + seq), len = __ldcg(a.seq_starts + seq + 1) - t0;
  const bool bad = len > 0 && (t0 < 0 || t0 + (long long)len > a.n_tokens);
  if (bad && threadIdx.x == 0) report(a.status, kBadStarts);
  const bool final = a.n_rec == a.rec0 + 1;
  const uint32_t mine = smem_u32(few_smem) + warp * S::kStages * 2 * S::kTile;
  float* joint = reinterpret_cast<float*>(few_smem);                            // [warp][16 rows][D], then [warp][16][2]
  float* joint_ml = joint + kFewWarps * 16 * D;
  FewRows<D> rows;
  bool waited = !early;
  for (int i = 0; i < (bad ? 0 : len); ++i) {
    const int token = t0 + i;
    long long limit = (long long)(token == seq ? position_guess : __ldcg(a.positions + token)) + 1;
    if (limit > (long long)a.table_ld * a.page_size) {
      if (threadIdx.x == 0) report(a.status, kBadPage);
      limit = (long long)a.table_ld * a.page_size;
    }
    const int hi = (int)(piece + 1 < a.pieces ? min(limit, from + a.piece_keys) : limit);
    // this warp's chunks: 16 keys from lo + 16 (warp + 4 c) on
    const int n = hi > lo ? ((hi - lo + 15) / 16 - warp + kFewWarps - 1) / kFewWarps : 0;
    auto key_of = [&](int c) { return lo + 16 * (warp + kFewWarps * c); };
    auto page_of = [&](int c) { return c == 0 ? page_first : c < n ? few_page(a, table, key_of(c) + (lane & 15)) : -1; };
    auto place_of = [&](int c, int page) { return c < n ? few_row(a, page, kvh, key_of(c) + (lane & 15), hi) : -1; };
    int page = page_of(0);
#pragma unroll
    for (int c = 0; c < S::kStages - 1; ++c) {
      if (c < n) few_fetch<D>(a, mine + c * 2 * S::kTile, mine + (c * 2 + 1) * S::kTile, place_of(c, page));
      cp_async_commit();
      page = page_of(c + 1);
    }
    const int g = lane >> 2;
    const elem_t* q = a.q + (long long)token * a.ld_q + (long long)kvh * G * D;
    rows.start(g < G ? q + g * D : nullptr, g + 8 < G ? q + (g + 8) * D : nullptr);
    for (int c = 0; c < n; ++c) {
      cp_async_wait<S::kStages - 2>();
      __syncwarp();
      const uint8_t* tile = few_smem + (warp * S::kStages + c % S::kStages) * 2 * S::kTile;
      rows.keys(tile, tile + S::kTile, hi - key_of(c), hi - key_of(c), a.scale_log2);
      __syncwarp();
      const int next = c + S::kStages - 1;
      if (next < n) {
        const uint32_t dst = mine + (next % S::kStages) * 2 * S::kTile;
        few_fetch<D>(a, dst, dst + S::kTile, place_of(next, page));
      }
      cp_async_commit();
      page = page_of(next + 1);
    }
    cp_async_wait<0>();
    rows.sum_lanes();
    __syncthreads();                                                            // (every warp has left its ring)
#pragma unroll
    for (int d = 0; d < D / 8; ++d) {
      float* dst = joint + (warp * 16 + g) * D + 8 * d + (lane & 3) * 2;
      *reinterpret_cast<float2*>(dst) = make_float2(rows.o[d][0], rows.o[d][1]);
      *reinterpret_cast<float2*>(dst + 8 * D) = make_float2(rows.o[d][2], rows.o[d][3]);
    }
    if ((lane & 3) == 0) {
      float* ml = joint_ml + (warp * 16 + g) * 2;
      ml[0] = rows.m[0];
      ml[1] = rows.l[0];
      ml[16] = rows.m[1];
      ml[17] = rows.l[1];
    }
    __syncthreads();
    if (!waited && final) {                                                     // the prefix's records
      chain_wait();
      waited = true;
    }
    constexpr int E = D / 32;
    for (int r = warp; r < G; r += kFewWarps) {
      float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w)
        if (joint_ml[(w * 16 + r) * 2 + 1] != 0.f) m = fmaxf(m, joint_ml[(w * 16 + r) * 2]);
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float lw = joint_ml[(w * 16 + r) * 2 + 1];
        if (lw == 0.f) continue;
        const float f = fast_exp2(joint_ml[(w * 16 + r) * 2] - m);
        l = fmaf(lw, f, l);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(joint[(w * 16 + r) * D + lane + 32 * e], f, o[e]);
      }
      few_result<D>(a, token, kvh * G + r, piece, final, m, l, o);
    }
    __syncthreads();
  }
  if (!waited) chain_wait();      // (a kernel after this one may count on the one over the prefix being done, too)
}

template <int D> struct FewRowsSmem {
  static constexpr int kKeys = 32, kStages = 4;
  static constexpr uint32_t kTile = kKeys * D * 2, kBytes = kStages * 2 * kTile;       // (64 rows of float results fit as well)
  static_assert(kBytes >= kFewRows * D * 4, "the results' rows lie over the ring");
};

template <int D>
__global__ void __launch_bounds__(kFewThreads) attention_own_rows_kernel(const PackedArgs a, const int early) {
  using S = FewRowsSmem<D>;
  extern __shared__ __align__(128) uint8_t few_smem[];
  __shared__ int s_hi, s_min, s_bad;
  if (!early) chain_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, G = a.nq / a.nkv, kvh = blockIdx.x, piece = blockIdx.z;
  int seq, tile, t0 = 0, len = 0;
  find_tile(a.seq_starts, a.n_seqs, G, kFewRows, blockIdx.y, seq, tile);
  if (seq >= 0) {
    t0 = __ldcg(a.seq_starts + seq);
    len = __ldcg(a.seq_starts + seq + 1) - t0;
    if (t0 < 0 || t0 + (long long)len > a.n_tokens) {
      if (tid == 0) report(a.status, kBadStarts);
      len = 0;
    }
  }
  const int r0 = tile * kFewRows, n_rows = (int)min((long long)kFewRows, (long long)len * G - r0);
  if (seq < 0 || len <= 0 || n_rows <= 0) {
    if (early) chain_wait();
    return;
  }
  const int* table = a.tables + (size_t)seq * a.table_ld;
  const bool final = a.n_rec == a.rec0 + 1;
  if (tid == 0) { s_hi = 0; s_min = INT_MAX; s_bad = 0; }
  __syncthreads();
  int lim[2], token[2], head[2];
  const elem_t* q[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = 16 * warp + g + 8 * h;
    const bool mine = r < n_rows;
    token[h] = t0 + (r0 + r) / G;
    head[h] = kvh * G + (r0 + r) % G;
    q[h] = mine ? a.q + (long long)token[h] * a.ld_q + (long long)head[h] * D : nullptr;
    long long limit = mine ? (long long)__ldcg(a.positions + token[h]) + 1 : 0;
    if (limit > (long long)a.table_ld * a.page_size) {
      report(a.status, kBadPage);
      limit = (long long)a.table_ld * a.page_size;
    }
    lim[h] = max((int)limit, 0);
    const int most = __reduce_max_sync(0xffffffffu, lim[h]), least = __reduce_min_sync(0xffffffffu, mine ? lim[h] : INT_MAX);
    if (lane == 0) { atomicMax(&s_hi, most); atomicMin(&s_min, least); }
  }
  __syncthreads();
  const long long from = (long long)a.prefix_len + (long long)piece * a.piece_keys;
  const int lo = (int)min(from, (long long)INT_MAX), hi = (int)(piece + 1 < a.pieces ? min((long long)s_hi, from + a.piece_keys) : (long long)s_hi);
  const int n = hi > lo ? (hi - lo + S::kKeys - 1) / S::kKeys : 0, least = s_min;
  // warp w fetches keys 16 (w & 1) .. of a stage, warps 0 and 1 their keys, 2 and 3 their values
  const uint32_t ring = smem_u32(few_smem);
  auto place_of = [&](int c) {
    const int key = lo + S::kKeys * c + 16 * (warp & 1) + (lane & 15);
    return c < n && key < hi ? few_row(a, few_page(a, table, key), kvh, key, hi) : -1;
  };
  auto fetch = [&](int c, int place) {
    constexpr int PIECES = D / 8, AT_ONCE = 32 / PIECES;
    const elem_t* pool = warp >= 2 ? a.v : a.k;
    const uint32_t dst = ring + (c % S::kStages) * 2 * S::kTile + (warp >= 2 ? S::kTile : 0);
    const int p = lane % PIECES;
#pragma unroll
    for (int r1 = 0; r1 < 16; r1 += AT_ONCE) {
      const int r = r1 + lane / PIECES;
      const int row = __shfl_sync(0xffffffffu, place, r);
      cp_async16(dst + few_at<D>(16 * (warp & 1) + r, p), pool + (long long)max(row, 0) * D + p * 8, row >= 0);
    }
  };
  int place = place_of(0);
#pragma unroll
  for (int c = 0; c < S::kStages - 1; ++c) {
    if (c < n) fetch(c, place);
    cp_async_commit();
    place = place_of(c + 1);
  }
  FewRows<D> rows;
  rows.start(q[0], q[1]);
  for (int c = 0; c < n; ++c) {
    cp_async_wait<S::kStages - 2>();
    __syncthreads();                              // this stage is there, and every warp has left the one before
    const int key0 = lo + S::kKeys * c, next = c + S::kStages - 1;
    if (next < n) fetch(next, place);
    cp_async_commit();
    place = place_of(next + 1);
    uint8_t* tile_k = few_smem + (c % S::kStages) * 2 * S::kTile;
    uint8_t* tile_v = tile_k + S::kTile;
    if (key0 + S::kKeys > least) {                // some row sees fewer keys: values that are no numbers become zeros for now
      for (int i = tid; i < (int)S::kTile / 16; i += kFewThreads) {
        uint4* p = reinterpret_cast<uint4*>(tile_v) + i;
        uint4 w = *p;
        uint32_t* e = &w.x;
        bool off = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if ((e[k] & 0x7f80u) == 0x7f80u) { e[k] &= 0xffff0000u; off = true; }
          if ((e[k] & 0x7f800000u) == 0x7f800000u) { e[k] &= 0xffffu; off = true; }
        }
        if (off) {
          *p = w;
          s_bad = 1;
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int h = 0; h < S::kKeys / 16; ++h)
      rows.keys(tile_k + h * 16 * D * 2, tile_v + h * 16 * D * 2, min(lim[0], hi) - key0 - 16 * h, min(lim[1], hi) - key0 - 16 * h, a.scale_log2);
  }
  cp_async_wait<0>();
  rows.sum_lanes();
  __syncthreads();                                // every warp has left the ring, every value has been looked at
  if (s_bad) {                                    // what a row does see of the values that were taken out
    for (int c = 0; c < n; ++c) {
      const int key0 = lo + S::kKeys * c;
      if (key0 + S::kKeys <= least) continue;
      for (int key = key0; key < min(key0 + S::kKeys, hi); ++key) {
        const elem_t *kr, *vr;
        key_rows<kOwn>(a, table, 0, kvh, key, kr, vr);
        if (!vr) continue;
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = __bfloat162float(vr[8 * d + (lane & 3) * 2 + (e & 1)]);
            if (!isfinite(v) && key < lim[e >> 1]) rows.o[d][e] += v;
          }
      }
    }
  }
  float* mine = reinterpret_cast<float*>(few_smem) + warp * 16 * D;             // this warp's rows
#pragma unroll
  for (int d = 0; d < D / 8; ++d) {
    float* dst = mine + g * D + 8 * d + (lane & 3) * 2;
    *reinterpret_cast<float2*>(dst) = make_float2(rows.o[d][0], rows.o[d][1]);
    *reinterpret_cast<float2*>(dst + 8 * D) = make_float2(rows.o[d][2], rows.o[d][3]);
  }
  __syncwarp();
  if (early) chain_wait();                        // the prefix's records
  constexpr int E = D / 32;
  for (int r = 0; r < min(16, n_rows - 16 * warp); ++r) {
    const int from_lane = (r & 7) * 4;
    const float m = __shfl_sync(0xffffffffu, r < 8 ? rows.m[0] : rows.m[1], from_lane), l = __shfl_sync(0xffffffffu, r < 8 ? rows.l[0] : rows.l[1], from_lane);
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = mine[r * D + lane + 32 * e];
    const int index = r0 + 16 * warp + r;
    few_result<D>(a, t0 + index / G, kvh * G + index % G, piece, final, m, l, o);
  }
}

}  // namespace erb
