// Attention over whole prompts packed one behind the other, and of a batch whose requests share a long prefix in the cache (what the calls
// are: packed.cuh): the kernels on CUDA cores, for both element types, any head size up to 256, any page size, strides and alignment; and
// the merge of the pieces that a call's keys were cut into.  attention_packed_tc.cu has the tensor-core forms.
//
// A block owns 32 rows of one kv head and walks its keys 64 at a time with the running maximum and sum of the softmax.  Queries, keys and
// values lie in shared memory as floats; a thread of the 128 owns 4 x 4 scores and then 4 rows x D / 16 entries of the result, so that
// 16 products take 8 floats from shared memory.  What bounds it: the longest row tile's walk, 11 steps of 7 us for 5 prompts of up to 701 tokens, 15
// heads of 64 (the multiprocessors are at work 62 % of that time), and in a step shared loads and instructions, with two blocks of four warps on a
// multiprocessor: instructions in 48 % of its cycles, multiply-adds in 32 % (tiles of 64 rows 113 us, of 32 84 us; with four steps of the scores'
// loop unrolled, so that the next floats are asked for before these are used, 78 us; two multiply-adds an instruction: 80 us).
//
// A request's own keys behind a prefix are walked by one block a piece and kv head, which takes the request's row tiles one after the other: made
// for a few rows a request.  15 heads on 5 of 64 behind 1,000 keys: 8 requests of 200 new tokens 0.36 ms, one of 2,000 3.4 ms.
//
// Keys that no row of the block may see are zeros in shared memory, whatever their memory holds; where only some rows may see a key, its
// product is left out for the others, not multiplied by zero, so that an infinity or NaN there stays unseen.
#include <limits.h>
#include <stdarg.h>

#include "packed.cuh"

using namespace erb;

ERB_DEFINE_LAST_ERROR(erb_last_error)

namespace {

constexpr int BM = 32, BN = 64, kThreads = 4 * BM, RS = BM / 4;      // (a thread's rows are RS apart)

// Floats on 16-byte boundaries are copied asynchronously, the next keys while these are worked on: two places for keys and values where
// two blocks still fit a multiprocessor (heads up to 64) or one does (128).
template <int DMAX> struct Smem {
  static constexpr int kLd = DMAX + 4, kLdP = BN + 4, kBufs = sizeof(elem_t) == 4 && DMAX <= 128 ? 2 : 1;
  float q[BM * kLd], k[kBufs][BN * kLd], v[kBufs][BN * DMAX], p[BM * kLdP];
  int limit[BM], any[2];
  const elem_t* krow[kBufs][BN];
  const elem_t* vrow[kBufs][BN];
};

// Four entries from column c on of a row as floats, zeros behind column D; `wide`: rows lie on four entries' boundaries.
__device__ __forceinline__ float4 load_four(const elem_t* row, int c, int D, bool wide) {
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (wide) {
    if (c < D) Pack4<elem_t>::load(row + c, x);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < D) x[j] = Elem<elem_t>::load(row + c + j);
  }
  return make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void copy16(float* dst, const void* src, bool real) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(real ? 16 : 0) : "memory");
}

template <int DMAX, int MODE>
__device__ __forceinline__ void work_on(const PackedArgs& a, const int wide) {
  extern __shared__ __align__(16) uint8_t raw[];
  Smem<DMAX>& sm = *reinterpret_cast<Smem<DMAX>*>(raw);
  constexpr int LD = Smem<DMAX>::kLd, LDP = Smem<DMAX>::kLdP, NC = DMAX / 64;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, D = a.D, G = a.nq / a.nkv, kvh = MODE == kPrompt ? blockIdx.x % a.nkv : blockIdx.y;

  // the rows of this block: tokens t0 .. of one sequence (kPrefix: of all), rows r0 .. of them
  int seq = 0, tile = blockIdx.x, t0, len;
  if (MODE == kPrompt) {           // the tiles that see the most keys first, each one's kv heads side by side
    const TileList list(a.seq_starts, a.n_seqs, G, BM);
    if ((int)(blockIdx.x / a.nkv) >= list.total) return;
    list.find(blockIdx.x / a.nkv, seq, tile);
  }
  if (MODE == kOwn) { seq = blockIdx.x / a.pieces; tile = 0; }
  if (seq < 0) return;
  if (MODE == kPrefix) {
    t0 = a.seq_starts[0];
    len = a.seq_starts[a.n_seqs] - t0;
  } else {
    t0 = a.seq_starts[seq];
    len = a.seq_starts[seq + 1] - t0;
  }
  if (len <= 0) return;
  if (t0 < 0 || t0 + (long long)len > a.n_tokens) {
    if (tid == 0) report(a.status, kBadStarts);
    return;
  }
  const int piece = MODE == kOwn ? blockIdx.x % a.pieces : blockIdx.z;
  const int* table = MODE == kOwn ? a.tables + (size_t)seq * a.table_ld : a.prefix_pages;
  const bool direct = a.n_rec <= 1;

  // (kOwn: blocks of one sequence are few, so one of them takes its row tiles in turn)
  for (int r0 = tile * BM; r0 < (long long)len * G; r0 += BM) {
    const int rows = (int)min((long long)BM, (long long)len * G - r0);
    __syncthreads();
    if (tid < 2) sm.any[tid] = 0;
    __syncthreads();
    if (tid < BM) {
      int lim = 0;
      if (tid < rows) {
        const int token = (r0 + tid) / G;
        if (MODE == kPrompt) lim = token + 1;
        else {
          lim = max(0, min(a.positions[t0 + token], INT_MAX - 1) + 1);
          if (MODE == kPrefix) lim = min(lim, a.prefix_len);
          if (MODE == kOwn && lim > (long long)a.table_ld * a.page_size) { report(a.status, kBadPage); lim = a.table_ld * a.page_size; }
        }
      }
      sm.limit[tid] = lim;
      atomicMax(&sm.any[0], lim);
    }
#pragma unroll 4
    for (int i = tid; i < BM * (DMAX / 4); i += kThreads) {
      const int r = i / (DMAX / 4), c = (i % (DMAX / 4)) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows) x = load_four(a.q + (long long)(t0 + (r0 + r) / G) * a.ld_q + (long long)(kvh * G + (r0 + r) % G) * D, c, D, wide);
      *reinterpret_cast<float4*>(sm.q + r * LD + c) = make_float4(x.x * a.scale_log2, x.y * a.scale_log2, x.z * a.scale_log2, x.w * a.scale_log2);
    }
    __syncthreads();
    // the keys of this block's piece, [lo, hi)
    int lo = MODE == kOwn ? a.prefix_len : 0, hi = sm.any[0];
    if (MODE == kPrefix) {
      const int n_tiles = (hi + BN - 1) / BN, per = (n_tiles + a.pieces - 1) / a.pieces;
      lo = min(hi, piece * per * BN);
      hi = min(hi, lo + per * BN);
    }
    if (MODE == kOwn) {
      const long long from = lo + (long long)piece * a.piece_keys;
      if (piece + 1 < a.pieces) hi = (int)min((long long)hi, from + a.piece_keys);
      lo = (int)min((long long)max(hi, lo), from);
    }

    float m[4], l[4], o[4][4 * NC];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < 4 * NC; ++c) o[i][c] = 0.f;
    }
    constexpr int BUFS = Smem<DMAX>::kBufs;
    const bool async = BUFS == 2 && wide;
    auto find_rows = [&](int key0, int buf) {
      if (tid < BN) {
        const elem_t *kr = nullptr, *vr = nullptr;
        if (key0 + tid < hi) key_rows<MODE>(a, table, t0, kvh, key0 + tid, kr, vr);
        sm.krow[buf][tid] = kr;
        sm.vrow[buf][tid] = vr;
      }
    };
    auto fetch = [&](int buf) {                    // the rows found, asynchronously
      constexpr int N = BN * (DMAX / 4) / kThreads;
#pragma unroll 4
      for (int n = 0; n < N; ++n) {
        const int i = tid + n * kThreads, r = i / (DMAX / 4), c = (i % (DMAX / 4)) * 4;
        const elem_t *kr = sm.krow[buf][r], *vr = sm.vrow[buf][r];
        const bool real = kr && c < D;
        copy16(sm.k[buf] + r * LD + c, real ? kr + c : a.k, real);
        copy16(sm.v[buf] + r * DMAX + c, real ? vr + c : a.v, real);
      }
    };
    int buf = 0;
    if (async && lo < hi) {
      find_rows(lo, 0);
      __syncthreads();
      fetch(0);
    }
    if (async) asm volatile("cp.async.commit_group;" ::: "memory");
    for (int key0 = lo; key0 < hi; key0 += BN) {
      if (async) {
        buf = ((key0 - lo) / BN) & 1;
        __syncthreads();                           // (the other place has been left)
        find_rows(key0 + BN, buf ^ 1);
        __syncthreads();
        if (key0 + BN < hi) fetch(buf ^ 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();
      } else {
        __syncthreads();
        find_rows(key0, 0);
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < BN * (DMAX / 4); i += kThreads) {
          const int r = i / (DMAX / 4), c = (i % (DMAX / 4)) * 4;
          const elem_t *kr = sm.krow[0][r], *vr = sm.vrow[0][r];
          const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
          *reinterpret_cast<float4*>(sm.k[0] + r * LD + c) = kr ? load_four(kr, c, D, wide) : none;
          *reinterpret_cast<float4*>(sm.v[0] + r * DMAX + c) = kr ? load_four(vr, c, D, wide) : none;
        }
        __syncthreads();
      }
      const float *tile_k = sm.k[buf], *tile_v = sm.v[buf];
      // scores: rows ty + 16 i, keys tx + 16 j
      float s[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
      for (int c = 0; c < D; c += 4) {
        float4 qa[4], ka[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          qa[i] = *reinterpret_cast<const float4*>(sm.q + (ty + RS * i) * LD + c);
          ka[i] = *reinterpret_cast<const float4*>(tile_k + (tx + 16 * i) * LD + c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s[i][j] = fmaf(qa[i].x, ka[j].x, fmaf(qa[i].y, ka[j].y, fmaf(qa[i].z, ka[j].z, fmaf(qa[i].w, ka[j].w, s[i][j]))));
      }
      bool partly = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int lim = min(sm.limit[ty + RS * i], hi);
        partly |= lim < key0 + BN;
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (key0 + tx + 16 * j >= lim) s[i][j] = -INFINITY;
          top = fmaxf(top, s[i][j]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float m_new = fmaxf(m[i], top), base = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = exp2f(m[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2f(s[i][j] - base);
          sum += p;
          sm.p[(ty + RS * i) * LDP + tx + 16 * j] = p;
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        m[i] = m_new;
        l[i] = l[i] * alpha + sum;
#pragma unroll
        for (int c = 0; c < 4 * NC; ++c) o[i][c] *= alpha;
      }
      __syncwarp();                            // (a row's scores are made and used by one warp)
      if (!__any_sync(0xffffffffu, partly)) {
        for (int j = 0; j < BN; j += 4) {
          float4 pa[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) pa[i] = *reinterpret_cast<const float4*>(sm.p + (ty + RS * i) * LDP + j);
#pragma unroll
          for (int jj = 0; jj < 4; ++jj)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              const float4 va = *reinterpret_cast<const float4*>(tile_v + (j + jj) * DMAX + 64 * c + 4 * tx);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float p = jj == 0 ? pa[i].x : jj == 1 ? pa[i].y : jj == 2 ? pa[i].z : pa[i].w;
                o[i][4 * c] = fmaf(p, va.x, o[i][4 * c]);
                o[i][4 * c + 1] = fmaf(p, va.y, o[i][4 * c + 1]);
                o[i][4 * c + 2] = fmaf(p, va.z, o[i][4 * c + 2]);
                o[i][4 * c + 3] = fmaf(p, va.w, o[i][4 * c + 3]);
              }
            }
        }
      } else {
        const int n = min(BN, hi - key0);
        for (int j = 0; j < n; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (key0 + j >= sm.limit[ty + RS * i]) continue;
            const float p = sm.p[(ty + RS * i) * LDP + j];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              const float4 va = *reinterpret_cast<const float4*>(tile_v + j * DMAX + 64 * c + 4 * tx);
              o[i][4 * c] = fmaf(p, va.x, o[i][4 * c]);
              o[i][4 * c + 1] = fmaf(p, va.y, o[i][4 * c + 1]);
              o[i][4 * c + 2] = fmaf(p, va.z, o[i][4 * c + 2]);
              o[i][4 * c + 3] = fmaf(p, va.w, o[i][4 * c + 3]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = ty + RS * i;
      if (r >= rows) continue;
      const int token = t0 + (r0 + r) / G, head = kvh * G + (r0 + r) % G;
      if (direct) {
        const float inv = l[i] != 0.f ? 1.f / l[i] : 0.f;      // (a row that sees no key: zeros)
        elem_t* dst = a.out + (long long)token * a.ld_out + (long long)head * D;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (64 * c + 4 * tx + j < D) Elem<elem_t>::store(dst + 64 * c + 4 * tx + j, o[i][4 * c + j] * inv);
      } else {
        const size_t record = ((size_t)token * a.nq + head) * a.n_rec + a.rec0 + piece;
        if (tx == 0) {
          a.part_ml[2 * record] = m[i];
          a.part_ml[2 * record + 1] = l[i];
        }
        if (l[i] == 0.f) continue;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (64 * c + 4 * tx + j < D) a.part_o[record * D + 64 * c + 4 * tx + j] = o[i][4 * c + j];
      }
    }
    if (MODE != kOwn) break;
  }
}

template <int DMAX, int MODE>
__global__ void __launch_bounds__(kThreads) attention_packed_kernel(const PackedArgs a, const int wide) {
  const bool early = MODE == kOwn && a.early;
  if (!early) chain_wait();
  work_on<DMAX, MODE>(a, wide);
  if (early) chain_wait();         // (a kernel after this one may count on the one over the prefix being done, too)
}

template <int DMAX, int MODE>
int launch_tiles(const PackedArgs& a, dim3 grid, cudaStream_t stream, const char* who) {
  const int bytes = (int)sizeof(Smem<DMAX>);
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(ERB_ERR_CUDA, "%s: no device", who);
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attention_packed_kernel<DMAX, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return fail(ERB_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    configured[dev] = true;
  }
  // whether every row starts on a boundary of four entries (floats: of 16 bytes)
  const uintptr_t starts = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v;
  const int wide = !(starts & (4 * sizeof(elem_t) - 1)) && !((a.ld_q | a.D | (MODE == kPrompt ? a.ld_k | a.ld_v : 0)) & 3);
  launch_chained(attention_packed_kernel<DMAX, MODE>, grid, dim3(kThreads), bytes, stream, a, wide);
  return check_launch(who);
}

template <int MODE>
int launch_by_size(const PackedArgs& a, dim3 grid, cudaStream_t stream, const char* who) {
  if (grid.x > 0x7fffffffu || grid.y > 65535u || grid.z > 65535u) return fail(ERB_ERR_UNSUPPORTED, "%s: too many blocks", who);
  if (a.D <= 64) return launch_tiles<64, MODE>(a, grid, stream, who);
  if (a.D <= 128) return launch_tiles<128, MODE>(a, grid, stream, who);
  return launch_tiles<256, MODE>(a, grid, stream, who);
}

}  // namespace

// Whole prompts: row t of q, k, v and out is token t; sequence s is rows seq_starts[s] .. seq_starts[s + 1] (int32 [n_seqs + 1]).
ERB_EXPORT int erb_attention_prompt(const void* q, long long ld_q, const void* k, long long ld_k, const void* v, long long ld_v,
                                    const int* seq_starts, int n_seqs, int n_tokens, void* out, long long ld_out, int nq, int nkv,
                                    int head_dim, float scale, int* status, void* stream) {
  if (n_seqs <= 0 || n_tokens <= 0) return ERB_OK;
  if (nq <= 0 || nkv <= 0 || nq % nkv || head_dim <= 0 || head_dim > 256 || !status) return fail(ERB_ERR_ARG, "attention_prompt: bad sizes");
  PackedArgs a = {};
  a.q = (const elem_t*)q; a.k = (const elem_t*)k; a.v = (const elem_t*)v; a.out = (elem_t*)out;
  a.ld_q = ld_q; a.ld_k = ld_k; a.ld_v = ld_v; a.ld_out = ld_out;
  a.seq_starts = seq_starts; a.n_seqs = n_seqs; a.n_tokens = n_tokens; a.nq = nq; a.nkv = nkv; a.D = head_dim;
  a.scale_log2 = scale * 1.4426950408889634f; a.n_rec = 1; a.pieces = 1; a.status = status; a.page_size = 1;
  const long long tiles = (long long)n_tokens * (nq / nkv) / BM + n_seqs;      // (a sequence has at most one tile that is not full)
  if (tiles * nkv > 0x7fffffffLL) return fail(ERB_ERR_UNSUPPORTED, "attention_prompt: too many rows");
  return launch_by_size<kPrompt>(a, dim3((unsigned)(tiles * nkv), 1, 1), (cudaStream_t)stream, "attention_prompt");
}

// A batch that shares a prefix: keys 0 .. prefix_len - 1 of every sequence lie in the pages prefix_pages (int32), those from prefix_len on
// in the sequence's own pages (row s of tables, entry i the page of keys i * page_size ..).  Row t of q and out is token t, at positions[t] of
// its sequence; it sees the keys up to there.  The prefix is cut into prefix_pieces, a sequence's own keys into own_pieces of piece_keys (the
// last takes the rest); with more than one piece in all, part_o has room for n_tokens * nq * pieces * head_dim floats and part_ml for
// n_tokens * nq * pieces * 2.
ERB_EXPORT int erb_attention_shared_prefix(const void* q, long long ld_q, const void* k_pages, const void* v_pages, int n_pages, int page_size,
                                           const int* prefix_pages, int prefix_len, const int* tables, int table_ld, const int* seq_starts,
                                           const int* positions, int n_seqs, int n_tokens, void* out, long long ld_out, int nq, int nkv,
                                           int head_dim, float scale, int prefix_pieces, int own_pieces, int piece_keys, float* part_o,
                                           float* part_ml, int* status, void* stream) {
  if (n_seqs <= 0 || n_tokens <= 0) return ERB_OK;
  if (nq <= 0 || nkv <= 0 || nq % nkv || head_dim <= 0 || head_dim > 256 || !status || n_pages <= 0 || page_size <= 0 || prefix_len < 0 ||
      table_ld <= 0 || prefix_pieces < (prefix_len > 0 ? 1 : 0) || own_pieces < 1 || piece_keys <= 0 || piece_keys > kMostPieceKeys ||
      prefix_len > kMostKeys || (long long)table_ld * page_size > kMostKeys)
    return fail(ERB_ERR_ARG, "attention_shared_prefix: bad sizes");
  const int n_rec = (prefix_len > 0 ? prefix_pieces : 0) + own_pieces;
  if (n_rec > 1 && (!part_o || !part_ml)) return fail(ERB_ERR_ARG, "attention_shared_prefix: pieces need scratch");
  PackedArgs a = {};
  a.q = (const elem_t*)q; a.k = (const elem_t*)k_pages; a.v = (const elem_t*)v_pages; a.out = (elem_t*)out;
  a.ld_q = ld_q; a.ld_out = ld_out; a.n_pages = n_pages; a.page_size = page_size; a.tables = tables; a.table_ld = table_ld;
  a.prefix_pages = prefix_pages; a.prefix_len = prefix_len; a.seq_starts = seq_starts; a.positions = positions;
  a.n_seqs = n_seqs; a.n_tokens = n_tokens; a.nq = nq; a.nkv = nkv; a.D = head_dim; a.scale_log2 = scale * 1.4426950408889634f;
  a.part_o = part_o; a.part_ml = part_ml; a.n_rec = n_rec; a.status = status; a.piece_keys = piece_keys;
  cudaStream_t s = (cudaStream_t)stream;
  const long long rows = (long long)n_tokens * (nq / nkv);
  if ((rows + BM - 1) / BM > 0x7fffffffLL || (long long)n_seqs * own_pieces > 0x7fffffffLL)
    return fail(ERB_ERR_UNSUPPORTED, "attention_shared_prefix: too many rows");
  if (prefix_len > 0) {
    a.rec0 = 0;
    a.pieces = prefix_pieces;
    const int rc = launch_by_size<kPrefix>(a, dim3((unsigned)((rows + BM - 1) / BM), nkv, prefix_pieces), s, "attention_shared_prefix");
    if (rc) return rc;
  }
  a.rec0 = prefix_len > 0 ? prefix_pieces : 0;
  a.pieces = own_pieces;
  a.early = prefix_len > 0;
  const int rc = launch_by_size<kOwn>(a, dim3((unsigned)(n_seqs * own_pieces), nkv, 1), s, "attention_shared_prefix");
  if (rc || n_rec <= 1) return rc;
  return launch_merge(a, s, "attention_shared_prefix");
}
