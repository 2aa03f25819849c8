// Attention over packed whole prompts, and of a batch behind a shared prefix (what the calls are: packed.cuh), on the 5th-generation tensor
// cores (tcgen05 + TMEM): bfloat16, heads of 64 and 128, cache pages of 8 to 128 tokens (a power of two).
//
// A block owns up to 256 rows of one kv head, (token, head of its group) pairs, as two query tiles A and B of 128 rows, and walks the
// keys in tiles of 128.  Every byte of K and V that reaches shared memory serves all its rows; with G query heads a kv head a prompt's
// block spans 256 / G tokens, so little of the last tile on the diagonal is hidden.  A call whose rows all fit one tile (`dual`) gives both
// tiles the same rows and every other key tile each, and leaves a record of its sums for each of them.
//
//   warp 10 (copy)    brings K and V tiles in turn into one ring of shared memory by TMA tensor copies, 128-byte swizzle: from the pages, one
//                     copy per page and 64 columns, or from rows beside the queries
//   warps 8, 9        issue S_t = Q_t K^T (M 128, N 128) and O_t += P_t V (M 128, N D, P from TMEM), one warp for each query tile
//   warps 0-3, 4-7    softmax of tile A and of tile B: a thread owns a row, takes its 128 scores into registers, and writes P back
//                     rounded to bfloat16 (the second product's operand type; the sum of P is taken before that rounding, in float)
//
// A row's reference maximum moves only when a tile's maximum is 2^8 above it; O is rescaled in TMEM then.  P is a floating-point number, so
// a reference that is low by eight powers of two costs no precision.
//
// TMEM, 512 columns: S 2 x 128, O 2 x D.  With heads of 64 P has 2 x 64 columns of its own, so the next scores are issued as soon as a
// tile's are in registers; with heads of 128 P takes its scores' place and the next scores wait for P V.
//
// Hidden keys.  Scores are masked where some row of a warp sees fewer keys than its tile has.  P is then zero, but zero times a value
// that is no number would spoil rows that do not see it; so in such tiles the softmax threads look the values over: rows nobody sees
// become zeros, and an infinity or NaN that only some rows see becomes zero and is added to exactly those rows at the end.
//
// Every wait is bounded: a thread that gives up raises a block-wide flag, every other wait of the block then ends too, the block records a
// code in *status, lets its copies land, frees its TMEM and returns.
#include <limits.h>
#include <stdarg.h>
#include <stdio.h>

#undef ERB_ELEM
#define ERB_ELEM 1
#include "packed.cuh"
#include "packed_few.cuh"
#include "tc_common.cuh"

using namespace erb;

ERB_DEFINE_LAST_ERROR(erb_last_error)

namespace {

constexpr int BM = 128, BN = 128;
constexpr int kSoftmaxWarps = 8, kIssueWarp = 8, kCopyWarp = 10, kThreads = 352;
constexpr float kMoveFrom = 8.f;          // powers of two by which a tile's maximum is above the reference before that moves
constexpr int kOwnMany = 0, kOwnToken = 1, kOwnRows = 2;      // kernels for a request's own keys
constexpr int kGaveUp = 9100000;          // status code of a wait that ran out

template <int D> struct Cfg {
  static constexpr int kHalves = D / 64;                         // blocks of 64 columns (128 bytes of a row)
  static constexpr uint32_t kBlock = BM * 128, kTile = kHalves * kBlock;
  static constexpr int kStages = D == 64 ? 10 : 5;               // tiles of K or V in the ring
  static constexpr bool kPlaceForP = D == 64;
  static constexpr uint32_t kColP = 256, kColO = D == 64 ? 384 : 256;
  // barriers: ring full, ring empty; per query tile: scores there, scores in registers, P written, P V done
  static constexpr int kFull = 0, kEmpty = kStages, kS = 2 * kStages, kRead = kS + 2, kP = kS + 4, kPv = kS + 6, kNumBars = kS + 8;
  static constexpr uint32_t kSmemTiles = (2 + kStages) * kTile, kSmemBytes = kSmemTiles + 8 * kNumBars + 64 + 1024;
};

struct Shared {
  int abort, bad;                 // bad: some value of a tile on an edge is no number
  uint32_t tmem;
  int hi[2], lim_min[2];          // per query tile: one behind the last key any row sees, the smallest such of a row
};

__device__ __forceinline__ bool not_finite2(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }

template <int D, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
attention_packed_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PackedArgs a, const int dual) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const uint32_t sQ = base, sRing = base + 2 * C::kTile, bars = base + C::kSmemTiles;
  Shared* sh = reinterpret_cast<Shared*>(smem + C::kSmemTiles + 8 * C::kNumBars);
  volatile int* s_abort = &sh->abort;
  auto bar = [&](int which) { return bars + 8u * (uint32_t)which; };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  chain_wait();
  const int code = tid == 0 ? *reinterpret_cast<volatile int*>(a.status) : 0;
  if (__syncthreads_or(code >= 1000000 && code != kBadPage && code != kBadStarts)) return;      // an earlier block gave up: do not pile on

  // --- the rows of this block: r0 .. of the (token, head) pairs of tokens t0 .. t0 + len ---
  const int kvh = blockIdx.x, G = a.nq / a.nkv, per_block = dual ? BM : 2 * BM;
  int seq = 0, tile = blockIdx.y, t0, len;
  if (MODE != kPrefix) find_tile(a.seq_starts, a.n_seqs, G, per_block, (int)(gridDim.y - 1 - blockIdx.y), seq, tile);
  if (seq < 0) return;
  if (MODE == kPrefix) {
    t0 = a.seq_starts[0];
    len = a.seq_starts[a.n_seqs] - t0;
  } else {
    t0 = a.seq_starts[seq];
    len = a.seq_starts[seq + 1] - t0;
  }
  const long long r0 = (long long)tile * per_block;
  if (len <= 0 || r0 >= (long long)len * G) return;
  if (t0 < 0 || t0 + (long long)len > a.n_tokens) {
    if (tid == 0) report(a.status, kBadStarts);
    return;
  }
  const int rows = (int)min((long long)per_block, (long long)len * G - r0);
  const int* table = MODE == kOwn ? a.tables + (size_t)seq * a.table_ld : a.prefix_pages;

  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) { mbar_init(bar(C::kFull + s), 1); mbar_init(bar(C::kEmpty + s), dual ? 1 : 2); }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar(C::kS + t), 1);
      mbar_init(bar(C::kRead + t), 4);
      mbar_init(bar(C::kP + t), 4);
      mbar_init(bar(C::kPv + t), 1);
      sh->hi[t] = 0;
      sh->lim_min[t] = INT_MAX;
    }
    sh->abort = sh->bad = 0;
    mbar_init_fence();
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  __syncthreads();
  // the keys each row sees: up to `lim` (softmax threads; a row that is none sees everything and costs no mask)
  const int my_tile = (warp >> 2) & 1, my_row = tid & (BM - 1), my_index = dual ? my_row : tid;
  int lim = INT_MAX, my_token = 0, my_head = 0;
  if (warp < kSoftmaxWarps) {
    const bool mine = my_index < rows;
    if (mine) {
      const int r = (int)(r0 + my_index);
      my_token = t0 + r / G;
      my_head = kvh * G + r % G;
      if (MODE == kPrompt) lim = r / G + 1;
      else {
        lim = a.positions[my_token] + 1;
        if (MODE == kPrefix) lim = min(lim, a.prefix_len);
        else if (lim > (long long)a.table_ld * a.page_size) { report(a.status, kBadPage); lim = a.table_ld * a.page_size; }
        lim = max(lim, 0);
      }
    }
    const int most = __reduce_max_sync(0xffffffffu, mine ? lim : 0), least = __reduce_min_sync(0xffffffffu, lim);
    if (lane == 0) { atomicMax(&sh->hi[my_tile], most); atomicMin(&sh->lim_min[my_tile], least); }
    // Q tiles: 16-byte pieces, rows behind the last one zeros
    constexpr int kPieces = D / 8, kRowsAtOnce = 256 / kPieces;
    const int piece = tid % kPieces, n_q = dual ? BM : 2 * BM;
    const __nv_bfloat16* q_head = a.q + (size_t)kvh * G * D + piece * 8;
#pragma unroll 4
    for (int r = tid / kPieces; r < n_q; r += kRowsAtOnce) {
      const bool valid = r < rows;
      const int idx = valid ? (int)(r0 + r) : (int)r0, token = idx / G;
      cp_async16(sQ + (r >> 7) * C::kTile + (piece >> 3) * C::kBlock + swz(r & (BM - 1), piece & 7),
                 q_head + (long long)(t0 + token) * a.ld_q + (idx - token * G) * D, valid);
    }
    cp_async_commit();
    cp_async_wait<0>();
    fence_async_proxy();
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = sh->tmem;

  // --- the walk: key tiles j0 .. j0 + n_copied, of which query tile t takes n_of(t) ---
  const int lo = MODE == kOwn ? a.prefix_len : 0, hi = max(sh->hi[0], sh->hi[1]);
  const int j_first = lo / BN, j_end = hi > lo ? (hi + BN - 1) / BN : j_first;
  int j0 = j_first, j1 = j_end;
  if (MODE != kPrompt) {
    const int piece = blockIdx.z, per = MODE == kOwn ? (a.piece_keys + BN - 1) / BN : (j_end - j_first + a.pieces - 1) / a.pieces;
    j0 = (int)min((long long)j_end, j_first + (long long)piece * per);
    if (MODE == kPrefix || piece + 1 < a.pieces) j1 = min(j_end, j0 + per);
  }
  const int n_copied = j1 - j0;
  auto n_of = [&](int t) { return dual ? (n_copied - t + 1) / 2 : max(0, min(n_copied, (sh->hi[t] + BN - 1) / BN - j0)); };
  auto copy_of = [&](int t, int i) { return dual ? 2 * i + t : i; };
  int copies = 0;                        // tiles of the ring that the copy warp has asked for

  if (warp == kCopyWarp) {
    bool ok = true;
    auto wait_empty = [&](int n) {
      bool mine = true;
      if (n >= C::kStages && lane == 0) mine = mbar_wait_or_abort(bar(C::kEmpty + n % C::kStages), (n / C::kStages - 1) & 1, s_abort);
      return __all_sync(0xffffffffu, mine) != 0;
    };
    if (MODE == kPrompt) {
      for (int n = 0; n < 2 * n_copied && ok; ++n) {
        ok = wait_empty(n);
        if (!ok) break;
        const uint32_t full = bar(C::kFull + n % C::kStages), dst = sRing + (n % C::kStages) * C::kTile;
        if (lane == 0) mbar_expect(full, C::kTile);
        __syncwarp();
        if (lane < C::kHalves) tma_load_box(dst + lane * C::kBlock, (n & 1) ? &map_v : &map_k, kvh * D + 64 * lane, t0 + (j0 + (n >> 1)) * BN, full);
        copies = n + 1;
      }
    } else {
      // lane i brings page i % 16 of a tile, columns 64 (i / 16) ..; its number is read one tile ahead
      const int ps = a.page_size, slot = lane & 15, half = lane >> 4;
      const uint32_t bytes = (uint32_t)ps * 128u;
      auto page_of = [&](int c) {
        const int key = (j0 + c) * BN + slot * ps;
        if (c >= n_copied || half >= C::kHalves || slot * ps >= BN || key >= hi || key + ps <= lo) return -1;
        const int page = table[key / ps];
        if (page >= 0 && page < a.n_pages) return page;
        report(a.status, kBadPage);
        return -1;
      };
      int page_next = page_of(0);
      for (int c = 0; c < n_copied && ok; ++c) {
        const int page = page_next;
        page_next = page_of(c + 1);
        const uint32_t n_pages = __popc(__ballot_sync(0xffffffffu, page >= 0));
        for (int kv = 0; kv < 2; ++kv) {
          const int n = 2 * c + kv;
          ok = wait_empty(n);
          if (!ok) break;
          const uint32_t full = bar(C::kFull + n % C::kStages), dst = sRing + (n % C::kStages) * C::kTile;
          if (lane == 0) mbar_expect(full, n_pages * bytes);
          __syncwarp();
          if (page >= 0) tma_load_box(dst + half * C::kBlock + slot * bytes, kv ? &map_v : &map_k, 64 * half, (page * a.nkv + kvh) * ps, full);
          copies = n + 1;
        }
      }
    }
  } else if (warp >= kIssueWarp) {
    const bool elected = elect_one();
    const int t = __shfl_sync(0xffffffffu, warp - kIssueWarp, 0), n = __shfl_sync(0xffffffffu, n_of(t), 0), all = __shfl_sync(0xffffffffu, n_copied, 0);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), d_s = tm + t * BN, a_p = C::kPlaceForP ? tm + C::kColP + t * 64 : d_s, d_o = tm + C::kColO + t * D;
    constexpr uint32_t kIdescS = mma_idesc(BM, BN, false), kIdescO = mma_idesc(BM, D, true);
    const uint64_t dq = make_desc(sQ + (dual ? 0 : t) * C::kTile), dk0 = make_desc(sRing);
    const uint64_t dv0 = (dk0 & ~((uint64_t)0x3fff << 16)) | ((uint64_t)(C::kBlock >> 4) << 16);      // 64 columns of V apart: a block
    bool ok = true;
    auto wait = [&](int which, int phase) {
      if (ok) ok = mbar_wait_or_abort(bar(which), phase & 1, s_abort);
      ok = __all_sync(0xffffffffu, ok) != 0;
      return ok;
    };
    auto scores = [&](int i) {
      const int slot = 2 * copy_of(t, i), st = slot % C::kStages;
      if (!wait(C::kFull + st, slot / C::kStages)) return;
      fence_after_sync();
      if (elected) {
        const uint64_t dk = dk0 + (uint64_t)(st * (C::kTile >> 4));
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t step = (k >> 2) * (C::kBlock >> 4) + 2 * (k & 3);
          mma_bf16(d_s, dq + step, dk + step, kIdescS, k > 0);
        }
        mma_commit(bar(C::kEmpty + st));
        mma_commit(bar(C::kS + t));
      }
      __syncwarp();
    };
    if (n > 0) scores(0);
    for (int i = 0; i < n && ok; ++i) {
      if (C::kPlaceForP && i + 1 < n && wait(C::kRead + t, i)) scores(i + 1);
      const int slot = 2 * copy_of(t, i) + 1, st = slot % C::kStages;
      if (!wait(C::kP + t, i) || !wait(C::kFull + st, slot / C::kStages)) break;
      fence_after_sync();
      if (elected) {
        const uint64_t dv = dv0 + (uint64_t)(st * (C::kTile >> 4));
#pragma unroll
        for (int k = 0; k < BN / 16; ++k) mma_bf16_a_tmem(d_o, a_p + k * 8, dv + (uint64_t)(k * (2048 >> 4)), kIdescO, (k > 0 || i > 0) ? 1u : 0u);
        mma_commit(bar(C::kEmpty + st));
        mma_commit(bar(C::kPv + t));
      }
      __syncwarp();
      if (!C::kPlaceForP && i + 1 < n && wait(C::kPv + t, i)) scores(i + 1);
    }
    if (!dual)                            // tiles that only the other query tile uses: free for this one, each once it is there
      for (int s = 2 * n; s < 2 * all && ok; ++s)
        if (wait(C::kFull + s % C::kStages, s / C::kStages) && lane == 0) mbar_arrive(bar(C::kEmpty + s % C::kStages));
  } else {
    // --- the softmax groups ---
    const int t = my_tile, n = n_of(t);
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + t * BN, t_p = C::kPlaceForP ? t_lane + C::kColP + t * 64 : t_s, t_o = t_lane + C::kColO + t * D;
    const int lim_warp = __reduce_min_sync(0xffffffffu, lim);
    const bool busy = (my_index & ~31) < rows;               // this warp has rows (the others' P may be anything: rows do not meet)
    auto on_edge = [&](int g, int key0) { return key0 + BN > sh->lim_min[g] || key0 < lo; };
    bool ok = true;
    auto wait = [&](int which, int phase) {
      if (ok) ok = mbar_wait_or_abort(bar(which), phase & 1, s_abort);
      ok = __all_sync(0xffffffffu, ok) != 0;
      return ok;
    };
    float m_ref = -INFINITY, l = 0.f;
    for (int i = 0; i < n; ++i) {
      const int key0 = (j0 + copy_of(t, i)) * BN;
      if (!wait(C::kS + t, i)) break;
      fence_after_sync();
      if (busy) {
        float s[BN];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + 32 * c, s + 32 * c);
        tmem_ld_wait();
        if (C::kPlaceForP) {
          fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::kRead + t));
        }
        if (key0 + BN > lim_warp || key0 < lo) {
          const int from = lo - key0, to = lim - key0;
#pragma unroll
          for (int c = 0; c < BN; ++c) s[c] = (c >= from && c < to) ? s[c] : -INFINITY;
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < BN; ++c) m4[c & 3] = fmaxf(m4[c & 3], s[c]);
        const float m_tile = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * a.scale_log2;
        const bool move = m_tile > m_ref + kMoveFrom;
        if (__any_sync(0xffffffffu, move)) {
          const float alpha = move ? fast_exp2(m_ref - m_tile) : 1.f;       // 0 on the first tile
          if (move) m_ref = m_tile;
          l *= alpha;
          if (i > 0) {
            if (!wait(C::kPv + t, i - 1)) break;
            fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float o[32];
              tmem_ld32(t_o + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= alpha;
              tmem_st32(t_o + c, o);
            }
            tmem_st_wait();
          }
        }
        const Two scale2(a.scale_log2), minus2(m_ref == -INFINITY ? 0.f : -m_ref);
        Two sum2[2] = {Two(0.f), Two(0.f)};
        if (C::kPlaceForP && i > 0 && !wait(C::kPv + t, i - 1)) break;      // the tile before's P has been used
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t packed[BN / 4];
#pragma unroll
          for (int c = 0; c < BN / 4; ++c) {
            float x, y;
            fma2(Two(s[64 * h + 2 * c], s[64 * h + 2 * c + 1]), scale2, minus2).get(x, y);
            x = fast_exp2(x);
            y = fast_exp2(y);
            sum2[c & 1] = sum2[c & 1] + Two(x, y);
            const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
            packed[c] = *reinterpret_cast<const uint32_t*>(&b);
          }
          tmem_st32(t_p + 32 * h, reinterpret_cast<const float*>(packed));
        }
        float x, y;
        (sum2[0] + sum2[1]).get(x, y);
        l += x + y;
        tmem_st_wait();
      } else if (C::kPlaceForP) {
        if (lane == 0) mbar_arrive(bar(C::kRead + t));
        if (i > 0 && !wait(C::kPv + t, i - 1)) break;                       // (its arrival below must not count for the tile before)
      }
      if (on_edge(t, key0)) {
        // rows of V that nobody sees, and values that are no numbers, become zeros
        const int slot = 2 * copy_of(t, i) + 1, st = slot % C::kStages;
        if (!wait(C::kFull + st, slot / C::kStages)) break;
        uint8_t* v_tile = smem + 2 * C::kTile + st * C::kTile;
        for (int piece = tid & 127; piece < BN * D / 8; piece += 128) {
          const int r = piece >> 3 & (BN - 1), key = key0 + r;
          uint4* p = reinterpret_cast<uint4*>(v_tile + (piece >> 10) * C::kBlock + swz(r, piece & 7));
          if (key < lo || key >= hi) {
            *p = make_uint4(0, 0, 0, 0);
            continue;
          }
          uint4 w = *p;
          if (not_finite2(w.x) || not_finite2(w.y) || not_finite2(w.z) || not_finite2(w.w)) {
            *reinterpret_cast<volatile int*>(&sh->bad) = 1;
            __threadfence_block();
            uint32_t* e = &w.x;
            for (int k = 0; k < 4; ++k) {
              if ((e[k] & 0x7f80u) == 0x7f80u) e[k] &= 0xffff0000u;
              if ((e[k] & 0x7f800000u) == 0x7f800000u) e[k] &= 0xffffu;
            }
            *p = w;
          }
        }
        fence_async_proxy();
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::kP + t));
    }
    if (n > 0) wait(C::kPv + t, n - 1);
    fence_after_sync();
    const bool mine = my_index < rows, direct = a.n_rec <= 1;
    const bool fix = *reinterpret_cast<volatile int*>(&sh->bad) != 0;
    if (ok && busy) {
      const size_t record = ((size_t)my_token * a.nq + my_head) * a.n_rec + a.rec0 + (dual ? 2 * blockIdx.z + t : blockIdx.z);
      const float inv = l != 0.f ? 1.f / l : 0.f;                        // (a row that sees no key: zeros)
      if (!direct && mine) {
        a.part_ml[2 * record] = m_ref;
        a.part_ml[2 * record + 1] = l;
      }
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        float o[32];
        __syncwarp();
        if (n > 0) {
          tmem_ld32(t_o + c0, o);
          tmem_ld_wait();
        }
        if (!mine) continue;
        if (n == 0 || l == 0.f) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        } else if (fix) {
          // what this row does see of the values that were taken out
          for (int i = 0; i < n; ++i) {
            const int key0 = (j0 + copy_of(t, i)) * BN;
            if (!on_edge(0, key0) && !on_edge(1, key0)) continue;
            for (int key = max(key0, lo); key < min(key0 + BN, lim); ++key) {
              const elem_t *kr, *vr;
              key_rows<MODE>(a, table, t0, kvh, key, kr, vr);
              if (!vr) continue;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float v = __bfloat162float(vr[c0 + e]);
                if (!isfinite(v)) o[e] += v;
              }
            }
          }
        }
        if (direct) {
          uint4* dst = reinterpret_cast<uint4*>(a.out + (long long)my_token * a.ld_out + my_head * D + c0);
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(o[e + 2 * k] * inv, o[e + 2 * k + 1] * inv);
              w[k] = *reinterpret_cast<const uint32_t*>(&b);
            }
            dst[e / 8] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else if (l != 0.f) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + record * D + c0);
#pragma unroll
          for (int e = 0; e < 8; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
    }
  }

  fence_before_sync();
  __syncthreads();
  if (*s_abort) {
    // copies that were asked for land before the shared memory is given back (each wait bounded on its own)
    if (warp == kCopyWarp && lane == 0)
      for (int n = max(0, copies - C::kStages); n < copies; ++n) mbar_wait(bar(C::kFull + n % C::kStages), (n / C::kStages) & 1);
    if (tid == 0) report(a.status, kGaveUp);
    __syncthreads();
  }
  if (warp == kIssueWarp) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

template <int D, int MODE>
int launch_one(const PackedArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, dim3 grid, int dual, cudaStream_t stream, const char* who) {
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(ERB_ERR_CUDA, "%s: no device", who);
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attention_packed_tc_kernel<D, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<D>::kSmemBytes);
    if (e != cudaSuccess) return fail(ERB_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    configured[dev] = true;
  }
  if (grid.y > 65535u || grid.z > 65535u) return fail(ERB_ERR_UNSUPPORTED, "%s: too many rows", who);
  launch_chained(attention_packed_tc_kernel<D, MODE>, grid, dim3(kThreads), Cfg<D>::kSmemBytes, stream, mk, mv, a, dual);
  return check_launch(who);
}

template <int MODE>
int launch_tc(const PackedArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, dim3 grid, int dual, cudaStream_t stream, const char* who) {
  return a.D == 64 ? launch_one<64, MODE>(a, mk, mv, grid, dual, stream, who) : launch_one<128, MODE>(a, mk, mv, grid, dual, stream, who);
}

// A request's own keys by the kernels for few rows: rows 1: one token a request (or one after the other), up to 16 query heads a kv head.
template <int D>
int launch_few(const PackedArgs& a, bool one_token, int early, cudaStream_t stream, const char* who) {
  auto kern = one_token ? attention_own_token_kernel<D> : attention_own_rows_kernel<D>;
  const int bytes = one_token ? (int)FewSmem<D>::kBytes : (int)FewRowsSmem<D>::kBytes;
  static bool configured[64][2] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(ERB_ERR_CUDA, "%s: no device", who);
  if (!configured[dev][one_token]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return fail(ERB_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    configured[dev][one_token] = true;
  }
  const long long tiles = one_token ? a.n_seqs : (long long)a.n_tokens * (a.nq / a.nkv) / kFewRows + a.n_seqs;
  if (tiles > 65535 || a.pieces > 65535) return fail(ERB_ERR_UNSUPPORTED, "%s: too many rows", who);
  launch_chained(kern, dim3(a.nkv, (unsigned)tiles, a.pieces), dim3(kFewThreads), bytes, stream, a, early);
  return check_launch(who);
}

bool aligned(const void* p, long long ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

}  // namespace

// The arguments of erb_attention_prompt (attention_packed.cu); heads of 64 or 128, rows and their strides on 16-byte boundaries.
ERB_EXPORT int erb_attention_prompt_tc(const void* q, long long ld_q, const void* k, long long ld_k, const void* v, long long ld_v,
                                       const int* seq_starts, int n_seqs, int n_tokens, void* out, long long ld_out, int nq, int nkv,
                                       int head_dim, float scale, int* status, void* stream) {
  if (n_seqs <= 0 || n_tokens <= 0) return ERB_OK;
  if (nq <= 0 || nkv <= 0 || nq % nkv || !status || !(scale > 0.f)) return fail(ERB_ERR_ARG, "attention_prompt_tc: bad sizes");
  if ((head_dim != 64 && head_dim != 128) || !aligned(q, ld_q) || !aligned(k, ld_k) || !aligned(v, ld_v) || !aligned(out, ld_out))
    return fail(ERB_ERR_UNSUPPORTED, "attention_prompt_tc: takes heads of 64 and 128 with rows on 16-byte boundaries");
  PackedArgs a = {};
  a.q = (const elem_t*)q; a.k = (const elem_t*)k; a.v = (const elem_t*)v; a.out = (elem_t*)out;
  a.ld_q = ld_q; a.ld_k = ld_k; a.ld_v = ld_v; a.ld_out = ld_out; a.page_size = 1;
  a.seq_starts = seq_starts; a.n_seqs = n_seqs; a.n_tokens = n_tokens; a.nq = nq; a.nkv = nkv; a.D = head_dim;
  a.scale_log2 = scale * 1.4426950408889634f; a.n_rec = 1; a.pieces = 1; a.status = status;
  CUtensorMap mk, mv;
  int rc;
  if ((rc = rows_map(&mk, k, n_tokens, nkv * head_dim, ld_k, BN, "attention_prompt_tc")) ||
      (rc = rows_map(&mv, v, n_tokens, nkv * head_dim, ld_v, BN, "attention_prompt_tc")))
    return rc;
  const long long tiles = (long long)n_tokens * (nq / nkv) / (2 * BM) + n_seqs;      // (a sequence has at most one block that is not full)
  return launch_tc<kPrompt>(a, mk, mv, dim3(nkv, (unsigned)min(tiles, 1LL << 20), 1), 0, (cudaStream_t)stream, "attention_prompt_tc");
}

// The arguments of erb_attention_shared_prefix (attention_packed.cu); heads of 64 or 128, rows, their strides and the pools on 16-byte
// boundaries, pages of 8 to 128 tokens, a power of two.  prefix_dual: blocks own 128 rows and leave two records each, so that prefix_pieces
// is twice the blocks' pieces.  own: the kernel for a request's own keys (kOwnMany: this file's for many rows; kOwnToken, kOwnRows:
// packed_few.cuh's, which join the records themselves where own_pieces is 1).
ERB_EXPORT int erb_attention_shared_prefix_tc(const void* q, long long ld_q, const void* k_pages, const void* v_pages, int n_pages, int page_size,
                                              const int* prefix_pages, int prefix_len, const int* tables, int table_ld, const int* seq_starts,
                                              const int* positions, int n_seqs, int n_tokens, void* out, long long ld_out, int nq, int nkv,
                                              int head_dim, float scale, int prefix_pieces, int own_pieces, int piece_keys, int prefix_dual,
                                              int own, float* part_o, float* part_ml, int* status, void* stream) {
  if (n_seqs <= 0 || n_tokens <= 0) return ERB_OK;
  if (nq <= 0 || nkv <= 0 || nq % nkv || !status || n_pages <= 0 || prefix_len < 0 || table_ld <= 0 || prefix_pieces < (prefix_len > 0 ? 1 : 0) ||
      own_pieces < 1 || piece_keys <= 0 || !(scale > 0.f) || prefix_pieces > 64 ||
      (prefix_dual && prefix_pieces % 2) || own < kOwnMany || own > kOwnRows || (own == kOwnToken && nq / nkv > 16))
    return fail(ERB_ERR_ARG, "attention_shared_prefix_tc: bad sizes");
  if ((head_dim != 64 && head_dim != 128) || !aligned(q, ld_q) || !aligned(out, ld_out) || !aligned(k_pages, 0) || !aligned(v_pages, 0) ||
      page_size < 8 || page_size > BN || (page_size & (page_size - 1)) || (unsigned long long)n_pages * nkv * page_size > 0x7fffffffull)
    return fail(ERB_ERR_UNSUPPORTED, "attention_shared_prefix_tc: takes heads of 64 and 128, 16-byte boundaries, pages of 8 to 128 tokens (a power of two)");
  const int n_rec = (prefix_len > 0 ? prefix_pieces : 0) + own_pieces;
  if (n_rec > 1 && (!part_o || !part_ml || ((uintptr_t)part_o & 15))) return fail(ERB_ERR_ARG, "attention_shared_prefix_tc: pieces need scratch");
  PackedArgs a = {};
  a.q = (const elem_t*)q; a.k = (const elem_t*)k_pages; a.v = (const elem_t*)v_pages; a.out = (elem_t*)out;
  a.ld_q = ld_q; a.ld_out = ld_out; a.n_pages = n_pages; a.page_size = page_size; a.tables = tables; a.table_ld = table_ld;
  a.prefix_pages = prefix_pages; a.prefix_len = prefix_len; a.seq_starts = seq_starts; a.positions = positions;
  a.n_seqs = n_seqs; a.n_tokens = n_tokens; a.nq = nq; a.nkv = nkv; a.D = head_dim; a.scale_log2 = scale * 1.4426950408889634f;
  a.part_o = part_o; a.part_ml = part_ml; a.n_rec = n_rec; a.status = status; a.piece_keys = piece_keys;
  cudaStream_t s = (cudaStream_t)stream;
  const char* who = "attention_shared_prefix_tc";
  const unsigned long long pool_rows = (unsigned long long)n_pages * nkv * page_size;
  CUtensorMap mk, mv;
  int rc;
  if ((rc = rows_map(&mk, k_pages, pool_rows, head_dim, head_dim, page_size, who)) || (rc = rows_map(&mv, v_pages, pool_rows, head_dim, head_dim, page_size, who)))
    return rc;
  const long long rows = (long long)n_tokens * (nq / nkv);
  if (prefix_len > 0) {
    a.rec0 = 0;
    a.pieces = prefix_dual ? prefix_pieces / 2 : prefix_pieces;
    if ((rc = launch_tc<kPrefix>(a, mk, mv, dim3(nkv, (unsigned)min(rows / (prefix_dual ? BM : 2 * BM) + 1, 1LL << 20), a.pieces), prefix_dual, s, who))) return rc;
  }
  a.rec0 = prefix_len > 0 ? prefix_pieces : 0;
  a.pieces = own_pieces;
  if (own == kOwnMany) {
    if ((rc = launch_tc<kOwn>(a, mk, mv, dim3(nkv, (unsigned)min(rows / (2 * BM) + n_seqs, 1LL << 20), a.pieces), 0, s, who)) || n_rec <= 1) return rc;
  } else {
    rc = head_dim == 64 ? launch_few<64>(a, own == kOwnToken, prefix_len > 0, s, who) : launch_few<128>(a, own == kOwnToken, prefix_len > 0, s, who);
    if (rc || own_pieces == 1) return rc;
  }
  const long long blocks = ((long long)n_tokens * nq + 3) / 4;
  if (blocks > 0x7fffffffLL) return fail(ERB_ERR_UNSUPPORTED, "%s: too many rows", who);
  launch_chained(attention_merge_kernel, dim3((unsigned)blocks), dim3(128), 0, s, (const float*)part_o, (const float*)part_ml, (elem_t*)out, ld_out,
                 seq_starts, n_seqs, n_tokens, nq, head_dim, n_rec);
  return check_launch(who);
}
