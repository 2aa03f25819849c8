// Attention over packed whole prompts, and of a batch behind a shared prefix (what the calls are: packed.cuh), on the 5th-generation tensor
// cores (tcgen05 + TMEM): bfloat16, heads of 64 and 128, cache pages of 8 to 128 tokens (a power of two).
//
// A piece of work is up to 256 rows of one kv head, (token, head of its group) pairs, as two query tiles A and B of up to 128 rows, and a
// walk over its keys in tiles of 128.  Every byte of K and V that reaches shared memory serves all its rows; with G query heads a kv head
// a prompt's piece spans 256 / G tokens, so little of the last tile on the diagonal is hidden.  (Rows that all fit one tile leave the other idle:
// with the same rows in both and every other key tile each, the ring is too short for two walks, and 128 rows over 16,384 keys took 40 us, not 32.)
//
// One block a multiprocessor takes pieces in turn, longest first (forwards and backwards through the list, so that the blocks' sums are
// alike).  Its warps work by role, each as far ahead as the barriers let it, so that a piece's first copies and products run while the
// one before is being finished:
//
//   warp 10 (copy)      finds the pieces and describes them to the others; brings Q tiles, and K and V tiles in turn into one ring of
//                       shared memory, by TMA tensor copies (128-byte swizzle): from the pages, one copy per page and 64 columns, or from
//                       rows beside the queries
//   warps 8, 9 (issue)  S_t = Q_t K^T (M 128, N 64) and O_t += P_t V (M 128, N D, K 64, P from TMEM), a warp for each query tile: a product
//                       starts some 300 clocks after what it waits for, which one warp for both would leave the tensor cores idle
//   warps 0-3, 4-7      softmax of tile A and of tile B: a thread owns a row, takes 64 of its scores into registers, and writes P back
//                       rounded to bfloat16 (the second product's operand type; the sum of P is taken before that rounding, in float)
//   warp 11 (look)      looks over the values of tiles with hidden keys (below)
//
// A row's reference maximum moves only when a tile's maximum is 2^8 above it; O is rescaled in TMEM then.  P is a floating-point number, so
// a reference that is low by eight powers of two costs no precision.  (References of scores past 2^20: kFarScore in packed.cuh.  The look for
// them costs 1 to 2 %: prompts of 8,192 tokens of 32 heads of 64 409 -> 415 us, of 32 on 8 of 128 481 -> 483.)
//
// A tile's keys are worked on in two halves of 64, each with a place of its own for its scores in TMEM (512 columns: S 2 x 2 x 64, O 2 x D),
// and P takes the place of the scores it was made of: the next tile's scores of a half are made behind P V of this tile's, while the softmax
// is at the other half.
//
// Hidden keys.  Scores are masked where some row of a warp sees fewer keys than its tile has.  P is then zero, but zero times a value
// that is no number would spoil rows that do not see it; so the values of such tiles are looked over before they are used: rows of V that
// nobody sees become zeros, and an infinity or NaN that only some rows see becomes zero and is added to exactly those rows at the end.
//
// What bounds it: a half step's chain, scores -> softmax -> P V, that two query tiles only partly hide from each other (polynomial exponentials,
// sixteen softmax warps and smaller chunks of P made it slower), and the tail of uneven pieces.  8,192 tokens, 32 query heads on 8 of 128: 483 us,
// 1.14 PFLOP/s, 0.69 of a library product's rate (550 us and 0.60 called without a pause, under the power limit; in steps as they were built: a block
// for each piece 700, one issuing warp 583, one tile of 128 keys at a time 545, as it is 489; CUDA cores 20,650); of heads of 64, 32 of them, 415 us.
// 23 prompts of up to 2,001 tokens, 32 heads of 64: 153 us.  16,384 keys of 8 heads of 128 before 1 row 27 us (2.5 TB/s), 8 30, 64 45, with the
// pieces' records written and joined.
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
constexpr int kSoftmaxWarps = 8, kIssueWarp = 8, kCopyWarp = 10, kLookWarp = 11, kThreads = 384;
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
constexpr float kMoveFrom = 8.f;          // powers of two by which a tile's maximum is above the reference before that moves
constexpr int kOwnMany = 0, kOwnToken = 1, kOwnRows = 2;      // kernels for a request's own keys
constexpr int kGaveUp = 9100000;          // status code of a wait that ran out
constexpr int kPieces = 4;                // descriptions of pieces of work on their way

template <int D> struct Cfg {
  static constexpr int kHalves = D / 64;                         // blocks of 64 columns (128 bytes of a row)
  static constexpr uint32_t kBlock = BM * 128, kTile = kHalves * kBlock;
  static constexpr int kStages = D == 64 ? 8 : 4;                // tiles of K or V in the ring (a power of two)
  static constexpr int kSets = D == 64 ? 2 : 1;                  // pairs of Q tiles
  static constexpr uint32_t kColO = 256;
  static constexpr uint32_t kOutBytes = 2048;                    // a softmax warp's place for results on their way out: 32 rows of 64 bytes
  static_assert(kStages % 2 == 0, "a place of the ring holds keys or values, never both");
  // barriers: ring full and empty; descriptions full and empty; a ring place's values looked over; per query tile: queries there and used;
  // per query tile t and half u of a tile's keys, at + 2 u + t: scores there, P written, P V done
  static constexpr int kFull = 0, kEmpty = kStages, kTold = 2 * kStages, kTaken = kTold + kPieces, kClean = kTaken + kPieces, kQ = kClean + kStages,
                       kQUsed = kQ + 2 * kSets, kS = kQUsed + 2 * kSets, kP = kS + 4, kPv = kS + 8, kNumBars = kS + 12;
  static constexpr uint32_t kRing = 2 * kSets * kTile, kSmemTiles = kRing + kStages * kTile, kSmemOut = kSmemTiles + kSoftmaxWarps * kOutBytes;
  static constexpr uint32_t kSmemBytes = kSmemOut + 8 * kNumBars + 16 + kPieces * 64 + 1024;
};

// A piece of work: rows r0 .. r0 + rows of the (token, head) pairs of the tokens from t0 on, key tiles j0 .. j0 + copied.
struct Piece {
  int seq, t0, token0, rows;      // token0: the first row's token
  int kvh, part, j0, copied;
  int lo, hi;                     // keys that any row sees lie in [lo, hi)
  int n[2], least[2];             // per query tile: key tiles it takes, the smallest number of keys one of its rows sees
  int bad;                        // some value that only some rows see is no number
  int more;                       // 0: there is no further piece
};
static_assert(sizeof(Piece) <= 64, "a description's place");

// acc + 0 * w for eight values: stays zero unless one of them is no number.
__device__ __forceinline__ void gather_not_finite(__nv_bfloat162& acc, const uint4& w) {
  const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
  acc = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.x), zero, acc);
  acc = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.y), zero, acc);
  acc = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.z), zero, acc);
  acc = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.w), zero, acc);
}

// Some tries of a phase, without a look at anything else: a wait that finds its phase complete costs a try and a vote.
__device__ __forceinline__ bool mbar_try_some(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .u32 n;\n\tmov.u32 n, 0;\n"
      "TRY_AGAIN:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra TRY_DONE;\n\t"
      "add.u32 n, n, 1;\n\tsetp.lt.u32 p, n, 64;\n\t@p bra TRY_AGAIN;\n\tsetp.ne.u32 p, n, n;\n"
      "TRY_DONE:\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// The rest of a wait: until the phase is there, another warp has given up, or the limit is reached.  The same answer for every lane.
__device__ __forceinline__ bool wait_long(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t i = 0; i < kSpinLimit / 64; ++i) {
    if (__all_sync(0xffffffffu, mbar_try_some(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
  }
  *abort_flag = 1;
  return false;
}

// The largest of three, NaN if one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

template <int D, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
attention_packed_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           const PackedArgs a) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const uint32_t sQ = base, sRing = base + C::kRing, bars = base + C::kSmemOut;
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + C::kSmemOut + 8 * C::kNumBars);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::kSmemOut + 8 * C::kNumBars + 8);
  auto bar = [&](int which) { return bars + 8u * (uint32_t)which; };
  auto piece_at = [&](int k) { return reinterpret_cast<Piece*>(smem + C::kSmemOut + 8 * C::kNumBars + 16 + (k % kPieces) * 64); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.nq / a.nkv, RT = BM / G * G, per_piece = 2 * RT;      // rows of a query tile (whole tokens), of a piece

  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) { mbar_init(bar(C::kFull + s), 1); mbar_init(bar(C::kEmpty + s), 2); mbar_init(bar(C::kClean + s), 1); }
    for (int k = 0; k < kPieces; ++k) { mbar_init(bar(C::kTold + k), 1); mbar_init(bar(C::kTaken + k), kSoftmaxWarps + 3); }
    for (int t = 0; t < 2; ++t) {
      for (int s = 0; s < C::kSets; ++s) { mbar_init(bar(C::kQ + 2 * s + t), 1); mbar_init(bar(C::kQUsed + 2 * s + t), 1); }
      for (int u = 0; u < 2; ++u) {
        mbar_init(bar(C::kS + 2 * u + t), 1);
        mbar_init(bar(C::kP + 2 * u + t), 4);
        mbar_init(bar(C::kPv + 2 * u + t), 1);
      }
    }
    *s_abort = 0;
    mbar_init_fence();
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *s_tmem;
  const bool early = MODE == kOwn && a.early;
  if (!early) chain_wait();

  bool ok = true;                        // the same for a whole warp
  auto wait = [&](int which, int phase) {
    if (ok && !__all_sync(0xffffffffu, mbar_try_some(bar(which), phase & 1))) ok = wait_long(bar(which), phase & 1, s_abort);
    return ok;
  };
  auto on_edge = [&](const Piece& p, int c) {          // some row sees only some of the tile's keys
    const int key0 = (p.j0 + c) * BN;
    return key0 < p.lo || key0 + BN > min(p.least[0], p.least[1]);
  };
  auto taken = [&](int k) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(C::kTaken + k % kPieces));
  };
  int copies = 0;                        // tiles of the ring, Q tiles that the copy warp has asked for
  int copies_q[2] = {0, 0};

  // The softmax warps hold a row's scores in registers; the four others give theirs up for it (together no more than the block was
  // launched with, 384 x 168: the launch looks).
  if (warp >= kSoftmaxWarps) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp == kCopyWarp) {
    // ---- finds the pieces of this block, describes them, and brings their tiles ----
    const int code = __ldcg(a.status);
    const int first = MODE == kPrefix ? __ldcg(a.seq_starts) : 0, end = MODE == kPrefix ? __ldcg(a.seq_starts + a.n_seqs) : 0;
    long long total;
    if (code >= 1000000 && code != kBadPage && code != kBadStarts) {        // an earlier block gave up: do not pile on
      *s_abort = 1;
      ok = false;
    }
    if (MODE == kPrefix) {
      if (first < 0 || end > a.n_tokens) {
        if (lane == 0) report(a.status, kBadStarts);
        total = 0;
      } else {
        total = ((long long)max(0, end - first) * G + per_piece - 1) / per_piece;
      }
    }
    const TileList list(a.seq_starts, MODE == kPrefix ? 0 : a.n_seqs, G, per_piece);
    if (MODE != kPrefix) total = list.total;
    total = min(total * a.nkv * a.pieces, 0x7fffffffLL - (long long)gridDim.x);        // (the launch refuses more)
    int n_told = 0;
    for (int round = 0; ok; ++round) {
      const int base_index = round * (int)gridDim.x, index = base_index + (int)((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      Piece p = {};
      p.more = base_index < total;
      if (p.more) {
        if (index >= total) continue;
        const int rest = index / a.nkv;
        p.kvh = index - rest * a.nkv;
        int tile = rest / a.pieces, len;
        p.part = rest - tile * a.pieces;
        if (MODE == kPrefix) {
          p.t0 = first;
          len = end - first;
        } else {
          list.find(tile, p.seq, tile);
          if (p.seq < 0) continue;
          if (p.seq < 32) {
            p.t0 = __shfl_sync(0xffffffffu, list.start_of_lane, p.seq);
            len = __shfl_sync(0xffffffffu, list.len_of_lane, p.seq);
          } else {
            p.t0 = __ldcg(a.seq_starts + p.seq);
            len = __ldcg(a.seq_starts + p.seq + 1) - p.t0;
          }
          if (p.t0 < 0 || p.t0 + (long long)len > a.n_tokens) {
            if (lane == 0) report(a.status, kBadStarts);
            continue;
          }
        }
        const int r0 = tile * per_piece, token_tile = RT / G;                  // (tokens times G is below 2^30)
        p.rows = min(per_piece, len * G - r0);
        p.token0 = p.t0 + tile * 2 * token_tile;
        // the keys that the rows of each query tile see
        int most[2] = {0, 0};
        p.least[0] = p.least[1] = INT_MAX;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int before = t * token_tile, n_tokens = max(0, min(token_tile, p.t0 + len - p.token0 - before));
          if (MODE == kPrompt) {
            if (n_tokens > 0) {
              p.least[t] = p.token0 - p.t0 + before + 1;
              most[t] = p.least[t] + n_tokens - 1;
            }
          }
          for (int i0 = 0; MODE != kPrompt && i0 < n_tokens; i0 += 32) {
            int lim = 0;
            const bool mine = i0 + lane < n_tokens;
            if (mine) {
              lim = max(0, min(__ldcg(a.positions + p.token0 + before + i0 + lane), INT_MAX - 1) + 1);
              if (MODE == kPrefix) lim = min(lim, a.prefix_len);
              else if (lim > (long long)a.table_ld * a.page_size) { report(a.status, kBadPage); lim = a.table_ld * a.page_size; }
            }
            most[t] = max(most[t], __reduce_max_sync(0xffffffffu, lim));
            p.least[t] = min(p.least[t], __reduce_min_sync(0xffffffffu, mine ? lim : INT_MAX));
          }
        }
        p.lo = MODE == kOwn ? a.prefix_len : 0;
        p.hi = max(most[0], most[1]);
        const int j_first = p.lo / BN, j_end = p.hi > p.lo ? (p.hi + BN - 1) / BN : j_first;
        int j1 = j_end;
        p.j0 = j_first;
        if (MODE != kPrompt) {
          const int per = MODE == kOwn ? (a.piece_keys + BN - 1) / BN : (j_end - j_first + a.pieces - 1) / a.pieces;
          p.j0 = (int)min((long long)j_end, j_first + (long long)p.part * per);
          if (MODE == kPrefix || p.part + 1 < a.pieces) j1 = min(j_end, p.j0 + per);
        }
        p.copied = j1 - p.j0;
#pragma unroll
        for (int t = 0; t < 2; ++t) p.n[t] = max(0, min(p.copied, (most[t] + BN - 1) / BN - p.j0));
        p.copied = max(p.n[0], p.n[1]);
      }
      if (n_told >= kPieces && !wait(C::kTaken + n_told % kPieces, n_told / kPieces - 1)) break;
      if (lane == 0) {
        *piece_at(n_told) = p;
        mbar_arrive(bar(C::kTold + n_told % kPieces));
      }
      ++n_told;
      if (!p.more) break;
      // queries: whole tokens, the heads of the group in order (tokens behind the sequence's last one are rows that nobody stores)
      for (int t = 0; t < 2; ++t) {
        if (p.n[t] == 0) continue;
        const int set = copies_q[t] % C::kSets, use = copies_q[t] / C::kSets;
        if (use > 0 && !wait(C::kQUsed + 2 * set + t, use - 1)) break;
        if (lane == 0) mbar_expect(bar(C::kQ + 2 * set + t), C::kHalves * RT * 128);
        __syncwarp();
        if (lane < C::kHalves)
          tma_load_3d(sQ + (2 * set + t) * C::kTile + lane * C::kBlock, &map_q, 64 * lane, p.kvh * G, p.token0 + t * (RT / G), bar(C::kQ + 2 * set + t));
        ++copies_q[t];
      }
      auto wait_empty = [&](int n) { return n < C::kStages ? ok : wait(C::kEmpty + n % C::kStages, n / C::kStages - 1); };
      if (MODE == kPrompt) {
        for (int n = 0; n < 2 * p.copied; ++n) {
          if (!wait_empty(copies)) break;
          const uint32_t full = bar(C::kFull + copies % C::kStages), dst = sRing + (copies % C::kStages) * C::kTile;
          if (lane == 0) mbar_expect(full, C::kTile);
          __syncwarp();
          if (lane < C::kHalves) tma_load_box(dst + lane * C::kBlock, (n & 1) ? &map_v : &map_k, p.kvh * D + 64 * lane, p.t0 + (p.j0 + (n >> 1)) * BN, full);
          ++copies;
        }
      } else {
        // lane i brings page i % 16 of a tile, columns 64 (i / 16) ..; its number is read one tile ahead
        const int* table = MODE == kOwn ? a.tables + (size_t)p.seq * a.table_ld : a.prefix_pages;
        const int ps = a.page_size, slot = lane & 15, half = lane >> 4;
        const uint32_t bytes = (uint32_t)ps * 128u;
        auto page_of = [&](int c) {
          const int key = (p.j0 + c) * BN + slot * ps;
          if (c >= p.copied || half >= C::kHalves || slot * ps >= BN || key >= p.hi || key + ps <= p.lo) return -1;
          const int page = __ldcg(table + key / ps);
          if (page >= 0 && page < a.n_pages) return page;
          report(a.status, kBadPage);
          return -1;
        };
        int page_next = page_of(0);
        for (int c = 0; c < p.copied && ok; ++c) {
          const int page = page_next;
          page_next = page_of(c + 1);
          const uint32_t n_pages = __popc(__ballot_sync(0xffffffffu, page >= 0));
          for (int kv = 0; kv < 2; ++kv) {
            if (!wait_empty(copies)) break;
            const uint32_t full = bar(C::kFull + copies % C::kStages), dst = sRing + (copies % C::kStages) * C::kTile;
            if (lane == 0) mbar_expect(full, n_pages * bytes);
            __syncwarp();
            if (page >= 0) tma_load_box(dst + half * C::kBlock + slot * bytes, kv ? &map_v : &map_k, 64 * half, (page * a.nkv + p.kvh) * ps, full);
            ++copies;
          }
        }
      }
    }
  } else if (warp < kCopyWarp) {
    // ---- the products of a query tile; an elected lane issues, with what a product takes in uniform registers (a shuffle from lane 0 makes them so: a
    // lane that moves its own values there takes sixty clocks a product) ----
    const bool elected = elect_one();
    auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
    const uint32_t tm = uniform(tmem);
    constexpr uint32_t kIdescS = mma_idesc(BM, BN / 2, false), kIdescO = mma_idesc(BM, D, true);
    const uint64_t like = make_desc(0);                        // a descriptor without its address, which is the low 14 bits
    const uint32_t dq0 = uniform(sQ >> 4), dk0 = uniform(sRing >> 4);
    auto desc = [&](uint32_t address) { return like | (uint64_t)address; };
    auto desc_v = [&](uint32_t address) {                      // 64 columns of V apart: a block
      return (like & ~((uint64_t)0x3fff << 16)) | ((uint64_t)(C::kBlock >> 4) << 16) | (uint64_t)address;
    };
    const int t = uniform(warp - kIssueWarp);
    const uint32_t d_s = tm + t * BN, d_o = tm + C::kColO + t * D;        // (P in the first half of its scores' place)
    int ring = 0, steps = 0, queries = 0;                      // ring tiles, steps, Q tiles of the pieces before
    for (int k = 0; wait(C::kTold + k % kPieces, k / kPieces); ++k) {
      const Piece& p = *piece_at(k);
      if (!p.more) break;
      const int n = uniform(p.n[t]), copied = uniform(p.copied), set = queries % C::kSets;
      const uint32_t dq = dq0 + uniform(2 * set + t) * (C::kTile >> 4);
      // scores of half u of step i's keys; their place is free behind P V of the half that was there
      auto scores = [&](int i, int u) {
        const int slot = ring + 2 * i, st = uniform(slot % C::kStages);
        if (!wait(C::kFull + st, slot / C::kStages)) return;
        if (steps + i > 0 && !wait(C::kPv + 2 * u + t, steps + i - 1)) return;
        fence_after_sync();
        const uint32_t dk = dk0 + st * (C::kTile >> 4) + uniform(u) * (64 * 128 >> 4), to = d_s + uniform(u) * 64;
        if (elected) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t step = (k >> 2) * (C::kBlock >> 4) + 2 * (k & 3);
            mma_bf16(to, desc(dq + step), desc(dk + step), kIdescS, k > 0);
          }
          mma_commit(bar(C::kS + 2 * u + t));
          if (u) mma_commit(bar(C::kEmpty + st));
          if (u && i + 1 == n) mma_commit(bar(C::kQUsed + 2 * set + t));
        }
        __syncwarp();
      };
      if (n > 0) {
        wait(C::kQ + 2 * set + t, queries / C::kSets);
        ++queries;
      }
      if (ok && n > 0) scores(0, 0);
      if (ok && n > 0) scores(0, 1);
      for (int i = 0; i < n && ok; ++i) {
        const int slot = ring + 2 * i + 1, st = uniform(slot % C::kStages);
        if (!wait(C::kClean + st, slot / C::kStages)) break;
        const uint32_t dv = dk0 + st * (C::kTile >> 4), more = uniform(i > 0);
#pragma unroll 1
        for (int u = 0; u < 2; ++u) {
          if (!wait(C::kP + 2 * u + t, steps + i)) break;
          fence_after_sync();
          const uint32_t from = dv + uniform(u) * (64 * 128 >> 4), a_p = d_s + uniform(u) * 64, first = uniform(u) | more;
          if (elected) {
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_bf16_a_tmem(d_o, a_p + k * 8, desc_v(from + k * (2048 >> 4)), kIdescO, k > 0 ? 1u : first);
            mma_commit(bar(C::kPv + 2 * u + t));
            if (u) mma_commit(bar(C::kEmpty + st));
          }
          __syncwarp();
          if (i + 1 < n) scores(i + 1, u);
          if (!ok) break;
        }
      }
      // tiles that only the other query tile uses: free for this one, each once it is there
      for (int c = 2 * n; c < 2 * copied && ok; ++c)
        if (wait(C::kFull + (ring + c) % C::kStages, (ring + c) / C::kStages) && lane == 0) mbar_arrive(bar(C::kEmpty + (ring + c) % C::kStages));
      steps += n;
      ring += 2 * copied;
      taken(k);
      if (!ok) break;
    }
  } else {
    // ---- rows of V that nobody sees, and values that are no numbers, become zeros ----
    int ring = 0;
    for (int k = 0; wait(C::kTold + k % kPieces, k / kPieces); ++k) {
      Piece& p = *piece_at(k);
      if (!p.more) break;
      for (int c = 0; c < p.copied; ++c) {
        const int slot = ring + 2 * c + 1, st = slot % C::kStages, key0 = (p.j0 + c) * BN, lo = p.lo, hi = p.hi;
        if (!wait(C::kFull + st, slot / C::kStages)) break;
        uint8_t* v_tile = smem + C::kRing + st * C::kTile;
        if (on_edge(p, c)) {
          // a lane the same piece of every fourth row, eight rows at a time
          auto at = [&](int i) { return reinterpret_cast<uint4*>(v_tile + (i >> 5) * C::kBlock + swz((i & 31) * 4 + (lane >> 3), lane & 7)); };
#pragma unroll 1
          for (int i0 = 0; i0 < 32 * C::kHalves; i0 += 8) {
            uint4 w[8];
            __nv_bfloat162 acc = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int key = key0 + ((i0 + i) & 31) * 4 + (lane >> 3);
              w[i] = *at(i0 + i);
              if (key < lo || key >= hi) *at(i0 + i) = w[i] = make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) gather_not_finite(acc, w[i]);
            if (__low2float(acc) == 0.f && __high2float(acc) == 0.f) continue;
#pragma unroll 1
            for (int i = i0; i < i0 + 8; ++i) {
              uint4 x = *at(i);
              uint32_t* e = &x.x;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                if ((e[q] & 0x7f80u) == 0x7f80u) e[q] &= 0xffff0000u;
                if ((e[q] & 0x7f800000u) == 0x7f800000u) e[q] &= 0xffffu;
              }
              *at(i) = x;
            }
            *reinterpret_cast<volatile int*>(&p.bad) = 1;
          }
          fence_async_proxy();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kClean + st));
      }
      if (!ok) break;
      ring += 2 * p.copied;
      taken(k);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---- the softmax groups ----
    const int t = warp >> 2, row = tid & (BM - 1);
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + t * BN, t_o = t_lane + C::kColO + t * D;
    const int local_token = row / G, local_head = row - local_token * G;      // of this thread's row in a query tile
    uint8_t* out_place = smem + C::kSmemTiles + warp * C::kOutBytes;
    const bool direct = a.n_rec <= 1;
    int steps = 0;
    for (int k = 0; wait(C::kTold + k % kPieces, k / kPieces); ++k) {
      const Piece& p = *piece_at(k);
      if (!p.more) break;
      const int index = t * RT + row, rows = p.rows, n = p.n[t], lo = p.lo, j0 = p.j0;
      const bool mine = row < RT && index < rows, busy = __any_sync(0xffffffffu, mine);    // (rows do not meet: P of the others may be anything)
      const int token = p.token0 + t * (RT / G) + local_token, head = p.kvh * G + local_head;
      int lim = INT_MAX;                                             // (a row that is none costs no mask)
      if (mine) {
        if (MODE == kPrompt) lim = token - p.t0 + 1;
        else {
          lim = max(0, min(__ldcg(a.positions + token), INT_MAX - 1) + 1);
          lim = MODE == kPrefix ? min(lim, a.prefix_len) : (int)min((long long)lim, (long long)a.table_ld * a.page_size);
        }
      }
      const int lim_warp = __reduce_min_sync(0xffffffffu, lim);
      float m_ref = -INFINITY, at_ref = -INFINITY, l = 0.f;        // the reference maximum, and the score that it is the scaled one of
#pragma unroll 1
      for (int half = 0; half < 2 * n; ++half) {                   // 64 keys at a time
        const int i = half >> 1, u = half & 1, key0 = (j0 + i) * BN + 64 * u, g = steps + i;
        if (!wait(C::kS + 2 * u + t, g)) break;
        fence_after_sync();
        if (busy) {
          float x[64];
          tmem_ld32(t_s + 64 * u, x);
          tmem_ld32(t_s + 64 * u + 32, x + 32);
          tmem_ld_wait();
          if (key0 + 64 > lim_warp || key0 < lo) {
            const int from = lo - key0, to = lim - key0;
#pragma unroll
            for (int c = 0; c < 64; ++c) x[c] = (c >= from && c < to) ? x[c] : -INFINITY;
          }
          float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int c = 4; c < 64; c += 2) top[(c >> 1) & 3] = max3_nan(top[(c >> 1) & 3], x[c], x[c + 1]);
          const float highest = max3_nan(max3_nan(top[0], top[1], top[2]), top[3], top[3]), m_new = highest * a.scale_log2;
          float minus = m_ref;
          if (__any_sync(0xffffffffu, !(m_new <= m_ref + kMoveFrom) || fabsf(m_new) > kFarScore)) {
            const bool move = !(m_new <= m_ref + kMoveFrom) || (far_score(m_new) && highest > at_ref);
            // (0 for the first keys.  A row with a score that is no number, or infinite, becomes NaN as a whole.)
            const float alpha = move ? fast_exp2(far_score(m_new) || far_score(m_ref) ? (at_ref - highest) * a.scale_log2 : m_ref - m_new) : 1.f;
            if (move) {
              m_ref = m_new < INFINITY ? m_new : NAN;
              at_ref = highest;
            }
            const bool far = far_score(m_ref);
            if (__any_sync(0xffffffffu, far)) {
              const float from = far ? at_ref : 0.f;
#pragma unroll
              for (int c = 0; c < 64; ++c) x[c] -= from;
            }
            minus = far ? 0.f : m_ref;
            l *= alpha;
            if (half > 0 && __any_sync(0xffffffffu, move)) {
              if (!wait(C::kPv + 2 * (u ^ 1) + t, u ? g : g - 1)) break;      // P V of the half before
              fence_after_sync();
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                float o[16];
                tmem_ld16(t_o + c, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= alpha;
                tmem_st16(t_o + c, reinterpret_cast<const uint32_t*>(o));
              }
              tmem_st_wait();
            }
          }
          const Two scale2(a.scale_log2), minus2(minus == -INFINITY ? 0.f : -minus);
          Two sum2[2] = {Two(0.f), Two(0.f)};
          uint32_t packed[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            float p0, p1;
            fma2(Two(x[2 * c], x[2 * c + 1]), scale2, minus2).get(p0, p1);
            p0 = fast_exp2(p0);
            p1 = fast_exp2(p1);
            sum2[c & 1] = sum2[c & 1] + Two(p0, p1);
            const __nv_bfloat162 b = __floats2bfloat162_rn(p0, p1);
            packed[c] = *reinterpret_cast<const uint32_t*>(&b);
          }
          tmem_st32(t_s + 64 * u, reinterpret_cast<const float*>(packed));
          float s0, s1;
          (sum2[0] + sum2[1]).get(s0, s1);
          l += s0 + s1;
          tmem_st_wait();
        }
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kP + 2 * u + t));
      }
      steps += n;
      if (n > 0) wait(C::kPv + 2 + t, steps - 1);
      if (!ok) break;
      fence_after_sync();
      if (busy) {
        const bool fix = *reinterpret_cast<const volatile int*>(&p.bad) != 0;
        const float inv = l != 0.f ? 1.f / l : 0.f;                           // (a row that sees no key: zeros)
        const size_t record = ((size_t)token * a.nq + head) * a.n_rec + a.rec0 + p.part;
        if (!direct && mine) {
          a.part_ml[2 * record] = m_ref;
          a.part_ml[2 * record + 1] = l;
        }
        // Rows leave through shared memory, 64 bytes of each at a time: four lanes then write a row's piece side by side.
        const long long place = direct ? (long long)token * a.ld_out + (long long)head * D : (long long)record * D;
        const bool stored = mine && (direct || l != 0.f);
        long long to[4];                                                      // the four rows that this lane writes a quarter of
        unsigned store = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          to[q] = __shfl_sync(0xffffffffu, place, 8 * q + (lane >> 2));
          store |= (unsigned)__shfl_sync(0xffffffffu, (int)stored, 8 * q + (lane >> 2)) << q;
        }
        auto leave = [&](const uint4* w, int col) {
#pragma unroll
          for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(out_place + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = w[q];
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int r = 8 * q + (lane >> 2), part = lane & 3;
            const uint4 x = *reinterpret_cast<const uint4*>(out_place + r * 64 + ((part ^ ((r >> 1) & 3)) << 4));
            if (!(store >> q & 1)) continue;
            if (direct) *reinterpret_cast<uint4*>(a.out + to[q] + col + 8 * part) = x;
            else *reinterpret_cast<uint4*>(a.part_o + to[q] + col + 4 * part) = x;
          }
          __syncwarp();
        };
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          float o[32];
          if (n > 0) {
            tmem_ld32(t_o + c0, o);
            tmem_ld_wait();
          }
          if (n == 0 || l == 0.f) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          } else if (fix && mine) {
            // what this row does see of the values that were taken out
            const int* table = MODE == kOwn ? a.tables + (size_t)p.seq * a.table_ld : a.prefix_pages;
            for (int i = 0; i < n; ++i) {
              if (!on_edge(p, i)) continue;
              const int key0 = (j0 + i) * BN;
              for (int key = max(key0, lo); key < min(key0 + BN, lim); ++key) {
                const elem_t *kr, *vr;
                key_rows<MODE>(a, table, p.t0, p.kvh, key, kr, vr);
                if (!vr) continue;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float v = __bfloat162float(vr[c0 + e]);
                  if (!isfinite(v)) o[e] += v;
                }
              }
            }
          }
          __syncwarp();
          if (direct) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(o[2 * e] * inv, o[2 * e + 1] * inv);
              w[e] = *reinterpret_cast<const uint32_t*>(&b);
            }
            leave(reinterpret_cast<const uint4*>(w), c0);
          } else {
            leave(reinterpret_cast<const uint4*>(o), c0);
            leave(reinterpret_cast<const uint4*>(o + 16), c0 + 16);
          }
        }
      }
      fence_before_sync();                // (O has been read before this group's next P is announced)
      taken(k);
    }
  }

  fence_before_sync();
  __syncthreads();
  if (*s_abort) {
    // copies that were asked for land before the shared memory is given back (each wait bounded on its own)
    if (warp == kCopyWarp && lane == 0) {
      for (int n = max(0, copies - C::kStages); n < copies; ++n) mbar_wait(bar(C::kFull + n % C::kStages), (n / C::kStages) & 1);
      for (int t = 0; t < 2; ++t)
        for (int n = max(0, copies_q[t] - C::kSets); n < copies_q[t]; ++n) mbar_wait(bar(C::kQ + 2 * (n % C::kSets) + t), (n / C::kSets) & 1);
    }
    if (tid == 0) report(a.status, kGaveUp);
    __syncthreads();
  }
  if (warp == kIssueWarp) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (early) chain_wait();         // (a kernel after this one may count on the one over the prefix being done, too)
}

// A tensor map over the queries [tokens][heads][D], boxes of 64 columns, the G heads of a kv head and as many whole tokens as 128 rows hold.
int query_map(CUtensorMap* out, const PackedArgs& a, const char* who) {
  const int G = a.nq / a.nkv;
  const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.nq, (cuuint64_t)a.n_tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)a.D * 2, (cuuint64_t)a.ld_q * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(BM / G)};
  const cuuint32_t elem[3] = {1, 1, 1};
  const CUresult r = cuTensorMapEncodeTiled(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<elem_t*>(a.q), dims, strides, box, elem,
                                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ERB_OK : fail(ERB_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", who, (int)r);
}

template <int D, int MODE>
int launch_one(const PackedArgs& a, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, long long pieces, cudaStream_t stream,
               const char* who) {
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(ERB_ERR_CUDA, "%s: no device", who);
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attention_packed_tc_kernel<D, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<D>::kSmemBytes);
    if (e != cudaSuccess) return fail(ERB_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    cudaFuncAttributes f;
    if (cudaFuncGetAttributes(&f, attention_packed_tc_kernel<D, MODE>) != cudaSuccess || f.numRegs * kThreads < 32 * (8 * kSoftmaxRegs + 4 * kOtherRegs))
      return fail(ERB_ERR_CUDA, "%s: built with too few registers for its split", who);
    configured[dev] = true;
  }
  if (pieces > 0x7f000000LL) return fail(ERB_ERR_UNSUPPORTED, "%s: too many rows", who);
  launch_chained(attention_packed_tc_kernel<D, MODE>, dim3((unsigned)(pieces < sm_count() ? pieces : sm_count())), dim3(kThreads), Cfg<D>::kSmemBytes, stream,
                 mq, mk, mv, a);
  return check_launch(who);
}

// pieces: a bound on the pieces of work.
template <int MODE>
int launch_tc(const PackedArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, long long pieces, cudaStream_t stream, const char* who) {
  CUtensorMap mq;
  if (const int rc = query_map(&mq, a, who)) return rc;
  return a.D == 64 ? launch_one<64, MODE>(a, mq, mk, mv, pieces, stream, who) : launch_one<128, MODE>(a, mq, mk, mv, pieces, stream, who);
}

// Rows of a piece of work: whole tokens of G heads in two query tiles.
long long rows_of_piece(int G) { return 2LL * (BM / G * G); }

// A request's own keys by the kernels for few rows: the one for a token a request (or one after the other) or the one for 64 rows.
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
  if ((head_dim != 64 && head_dim != 128) || nq / nkv > BM || !aligned(q, ld_q) || !aligned(k, ld_k) || !aligned(v, ld_v) || !aligned(out, ld_out))
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
  const long long pieces = ((long long)n_tokens * (nq / nkv) / rows_of_piece(nq / nkv) + n_seqs) * nkv;      // (a sequence has at most one that is not full)
  return launch_tc<kPrompt>(a, mk, mv, pieces, (cudaStream_t)stream, "attention_prompt_tc");
}

// The arguments of erb_attention_shared_prefix (attention_packed.cu); heads of 64 or 128, rows, their strides and the pools on 16-byte
// boundaries, pages of 8 to 128 tokens, a power of two.  own: the kernel for a request's own keys (kOwnMany: this file's for many rows; kOwnToken, kOwnRows:
// packed_few.cuh's, which join the records themselves where own_pieces is 1).
ERB_EXPORT int erb_attention_shared_prefix_tc(const void* q, long long ld_q, const void* k_pages, const void* v_pages, int n_pages, int page_size,
                                              const int* prefix_pages, int prefix_len, const int* tables, int table_ld, const int* seq_starts,
                                              const int* positions, int n_seqs, int n_tokens, void* out, long long ld_out, int nq, int nkv,
                                              int head_dim, float scale, int prefix_pieces, int own_pieces, int piece_keys, int own,
                                              float* part_o, float* part_ml, int* status, void* stream) {
  if (n_seqs <= 0 || n_tokens <= 0) return ERB_OK;
  if (nq <= 0 || nkv <= 0 || nq % nkv || !status || n_pages <= 0 || prefix_len < 0 || table_ld <= 0 || prefix_pieces < (prefix_len > 0 ? 1 : 0) ||
      own_pieces < 1 || piece_keys <= 0 || piece_keys > kMostPieceKeys || prefix_len > kMostKeys || (long long)table_ld * page_size > kMostKeys ||
      !(scale > 0.f) || prefix_pieces > 64 ||
      own < kOwnMany || own > kOwnRows || (own == kOwnToken && nq / nkv > 16))
    return fail(ERB_ERR_ARG, "attention_shared_prefix_tc: bad sizes");
  if ((head_dim != 64 && head_dim != 128) || nq / nkv > BM || !aligned(q, ld_q) || !aligned(out, ld_out) || !aligned(k_pages, 0) || !aligned(v_pages, 0) ||
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
    a.pieces = prefix_pieces;
    if ((rc = launch_tc<kPrefix>(a, mk, mv, (rows / rows_of_piece(nq / nkv) + 1) * nkv * a.pieces, s, who))) return rc;
  }
  a.rec0 = prefix_len > 0 ? prefix_pieces : 0;
  a.pieces = own_pieces;
  a.early = prefix_len > 0;
  if (own == kOwnMany) {
    if ((rc = launch_tc<kOwn>(a, mk, mv, (rows / rows_of_piece(nq / nkv) + n_seqs) * nkv * a.pieces, s, who)) || n_rec <= 1) return rc;
  } else {
    rc = head_dim == 64 ? launch_few<64>(a, own == kOwnToken, prefix_len > 0, s, who) : launch_few<128>(a, own == kOwnToken, prefix_len > 0, s, who);
    if (rc || own_pieces == 1) return rc;
  }
  return launch_merge(a, s, who);
}
