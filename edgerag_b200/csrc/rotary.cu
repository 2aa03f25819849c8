// Queries and keys on their way from the projections to attention, in one pass over them: an optional norm per head, the
// rotary position encoding scaled for long contexts, and the append of keys and values to the paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                               (with a norm; one weight vector for all heads)
//   (a, b) -> m (a cos - b sin, b cos + a sin)                       for pair i of the first rot_dim entries, m the multiplier
//
// Pair i is (i, i + rot_dim / 2) or, with `pairs`, (2i, 2i + 1).  All arithmetic in float, one rounding at the store.
//
// The angle.  position * frequency in float loses the angle of far positions: at position 10^6 the fastest pair is off by 0.06 radians.
// The kernel takes frequencies in turns per position as 64-bit fixed point (`turns`, units of 2^-64 turn), so the integer product with the
// position, modulo 2^64, is the angle modulo a full turn with an error below position * 2^-65 turns.  Its upper 32 bits are cut into a
// quadrant and a rest of at most an eighth of a turn, which a float holds to 5e-8 radians.
//
// Bytes bound it: every entry is read once and written once.  A thread moves 2 V entries that hold whole pairs (V: sixteen bytes of
// entries), so the lanes of a head exchange nothing but the norm's sum; a token's angles are taken once by the block that works on it.
#include <stdarg.h>

#include "common.cuh"

using namespace erb;

ERB_DEFINE_LAST_ERROR(erb_last_error)

namespace {

struct RotaryArgs {
  const elem_t* q;
  elem_t* q_out;
  long long ld_q, ld_qo;
  const elem_t* k;                 // null: queries only
  elem_t* k_out;                   // null: keys go to the cache only
  long long ld_k, ld_ko;
  const elem_t* v;
  long long ld_v;
  const float *q_norm, *k_norm;    // null: no norm
  float eps, multiplier;
  const int* positions;
  const unsigned long long* turns;
  int rot_dim, pairs;
  const int* slots;
  elem_t *k_pages, *v_pages;       // null: no cache
  long long n_slots;
  int page_size, n_tokens, nq, nkv, D;
  int* status;
};

// m cos and m sin of position * turns / 2^64 turns.
__device__ __forceinline__ void turn_of(int position, unsigned long long turns, float m, float& cs, float& sn) {
  const unsigned phase = (unsigned)(((unsigned long long)(long long)position * turns) >> 32);     // 2^-32 turns
  const unsigned quadrant = (phase + 0x20000000u) >> 30;                                          // the nearest quarter turn (0..3, 4 is 0)
  const int rest = (int)(phase - (quadrant << 30));                                               // [-2^29, 2^29)
  float s, c;
  sincospif((float)rest * 4.656612873077393e-10f, &s, &c);                                        // 2^-31: half turns
  const float c4 = (quadrant & 1) ? -s : c, s4 = (quadrant & 1) ? c : s;
  cs = m * ((quadrant & 2) ? -c4 : c4);
  sn = m * ((quadrant & 2) ? -s4 : s4);
}

// The token's place in the cache, or -1; a slot behind the pool is reported and left alone.
__device__ __forceinline__ long long slot_of(const RotaryArgs& a, int t, bool report) {
  if (!a.k_pages) return -1;
  const int slot = a.slots[t];
  if (slot >= a.n_slots) {
    if (report) atomicCAS(a.status, 0, t + 1);
    return -1;
  }
  return slot;
}

// Any head size, any alignment: a warp per (token, head).
__global__ void __launch_bounds__(128) rotary_general_kernel(const RotaryArgs a) {
  chain_wait();
  extern __shared__ float rows[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.D, half = a.rot_dim / 2;
  float* x = rows + warp * D;
  const int heads = a.nq + (a.k ? a.nkv : 0) + (a.v ? a.nkv : 0);
  const long long item = (long long)blockIdx.x * 4 + warp;
  if (item >= (long long)a.n_tokens * heads) return;
  const int t = (int)(item / heads), head = (int)(item % heads);
  const long long slot = slot_of(a, t, head == 0 && lane == 0);
  auto cache_row = [&](elem_t* pool, int h) { return pool + (((slot / a.page_size) * a.nkv + h) * a.page_size + slot % a.page_size) * D; };
  if (head >= a.nq + a.nkv) {                    // a value head: to the cache as it is
    if (slot < 0) return;
    const elem_t* src = a.v + t * a.ld_v + (long long)(head - a.nq - a.nkv) * D;
    elem_t* dst = cache_row(a.v_pages, head - a.nq - a.nkv);
    for (int i = lane; i < D; i += 32) dst[i] = src[i];
    return;
  }
  const bool is_q = head < a.nq;
  const int h = is_q ? head : head - a.nq;
  const elem_t* src = (is_q ? a.q + t * a.ld_q : a.k + t * a.ld_k) + (long long)h * D;
  const float* w = is_q ? a.q_norm : a.k_norm;
  float ss = 0.f;
  for (int i = lane; i < D; i += 32) {
    x[i] = Elem<elem_t>::load(src + i);
    ss = fmaf(x[i], x[i], ss);
  }
  if (w) {
    const float rs = rsqrtf(warp_sum(ss) / (float)D + a.eps);
    for (int i = lane; i < D; i += 32) x[i] = x[i] * rs * w[i];
  }
  __syncwarp();
  for (int i = lane; i < half; i += 32) {
    const int i0 = a.pairs ? 2 * i : i, i1 = a.pairs ? 2 * i + 1 : i + half;
    float cs, sn, lo, hi;
    turn_of(a.positions[t], a.turns[i], a.multiplier, cs, sn);
    rotate_pair(x[i0], x[i1], cs, sn, lo, hi);
    x[i0] = lo;
    x[i1] = hi;
  }
  __syncwarp();
  elem_t* to[2] = {is_q ? a.q_out + t * a.ld_qo + (long long)h * D : (a.k_out ? a.k_out + t * a.ld_ko + (long long)h * D : nullptr),
                   !is_q && slot >= 0 ? cache_row(a.k_pages, h) : nullptr};
#pragma unroll
  for (int n = 0; n < 2; ++n)
    if (to[n])
      for (int i = lane; i < D; i += 32) Elem<elem_t>::store(to[n] + i, x[i]);
}

}  // namespace

// q, k, v: rows of heads, ld_* elements apart (k null: queries only; v null: no values).  q_out / k_out: rows for the results, the inputs
// themselves allowed; k_out null: keys go to the cache only.  k_pages / v_pages [n_pages][nkv][page_size][D] with slots: the place of
// token t is page slots[t] / page_size, offset slots[t] % page_size; negative: the token has none; one behind the pool sets *status to
// the token's number plus one.
ERB_EXPORT int erb_rotary_append(const void* q, void* q_out, long long ld_q, long long ld_qo, const void* k, void* k_out, long long ld_k,
                                 long long ld_ko, const void* v, long long ld_v, const float* q_norm, const float* k_norm, float eps,
                                 float multiplier, const int* positions, const void* turns, int rot_dim, int pairs, const int* slots,
                                 void* k_pages, void* v_pages, int n_pages, int page_size, int n_tokens, int nq, int nkv, int head_dim,
                                 int* status, void* stream) {
  if (n_tokens <= 0) return ERB_OK;
  if (!q || !q_out || nq <= 0 || head_dim <= 0 || head_dim > 1024 || rot_dim < 0 || rot_dim > head_dim || rot_dim % 2 || (rot_dim && (!turns || !positions)))
    return fail(ERB_ERR_ARG, "rotary_append: bad sizes (rot_dim %d of head_dim %d)", rot_dim, head_dim);
  if ((k && nkv <= 0) || (v && !k) || (k_pages && (!k || !v || !v_pages || !slots || !status || page_size <= 0 || n_pages <= 0)))
    return fail(ERB_ERR_ARG, "rotary_append: keys, values, pages and slots come together");
  RotaryArgs a = {(const elem_t*)q, (elem_t*)q_out, ld_q, ld_qo, (const elem_t*)k, (elem_t*)k_out, ld_k, ld_ko, (const elem_t*)v, ld_v,
                  q_norm, k_norm, eps, multiplier, positions, (const unsigned long long*)turns, rot_dim, pairs, slots, (elem_t*)k_pages,
                  (elem_t*)v_pages, (long long)n_pages * page_size, page_size > 0 ? page_size : 1, n_tokens, nq, nkv, head_dim, status};
  const long long items = (long long)n_tokens * (nq + (k ? nkv : 0) + (v ? nkv : 0)), blocks = (items + 3) / 4;
  if (blocks > 0x7fffffffLL) return fail(ERB_ERR_UNSUPPORTED, "rotary_append: %d tokens of %d heads", n_tokens, nq);
  launch_chained(rotary_general_kernel, dim3((unsigned)blocks), dim3(128), 4 * head_dim * sizeof(float), (cudaStream_t)stream, a);
  return check_launch("rotary_append");
}
