// Queries and keys on their way from the projections to attention, in one pass over them: an optional norm per head, the
// rotary position encoding scaled for long contexts, and the append of keys and values to the paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                               (with a norm; one weight vector for all heads)
//   (a, b) -> m (a cos - b sin, b cos + a sin)                       for pair i of the first rot_dim entries, m the multiplier
//
// Pair i is (i, i + rot_dim / 2) or, with `pairs`, (2i, 2i + 1).  All arithmetic in float, one rounding at the store.
//
// The angle.  position * frequency in float loses the angle of far positions: at position 10^6 the fastest pair is off by 0.06 radians.
// The kernel takes frequencies in turns per position as 64-bit fixed point (`turns`, units of 2^-64 turn, rounded down), so the integer product
// with the position, modulo 2^64, is the angle modulo a full turn with an error below |position| * 2^-64 turns.  Its upper 32 bits (what is
// below them is less than 2^-32 turn, 1.5e-9 radians) are cut into a quadrant and a rest of at most an eighth of a turn, which a float holds to 5e-8 radians.
//
// Bytes bound it: every entry is read once and written once.  A thread moves 2 V entries that hold whole pairs (V: sixteen bytes of
// entries), so the lanes of a head exchange nothing but the norm's sum; a token's angles are taken once by the block that works on it.
// 8,192 tokens of 32 + 8 + 8 heads of 128, bfloat16, into the cache: 38 us, 201 MB read and written, 0.81 of what a copy moves; 2,501 tokens of
// 15 + 5 heads of 64, float, half of each turned: 6.7 us, 3.8 TB/s.
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

// Sixteen bytes of neighbouring entries as floats, and back.
template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <> struct Piece<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Rows on 16-byte boundaries, heads of UNITS * 2 N entries (N: sixteen bytes of entries), turned entries a multiple of 2 N.  A unit is two
// pieces of sixteen bytes that hold whole pairs: neighbours with `pairs`, else piece u of the first half of the turned part and its partner
// in the second half (behind the turned part: two neighbours).  UNITS neighbouring lanes make a head.  A block works on the units of one
// token, AHEAD for each thread, asked for before the token's angles are made, blockIdx.y telling apart the blocks that share a token.
constexpr int kFastThreads = 128;

template <int UNITS, bool PAIRS, int AHEAD>
__global__ void __launch_bounds__(kFastThreads) rotary_units_kernel(const RotaryArgs a) {
  using P = Piece<elem_t>;
  constexpr int N = P::N, D = UNITS * 2 * N;
  __shared__ float2 trig[D / 2];
  const int half = a.rot_dim / 2, turned = a.rot_dim / (2 * N);          // units of a head that are turned
  const int heads = a.nq + (a.k ? a.nkv : 0), q_units = heads * UNITS, all = q_units + (a.v ? a.nkv * UNITS : 0);
  const int t = blockIdx.x, stride = gridDim.y * kFastThreads;
  const int u = threadIdx.x % UNITS;                                     // this thread's unit of every head it works on
  const int o0 = PAIRS ? 2 * u * N : (u < turned ? u * N : a.rot_dim + (u - turned) * 2 * N);
  const int o1 = PAIRS || u >= turned ? o0 + N : half + u * N;
  chain_wait();
  const elem_t* q = a.q + t * a.ld_q;
  const elem_t* k = a.k + t * a.ld_k;
  const elem_t* v = a.v + t * a.ld_v;
  const int position = a.rot_dim ? a.positions[t] : 0;
  const long long slot = slot_of(a, t, blockIdx.y == 0 && threadIdx.x == 0);
  const long long cache_row = slot < 0 ? 0 : ((slot / a.page_size) * a.nkv * a.page_size + slot % a.page_size) * D;
  const long long head_step = (long long)a.page_size * D;                // from a kv head's row of a page to the next head's
  bool first = true;
  for (int w0 = blockIdx.y * kFastThreads; w0 < all; w0 += stride * AHEAD) {      // (uniform: the lanes of a head stay together)
    uint4 x0[AHEAD], x1[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) {
      const int w = w0 + n * stride + threadIdx.x, head = w / UNITS;
      x0[n] = x1[n] = make_uint4(0, 0, 0, 0);
      if (w >= all) continue;
      const elem_t* src = head < a.nq ? q + head * D : (head < heads ? k + (head - a.nq) * D : v + (head - heads) * D);
      const int p0 = w < q_units ? o0 : 2 * u * N, p1 = w < q_units ? o1 : p0 + N;
      x0[n] = *reinterpret_cast<const uint4*>(src + p0);
      x1[n] = *reinterpret_cast<const uint4*>(src + p1);
    }
    if (first) {
      for (int i = threadIdx.x; i < half; i += kFastThreads) turn_of(position, a.turns[i], a.multiplier, trig[i].x, trig[i].y);
      __syncthreads();
      first = false;
    }
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) {
      const int w = w0 + n * stride + threadIdx.x, head = w / UNITS;
      if (w0 + n * stride >= all) break;                                 // (the whole block)
      float lo[N], hi[N];
      P::unpack(x0[n], lo);
      P::unpack(x1[n], hi);
      const float* weight = w >= q_units ? nullptr : (head < a.nq ? a.q_norm : a.k_norm);
      if (a.q_norm || a.k_norm) {                                        // (every lane takes part in the exchange)
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) ss = fmaf(lo[i], lo[i], fmaf(hi[i], hi[i], ss));
#pragma unroll
        for (int o = UNITS / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (weight) {
          const float rs = rsqrtf(ss / (float)D + a.eps);
#pragma unroll
          for (int i = 0; i < N; ++i) { lo[i] = lo[i] * rs * weight[o0 + i]; hi[i] = hi[i] * rs * weight[o1 + i]; }
        }
      }
      if (w >= all) continue;
      if (w >= q_units) {                                                // values: to the cache as they are
        if (slot < 0) continue;
        elem_t* dst = a.v_pages + cache_row + (head - heads) * head_step + 2 * u * N;
        *reinterpret_cast<uint4*>(dst) = x0[n];
        *reinterpret_cast<uint4*>(dst + N) = x1[n];
        continue;
      }
      if (u < turned) {
        if (PAIRS) {
#pragma unroll
          for (int i = 0; i < N; i += 2) {
            const float2 c0 = trig[u * N + i / 2], c1 = trig[u * N + N / 2 + i / 2];
            rotate_pair(lo[i], lo[i + 1], c0.x, c0.y, lo[i], lo[i + 1]);
            rotate_pair(hi[i], hi[i + 1], c1.x, c1.y, hi[i], hi[i + 1]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float2 c = trig[u * N + i];
            rotate_pair(lo[i], hi[i], c.x, c.y, lo[i], hi[i]);
          }
        }
      }
      const uint4 y0 = P::pack(lo), y1 = P::pack(hi);
      auto store = [&](elem_t* dst) {
        *reinterpret_cast<uint4*>(dst + o0) = y0;
        *reinterpret_cast<uint4*>(dst + o1) = y1;
      };
      if (head < a.nq) store(a.q_out + t * a.ld_qo + head * D);
      else {
        if (a.k_out) store(a.k_out + t * a.ld_ko + (head - a.nq) * D);
        if (slot >= 0) store(a.k_pages + cache_row + (head - a.nq) * head_step);
      }
    }
  }
}

// As many blocks a token as its units fill, no more than give each multiprocessor sixteen (8,192 tokens: with 64 43.1 us, with 2 to 32 39.7).
template <int UNITS, int AHEAD>
void launch_ahead(const RotaryArgs& a, int work, cudaStream_t stream) {
  int share = (work + kFastThreads * AHEAD - 1) / (kFastThreads * AHEAD);
  const int want = (int)((sm_count() * 16LL + a.n_tokens - 1) / a.n_tokens);
  share = share < want ? share : want;
  const dim3 grid(a.n_tokens, share < 1 ? 1 : share);
  if (a.pairs) launch_chained(rotary_units_kernel<UNITS, true, AHEAD>, grid, dim3(kFastThreads), 0, stream, a);
  else launch_chained(rotary_units_kernel<UNITS, false, AHEAD>, grid, dim3(kFastThreads), 0, stream, a);
}
// Few tokens: one unit a thread, so that a token's work is in as many blocks as it has (16 tokens of 48 heads of 128, bfloat16: 2.4 us; two
// units 2.6, three 2.9; 128 tokens 2.7 and 2.8; but 256 3.8 and 3.3).  Many: a token's units in one block where it can, its angles made once
// (1,024 tokens of 48 heads: three 6.2 us, two 6.9; 8,192 38.6 and 39.8), and no more than it needs (8,192 tokens of 25 heads of 64: two 12.9 us,
// three 14.2: registers).
template <int UNITS>
void launch_units(const RotaryArgs& a, int work, cudaStream_t stream) {
  const long long blocks = (long long)a.n_tokens * ((work + kFastThreads - 1) / kFastThreads);
  if (blocks <= 3LL * sm_count()) launch_ahead<UNITS, 1>(a, work, stream);
  else if (work <= 2 * kFastThreads) launch_ahead<UNITS, 2>(a, work, stream);
  else launch_ahead<UNITS, 3>(a, work, stream);
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
  constexpr int N = Piece<elem_t>::N;
  const int units = head_dim / (2 * N);
  const uintptr_t all = (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)k_out | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages;
  if (head_dim % (2 * N) == 0 && rot_dim % (2 * N) == 0 && units >= 2 && units <= 32 && !(units & (units - 1)) && !(all & 15) &&
      !((ld_q | ld_qo | ld_k | ld_ko | ld_v) % N)) {
    const int work = (nq + (k ? nkv : 0) + (v ? nkv : 0)) * units;
    switch (units) {
      case 2: launch_units<2>(a, work, (cudaStream_t)stream); break;
      case 4: launch_units<4>(a, work, (cudaStream_t)stream); break;
      case 8: launch_units<8>(a, work, (cudaStream_t)stream); break;
      case 16: launch_units<16>(a, work, (cudaStream_t)stream); break;
      default: launch_units<32>(a, work, (cudaStream_t)stream);
    }
    return check_launch("rotary_append");
  }
  const long long items = (long long)n_tokens * (nq + (k ? nkv : 0) + (v ? nkv : 0)), blocks = (items + 3) / 4;
  if (blocks > 0x7fffffffLL) return fail(ERB_ERR_UNSUPPORTED, "rotary_append: %d tokens of %d heads", n_tokens, nq);
  launch_chained(rotary_general_kernel, dim3((unsigned)blocks), dim3(128), 4 * head_dim * sizeof(float), (cudaStream_t)stream, a);
  return check_launch("rotary_append");
}
