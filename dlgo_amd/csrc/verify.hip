// Verification of drafted tokens against the target model's logits, from given uniform numbers (speculative sampling).
//
// A sequence brings d drafted tokens x_0 .. x_{d-1} and the d + 1 rows of logits that the target model gave for the
// places of the drafts and the one after.  With p_j = softmax(row j / T) and q_j the distribution that draft j was drawn
// from (softmax of the draft model's logits / T, or all of it on x_j where the drafts were looked up), draft j is kept
// while u_j * q_j(x_j) < p_j(x_j).  The token after the first a kept drafts is drawn from max(p_a - q_a, 0), or from p_d
// where all were kept, as the first index whose running sum passes u_d times the whole (the sequence's last uniform
// number).  What comes out is then distributed as the target's own tokens would be.  T = 0: a draft is kept if it is the
// row's maximum (the lowest index among equals), and the token after is the maximum.
//
// Everything that decides is held in 64 bits: an index of a vocabulary of 128,256 flat weights owns 2^-17 of the sum, and
// a sum in 32 bits would put about one draw in a hundred beside its neighbour.  computerex/dlgo draws from float32
// probabilities in one pass over a sorted row (ops/sampling.go); it verifies no drafts.
//
// Bound by memory: every row of logits is read once, by blocks of 4,096 elements that each leave a maximum, its index and
// a sum; the row that the next token comes from (and its draft's) is read again where a draft was refused.
#include "common.h"
// everything here is float32 or float64 arithmetic: no approximation can be named (exact_begin.h)
#include "exact_begin.h"

#define CHUNK 4096                       // elements of a row that a block takes, 16 a thread
#define THREADS 256
#define PER (CHUNK / THREADS)

struct Piece16 {
  double sum;                            // of exp((x - max) / T) over the block's elements
  float max;
  int arg;                               // lowest index of the maximum, -1 if nothing was a number
};
struct Choice {                          // what the first block of a sequence found, for the last kernel
  int accepted, row, draft_row, drawn;   // draft_row: -1 where nothing is taken away; drawn: the token if it is settled
  int without;                           // a token that gets no weight (a refused draft that was certain), -1 for none
  float tmax, dmax;
  double tinv, dinv;                     // 1 / the rows' sums
};

struct Verify {
  const float* logits;
  const float* drafts;                   // the draft model's logits, null where the drafts are certain
  const int32_t* tokens;
  const int32_t* cu;
  const float* temperature;
  const float* uniform;
  int32_t* accepted;
  int32_t* token;
  float* probs;                          // may be null
  Piece16* pieces;                       // [target rows, then draft rows][parts]
  double* mass;                          // [sequences][parts]
  Choice* choice;                        // [sequences]
  long long ldl, ldd;
  int n, d, vocab, parts, most;
};

// exp(x) for x <= 0 (or NaN, which counts as nothing): Cody and Waite's reduction to |r| <= ln 2 / 2 and the Taylor series
// to r^12, whose remainder is below 2 * 10^-16 of the result.
__device__ __forceinline__ double exp_neg(double x) {
  x = fmax(x, -800.0);
  const double k = rint(x * 1.4426950408889634074);
  double r = fma(k, -0x1.62e42fee00000p-1, x);           // ln 2 in two parts, the first with 21 zero bits at its end
  r = fma(k, -0x1.a39ef35793c76p-33, r);
  double p = 1.0 / 479001600.0;
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)k);
}
// the weight of x in a row whose maximum is m: 1 for the maximum itself, infinite or not
__device__ __forceinline__ double weight(float x, float m, double inv_t) {
  return x == m ? 1.0 : exp_neg(((double)x - (double)m) * inv_t);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
  return v;
}
__device__ __forceinline__ void take_max(float& m, int& at, float m2, int at2) {
  if (at2 >= 0 && (at < 0 || m2 > m || (m2 == m && at2 < at))) {
    m = m2;
    at = at2;
  }
}
__device__ __forceinline__ void wave_max_at(float& m, int& at) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o, WAVE);
    const int at2 = __shfl_xor(at, o, WAVE);
    take_max(m, at, m2, at2);
  }
}

// Sixteen elements of a row, four runs of four a thread (element 4 * (256 k + thread) + e of the block's part), with
// nothing (NaN) past the row's end.
__device__ __forceinline__ void load16(const float* row, int first, int vocab, float (&x)[PER]) {
  const bool aligned = ((uintptr_t)row & 15) == 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = first + (k * THREADS + (int)threadIdx.x) * 4;
    if (aligned && i + 3 < vocab) {
      *(float4*)(x + 4 * k) = *(const float4*)(row + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * k + e] = i + e < vocab ? row[i + e] : __uint_as_float(0x7fc00000u);
    }
  }
}

// Sixteen consecutive elements from `first` on.
__device__ __forceinline__ void load_run(const float* row, int first, int vocab, float (&x)[PER]) {
  const bool aligned = ((uintptr_t)row & 15) == 0;
#pragma unroll
  for (int k = 0; k < PER; k += 4) {
    const int i = first + k;
    if (aligned && i + 3 < vocab) {
      *(float4*)(x + k) = *(const float4*)(row + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[k + e] = i + e < vocab ? row[i + e] : __uint_as_float(0x7fc00000u);
    }
  }
}

// A sequence's drafts [c0, c1) whatever the numbers on the device are.
__device__ __forceinline__ void drafts_of(const Verify& a, int seq, int& c0, int& c1) {
  c0 = a.cu[seq];
  c1 = a.cu[seq + 1];
  c0 = c0 < 0 ? 0 : (c0 > a.d ? a.d : c0);
  c1 = c1 < c0 ? c0 : (c1 > a.d ? a.d : c1);
  if (c1 - c0 > a.most) c1 = c0 + a.most;
}

// grid: rows * parts.  Maximum, its index and the sum of a part of a row.
__global__ __launch_bounds__(THREADS) void verify_rows_kernel(Verify a) {
  __shared__ float ms[THREADS / WAVE];
  __shared__ int as[THREADS / WAVE];
  __shared__ double ss[THREADS / WAVE];
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts, wave = threadIdx.x / WAVE;
  const bool target = row < a.d + a.n;
  const int at_row = target ? row : row - (a.d + a.n);
  float x[PER];
  load16(target ? a.logits + at_row * a.ldl : a.drafts + at_row * a.ldd, part * CHUNK, a.vocab, x);
  // the row's sequence: how many of the others begin no later
  int before = 0;
  for (int i0 = 1; i0 < a.n; i0 += THREADS) {
    const int i = i0 + (int)threadIdx.x;
    before += __syncthreads_count(i < a.n && a.cu[i < a.n ? i : 0] + (target ? i : 0) <= at_row);
  }
  const float t = a.temperature[before];
  const bool greedy = !(t > 0.f);
  float m = -INFINITY;
  int at = -1;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = x[4 * k + e];
      const bool more = v == v && (at < 0 || v > m);        // indices grow: the first of equals stays
      m = more ? v : m;
      at = more ? part * CHUNK + (k * THREADS + (int)threadIdx.x) * 4 + e : at;
    }
  wave_max_at(m, at);
  if ((threadIdx.x & 63) == 0) {
    ms[wave] = m;
    as[wave] = at;
  }
  __syncthreads();
  m = ms[0];
  at = as[0];
#pragma unroll
  for (int w = 1; w < THREADS / WAVE; ++w) take_max(m, at, ms[w], as[w]);
  double s = 0.0;
  if (!greedy) {
    const double inv_t = 1.0 / (double)t;
#pragma unroll
    for (int k = 0; k < PER; ++k) s += x[k] == x[k] ? weight(x[k], m, inv_t) : 0.0;
    s = wave_sum64(s);
    if ((threadIdx.x & 63) == 0) ss[wave] = s;
    __syncthreads();
    s = ss[0];
#pragma unroll
    for (int w = 1; w < THREADS / WAVE; ++w) s += ss[w];
  }
  if (threadIdx.x == 0) {
    Piece16 p;
    p.sum = s;
    p.max = m;
    p.arg = at;
    a.pieces[(size_t)row * a.parts + part] = p;
  }
}

// A whole row from its parts, by one wave: maximum, its index, sum.
__device__ __forceinline__ void whole_row(const Verify& a, int row, double inv_t, float& m, int& at, double& sum) {
  const Piece16* p = a.pieces + (size_t)row * a.parts;
  const int lane = threadIdx.x & 63;
  m = -INFINITY;
  at = -1;
  for (int i = lane; i < a.parts; i += WAVE) take_max(m, at, p[i].max, p[i].arg);
  wave_max_at(m, at);
  sum = 0.0;
  for (int i = lane; i < a.parts; i += WAVE)
    if (p[i].arg >= 0) sum += p[i].sum * weight(p[i].max, m, inv_t);
  sum = wave_sum64(sum);
}

struct Judged {       // a row's maxima and inverse sums, and whether its draft is kept
  double tinv, dinv;
  float tmax, dmax;
  int arg, keep;
};

// grid (parts, sequences).  Every block of a sequence judges its drafts (a few hundred numbers that the first kernel
// left) and sums the weights of its part of the row that the next token comes from.
__global__ __launch_bounds__(THREADS) void verify_judge_kernel(Verify a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  Judged* rows = (Judged*)lds;             // [most + 1]
  __shared__ double ss[THREADS / WAVE];
  const int part = blockIdx.x, seq = blockIdx.y, wave = threadIdx.x / WAVE, lane = threadIdx.x & 63;
  int c0, c1;
  drafts_of(a, seq, c0, c1);
  const int d = c1 - c0;
  const float t = a.temperature[seq];
  const bool greedy = !(t > 0.f);
  const double inv_t = greedy ? 1.0 : 1.0 / (double)t;
  for (int j = wave; j <= d; j += THREADS / WAVE) {
    const int row = c0 + seq + j;
    Judged r;
    double sum, dsum = 1.0;
    int darg;
    whole_row(a, row, inv_t, r.tmax, r.arg, sum);
    r.tinv = 1.0 / sum;
    r.dmax = 0.f;
    r.dinv = 0.0;
    r.keep = 0;
    if (j < d) {
      const int tok = a.tokens[c0 + j];
      const bool in = tok >= 0 && tok < a.vocab;
      double p = 0.0, q = 1.0;
      if (greedy) {
        p = in && tok == r.arg ? 1.0 : 0.0;
        r.keep = p > 0.0;
      } else {
        const float x = a.logits[row * a.ldl + (in ? tok : 0)];
        p = in && x == x ? weight(x, r.tmax, inv_t) * r.tinv : 0.0;
        if (a.drafts) {
          whole_row(a, a.d + a.n + c0 + j, inv_t, r.dmax, darg, dsum);
          r.dinv = 1.0 / dsum;
          const float y = a.drafts[(c0 + j) * a.ldd + (in ? tok : 0)];
          q = in && y == y ? weight(y, r.dmax, inv_t) * r.dinv : 0.0;
        }
        r.keep = (double)a.uniform[row] * q < p;
      }
      if (part == 0 && lane == 0 && a.probs) a.probs[c0 + j] = (float)p;
    }
    if (lane == 0) rows[j] = r;
  }
  __syncthreads();
  int kept = 0;
  while (kept < d && rows[kept].keep) ++kept;
  const Judged r = rows[kept];
  const bool refused = kept < d;
  const int row = c0 + seq + kept;
  Choice c;
  c.accepted = kept;
  c.row = row;
  c.draft_row = refused && !greedy && a.drafts ? c0 + kept : -1;
  c.without = refused && !greedy && !a.drafts ? a.tokens[c0 + kept] : -1;
  c.drawn = greedy ? (r.arg < 0 ? 0 : r.arg) : -1;
  c.tmax = r.tmax;
  c.dmax = r.dmax;
  c.tinv = r.tinv;
  c.dinv = r.dinv;
  if (part == 0 && threadIdx.x == 0) a.choice[seq] = c;
  if (greedy) return;
  double s = 0.0;
  if (!refused) {                          // the whole row: its parts' sums are known
    const Piece16 p = a.pieces[(size_t)row * a.parts + part];
    s = p.arg >= 0 ? p.sum * weight(p.max, r.tmax, inv_t) * r.tinv : 0.0;
  } else {
    float x[PER], y[PER];
    load16(a.logits + row * a.ldl, part * CHUNK, a.vocab, x);
    if (a.drafts) load16(a.drafts + (long long)c.draft_row * a.ldd, part * CHUNK, a.vocab, y);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      double w = x[k] == x[k] ? weight(x[k], r.tmax, inv_t) * r.tinv : 0.0;
      if (a.drafts) w -= y[k] == y[k] ? weight(y[k], r.dmax, inv_t) * r.dinv : 0.0;
      else if (part * CHUNK + ((k >> 2) * THREADS + (int)threadIdx.x) * 4 + (k & 3) == c.without) w = 0.0;
      s += fmax(w, 0.0);
    }
    s = wave_sum64(s);
    if (lane == 0) ss[wave] = s;
    __syncthreads();
    s = ss[0];
#pragma unroll
    for (int w = 1; w < THREADS / WAVE; ++w) s += ss[w];
  }
  if (threadIdx.x == 0) a.mass[(size_t)seq * a.parts + part] = s;
}

// grid (sequences).  The part whose running sum passes the target, then the element in it.
__global__ __launch_bounds__(THREADS) void verify_draw_kernel(Verify a) {
  __shared__ double run[THREADS];
  __shared__ int found;
  const int seq = blockIdx.x;
  const Choice c = a.choice[seq];
  if (threadIdx.x == 0) a.accepted[seq] = c.accepted;
  if (c.drawn >= 0) {
    if (threadIdx.x == 0) a.token[seq] = c.drawn;
    return;
  }
  int c0, c1;
  drafts_of(a, seq, c0, c1);
  const double inv_t = 1.0 / (double)a.temperature[seq];
  // every wave by itself: the parts' masses one a lane, their running sums
  const int lane = threadIdx.x & 63;
  const Piece16* p = a.pieces + (size_t)c.row * a.parts;
  auto total_of = [&](bool plain) {
    double v = 0.0;
    for (int i = lane; i < a.parts; i += WAVE)
      v += plain ? (p[i].arg >= 0 ? p[i].sum * weight(p[i].max, c.tmax, inv_t) * c.tinv : 0.0) : a.mass[(size_t)seq * a.parts + i];
    return wave_sum64(v);
  };
  double total = total_of(false);
  const bool plain = !(total > 0.0);       // nothing is left beside the draft's distribution: the target's own
  if (plain) total = total_of(true);
  const double target = (double)a.uniform[c1 + seq] * total;
  int part = -1, last_part = 0;
  double before = 0.0, last_before = 0.0, sum_so_far = 0.0;
  for (int i0 = 0; i0 < a.parts && part < 0; i0 += WAVE) {
    const int i = i0 + lane;
    double v = 0.0;
    if (i < a.parts) v = plain ? (p[i].arg >= 0 ? p[i].sum * weight(p[i].max, c.tmax, inv_t) * c.tinv : 0.0) : a.mass[(size_t)seq * a.parts + i];
    double incl = v;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
      const double u = __shfl_up(incl, o, WAVE);
      if (lane >= o) incl += u;
    }
    incl += sum_so_far;
    const double excl = incl - v;
    const unsigned long long over = __ballot(i < a.parts && v > 0.0 && incl > target), some = __ballot(v > 0.0);
    if (some) {
      const int at = 63 - __builtin_clzll(some);
      last_part = i0 + at;
      last_before = __shfl(excl, at, WAVE);
    }
    if (over) {
      const int at = __builtin_ctzll(over);
      part = i0 + at;
      before = __shfl(excl, at, WAVE);
    }
    sum_so_far = __shfl(incl, WAVE - 1, WAVE);
  }
  if (part < 0) {                          // the target lies behind the last sum by a rounding
    part = last_part;
    before = last_before;
  }
  if (threadIdx.x == 0) found = a.vocab;
  __syncthreads();
  const int first = part * CHUNK + (int)threadIdx.x * PER;         // consecutive elements a thread, for the running sum
  const float* row = a.logits + (long long)c.row * a.ldl;
  const bool less = !plain && c.draft_row >= 0;
  float x[PER], y[PER];
  load_run(row, first, a.vocab, x);
  if (less) load_run(a.drafts + (long long)c.draft_row * a.ldd, first, a.vocab, y);
  double w[PER], sum = 0.0;
  int last = -1;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = first + k;
    double v = x[k] == x[k] ? weight(x[k], c.tmax, inv_t) * c.tinv : 0.0;
    if (less) v -= y[k] == y[k] ? weight(y[k], c.dmax, inv_t) * c.dinv : 0.0;
    if (!plain && i == c.without) v = 0.0;
    w[k] = fmax(v, 0.0);
    if (w[k] > 0.0) last = i;
    sum += w[k];
  }
  run[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 1; o < THREADS; o <<= 1) {          // running sums over the threads
    const double v = (int)threadIdx.x >= o ? run[threadIdx.x - o] : 0.0;
    __syncthreads();
    run[threadIdx.x] += v;
    __syncthreads();
  }
  double at = before + (threadIdx.x > 0 ? run[threadIdx.x - 1] : 0.0);
  int hit = a.vocab;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    at += w[k];
    if (hit == a.vocab && w[k] > 0.0 && at > target) hit = first + k;
  }
  if (hit < a.vocab) atomicMin(&found, hit);
  __syncthreads();
  if (found < a.vocab) {
    if (threadIdx.x == 0) a.token[seq] = found;
    return;
  }
  // the target lies behind the last sum by a rounding: the last element that has a weight
  __syncthreads();
  if (threadIdx.x == 0) found = -1;
  __syncthreads();
  if (last >= 0) atomicMax(&found, last);
  __syncthreads();
  if (threadIdx.x == 0) a.token[seq] = found < 0 ? 0 : found;
}

static long long round16(long long n) { return (n + 15) / 16 * 16; }

// bytes of scratch for n sequences with d drafts in all, over a vocabulary
extern "C" long long dlgo_verify_drafts_scratch(int n, int d, int vocab, int model_drafts) {
  if (n <= 0 || d < 0 || vocab <= 0) return 0;
  const long long parts = (vocab + CHUNK - 1) / CHUNK, rows = (long long)d + n + (model_drafts ? d : 0);
  return round16(rows * parts * (long long)sizeof(Piece16)) + round16(n * parts * 8) + round16(n * (long long)sizeof(Choice));
}

extern "C" const char* dlgo_verify_drafts(const float* logits, long long ldl, const int32_t* tokens, const float* drafts, long long ldd,
                                          const int32_t* cu, const float* temperature, const float* uniform, int n, int d, int vocab,
                                          int most, int32_t* accepted, int32_t* token, float* probs, void* scratch,
                                          long long scratch_bytes, hipStream_t stream) {
  DLGO_REQUIRE(n >= 0 && d >= 0 && vocab > 0 && most >= 0, "verify_drafts: bad sizes");
  if (n == 0) return nullptr;
  DLGO_REQUIRE(most <= 1024, "verify_drafts: at most 1024 drafts a sequence, not %d", most);
  DLGO_REQUIRE(ldl >= vocab && (!drafts || ldd >= vocab), "verify_drafts: rows shorter than the vocabulary");
  const long long parts = (vocab + CHUNK - 1) / CHUNK, rows = (long long)d + n + (drafts ? d : 0);
  const long long need = dlgo_verify_drafts_scratch(n, d, vocab, drafts != nullptr);
  DLGO_REQUIRE(scratch && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0, "verify_drafts: %lld bytes of scratch are needed, %lld given", need, scratch ? scratch_bytes : 0ll);
  DLGO_REQUIRE(rows * parts < (1ll << 31) && n <= 65535, "verify_drafts: too many rows at once");
  char* at = (char*)scratch;
  Verify a = {logits, drafts, tokens, cu, temperature, uniform, accepted, token, probs, (Piece16*)at, nullptr, nullptr, ldl, ldd, n, d, vocab, (int)parts, most};
  at += round16(rows * parts * (long long)sizeof(Piece16));
  a.mass = (double*)at;
  at += round16(n * parts * 8);
  a.choice = (Choice*)at;
  hipLaunchKernelGGL(verify_rows_kernel, dim3((unsigned)(rows * parts)), dim3(THREADS), 0, stream, a);
  DLGO_LAUNCH_CHECK("verify_drafts");
  hipLaunchKernelGGL(verify_judge_kernel, dim3((unsigned)parts, (unsigned)n), dim3(THREADS), (most + 1) * (int)sizeof(Judged), stream, a);
  DLGO_LAUNCH_CHECK("verify_drafts");
  hipLaunchKernelGGL(verify_draw_kernel, dim3((unsigned)n), dim3(THREADS), 0, stream, a);
  DLGO_LAUNCH_CHECK("verify_drafts");
  return nullptr;
}

#include "exact_end.h"
