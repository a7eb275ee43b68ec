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
// Everything that decides is held in 64 bits, a logit's weight right to 1.1 * 10^-12 of itself (exp2_neg, 40 bits): an index of
// a vocabulary of 128,256 flat weights owns 2^-17 of the sum, and a sum in 32 bits would put about one draw in a hundred
// beside its neighbour.  computerex/dlgo draws from float32
// probabilities in one pass over a sorted row (ops/sampling.go); it verifies no drafts.
//
// Every row of logits is read once, by blocks of 4,096 elements that each leave a maximum, its index and a sum; the row that
// the next token comes from (and its draft's) is read again where a draft was refused.
//
// Bound by memory for many rows: 64 sequences with 5 drafts of a draft model and a vocabulary of 128,256, 361 MB: 85 us for the
// rows (4.2 TB/s; 65 us with the exponentials taken out, so these hide only in part), 26 for judging and what is left of the
// refused rows, 10 for the draws.  By latency for few: one sequence 5.3, 5 and 6.6 us, eight with looked-up drafts 9 and 12,
// a chain of four trips to memory in the later kernels.  Measured and not kept for the rows: 1, 2, 8 and 32 parts a block in
// turn (4 it is, from 8,192 parts on), registers for 6 or 8 waves a SIMD.
#include "common.h"
// everything here is float32 or float64 arithmetic: no approximation can be named (exact_begin.h)
#include "exact_begin.h"

#define CHUNK 4096                       // elements of a row that a block takes, 16 a thread
#define THREADS 256
#define PER (CHUNK / THREADS)
#define LOG2E 1.44269504088896340736

struct Piece16 {
  double sum;                            // of exp((x - max) / T) over the part's elements (not where T = 0)
  float max;
  int arg;                               // T = 0: lowest index of the maximum, -1 if nothing was a number; else 0
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
  int run, judge_run;                    // parts of a row that a block of the first (second) kernel takes in turn
};

// 2^y for y <= 0: y is taken apart into a whole number (the addition of 1.5 * 2^52 leaves it in the sum's low bits) and a
// rest of at most a half, whose power is the polynomial of degree 8 through the nine Chebyshev nodes of [-1/2, 1/2]: off
// by at most 1.07 * 10^-12 of itself.  Below 2^-1000 (-inf and NaN among it) it is 2^-1000.
__device__ __forceinline__ double exp2_neg(double y) {
  y = fmax(y, -1000.0);
  const double shifted = y + 0x1.8p52;
  const double f = y - (shifted - 0x1.8p52);
  double p = fma(1.3255224878668817e-06, f, 1.5310079402249296e-05);
  p = fma(p, f, 0.00015403455852453838);
  p = fma(p, f, 0.0013333450568000645);
  p = fma(p, f, 0.009618129159402558);
  p = fma(p, f, 0.05550410941205933);
  p = fma(p, f, 0.2402265069581299);
  p = fma(p, f, 0.6931471805459335);
  p = fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)(uint32_t)__double_as_longlong(shifted));
}
// The weight exp((x - m) / T) of a logit in a row whose maximum is m, c = log2 e / T: 1 for the maximum itself, infinite or
// not, and nothing at all for what lies 2^-1000 below it, -inf and NaN among it.
__device__ __forceinline__ double weight(float x, float m, double c) {
  const double y = ((double)x - (double)m) * c;
  return x == m ? 1.0 : (y > -1000.0 ? exp2_neg(y) : 0.0);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
  return v;
}
// the sum over the lanes up to this one
__device__ __forceinline__ double wave_running64(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const double u = __shfl_up(v, o, WAVE);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ void take_max(float& m, int& at, float m2, int at2) {        // the lowest index of equals
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

// four floats in a row in memory, at any float's address
struct __attribute__((packed, aligned(4))) Four {
  float x, y, z, w;
};

// Sixteen elements of a row, nothing (NaN) past the row's end: element k is `first` + at(k).  No load stands under a lane's
// condition: a part that reaches past the end reads the last element in place of what is not there.
template <typename At>
__device__ __forceinline__ void load_part(const float* row, int first, int vocab, float (&x)[PER], At at) {
  if (first + CHUNK <= vocab) {
#pragma unroll
    for (int k = 0; k < PER; k += 4) {
      const Four f = *(const Four*)(row + first + at(k));
      x[k] = f.x;
      x[k + 1] = f.y;
      x[k + 2] = f.z;
      x[k + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = first + at(k);
      x[k] = row[i < vocab ? i : vocab - 1];
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = first + at(k) < vocab ? x[k] : __uint_as_float(0x7fc00000u);
  }
}
// four runs of four a thread: what 64 lanes load is 1 KB in a row
__device__ __forceinline__ int in_runs(int k) { return ((k >> 2) * THREADS + (int)threadIdx.x) * 4 + (k & 3); }
__device__ __forceinline__ void load16(const float* row, int first, int vocab, float (&x)[PER]) { load_part(row, first, vocab, x, in_runs); }

// A sequence's drafts [c0, c1) whatever the numbers on the device are.
__device__ __forceinline__ void drafts_of(const Verify& a, int seq, int& c0, int& c1) {
  c0 = a.cu[seq];
  c1 = a.cu[seq + 1];
  c0 = c0 < 0 ? 0 : (c0 > a.d ? a.d : c0);
  c1 = c1 < c0 ? c0 : (c1 > a.d ? a.d : c1);
  if (c1 - c0 > a.most) c1 = c0 + a.most;
}

__device__ __forceinline__ float max_of(const float (&x)[PER]) {
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < PER; ++k) m = fmaxf(m, x[k]);
  return m;
}

// grid: rows * ceil(parts / run).  Maximum and sum (T = 0: its index) of `run` parts of a row one after the other, the next
// one's elements on their way while this one's are summed.  A wave's sum stands on the wave's own maximum; one barrier a
// part brings the four together.
__global__ __launch_bounds__(THREADS) void verify_rows_kernel(Verify a) {
  constexpr int NWV = THREADS / WAVE;
  __shared__ float ms[2][NWV];
  __shared__ int as[2][NWV];
  __shared__ double ss[2][NWV];
  const int runs = (a.parts + a.run - 1) / a.run;
  const int row = blockIdx.x / runs, part0 = blockIdx.x % runs * a.run, wave = threadIdx.x / WAVE;
  const int part1 = part0 + a.run < a.parts ? part0 + a.run : a.parts;
  const bool target = row < a.d + a.n;
  const int at_row = target ? row : row - (a.d + a.n);
  const float* src = target ? a.logits + at_row * a.ldl : a.drafts + at_row * a.ldd;
  float x[PER], y[PER];
  load16(src, part0 * CHUNK, a.vocab, x);
  // the row's sequence: how many of the others begin no later (every wave counts for itself)
  int before = 0;
  for (int i0 = 1; i0 < a.n; i0 += WAVE) {
    const int i = i0 + ((int)threadIdx.x & 63);
    before += __popcll(__ballot(i < a.n && a.cu[i < a.n ? i : 0] + (target ? i : 0) <= at_row));
  }
  const float t = a.temperature[before];
  const bool greedy = !(t > 0.f);
  const double c = greedy ? 1.0 : LOG2E / (double)t;
  auto one = [&](int part, float (&v)[PER], float (&next)[PER]) {
    if (part + 1 < part1) load16(src, (part + 1) * CHUNK, a.vocab, next);
    const int odd = part & 1;
    float m = max_of(v);
    int at = 0;
    double s = 0.0;
    if (greedy) {
      at = -1;
#pragma unroll
      for (int k = PER - 1; k >= 0; --k)                      // the first of equals stays
        if (v[k] == m) at = part * CHUNK + in_runs(k);
      wave_max_at(m, at);
    } else {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, WAVE));
      if (m < INFINITY) {
        // The difference first: v c - m c in one operation would lose it where T is near zero.  What is -inf or NaN counts
        // 2^-1000 here: nothing beside the maximum's 1, and more than nothing where a row holds no number.
#pragma unroll
        for (int k = 0; k < PER; ++k) s += exp2_neg(((double)v[k] - (double)m) * c);
      } else {
#pragma unroll
        for (int k = 0; k < PER; ++k) s += v[k] == m ? 1.0 : 0.0;
      }
      s = wave_sum64(s);
    }
    if ((threadIdx.x & 63) == 0) {
      ms[odd][wave] = m;
      as[odd][wave] = at;
      ss[odd][wave] = s;
    }
    __syncthreads();                       // the other place is written a part later, when everybody has read this one
    if (threadIdx.x == 0) {
      Piece16 p;
      p.max = ms[odd][0];
      p.arg = as[odd][0];
#pragma unroll
      for (int w = 1; w < NWV; ++w) {
        if (greedy) take_max(p.max, p.arg, ms[odd][w], as[odd][w]);
        else p.max = fmaxf(p.max, ms[odd][w]);
      }
      p.sum = 0.0;
      if (!greedy) {
#pragma unroll
        for (int w = 0; w < NWV; ++w) p.sum += ss[odd][w] * weight(ms[odd][w], p.max, c);
      }
      a.pieces[(size_t)row * a.parts + part] = p;
    }
  };
  for (int part = part0; part < part1; part += 2) {
    one(part, x, y);
    if (part + 1 < part1) one(part + 1, y, x);
  }
}

struct Whole {        // a row from its parts: 1 / sum, maximum, its index
  double inv;
  float max;
  int arg;
};

// what a part adds to its row's probability
__device__ __forceinline__ double share(const Piece16& p, float max, double inv, double c) { return p.sum * weight(p.max, max, c) * inv; }

// Writes what was found of a sequence.  Where a token is still to be drawn: the part whose running sum passes the target,
// then the element in it; mass(i) is what part i (the lane's number modulo 64) weighs.
template <typename Mass>
__device__ __forceinline__ void draw(const Verify& a, int seq, const Choice& ch, Mass mass) {
  __shared__ double wave_run[THREADS / WAVE];
  __shared__ int found;
  const int lane = threadIdx.x & 63, wave = threadIdx.x / WAVE;
  const float t = a.temperature[seq];
  int c0, c1;
  drafts_of(a, seq, c0, c1);
  const double u = (double)a.uniform[c1 + seq];
  if (threadIdx.x == 0) {
    a.accepted[seq] = ch.accepted;
    found = a.vocab;
  }
  if (ch.drawn >= 0) {
    if (threadIdx.x == 0) a.token[seq] = ch.drawn;
    return;
  }
  const double c = LOG2E / (double)t;
  // every wave by itself: the parts' masses one a lane, their running sums
  const Piece16* p = a.pieces + (size_t)ch.row * a.parts;
  bool plain = false;
  double run64 = 0.0, v64 = 0.0;           // of the first 64 parts
  auto mass_of = [&](int i) {              // of part i, whose number is the lane's modulo 64
    if (plain) return i < a.parts ? share(p[i], ch.tmax, ch.tinv, c) : 0.0;
    return i < a.parts ? mass(i) : 0.0;
  };
  auto total_of = [&]() {
    v64 = mass_of(lane);
    run64 = wave_running64(v64);
    double sum = __shfl(run64, WAVE - 1, WAVE);
    for (int i0 = WAVE; i0 < a.parts; i0 += WAVE) sum = __shfl(wave_running64(mass_of(i0 + lane)) + sum, WAVE - 1, WAVE);
    return sum;
  };
  double total = total_of();
  if (!(total > 0.0)) {                    // nothing is left beside the draft's distribution: the target's own
    plain = true;
    total = total_of();
  }
  const double target = u * total;
  int part = -1, last_part = 0;
  double before = 0.0, last_before = 0.0, sum_so_far = 0.0;
  for (int i0 = 0; i0 < a.parts && part < 0; i0 += WAVE) {
    const double v = i0 == 0 ? v64 : mass_of(i0 + lane);
    const double incl = i0 == 0 ? run64 : wave_running64(v) + sum_so_far, excl = incl - v;
    const unsigned long long over = __ballot(v > 0.0 && incl > target), some = __ballot(v > 0.0);
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
  const int first = part * CHUNK + (int)threadIdx.x * PER;
  const bool less = !plain && ch.draft_row >= 0;
  float x[PER], y[PER];
  auto consecutive = [](int k) { return (int)threadIdx.x * PER + k; };      // a thread's sixteen lie in a row, for the running sum
  load_part(a.logits + (long long)ch.row * a.ldl, part * CHUNK, a.vocab, x, consecutive);
  if (less) load_part(a.drafts + (long long)ch.draft_row * a.ldd, part * CHUNK, a.vocab, y, consecutive);
  double w[PER], sum = 0.0;
  int last = -1;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = first + k;
    double v = weight(x[k], ch.tmax, c) * ch.tinv;
    if (less) v -= weight(y[k], ch.dmax, c) * ch.dinv;
    if (!plain && i == ch.without) v = 0.0;
    w[k] = fmax(v, 0.0);
    if (w[k] > 0.0) last = i;
    sum += w[k];
  }
  const double run = wave_running64(sum);
  if (lane == WAVE - 1) wave_run[wave] = run;
  __syncthreads();
  double at = before + (run - sum);
#pragma unroll
  for (int i = 0; i < THREADS / WAVE; ++i)
    if (i < wave) at += wave_run[i];
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

// grid (ceil(parts / judge_run), sequences).  Every block of a sequence judges its drafts (from a few hundred numbers that
// the first kernel left, eight lanes a row) and sums the weights of its parts of the row that the next token comes from.
// CERTAIN, where the drafts are: a refused one's row is the target's without one token, so all parts but that token's
// weigh what the first kernel found, and one block a sequence does the rest, the draw included.
template <bool CERTAIN>
__global__ __launch_bounds__(THREADS) void verify_judge_kernel(Verify a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  Whole* rows = (Whole*)lds;               // [most + 1] of the target, [most] of the drafts
  __shared__ double ss[THREADS / WAVE];
  const int part0 = blockIdx.x * a.judge_run, seq = blockIdx.y, wave = threadIdx.x / WAVE, lane = threadIdx.x & 63;
  const int part1 = part0 + a.judge_run < a.parts ? part0 + a.judge_run : a.parts;
  int c0, c1;
  drafts_of(a, seq, c0, c1);
  const int d = c1 - c0;
  const float t = a.temperature[seq];
  const bool greedy = !(t > 0.f);
  const double c = greedy ? 1.0 : LOG2E / (double)t;
  // a lane for each draft (every wave judges all of them): its token and the two logits
  auto logits_of = [&](int j, bool& in, float& x, float& y) {
    const int tok = a.tokens[c0 + j];
    in = tok >= 0 && tok < a.vocab;
    x = a.logits[(c0 + seq + j) * a.ldl + (in ? tok : 0)];
    y = a.drafts ? a.drafts[(c0 + j) * a.ldd + (in ? tok : 0)] : 0.f;
  };
  bool in0 = false;
  float x0 = 0.f, y0 = 0.f, u0 = 0.f;
  if (lane < d) {
    u0 = a.uniform[c0 + seq + lane];
    logits_of(lane, in0, x0, y0);
  }
  const int n_rows = d + 1 + (a.drafts && !greedy ? d : 0), sub = threadIdx.x & 7;
  for (int q0 = 0; q0 < n_rows; q0 += THREADS / 8) {
    const int q = q0 + (int)threadIdx.x / 8, qc = q < n_rows ? q : n_rows - 1;
    const Piece16* p = a.pieces + (size_t)(qc <= d ? c0 + seq + qc : a.d + a.n + c0 + qc - d - 1) * a.parts;
    Whole w;
    w.max = -INFINITY;
    w.arg = -1;
    double sum = 0.0;
    // eight pieces a lane are asked for at once; a piece past the last is the last again and counts nothing
    for (int i0 = 0; i0 < a.parts; i0 += 64) {
      Piece16 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + 8 * k + sub;
        v[k] = p[i < a.parts ? i : a.parts - 1];
      }
      const float before = w.max;
#pragma unroll
      for (int k = 0; k < 8; ++k) take_max(w.max, w.arg, v[k].max, v[k].arg);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(w.max, o, WAVE);
        const int at2 = __shfl_xor(w.arg, o, WAVE);
        take_max(w.max, w.arg, m2, at2);
      }
      if (i0 > 0) sum *= weight(before, w.max, c);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += i0 + 8 * k + sub < a.parts ? v[k].sum * weight(v[k].max, w.max, c) : 0.0;
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor(sum, o, WAVE);
    w.inv = 1.0 / sum;
    if (sub == 0 && q < n_rows) rows[q] = w;
  }
  __syncthreads();
  int kept = d;
  for (int j0 = 0; j0 < d && kept == d; j0 += WAVE) {
    const int j = j0 + lane;
    if (j0 > 0 && j < d) {
      u0 = a.uniform[c0 + seq + j];
      logits_of(j, in0, x0, y0);
    }
    bool keep = true;
    if (j < d) {
      double p, q = 1.0;
      if (greedy) {
        p = in0 && a.tokens[c0 + j] == rows[j].arg ? 1.0 : 0.0;
        keep = p > 0.0;
      } else {
        p = in0 ? weight(x0, rows[j].max, c) * rows[j].inv : 0.0;
        if (a.drafts) q = in0 ? weight(y0, rows[d + 1 + j].max, c) * rows[d + 1 + j].inv : 0.0;
        keep = (double)u0 * q < p;
      }
      if (part0 == 0 && wave == 0 && a.probs) a.probs[c0 + j] = (float)p;
    }
    const unsigned long long refused = __ballot(!keep);
    if (refused) kept = j0 + __builtin_ctzll(refused);
  }
  if (part0 == 0 && wave == 0 && a.probs)             // the drafts behind the first 64 and a refused one have a probability too
    for (int j = (kept / WAVE + 1) * WAVE + lane; kept < d && j < d; j += WAVE) {
      logits_of(j, in0, x0, y0);
      a.probs[c0 + j] = !in0 ? 0.f : greedy ? (a.tokens[c0 + j] == rows[j].arg ? 1.f : 0.f) : (float)(weight(x0, rows[j].max, c) * rows[j].inv);
    }
  const bool refused = kept < d;
  const Whole r = rows[kept], less = rows[refused && a.drafts && !greedy ? d + 1 + kept : kept];
  const int row = c0 + seq + kept;
  Choice ch;
  ch.accepted = kept;
  ch.row = row;
  ch.draft_row = refused && !greedy && a.drafts ? c0 + kept : -1;
  ch.without = refused && !greedy && !a.drafts ? a.tokens[c0 + kept] : -1;
  ch.drawn = greedy ? (r.arg < 0 ? 0 : r.arg) : -1;
  ch.tmax = r.max;
  ch.dmax = less.max;
  ch.tinv = r.inv;
  ch.dinv = less.inv;
  const Piece16* own = a.pieces + (size_t)row * a.parts;
  const float* src = a.logits + row * a.ldl;
  if constexpr (CERTAIN) {
    const int special = ch.without >= 0 && ch.without < a.vocab ? ch.without / CHUNK : -1;
    double s = 0.0;
    if (special >= 0) {                    // the same in the whole block
      float x[PER];
      load16(src, special * CHUNK, a.vocab, x);
#pragma unroll
      for (int k = 0; k < PER; ++k) s += special * CHUNK + in_runs(k) == ch.without ? 0.0 : weight(x[k], r.max, c) * r.inv;
      s = wave_sum64(s);
      if (lane == 0) ss[wave] = s;
      __syncthreads();
      s = ss[0];
#pragma unroll
      for (int w = 1; w < THREADS / WAVE; ++w) s += ss[w];
    }
    draw(a, seq, ch, [&](int i) { return i == special ? s : share(own[i], r.max, r.inv, c); });
    return;
  }
  if (part0 == 0 && threadIdx.x == 0) a.choice[seq] = ch;
  if (greedy) return;
  if (!refused) {                          // the whole row: its parts' sums are known
    const int part = part0 + (int)threadIdx.x;
    if (part < part1) a.mass[(size_t)seq * a.parts + part] = share(own[part], r.max, r.inv, c);
    return;
  }
  const float* src2 = a.drafts + (long long)ch.draft_row * a.ldd;
  for (int part = part0; part < part1; ++part) {
    float x[PER], y[PER];
    load16(src, part * CHUNK, a.vocab, x);
    load16(src2, part * CHUNK, a.vocab, y);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const double w = weight(x[k], r.max, c) * r.inv - weight(y[k], less.max, c) * less.inv;
      s += fmax(w, 0.0);
    }
    s = wave_sum64(s);
    if (part > part0) __syncthreads();     // the part before has been read
    if (lane == 0) ss[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      s = ss[0];
#pragma unroll
      for (int w = 1; w < THREADS / WAVE; ++w) s += ss[w];
      a.mass[(size_t)seq * a.parts + part] = s;
    }
  }
}

// grid (sequences).  Draws from what the second kernel left.
__global__ __launch_bounds__(THREADS) void verify_draw_kernel(Verify a) {
  const int seq = blockIdx.x, lane = threadIdx.x & 63;
  const Choice ch = a.choice[seq];
  const double* mass = a.mass + (size_t)seq * a.parts;
  const double own = mass[lane < a.parts ? lane : 0];      // of the first 64 parts: asked for beside the choice
  draw(a, seq, ch, [&](int i) { return i < WAVE ? own : mass[i]; });
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
  Verify a = {logits, drafts, tokens, cu, temperature, uniform, accepted, token, probs, (Piece16*)at, nullptr, nullptr, ldl, ldd, n, d, vocab, (int)parts, most, 1, 1};
  at += round16(rows * parts * (long long)sizeof(Piece16));
  a.mass = (double*)at;
  at += round16(n * parts * 8);
  a.choice = (Choice*)at;
  // with many blocks a unit each takes several parts in turn; with few every part is a block of its own
  a.run = rows * parts >= 8192 ? 4 : 1;
  hipLaunchKernelGGL(verify_rows_kernel, dim3((unsigned)(rows * ((parts + a.run - 1) / a.run))), dim3(THREADS), 0, stream, a);
  DLGO_LAUNCH_CHECK("verify_drafts");
  if (!drafts) {
    hipLaunchKernelGGL(verify_judge_kernel<true>, dim3(1, (unsigned)n), dim3(THREADS), (most + 1) * (int)sizeof(Whole), stream, a);
    DLGO_LAUNCH_CHECK("verify_drafts");
    return nullptr;
  }
  a.judge_run = n * parts >= 1024 ? 2 : 1;
  hipLaunchKernelGGL(verify_judge_kernel<false>, dim3((unsigned)((parts + a.judge_run - 1) / a.judge_run), (unsigned)n), dim3(THREADS), (2 * most + 1) * (int)sizeof(Whole), stream, a);
  DLGO_LAUNCH_CHECK("verify_drafts");
  hipLaunchKernelGGL(verify_draw_kernel, dim3((unsigned)n), dim3(THREADS), 0, stream, a);
  DLGO_LAUNCH_CHECK("verify_drafts");
  return nullptr;
}

#include "exact_end.h"
