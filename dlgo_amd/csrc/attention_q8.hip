// Attention over the 8-bit cache (q8_page.h): softmax(q k^T * scale) v with the keys and values that the pages hold,
// for the rows of a step, each row seeing its sequence's tokens up to its own position (and no further back than the
// window).  One library per head size.  Queries and results are bfloat16; scores, softmax statistics and sums float32.
//
// A byte becomes a bfloat16 number exactly (one conversion instruction for two, the keys' power of two among its
// operands), so the products round nothing that the cache has not rounded already, except the probabilities: they are
// rounded to bfloat16 (half a step: 2^-9 of each, in the sum over the keys less than the result's own rounding) for the
// matrix instructions, as in the attention over a bfloat16 cache; the softmax's sum takes them unrounded.
//
//   attn_decode_kernel   steps that bring a few rows a sequence (a single token, drafted tokens): the pages of one
//                        (sequence, kv head) are dealt to the waves of a block, and to several blocks where there are
//                        too few; the columns of the matrix products are the group's heads of the sequence's rows.
//   attn_combine_kernel  joins what several blocks left for a row.
//   attn_prefill_kernel  prompts and pieces of prompts (more than 32 rows * heads of a group): 128 columns a block, pages
//                        turned to bfloat16 on their way into LDS.
//
// computerex/dlgo attends over float32 rows of the cache, one query at a time (models/llm/forward.go:258-278).
#include "q8_page.h"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 256, "head sizes come in steps of 16, up to 256");

#define HD HEAD_DIM
#define PIECES (HD / 16)                    // 16-byte pieces of a key, and rows of 16 of the turned values
#define KLOADS ((PIECES + 3) / 4)           // loads of a wave that bring 16 keys
#define PART_ROW (HD + 4)                   // floats of a partial result: values, maximum, sum

struct AttnQ8 {
  const bf16_t* q;
  bf16_t* out;
  float* part;
  const int32_t* cu_q;
  const int32_t* start_pos;
  const int32_t* slots;          // null: row i of page_table belongs to sequence i
  const int32_t* page_table;
  const uint8_t* cache;
  long long page_stride;
  int ldq, ldo, n_rows, n_seq, n_heads, n_kv, group, n_slots, max_pages, n_pages, window;
  float scale_log2e;             // not negative; `flip` is its sign
  uint32_t flip;
  int max_q, shared;             // rows of a sequence that are looked at; blocks that take one share of its pages (kv heads * chunks)
  int dealt, fill, most;         // how a sequence's pages are dealt to blocks: see Plan
  int tokens;                    // prompts: tokens of a tile
  const float* cos_t;            // FUSED: the rotation's tables
  const float* sin_t;
  int table_rows;
};
enum { WHOLE, EVENLY, BY_TILE };

// Waves of a block: four.  Eight leave room for one block a compute unit (a block's own start, its first trips to memory,
// is then nobody's time to use): 64 sequences of 2,300 tokens 31.1 against 29.3 us, 16 sequences with drafts 21.6 against 18.7.
#define WAVES 4

// The rows and pages of a sequence, from numbers that live on the device; nothing outside the buffers whatever they are.
struct Span {
  int row0, rows, start, len, slot, first_page, n_pages;
};
__device__ __forceinline__ Span span_of(const AttnQ8& a, int seq) {
  Span s;
  s.row0 = a.cu_q[seq];
  int row1 = a.cu_q[seq + 1];
  s.start = a.start_pos[seq];
  s.slot = a.slots ? a.slots[seq] : seq;
  if (s.row0 < 0) s.row0 = 0;
  if (row1 > a.n_rows) row1 = a.n_rows;
  s.rows = row1 - s.row0;
  if (s.rows > a.max_q) s.rows = a.max_q;
  if (s.start < 0 || s.slot < 0 || s.slot >= a.n_slots) s.rows = 0;
  if (s.rows < 0) s.rows = 0;
  s.len = s.start + s.rows;
  const int lo = a.window > 0 && s.start - a.window + 1 > 0 ? s.start - a.window + 1 : 0;
  s.first_page = lo / Q8_PAGE;
  int last = (s.len - 1) / Q8_PAGE;
  if (last >= a.max_pages) last = a.max_pages - 1;
  s.n_pages = s.rows > 0 && last >= s.first_page ? last - s.first_page + 1 : 0;
  return s;
}

// EVENLY: the blocks that share a sequence of n pages: enough to fill the chip, but not more than leave each wave a page, and so
// many that a wave has at most 16 pages, as far as the launch has them (`most`; else a wave has n / (4 * most) pages: 64 of
// a sequence of 2,048 pages among so many others that each goes to eight blocks at most).
__device__ __forceinline__ int even_shares(const AttnQ8& a, int n) {
  const int by_wave = (n + WAVES - 1) / WAVES, by_16 = (n + 16 * WAVES - 1) / (16 * WAVES);
  int s = a.fill < by_wave ? a.fill : by_wave;
  if (n < 16) s = 1;
  if (s < by_16) s = by_16;
  return s < 1 ? 1 : (s > a.most ? a.most : s);
}
#define TILE_PAGES 12            // a tile that sees fewer pages is one block's
// BY_TILE: the pages that a tile of a prompt sees ([lo, hi], nothing if hi < lo), and how many blocks share them.
__device__ __forceinline__ void tile_pages(const AttnQ8& a, const Span& s, int t0, int t1, int& lo, int& hi) {
  const int first = a.window > 0 && s.start + t0 - a.window + 1 > 0 ? s.start + t0 - a.window + 1 : 0;
  lo = first / Q8_PAGE;
  hi = (s.start + t1 - 1) / Q8_PAGE;
  if (hi >= a.max_pages) hi = a.max_pages - 1;
}
__device__ __forceinline__ int tile_shares(const AttnQ8& a, int pages) {
  const int n = pages / 4;
  return pages < TILE_PAGES ? 1 : (n < a.most ? n : a.most);
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// The maximum of a lane's value and that of the lane 32 (16) away.
__device__ __forceinline__ float max_32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// Sums are rescaled only where a maximum has grown by more than 2^8 over the one that they stand for: a probability is
// then at most 2^8, which costs float32 and bfloat16 none of their places.  (It takes 2^8 of their range: values from
// 2^119 on may overflow the sums.)
__device__ __forceinline__ bool has_grown(float mx, float m, float scale_log2e) { return (mx - m) * scale_log2e > 8.f; }

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
template <bool HI> __device__ __forceinline__ uint32_t pair_of(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, scale, HI));
}
// eight bytes -> eight bfloat16, times one power of two
__device__ __forceinline__ bf16x8_t eight(uint32_t w0, uint32_t w1, float scale) {
  uint4 u;
  u.x = pair_of<false>(w0, scale);
  u.y = pair_of<true>(w0, scale);
  u.z = pair_of<false>(w1, scale);
  u.w = pair_of<true>(w1, scale);
  return __builtin_bit_cast(bf16x8_t, u);
}
// the first `n` of a word's four bytes (n may be anything)
__device__ __forceinline__ uint32_t first_bytes(uint32_t w, int n) { return n >= 4 ? w : (n <= 0 ? 0u : w & ((1u << (8 * n)) - 1u)); }

// ---------------------------------------------------------------------------------------------------------------------
// Few rows a sequence.  grid: shares * sequences * chunks of columns * kv heads, WAVES waves.  A wave holds a whole page of
// its head in registers: the keys of 16 tokens are KLOADS loads of 16 bytes a lane, the values of 16 elements one, all
// of them consecutive in memory, and each is an operand of the matrix instructions as it lies once its bytes are
// converted.  The next page's loads are on their way while this one is multiplied.  The scores come out with a lane
// holding four neighbouring tokens of a column, which is the order of the values' bytes: no lane hands anything to
// another but the two exchanges of the maximum.
//
// Bound by memory where there is much of it: 64 sequences of 2,048 to 2,303 tokens, 32 heads of 64 over 8: 145 MB in 28.7 us,
// 5.1 TB/s, what a large copy reaches on this chip; 32 sequences of 64 to 8,192 tokens, heads of 128: 273 MB in 58 us, 4.7
// TB/s.  By latency where there is little: a block needs three trips to memory before its first product
// (the sequence's numbers, its page numbers, the page) and hands its result over, 5 us in all: one sequence of 2,300
// tokens takes 5.2 us and 4 for the join; 16 with up to six drafted tokens each (35 MB) 14.7 and 4.
// Measured and not kept: eight waves a block (see WAVES), one page's registers in place of two (the same), 128 registers
// a lane (spills), 4 or 8 pages a wave at least (slower from 8 sequences on), shares of about equal length worked out by
// every wave from the lengths on the device (0.7 us a kernel, and up to twice the time where the lengths are equal).
#define COLS(NC) (16 * (NC))
#define NC_MOST (HD <= 128 ? 2 : 1)                        // blocks of 16 columns whose sums a wave's registers hold beside two pages

struct PageRegs {
  uint4 k[4][KLOADS];
  uint4 v[PIECES];
  uint32_t ks;          // the scales of the keys of tokens 16 t + (lane % 16), t = 0 .. 3
  uint4 vs;             // the scales of the values of tokens 16 t + 4 (lane / 16) + r
};

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
static __device__ __forceinline__ uint4 buffer16(__amdgpu_buffer_rsrc_t r, int at, int fixed) {
  const u32x4_t v = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, at, fixed, 0));
  return make_uint4(v.x, v.y, v.z, v.w);
}

// Asks for a page.  Through a buffer descriptor: what lies beyond `bytes` (all of it, if that is 0: no such page) comes
// back as zeros without a trip to memory, so no load stands under a condition, and the loads of the next page stay in
// flight while this one is used.
static __device__ __forceinline__ void fetch_page(PageRegs& p, const uint8_t* head, int bytes, int lane) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)head, 0, bytes, 0x00027000);
  const int at = lane * 16;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int j = 0; j < KLOADS; ++j) p.k[t][j] = buffer16(r, at, (t * PIECES + 4 * j) * 256);
  p.ks = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (lane & 15) * 4, 2 * Q8_PAGE * HD, 0);
#pragma unroll
  for (int c = 0; c < PIECES; ++c) p.v[c] = buffer16(r, at, Q8_PAGE * HD + c * 1024);
  p.vs = buffer16(r, (lane >> 4) * 16, 2 * Q8_PAGE * HD + 64);
}

// Waves a SIMD that the registers are to allow: two places for a page, the sums and the queries.
#define EU(NC) ((NC) == 1 ? (HD <= 64 ? 3 : (HD <= 128 ? 2 : 1)) : ((NC) == 2 && HD <= 64 ? 2 : 1))

// The key and value of a step's own token, in the lanes in which a page has its places.
struct NewToken {
  uint4 k[KLOADS];               // piece 4 j + lane / 16 of the key (the lanes of a piece have the same)
  uint32_t v[PIECES];            // the byte of element 16 c + lane % 16 of the value
  uint32_t ks, vs;
};
// FUSED: rows of single tokens come unrotated, with their key and value behind the queries.  A wave rotates its own columns'
// queries, and the one that has the token's page rotates, rounds and stores the key and the value (as kv_q8.hip does, bit
// for bit) and puts them in their places in its registers; split halves over the whole head.  (Rows that a product left
// unsummed, added up here: 0.660 against 0.612 ms a step of 24 sequences with the sum in a launch of its own.)
#define FUSES (HD % 32 == 0 && HD <= 128)       // (larger ones do not fit the registers)
#define EU_OF(NC, FUSED) ((FUSED) ? (HD <= 64 ? 2 : 1) : EU(NC))

template <int NC, bool FUSED>
__global__ __launch_bounds__(WAVES* WAVE) __attribute__((amdgpu_waves_per_eu(EU_OF(NC, FUSED)))) void attn_decode_kernel(AttnQ8 a) {
  constexpr int QK = 2 * KLOADS;                         // matrix instructions for the scores of 16 tokens
  extern __shared__ __attribute__((aligned(16))) float merge[];    // [WAVES][COLS][HD], then [WAVES][COLS] maxima and sums
  const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);        // known to be the same in all lanes, as all that follows from it
  const int in_share = blockIdx.x % a.shared, kvh = in_share % a.n_kv, chunk = in_share / a.n_kv, item = blockIdx.x / a.shared;
  const int seq = item % a.n_seq, split = item / a.n_seq;
  const Span s = span_of(a, seq);
  const int used = a.dealt == EVENLY ? even_shares(a, s.n_pages) : 1;
  if (split >= used) return;
  const int cols = s.rows * a.group, col0 = chunk * COLS(NC);
  if (col0 >= cols) return;
  const int per = (s.n_pages + used - 1) / used;
  const int pg0 = s.first_page + split * per;
  const int pg1 = pg0 + per < s.first_page + s.n_pages ? pg0 + per : s.first_page + s.n_pages;      // pages [pg0, pg1)

  // The numbers of the wave's first 64 pages, one a lane, asked for together with the queries: page k of the wave is
  // first + k * WAVES.
  const int32_t* table = a.page_table + (size_t)s.slot * a.max_pages;
  const int turns = pg1 - pg0 > wave ? (pg1 - pg0 - wave + WAVES - 1) / WAVES : 0;
  const int first = turns > 0 ? pg0 + wave : 0;
  int ids = table[first + (lane < turns ? lane : 0) * WAVES];

  // this lane's column of each of the NC blocks of 16: a row of the step and a head (a column past the last reads the last)
  uint4 qraw[NC][QK];
  [[maybe_unused]] uint4 partner[FUSED ? QK : 1];
  [[maybe_unused]] float4 cs[FUSED ? 2 * QK : 1], sn[FUSED ? 2 * QK : 1];
  int pos[NC], lo[NC];
#pragma unroll
  for (int b = 0; b < NC; ++b) {
    const int col = col0 + 16 * b + n;
    const bool real = col < cols;
    const int at = real ? col : cols - 1, row = at / a.group, hig = at % a.group;
    pos[b] = real ? s.start + row : -1;
    lo[b] = a.window > 0 && pos[b] - a.window + 1 > 0 ? pos[b] - a.window + 1 : 0;
    const bf16_t* src = a.q + (size_t)(s.row0 + row) * a.ldq + (size_t)(kvh * a.group + hig) * HD;
#pragma unroll
    for (int j = 0; j < KLOADS; ++j)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int piece = 4 * j + g;
        const int d = piece < PIECES ? piece * 16 + m * 8 : 0;
        qraw[b][2 * j + m] = *(const uint4*)(src + d);
        if constexpr (FUSED) partner[2 * j + m] = *(const uint4*)(src + (d < HD / 2 ? d + HD / 2 : d - HD / 2));
      }
  }
  if constexpr (FUSED) {
    const size_t at = (size_t)(s.start < a.table_rows ? s.start : a.table_rows - 1) * (HD / 2);
#pragma unroll
    for (int j = 0; j < QK; ++j) {
      const int piece = 4 * (j / 2) + g, d = (piece < PIECES ? piece * 16 + (j & 1) * 8 : 0) % (HD / 2);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        cs[2 * j + e] = *(const float4*)(a.cos_t + at + d + 4 * e);
        sn[2 * j + e] = *(const float4*)(a.sin_t + at + d + 4 * e);
      }
    }
  }
  // eight elements of a head's piece (of this lane's j-th eight), rotated
  auto rotated = [&](int j, const uint4& own, const uint4& other, float* y) {
    const bool low = (4 * (j / 2) + g) * 16 < HD / 2;
    const uint32_t w[4] = {own.x, own.y, own.z, own.w}, o[4] = {other.x, other.y, other.z, other.w};
    const float c[8] = {cs[2 * j].x, cs[2 * j].y, cs[2 * j].z, cs[2 * j].w, cs[2 * j + 1].x, cs[2 * j + 1].y, cs[2 * j + 1].z, cs[2 * j + 1].w};
    const float sn8[8] = {sn[2 * j].x, sn[2 * j].y, sn[2 * j].z, sn[2 * j].w, sn[2 * j + 1].x, sn[2 * j + 1].y, sn[2 * j + 1].z, sn[2 * j + 1].w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16), z = __uint_as_float(e & 1 ? o[e / 2] & 0xffff0000u : o[e / 2] << 16);
      y[e] = low ? rotated_lo(x, z, c[e], sn8[e]) : rotated_hi(z, x, c[e], sn8[e]);
    }
  };
  f32x4_t o[NC][PIECES];
  float m[NC], l[NC];
#pragma unroll
  for (int b = 0; b < NC; ++b) {
    m[b] = -INFINITY;
    l[b] = 0.f;
#pragma unroll
    for (int c = 0; c < PIECES; ++c) o[b][c] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }
  bf16x8_t qf[NC][QK];
  auto queries = [&]() {
#pragma unroll
    for (int b = 0; b < NC; ++b)
#pragma unroll
      for (int j = 0; j < QK; ++j) {
        // pieces beyond the head count as zero (the keys' lanes then hold bytes of the next piece, never NaN)
        const bool ok = PIECES % 4 == 0 || 4 * (j / 2) + g < PIECES;
        uint4 u = qraw[b][j];
        if constexpr (FUSED) {
          float y[8];
          rotated(j, u, partner[j], y);
          u = make_uint4(Elem<bf16_t>::pair(y[0], y[1]), Elem<bf16_t>::pair(y[2], y[3]), Elem<bf16_t>::pair(y[4], y[5]), Elem<bf16_t>::pair(y[6], y[7]));
        }
        qf[b][j] = __builtin_bit_cast(bf16x8_t, ok ? make_uint4(u.x ^ a.flip, u.y ^ a.flip, u.z ^ a.flip, u.w ^ a.flip) : make_uint4(0, 0, 0, 0));
      }
  };

  const uint8_t* head = a.cache + (size_t)kvh * q8_head_bytes(HD);

  // the token's own page is this wave's last, or another wave's or nobody's
  [[maybe_unused]] const int own_page = s.start / Q8_PAGE, in = s.start & (Q8_PAGE - 1);
  [[maybe_unused]] const bool owner = FUSED && turns > 0 && first + (turns - 1) * WAVES == own_page;
  [[maybe_unused]] NewToken fresh;
  auto new_token = [&]() {
    if constexpr (FUSED) {
      const bf16_t* key = a.q + (size_t)s.row0 * a.ldq + (size_t)(a.n_heads + kvh) * HD;
      const bf16_t* val = key + (size_t)a.n_kv * HD;
      uint4 own[QK], other[QK];
      float v[PIECES];
#pragma unroll
      for (int j = 0; j < QK; ++j) {
        const int piece = 4 * (j / 2) + g, d = piece < PIECES ? piece * 16 + (j & 1) * 8 : 0;
        own[j] = *(const uint4*)(key + d);
        other[j] = *(const uint4*)(key + (d < HD / 2 ? d + HD / 2 : d - HD / 2));
      }
#pragma unroll
      for (int c = 0; c < PIECES; ++c) v[c] = bf16_to_f32(val[16 * c + n]);
      float y[QK][8];
      uint32_t kt = 0, vt = 0;
#pragma unroll
      for (int j = 0; j < QK; ++j) {
        rotated(j, own[j], other[j], y[j]);
        const uint32_t top = PIECES % 4 == 0 || 4 * (j / 2) + g < PIECES ? q8_top_bits(y[j]) : 0u;
        kt = top > kt ? top : kt;
      }
#pragma unroll
      for (int c = 0; c < PIECES; ++c) {
        const uint32_t top = __float_as_uint(v[c]) & 0x7fffffffu;
        vt = top > vt ? top : vt;
      }
#pragma unroll
      for (int o = 1; o < WAVE; o <<= 1) {
        uint32_t& m = o < 16 ? vt : kt;
        const uint32_t other_m = (uint32_t)__shfl_xor((int)m, o, WAVE);
        m = other_m > m ? other_m : m;
      }
      const bool finite = kt < 0x7f800000u && vt < 0x7f800000u;
      const int ke = q8_power_for(kt), ve = q8_power_for(vt);
      const float vf = __uint_as_float((uint32_t)(127 - ve) << 23);
#pragma unroll
      for (int j = 0; j < KLOADS; ++j) {
        const uint2 lo8 = q8_to_e4m3(y[2 * j], ke), hi8 = q8_to_e4m3(y[2 * j + 1], ke);
        fresh.k[j] = finite ? make_uint4(lo8.x, lo8.y, hi8.x, hi8.y) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < PIECES; ++c) fresh.v[c] = finite ? (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[c] * vf, v[c] * vf, 0, false) & 255u : 0u;
      fresh.ks = finite ? ke + 127 : Q8_NAN;
      fresh.vs = finite ? ve + 127 : 127;
    }
  };
  // into the page's bytes and into what this wave has of them
  auto take_in = [&](PageRegs& cur, int id) {
    if constexpr (FUSED) {
      const int t16 = in >> 4, i = in & 15, g0 = i >> 2, r8 = 8 * (i & 3);
      uint8_t* to = (uint8_t*)head + (size_t)id * a.page_stride;
      auto with = [&](uint32_t w, uint32_t byte, int at) { return (w & ~(255u << at)) | (byte << at); };
      if (n == i) {
#pragma unroll
        for (int j = 0; j < KLOADS; ++j)
          if (PIECES % 4 == 0 || 4 * j + g < PIECES) *(uint4*)(to + (t16 * PIECES + 4 * j + g) * 256 + 16 * i) = fresh.k[j];
        if (g == 0) to[2 * Q8_PAGE * HD + 4 * i + t16] = (uint8_t)fresh.ks;
      }
      if (g == g0) {
#pragma unroll
        for (int c = 0; c < PIECES; ++c) to[Q8_PAGE * HD + ((c * 4 + g0) * 16 + n) * 16 + 4 * t16 + (i & 3)] = (uint8_t)fresh.v[c];
        if (n == 0) to[2 * Q8_PAGE * HD + 64 + 16 * g0 + 4 * t16 + (i & 3)] = (uint8_t)fresh.vs;
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < KLOADS; ++j) {
          const bool here = t == t16 && n == i;
          cur.k[t][j] = make_uint4(here ? fresh.k[j].x : cur.k[t][j].x, here ? fresh.k[j].y : cur.k[t][j].y, here ? fresh.k[j].z : cur.k[t][j].z,
                                   here ? fresh.k[j].w : cur.k[t][j].w);
        }
      if (n == i) cur.ks = with(cur.ks, fresh.ks, 8 * t16);
      if (g == g0) {
#pragma unroll
        for (int c = 0; c < PIECES; ++c)
          cur.v[c] = make_uint4(t16 == 0 ? with(cur.v[c].x, fresh.v[c], r8) : cur.v[c].x, t16 == 1 ? with(cur.v[c].y, fresh.v[c], r8) : cur.v[c].y,
                                t16 == 2 ? with(cur.v[c].z, fresh.v[c], r8) : cur.v[c].z, t16 == 3 ? with(cur.v[c].w, fresh.v[c], r8) : cur.v[c].w);
        cur.vs = make_uint4(t16 == 0 ? with(cur.vs.x, fresh.vs, r8) : cur.vs.x, t16 == 1 ? with(cur.vs.y, fresh.vs, r8) : cur.vs.y,
                            t16 == 2 ? with(cur.vs.z, fresh.vs, r8) : cur.vs.z, t16 == 3 ? with(cur.vs.w, fresh.vs, r8) : cur.vs.w);
      }
    }
  };

  auto page = [&](PageRegs& cur, int key0) {
      f32x4_t sc[NC][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float ksc = q8_scale((cur.ks >> (8 * t)) & 255u);
#pragma unroll
        for (int b = 0; b < NC; ++b) sc[b][t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KLOADS; ++j) {
          uint4 u = cur.k[t][j];
          if (PIECES % 4 != 0 && 4 * j + g >= PIECES) u = make_uint4(0, 0, 0, 0);
          const bf16x8_t k0 = eight(u.x, u.y, ksc), k1 = eight(u.z, u.w, ksc);
#pragma unroll
          for (int b = 0; b < NC; ++b) {
            sc[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qf[b][2 * j], sc[b][t], 0, 0, 0);
            sc[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qf[b][2 * j + 1], sc[b][t], 0, 0, 0);
          }
        }
      }
      // element r of sc[b][t] is key  key0 + 16 t + 4 g + r  of column n
      const bool mask = key0 + Q8_PAGE - 1 > s.start || a.window > 0;
      bf16x8_t pf[NC][2];
#pragma unroll
      for (int b = 0; b < NC; ++b) {
        if (mask) {
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int key = key0 + 16 * t + 4 * g + r;
              sc[b][t][r] = key <= pos[b] && key >= lo[b] ? sc[b][t][r] : -INFINITY;
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[b][t][r]);
        mx = max_32(max_16(mx));
        if (__any(has_grown(mx, m[b], a.scale_log2e))) {
          const float m_new = fmaxf(m[b], mx);
          const float keep = m[b] == -INFINITY ? 0.f : fast_exp2((m[b] - m_new) * a.scale_log2e);
          l[b] *= keep;
#pragma unroll
          for (int c = 0; c < PIECES; ++c) o[b][c] *= keep;
          m[b] = m_new;
        }
        const float off = m[b] == -INFINITY ? 0.f : -m[b] * a.scale_log2e;
        float p[16];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = fast_exp2(fmaf(sc[b][t][r], a.scale_log2e, off));       // 0 where the score is -inf
            l[b] += e;
            // the value's power of two goes into the probability: exact, and its own bits are at hand
            const uint32_t w = t == 0 ? cur.vs.x : (t == 1 ? cur.vs.y : (t == 2 ? cur.vs.z : cur.vs.w));
            p[4 * t + r] = e * q8_scale((w >> (8 * r)) & 255u);
          }
        if (mask) {                                    // the power of a token that nobody sees may be anything
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = sc[b][i >> 2][i & 3] == -INFINITY ? 0.f : p[i];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 8; ++e) pf[b][h][e] = (__bf16)p[8 * h + e];
      }
      if (key0 + Q8_PAGE > s.len) {                    // tokens that the sequence does not hold: their bytes are anybody's
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
          const int k0 = s.len - key0 - 4 * g;
          cur.v[c] = make_uint4(first_bytes(cur.v[c].x, k0), first_bytes(cur.v[c].y, k0 - 16), first_bytes(cur.v[c].z, k0 - 32),
                                first_bytes(cur.v[c].w, k0 - 48));
        }
      }
#pragma unroll
      for (int c = 0; c < PIECES; ++c) {
        const bf16x8_t v0 = eight(cur.v[c].x, cur.v[c].y, 1.f), v1 = eight(cur.v[c].z, cur.v[c].w, 1.f);
#pragma unroll
        for (int b = 0; b < NC; ++b) {
          o[b][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, pf[b][0], o[b][c], 0, 0, 0);
          o[b][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, pf[b][1], o[b][c], 0, 0, 0);
        }
      }
  };

  // two places in registers, one filling while the other is used
  for (int k0 = 0; k0 < turns; k0 += 64) {
    const int pg = first + k0 * WAVES;
    const int here = turns - k0 < 64 ? turns - k0 : 64;
    if (k0 > 0) ids = table[pg + (lane < here ? lane : 0) * WAVES];
    bool real[2];
    PageRegs regs[2];
    auto fetch = [&](int k, int which) {
      const int id = __builtin_amdgcn_readlane(ids, k < here ? k : 0);
      real[which] = k < here && id >= 0 && id < a.n_pages;             // a hole counts nothing
      fetch_page(regs[which], (const uint8_t*)uniform_ptr(head + (size_t)(real[which] ? id : 0) * a.page_stride),
                 real[which] ? (int)q8_head_bytes(HD) : 0, lane);
    };
    fetch(0, 0);
    if (k0 == 0) {
      __builtin_amdgcn_sched_barrier(0);               // the queries are not waited for before the first page is asked for
      queries();
      if constexpr (FUSED)
        if (owner) new_token();
    }
    for (int k = 0; k < here; k += 2) {
      fetch(k + 1, 1);
      if constexpr (FUSED)
        if (real[0] && owner && k0 + k == turns - 1) take_in(regs[0], __builtin_amdgcn_readlane(ids, k));
      if (real[0]) page(regs[0], (pg + k * WAVES) * Q8_PAGE);
      fetch(k + 2, 0);
      if constexpr (FUSED)
        if (real[1] && owner && k0 + k + 1 == turns - 1) take_in(regs[1], __builtin_amdgcn_readlane(ids, k + 1));
      if (real[1]) page(regs[1], (pg + (k + 1) * WAVES) * Q8_PAGE);
    }
  }

  // the waves' results meet in LDS: element 4 g + r of o[b][c] is element 16 c + 4 g + r of the head, of column n
  float* mw = merge + WAVES * COLS(NC) * HD;
  float* lw = mw + WAVES * COLS(NC);
#pragma unroll
  for (int b = 0; b < NC; ++b) {
    l[b] += __shfl_xor(l[b], 16, WAVE);
    l[b] += __shfl_xor(l[b], 32, WAVE);
    const int col = 16 * b + n;
    if (g == 0) {
      mw[wave * COLS(NC) + col] = m[b];
      lw[wave * COLS(NC) + col] = l[b];
    }
    // 16 columns a row of the head apart would all fall on the same banks: pieces of 4 floats are moved by the column
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
      *(f32x4_t*)(merge + (size_t)(wave * COLS(NC) + col) * HD + (((4 * c + g) + col) % (HD / 4)) * 4) = o[b][c];
  }
  __syncthreads();
  const int left = cols - col0 < COLS(NC) ? cols - col0 : COLS(NC);
  for (int i = threadIdx.x; i < left * (HD / 4); i += WAVES * WAVE) {
    const int col = i / (HD / 4), e4 = i % (HD / 4);
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) M = fmaxf(M, mw[w * COLS(NC) + col]);
    float L = 0.f;
    f32x4_t acc = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float mm = mw[w * COLS(NC) + col], ll = lw[w * COLS(NC) + col];
      const float f = mm == -INFINITY ? 0.f : fast_exp2((mm - M) * a.scale_log2e);
      const f32x4_t v = *(const f32x4_t*)(merge + (size_t)(w * COLS(NC) + col) * HD + ((e4 + col) % (HD / 4)) * 4);
      // a wave whose scores are all NaN has no maximum but a sum that is NaN: it must reach the row
      L += mm == -INFINITY ? ll : f * ll;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += mm == -INFINITY ? v[e] : f * v[e];
    }
    const int row = s.row0 + (col0 + col) / a.group, h = kvh * a.group + (col0 + col) % a.group;
    if (used == 1) {
      const float inv = L == 0.f ? 0.f : 1.0f / L;       // a row that sees no token at all (its pages are missing): zeros
      Elem<bf16_t>::store4(a.out + (size_t)row * a.ldo + (size_t)h * HD + e4 * 4, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    } else {
      float* dst = a.part + (((size_t)row * a.n_heads + h) * a.most + split) * PART_ROW;
      *(f32x4_t*)(dst + e4 * 4) = acc;
      if (e4 == 0) {
        dst[HD] = M;
        dst[HD + 1] = L;
      }
    }
  }
}

// One wave for each row and head that several blocks left results of.  grid (most rows a sequence * heads, sequences).
#include "exact_begin.h"
__global__ __launch_bounds__(WAVE) void attn_combine_kernel(AttnQ8 a) {
  const int lane = threadIdx.x, h = blockIdx.x % a.n_heads, r = blockIdx.x / a.n_heads, seq = blockIdx.y;
  const Span s = span_of(a, seq);
  if (r >= s.rows) return;
  int pages = s.n_pages, used;                         // the pages that are shared, and by how many blocks
  if (a.dealt == BY_TILE) {
    const int t0 = r / a.tokens * a.tokens, t1 = t0 + a.tokens < s.rows ? t0 + a.tokens : s.rows;
    int lo, hi;
    tile_pages(a, s, t0, t1, lo, hi);
    pages = hi - lo + 1;
    used = tile_shares(a, pages);
  } else {
    used = even_shares(a, pages);
  }
  if (used == 1) return;                               // written by its block
  const int row = s.row0 + r;
  const float* base = a.part + ((size_t)row * a.n_heads + h) * a.most * PART_ROW;
  const int per = (pages + used - 1) / used;
  const int filled = (pages + per - 1) / per;          // shares that were given pages
  float M = -INFINITY;
  for (int i = lane; i < filled; i += WAVE) M = fmaxf(M, base[(size_t)i * PART_ROW + HD]);
  M = wave_max(M);
  constexpr int NE = (HD + WAVE - 1) / WAVE;
  float L = 0.f, acc[NE];
#pragma unroll
  for (int e = 0; e < NE; ++e) acc[e] = 0.f;
  // eight results at a time are asked for at once; what lies past the last is the last again, with no weight
  for (int i0 = 0; i0 < filled; i0 += 8) {
    float mm[8], ll[8], v[8][NE];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* p = base + (size_t)(i0 + i < filled ? i0 + i : filled - 1) * PART_ROW;
      mm[i] = p[HD];
      ll[i] = p[HD + 1];
#pragma unroll
      for (int e = 0; e < NE; ++e) v[i][e] = p[e * WAVE + lane < HD ? e * WAVE + lane : 0];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < filled) {
        const float f = mm[i] == -INFINITY ? 1.f : exp2f((mm[i] - M) * a.scale_log2e);       // -inf: zeros, or NaN
        L = fmaf(f, ll[i], L);
#pragma unroll
        for (int e = 0; e < NE; ++e) acc[e] = fmaf(f, v[i][e], acc[e]);
      }
  }
  const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
  for (int e = 0; e < NE; ++e)
    if (e * WAVE + lane < HD) a.out[(size_t)row * a.ldo + (size_t)h * HD + e * WAVE + lane] = f32_to_bf16(acc[e] * inv);
}
#include "exact_end.h"

// ---------------------------------------------------------------------------------------------------------------------
// Prompts.  A block of four waves takes 128 columns (tokens x the heads of a group) of a sequence and walks the pages.
// A page's bytes are turned to bfloat16 once for all its columns on the way into LDS (keys and values with their powers
// of two: exact), the next page's bytes are on their way meanwhile, and the two places in LDS are used in turn, so that
// a page costs one barrier.  Scores are kept transposed (keys x columns): a lane owns a column.
//
// Bound by instruction issue: a page is 32 scores a lane to scale, compare, raise and round beside 16 (head size 64) or 32
// (128) matrix instructions, and one wave a SIMD finds the two of little help to each other, two waves do (381 us, not 768,
// for 8 prompts of 64 to 2,048 tokens behind up to 2,048, 32 heads of 128 over 8).  Operands asked for four steps ahead: 366;
// sums rescaled only where a maximum has grown and maxima exchanged without LDS: 349; pages two ahead: 319 to 334, 660
// TFLOP/s.  A lone prompt of 2,048 tokens (heads of 64, 38.8 us) waits for its last tiles, 32 pages of 1.1 us one after the
// other.  Measured on that prompt and not kept: 64 columns a wave (78 us), eight waves with 256 columns (50 to 59: there are too
// few tiles of that size; with many tiles it was not measured), two teams of waves on alternate pages (45), the scores of the
// next page beside this one's softmax (-3%, and spills with heads of 128).  On the eight prompts: wave priorities raised
// around the products or the softmax (337 to 360 against 336).
#define PF_WAVES 4
#define PF_EU (HD <= 128 ? 2 : 1)           // waves a SIMD that the registers are to allow
#define DT ((HD + 31) / 32)                 // tiles of 32 elements of the result
#define KS (HD / 16)                        // steps of 16 along the head
#define LDS_K (Q8_PAGE * HD * 2)            // [element / 8][token][8 elements]
#define LDS_V (4 * 2 * DT * 32 * 16)        // [t][h][element][8 tokens: 16 t + 8 a + 4 h + r]

__global__ __launch_bounds__(PF_WAVES* WAVE) __attribute__((amdgpu_waves_per_eu(PF_EU))) void attn_prefill_kernel(AttnQ8 a) {
  extern __shared__ __attribute__((aligned(16))) char pf_lds[];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Late tiles see more keys than early ones: every sequence's tiles are dealt from its last one on, 256 blocks (one a
  // compute unit) at a time, every other time in reverse, so that the blocks that share a unit add up to about the same
  // number of pages and the launch ends with short ones.
  const int tokens = a.tokens, total = gridDim.x / a.most, width = a.n_seq * a.n_kv, split = blockIdx.x / total, block = blockIdx.x % total;
  const int turn = block >> 8, in_turn = total - (turn << 8) < 256 ? total - (turn << 8) : 256;
  const int place = turn & 1 ? (turn << 8) + in_turn - 1 - (block & 255) : block;
  const int kvh = place % a.n_kv, seq = place % width / a.n_kv;
  const Span s = span_of(a, seq);
  const int tile = (s.rows + tokens - 1) / tokens - 1 - place / width, t0 = tile * tokens;
  if (tile < 0) return;
  const int t1 = t0 + tokens < s.rows ? t0 + tokens : s.rows;        // the block's rows of the sequence
  int pg_lo, pg_hi;
  tile_pages(a, s, t0, t1, pg_lo, pg_hi);
  const int used = tile_shares(a, pg_hi - pg_lo + 1);
  if (split >= used) return;
  if (used > 1) {
    const int per = (pg_hi - pg_lo + used) / used;
    pg_lo += split * per;
    if (pg_lo + per - 1 < pg_hi) pg_hi = pg_lo + per - 1;
  }

  // this lane's column: a row of the sequence and a head (one past the last reads the block's first row and counts nothing)
  const int col = wave * 32 + (lane & 31), trow = t0 + col / a.group, hig = col % a.group;
  const bool mine = trow < t1 && col < tokens * a.group;
  const int pos = mine ? s.start + trow : -1;
  const int lo = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
  bf16x8_t qf[KS];
  {
    const bf16_t* src = a.q + (size_t)(s.row0 + (mine ? trow : t0)) * a.ldq + (size_t)(kvh * a.group + hig) * HD + half * 8;
    uint4 u[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) u[k] = *(const uint4*)(src + k * 16);
#pragma unroll
    for (int k = 0; k < KS; ++k) qf[k] = __builtin_bit_cast(bf16x8_t, make_uint4(u[k].x ^ a.flip, u[k].y ^ a.flip, u[k].z ^ a.flip, u[k].w ^ a.flip));
  }
  // pages up to position all_see and from any_lo on are seen whole by every column of the wave: they need no mask; pages
  // behind last_pos and before first_lo by none
  const int c0 = wave * 32, c1 = c0 + 31 < tokens * a.group - 1 ? c0 + 31 : tokens * a.group - 1;
  const int all_see = s.start + t0 + c0 / a.group;
  const int last_pos = s.start + (t0 + c1 / a.group < t1 - 1 ? t0 + c1 / a.group : t1 - 1);
  const int any_lo = a.window > 0 && last_pos - a.window + 1 > 0 ? last_pos - a.window + 1 : 0;
  const int first_lo = a.window > 0 && all_see - a.window + 1 > 0 ? all_see - a.window + 1 : 0;
  const bool some = c0 < tokens * a.group && t0 + c0 / a.group < t1;

  f32x16_t o[DT];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.f;

  const int32_t* table = a.page_table + (size_t)s.slot * a.max_pages;
  const uint8_t* head = a.cache + (size_t)kvh * q8_head_bytes(HD);
  // The 8 * HD pieces of a page, its keys' and then its values', are shared out over the threads: a wave's 64 are of one kind.
  constexpr int THREADS = PF_WAVES * WAVE, NP = (8 * HD + THREADS - 1) / THREADS;
  struct Raw {
    uint4 piece[NP];
    uint32_t ks;                             // the scales of the keys of tokens 16 t + (lane % 16)
    uint4 vs;                                // the scales of the values of tokens 16 t + 4 (lane / 16) + r
    int there;                               // whether there is such a page
  };
  int id = table[pg_lo <= pg_hi ? pg_lo : 0];            // the number of the page that is asked for next, known a page ahead
  auto fetch = [&](Raw& x, int pg) {                     // pages are asked for in order
    const int after = table[pg < pg_hi ? pg + 1 : pg_hi];
    x.there = id >= 0 && id < a.n_pages;
    const uint8_t* p = head + (size_t)(x.there ? id : 0) * a.page_stride;
    x.ks = *(const uint32_t*)(p + 2 * Q8_PAGE * HD + (lane & 15) * 4);
    x.vs = *(const uint4*)(p + 2 * Q8_PAGE * HD + 64 + (lane >> 4) * 16);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int w0 = i * THREADS + wave * WAVE;
      x.piece[i] = *(const uint4*)(p + ((i + 1) * THREADS <= 8 * HD || w0 < 8 * HD ? w0 * 16 : 0) + lane * 16);
    }
    id = after;
  };
  auto stage = [&](Raw& x, char* lds, int key0) {
    // tokens that the sequence does not hold, or a page that is not there: zeros, with a power that leaves them zeros
    const int left = x.there ? s.len - key0 : 0;
    if (left < Q8_PAGE) {
      const int n = left - 4 * (lane >> 4);
      x.vs = make_uint4(first_bytes(x.vs.x, n), first_bytes(x.vs.y, n - 16), first_bytes(x.vs.z, n - 32), first_bytes(x.vs.w, n - 48));
#pragma unroll
      for (int i = 0; i < NP; ++i)
        if ((i + 1) * THREADS > 4 * HD && i * THREADS + wave * WAVE >= 4 * HD)
          x.piece[i] = make_uint4(first_bytes(x.piece[i].x, n), first_bytes(x.piece[i].y, n - 16), first_bytes(x.piece[i].z, n - 32), first_bytes(x.piece[i].w, n - 48));
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int w0 = i * THREADS + wave * WAVE;
      const uint4 u = x.piece[i];
      if ((i + 1) * THREADS <= 4 * HD || w0 < 4 * HD) {
        // piece p of token 16 t + (lane % 16)
        const int tp = w0 / 16 + (lane >> 4), t = tp / PIECES, p = tp % PIECES, token = 16 * t + (lane & 15);
        const float ksc = q8_scale((x.ks >> (8 * t)) & 255u);
        *(bf16x8_t*)(lds + ((2 * p) * Q8_PAGE + token) * 16) = eight(u.x, u.y, ksc);
        *(bf16x8_t*)(lds + ((2 * p + 1) * Q8_PAGE + token) * 16) = eight(u.z, u.w, ksc);
      } else if ((i + 1) * THREADS <= 8 * HD || w0 < 8 * HD) {
        // element d, tokens 16 t + 4 g + r
        const int d = (w0 / 64 - HD / 16) * 16 + (lane & 15), g = lane >> 4;
        char* dst = lds + LDS_K + ((g & 1) * (DT * 32) + d) * 16 + (g >> 1) * 8;
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4) {
          const uint32_t w = t4 == 0 ? u.x : (t4 == 1 ? u.y : (t4 == 2 ? u.z : u.w));
          const uint32_t sc = t4 == 0 ? x.vs.x : (t4 == 1 ? x.vs.y : (t4 == 2 ? x.vs.z : x.vs.w));
          // each of a word's four has a power of its own: convert a pair with either and keep the half that is meant
          const uint32_t a0 = pair_of<false>(w, q8_scale(sc & 255u)), a1 = pair_of<false>(w, q8_scale((sc >> 8) & 255u));
          const uint32_t b0 = pair_of<true>(w, q8_scale((sc >> 16) & 255u)), b1 = pair_of<true>(w, q8_scale(sc >> 24));
          *(uint2*)(dst + t4 * (2 * DT * 32 * 16)) = make_uint2((a0 & 0xffffu) | (a1 & 0xffff0000u), (b0 & 0xffffu) | (b1 & 0xffff0000u));
        }
      }
    }
  };

  // One page: its bytes lie in LDS; the next page's are in `soon` (asked for a page ago) and go there after it, those of
  // the page after that are asked for into `later`: a trip to memory takes longer than a page.
  int ok = 0;
  auto page = [&](int pg, Raw& soon, Raw& later) {
    fetch(later, pg + 2);
    const int key0 = pg * Q8_PAGE;
    const char* lds = pf_lds + ((pg - pg_lo) & 1) * (LDS_K + LDS_V);
    if (ok && some && key0 <= last_pos && key0 + Q8_PAGE > first_lo) {
      f32x16_t sc[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[kt][v] = 0.f;
      // the operands of four steps are asked for together, and the two tiles of keys take turns: nothing waits for the
      // instruction before it
#pragma unroll
      for (int k0 = 0; k0 < KS; k0 += 4) {
        bf16x8_t kf[4][2];
#pragma unroll
        for (int k = k0; k < KS && k < k0 + 4; ++k)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) kf[k - k0][kt] = *(const bf16x8_t*)(lds + ((2 * k + half) * Q8_PAGE + kt * 32 + (lane & 31)) * 16);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = k0; k < KS && k < k0 + 4; ++k)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) sc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[k - k0][kt], qf[k], sc[kt], 0, 0, 0);
      }
      // element v of sc[kt] is key  key0 + 32 kt + 8 (v / 4) + 4 half + v % 4  of the lane's column
      if (key0 + Q8_PAGE - 1 > all_see || key0 < any_lo) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int key = key0 + kt * 32 + 8 * (v >> 2) + 4 * half + (v & 3);
            sc[kt][v] = key <= pos && key >= lo ? sc[kt][v] : -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sc[kt][v]);
      mx = max_32(mx);
      if (__any(has_grown(mx, m, a.scale_log2e))) {
        const float m_new = fmaxf(m, mx);
        const float keep = m == -INFINITY ? 0.f : fast_exp2((m - m_new) * a.scale_log2e);
        l *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] *= keep;
        m = m_new;
      }
      const float off = m == -INFINITY ? 0.f : -m * a.scale_log2e;
      bf16x8_t pf[4];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const float e = fast_exp2(fmaf(sc[kt][v], a.scale_log2e, off));
          l += e;
          pf[2 * kt + (v >> 3)][v & 7] = (__bf16)e;
        }
      // element e of pf[t] is key  16 t + 8 (e / 4) + 4 half + e % 4: the values lie in LDS in that order
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const bf16x8_t vf = *(const bf16x8_t*)(lds + LDS_K + ((t * 2 + half) * (DT * 32) + d * 32 + (lane & 31)) * 16);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[t], o[d], 0, 0, 0);
        }
    }
    if (pg < pg_hi) {
      stage(soon, pf_lds + ((pg - pg_lo + 1) & 1) * (LDS_K + LDS_V), key0 + Q8_PAGE);
      ok = soon.there;
    }
    __syncthreads();
  };
  if (pg_lo <= pg_hi) {                      // else the window begins behind the table: nothing to see
    Raw x, y;
    fetch(x, pg_lo);
    fetch(y, pg_lo + 1);
    stage(x, pf_lds, pg_lo * Q8_PAGE);
    ok = x.there;
    __syncthreads();
    for (int pg = pg_lo; pg <= pg_hi; pg += 2) {
      page(pg, y, x);
      if (pg < pg_hi) page(pg + 1, x, y);
    }
  }
  l += __shfl_xor(l, 32, WAVE);
  if (!mine) return;
  if (used > 1) {
    float* to = a.part + (((size_t)(s.row0 + trow) * a.n_heads + kvh * a.group + hig) * a.most + split) * PART_ROW;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int qd = 0; qd < 4; ++qd) {
        const int e = d * 32 + 8 * qd + 4 * half;
        if (e < HD) *(f32x4_t*)(to + e) = (f32x4_t){o[d][4 * qd], o[d][4 * qd + 1], o[d][4 * qd + 2], o[d][4 * qd + 3]};
      }
    if (half == 0) {
      to[HD] = m;
      to[HD + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  bf16_t* dst = a.out + (size_t)(s.row0 + trow) * a.ldo + (size_t)(kvh * a.group + hig) * HD;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int qd = 0; qd < 4; ++qd) {
      const int e = d * 32 + 8 * qd + 4 * half;
      if (e < HD) Elem<bf16_t>::store4(dst + e, o[d][4 * qd] * inv, o[d][4 * qd + 1] * inv, o[d][4 * qd + 2] * inv, o[d][4 * qd + 3] * inv);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// What a launch looks like, from sizes that the host knows.  max_q_len and max_kv_len bound the sequences' rows and
// lengths (a recorded launch passes the context's).
struct Plan {
  int tiled, nc, chunks, dealt, fill, most, tokens;
  long long items;                           // shares of sequences that there may be
};
static Plan plan_of(int n_seq, int n_heads, int n_kv, int max_q_len, int max_kv_len, int window) {
  Plan p = {};
  const int group = n_heads / n_kv;
  const long long cols = (long long)max_q_len * group;
  int pages = (max_kv_len + Q8_PAGE - 1) / Q8_PAGE;
  if (window > 0) {
    const long long seen = ((long long)window + max_q_len + Q8_PAGE - 2) / Q8_PAGE + 1;      // a window may be any int
    if (seen < pages) pages = (int)seen;
  }
  const int chip = 512;
  // Up to 32 columns: with 20 and 32 of them the tiles are slower for heads of 64 (16 sequences with up to 24 columns behind
  // 128 to 4,089 tokens 28 against 18.5 us) and as fast for 128; with 36 to 64 they are faster from no past to 16,384 tokens
  // (16 sequences behind 1,024: 22 against 26 to 29, and 29 against 40 to 43), but for 48 and more behind 4,096 (96 against
  // 86 to 96, 133 against 115).
  p.tiled = cols > 32;
  if (p.tiled) {
    // Few tiles behind a long past (the next turn of a conversation, a piece of a prompt) would each walk all of it alone, a
    // page in 1.0 us (head size 64) to 1.4 (128): their pages are dealt to as many blocks as fill the chip.  Joining them costs
    // 5 us and, in full, 36 to 69 MB of partial results, some 8 pages and 16 more, which the dealing has to save.  17 rows
    // behind 16,384 tokens, 32 heads over 8: 260 -> 27 us and (128) 351 -> 33; 512 rows 266 -> 120, 362 -> 173; four
    // sequences of 17 rows 266 -> 40, 355 -> 54; 1,024 rows behind 2,048, where it does not: 54 against 65, 74 against 83.
    p.tokens = PF_WAVES * 32 / group;
    p.items = (long long)((max_q_len + p.tokens - 1) / p.tokens) * n_seq;
    const long long blocks = p.items * n_kv;
    p.most = (int)(chip / blocks < pages / 4 ? chip / blocks : pages / 4);
    if (p.most < 1) p.most = 1;
    const int halves = blocks * p.most > chip / 2 ? 3 : 2;       // two blocks a unit take 1.5 times as long a page
    p.dealt = pages - pages * halves / (2 * p.most) >= 8 + 16 * blocks * p.most / chip ? BY_TILE : WHOLE;
    if (p.dealt == WHOLE) p.most = 1;
    return p;
  }
  p.nc = cols <= 16 ? 1 : 2;
  if (p.nc > NC_MOST) p.nc = NC_MOST;
  p.chunks = (int)((cols + 16 * p.nc - 1) / (16 * p.nc));
  // How the pages are dealt.  One block a (sequence, kv head) takes `turn` ns for every page a wave; dealing them to as many
  // blocks as fill the chip costs a launch that joins their results, 4 us, and saves nothing of the time that the memory
  // needs (counted at 0.7 of the bound, since lengths differ).  Dealt and whole, us: one sequence of 24 and 40 pages 8.5 and
  // 8.0, 9.3 and 10.6 (head size 64), 9.6 and 10.0, 10.4 and 13.3 (128); 16 of 32 and 126 pages 12.1 and 10.5, 28.2 and 25.7,
  // 18.9 and 14.8, 46.3 and 41.5; 4 of 313 to 512 pages 27 and 88; 16 of up to 64 pages with drafts 18.3 and 20.9.  However
  // many sequences there are, one of more than 128 pages goes to up to eight blocks at least.
  const long long pairs = (long long)n_seq * n_kv * p.chunks, turn = (400 + 7 * HD / 2) * (p.nc == 2 ? 8 : 5) / 5;
  const int by_wave = (pages + WAVES - 1) / WAVES, by_16 = (pages + 16 * WAVES - 1) / (16 * WAVES);
  const bool pays = by_wave * turn - pairs * pages * q8_head_bytes(HD) / 5200 * 7 / 10 > 4000;
  p.fill = pays && pairs < chip ? (int)((chip + pairs - 1) / pairs) : 1;
  p.most = p.fill < by_wave ? p.fill : by_wave;
  if (pages > 128 && p.most < by_16) p.most = by_16 < 8 ? by_16 : (p.most < 8 ? 8 : p.most);       // (blocks that a short sequence has no use for)
  if (p.most < 1) p.most = 1;
  p.dealt = p.most > 1 ? EVENLY : WHOLE;
  p.items = (long long)n_seq * p.most;
  return p;
}

static long long scratch_of(const Plan& p, int n_rows, int n_heads) {
  return p.dealt == WHOLE ? 0 : (long long)n_rows * p.most * n_heads * PART_ROW;
}

extern "C" int dlgo_attention_q8_head_dim() { return HD; }

// floats of scratch that a launch needs (0: none)
extern "C" long long dlgo_attention_q8_scratch(int n_rows, int n_seq, int n_heads, int n_kv, int max_q_len, int max_kv_len, int window) {
  if (n_rows <= 0 || n_seq <= 0 || n_kv <= 0 || n_heads < n_kv || max_q_len <= 0 || max_kv_len <= 0) return 0;
  const Plan p = plan_of(n_seq, n_heads, n_kv, max_q_len, max_kv_len, window);
  return scratch_of(p, n_rows, n_heads);
}

template <int NC, bool FUSED>
static hipError_t launch_decode(const AttnQ8& a, dim3 grid, hipStream_t stream) {
  const int lds = WAVES * COLS(NC) * (HD + 2) * 4;       // the waves' results
  hipError_t e = hipSuccess;
  if (lds > 64 * 1024) e = hipFuncSetAttribute((const void*)attn_decode_kernel<NC, FUSED>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e == hipSuccess) hipLaunchKernelGGL((attn_decode_kernel<NC, FUSED>), grid, dim3(WAVES * WAVE), lds, stream, a);
  return e;
}

extern "C" const char* dlgo_attention_q8(const void* q, int ldq, void* out, int ldo, int n_rows, int n_seq, int n_heads, int n_kv, int head_dim,
                                         const int32_t* cu_q, const int32_t* start_pos, const int32_t* slots, const int32_t* page_table,
                                         int n_slots, int max_pages, const void* cache, long long page_stride, int n_pages, int max_q_len,
                                         int max_kv_len, int window, float scale, float* part, long long part_elems, const float* cos_t,
                                         const float* sin_t, int table_rows, hipStream_t stream) {
  DLGO_REQUIRE(head_dim == HD, "attention_q8: this library is built for a head size of %d, not %d", HD, head_dim);
  DLGO_REQUIRE(n_rows >= 0 && n_seq >= 0 && n_kv > 0 && n_heads >= n_kv && n_heads % n_kv == 0, "attention_q8: %d heads over %d kv heads", n_heads, n_kv);
  DLGO_REQUIRE(n_heads / n_kv <= 128, "attention_q8: at most 128 heads share a kv head, not %d", n_heads / n_kv);
  if (n_rows == 0 || n_seq == 0 || max_q_len == 0) return nullptr;
  DLGO_REQUIRE(max_q_len > 0 && max_kv_len > 0 && n_slots > 0 && max_pages > 0 && n_pages > 0, "attention_q8: bad bounds");
  DLGO_REQUIRE(scale - scale == 0.f && scale != 0.f, "attention_q8: the scale must be finite and not zero");
  DLGO_REQUIRE(((uintptr_t)q & 15) == 0 && ldq % 8 == 0 && ldq >= n_heads * HD && ((uintptr_t)out & 7) == 0 && ldo % 4 == 0 && ldo >= n_heads * HD,
               "attention_q8: query rows must be 16-byte aligned, result rows 8-byte aligned (strides %d and %d)", ldq, ldo);
  DLGO_REQUIRE(((uintptr_t)cache & 15) == 0 && page_stride % 16 == 0 && page_stride >= n_kv * q8_head_bytes(HD),
               "attention_q8: pages %lld bytes apart (16-byte aligned pages of at least %lld bytes are needed)", page_stride, n_kv * q8_head_bytes(HD));
  DLGO_REQUIRE(n_seq <= 65535, "attention_q8: at most 65535 sequences");
  DLGO_REQUIRE(!cos_t || (FUSES && sin_t && table_rows > 0 && max_q_len == 1 && n_heads / n_kv <= 16 && ldq >= (n_heads + 2 * n_kv) * HD &&
                          ((uintptr_t)cos_t & 15) == 0 && ((uintptr_t)sin_t & 15) == 0),
               "attention_q8: rotates single tokens of up to 16 heads a kv head, of sizes in steps of 32 up to 128 (head size %d, %d heads over %d)", HD, n_heads, n_kv);
  if (max_kv_len > max_pages * (long long)Q8_PAGE) max_kv_len = max_pages * Q8_PAGE;
  const Plan p = plan_of(n_seq, n_heads, n_kv, max_q_len, max_kv_len, window);
  AttnQ8 a = {(const bf16_t*)q, (bf16_t*)out, part, cu_q, start_pos, slots, page_table, (const uint8_t*)cache, page_stride, ldq, ldo, n_rows, n_seq,
              n_heads, n_kv, n_heads / n_kv, n_slots, max_pages, n_pages, window > 0 ? window : 0,
              (scale < 0 ? -scale : scale) * 1.44269504088896341f, scale < 0 ? 0x80008000u : 0u, max_q_len, n_kv * p.chunks, p.dealt, p.fill, p.most, p.tokens, cos_t, sin_t, table_rows};
  hipError_t e = hipSuccess;
  const long long need = scratch_of(p, n_rows, n_heads), blocks = p.items * (p.tiled ? (long long)n_kv * p.most : a.shared);
  DLGO_REQUIRE(need == 0 || (part && part_elems >= need && ((uintptr_t)part & 15) == 0), "attention_q8: scratch of %lld floats is needed, %lld given", need, part ? part_elems : 0ll);
  DLGO_REQUIRE(blocks < (1ll << 31), "attention_q8: too many rows at once");
  if (p.tiled) {
    const int lds = 2 * (LDS_K + LDS_V);
    if (lds > 64 * 1024) e = hipFuncSetAttribute((const void*)attn_prefill_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e == hipSuccess) hipLaunchKernelGGL(attn_prefill_kernel, dim3((unsigned)blocks), dim3(PF_WAVES * WAVE), lds, stream, a);
  } else {
    const dim3 grid((unsigned)blocks);
    e = hipErrorInvalidValue;
    if constexpr (FUSES) if (cos_t) e = launch_decode<1, true>(a, grid, stream);
    if (p.nc == 1 && !cos_t) e = launch_decode<1, false>(a, grid, stream);
    if constexpr (NC_MOST >= 2) if (p.nc == 2) e = launch_decode<2, false>(a, grid, stream);
  }
  if (e == hipSuccess && p.dealt) {
    DLGO_LAUNCH_CHECK("attention_q8");
    hipLaunchKernelGGL(attn_combine_kernel, dim3((unsigned)(max_q_len * n_heads), (unsigned)n_seq), dim3(WAVE), 0, stream, a);
  }
  DLGO_REQUIRE(e == hipSuccess, "attention_q8: %s", hipGetErrorString(e));
  DLGO_LAUNCH_CHECK("attention_q8");
  return nullptr;
}
