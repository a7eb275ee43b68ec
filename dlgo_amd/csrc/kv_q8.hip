// Rotation of a step's queries and keys, fused with the write of keys and values into the 8-bit cache (q8_page.h).
//
// For a token's key (rotated) or value x of one head:  e = the least integer with max|x| <= 448 * 2^e (at least -126),
//   byte_d = e4m3(x_d * 2^-e), to nearest, ties to even;  scale = e + 127.
// The multiplication is exact, so an element is rounded once, from float32: off by at most 2^-4 of itself (half a step
// of e4m3's 3 bits), or 2^-10 * 2^e below e4m3's smallest normal number.  computerex/dlgo keeps keys and values in
// float32 (memory/kvcache.go:5-9); its weights' 8-bit blocks carry a scale each (quant/dequant.go), as tokens do here.
//
// Bound by memory: a row is read once (the second read of a partner piece hits the cache), queries are written in
// bfloat16, keys and values in 8 bits: 17,408 rows of 24 heads of 128 over 8, 330 MB, in 65.5 us, 5.0 TB/s.  Eight single
// tokens take 4.5 us, a launch and three trips to memory.  A rotated width that is no multiple of 16, or rows that are not
// 16-byte aligned, go element by element: 82 us for eight tokens of those heads, 1.1 to 1.7 ms for the 17,408 rows.
#include "q8_page.h"
// everything here is float32 arithmetic whatever the storage type: no approximation can be named (exact_begin.h)
#include "exact_begin.h"

struct RopeQ8 {
  const bf16_t* qkv;
  bf16_t* q_out;
  uint8_t* cache;
  const float* cos_t;
  const float* sin_t;
  const int32_t* positions;
  const int32_t* tok_seq;
  const int32_t* slots;
  const int32_t* page_table;
  long long page_stride;
  int ld, ldq, n_tokens, n_heads, n_kv, hd, rot, interleaved, table_rows, n_seq, n_slots, max_pages, n_pages;
  const float* part;             // where the product that makes the rows left the runs of its inner sum unsummed: n_parts
  long long plane;               // planes of float32, `plane` apart, rows part_ld apart
  int n_parts, part_ld;
};

static __device__ __forceinline__ void load8(const bf16_t* p, float* f) {
  const uint4 u = *(const uint4*)p;
  f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
  f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
  f[4] = __uint_as_float(u.z << 16); f[5] = __uint_as_float(u.z & 0xffff0000u);
  f[6] = __uint_as_float(u.w << 16); f[7] = __uint_as_float(u.w & 0xffff0000u);
}

// The sum of the runs in their order, B of them asked for at once; one past the last is the last again and is not added.
template <int B>
static __device__ __forceinline__ void sum8(const RopeQ8& a, const float* p, float* f) {
  for (int s0 = 0; s0 < a.n_parts; s0 += B) {
    float4 v[B][2];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const float* q = p + (s0 + i < a.n_parts ? s0 + i : a.n_parts - 1) * a.plane;
      v[i][0] = *(const float4*)q;
      v[i][1] = *(const float4*)(q + 4);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const float w[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w, v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = s0 + i == 0 ? w[e] : (s0 + i < a.n_parts ? f[e] + w[e] : f[e]);
    }
  }
}
// Eight elements of row t from column `col` on: from the rows themselves or, SUMS, from the runs.
template <bool SUMS>
static __device__ __forceinline__ void row8(const RopeQ8& a, int t, int col, float* f) {
  if constexpr (!SUMS) {
    load8(a.qkv + (size_t)t * a.ld + col, f);
  } else {
    const float* p = a.part + (size_t)t * a.part_ld + col;
    if (a.n_parts <= 2) sum8<2>(a, p, f);
    else sum8<4>(a, p, f);
  }
}

static __device__ __forceinline__ void store8(bf16_t* p, const float* f) {
  *(uint4*)p = make_uint4(Elem<bf16_t>::pair(f[0], f[1]), Elem<bf16_t>::pair(f[2], f[3]), Elem<bf16_t>::pair(f[4], f[5]), Elem<bf16_t>::pair(f[6], f[7]));
}

// Eight elements of a head (from column `col` of row t on) from element d0 on, rotated.  PIECES: pairs lie in this piece (interleaved) or are this piece
// and the one half a rotated width away, all 16-byte aligned; else element by element.
template <bool PIECES, bool SUMS>
static __device__ __forceinline__ void rotated8(const RopeQ8& a, int t, int col, int pos, int d0, float* y) {
  const int half = a.rot / 2;
  // a position beyond the table is the caller's mistake: it must not become a read out of bounds
  const size_t at = (size_t)(pos < 0 ? 0 : (pos < a.table_rows ? pos : a.table_rows - 1)) * half;
  if constexpr (PIECES) {
    row8<SUMS>(a, t, col + d0, y);
    if (!a.cos_t || d0 >= a.rot) return;
    float c[8], s[8], x[8];
    if (a.interleaved) {
      *(float4*)c = *(const float4*)(a.cos_t + at + d0 / 2);
      *(float4*)s = *(const float4*)(a.sin_t + at + d0 / 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x0 = y[2 * i], x1 = y[2 * i + 1];
        y[2 * i] = rotated_lo(x0, x1, c[i], s[i]);
        y[2 * i + 1] = rotated_hi(x0, x1, c[i], s[i]);
      }
      return;
    }
    const bool low = d0 < half;
    const int i0 = low ? d0 : d0 - half;
    row8<SUMS>(a, t, col + (low ? d0 + half : d0 - half), x);
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      *(float4*)(c + e) = *(const float4*)(a.cos_t + at + i0 + e);
      *(float4*)(s + e) = *(const float4*)(a.sin_t + at + i0 + e);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = low ? rotated_lo(y[e], x[e], c[e], s[e]) : rotated_hi(x[e], y[e], c[e], s[e]);
  } else {
    const bf16_t* head = a.qkv + (size_t)t * a.ld + col;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e;
      float v = bf16_to_f32(head[d]);
      if (a.cos_t && d < a.rot) {
        const int i = a.interleaved ? d / 2 : (d < half ? d : d - half);
        const bool low = a.interleaved ? (d & 1) == 0 : d < half;
        const float o = bf16_to_f32(head[a.interleaved ? (d ^ 1) : (low ? d + half : d - half)]);
        const float c = a.cos_t[at + i], s = a.sin_t[at + i];
        v = low ? rotated_lo(v, o, c, s) : rotated_hi(o, v, c, s);
      }
      y[e] = v;
    }
  }
}

template <bool PIECES, bool SUMS>
static __device__ __forceinline__ void plain8(const RopeQ8& a, int t, int col, float* y) {
  if constexpr (PIECES) {
    row8<SUMS>(a, t, col, y);
  } else {
    const bf16_t* p = a.qkv + (size_t)t * a.ld + col;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) y[e] = bf16_to_f32(p[e]);
  }
}

// Where row t's token lies: its page's offset in the cache (-1 if there is no such page: nothing is written) and its
// place in the page.
static __device__ __forceinline__ long long page_of(const RopeQ8& a, int t, int pos) {
  const int seq = a.tok_seq[t];
  if (seq < 0 || seq >= a.n_seq || pos < 0 || pos / Q8_PAGE >= a.max_pages) return -1;
  const int slot = a.slots[seq];
  if (slot < 0 || slot >= a.n_slots) return -1;
  const int page = a.page_table[(size_t)slot * a.max_pages + pos / Q8_PAGE];
  return page < 0 || page >= a.n_pages ? -1 : (long long)page * a.page_stride;
}

// The queries.  A thread takes a piece of eight elements, or the two pieces whose elements are each other's partners, of
// QH (four) heads of a row: the angles are read once for all of them, and their loads are asked for together.  It writes only
// what it has read, so q_out may be the queries' own place in qkv.
// (One head where the rows are unsummed runs: those are the loads that count then.  64 tokens, two runs: 8.9 -> 6.3 us.)
struct QueryUnits {
  int far, per_head, groups;      // pairs of pieces half a rotated width apart; units a head; groups of QH heads
};
static __host__ __device__ __forceinline__ QueryUnits query_units(int QH, int n_heads, int hd, int rot, bool pieces, bool rotates, bool interleaved) {
  QueryUnits u;
  u.far = rotates && !interleaved ? rot / 16 : 0;
  u.per_head = pieces ? u.far + (hd - 16 * u.far) / 8 : 1;
  u.groups = (n_heads + QH - 1) / QH;
  return u;
}
template <bool PIECES, bool SUMS>
static __device__ __forceinline__ void queries(const RopeQ8& a, long long idx) {
  constexpr int QH = SUMS ? 1 : 4;
  const QueryUnits u = query_units(QH, a.n_heads, a.hd, a.rot, PIECES, a.cos_t != nullptr, a.interleaved != 0);
  const int per_row = u.groups * u.per_head;
  if (idx >= (long long)a.n_tokens * per_row) return;
  const int t = (int)(idx / per_row), c = (int)(idx % per_row), h0 = c / u.per_head * QH, unit = c % u.per_head;
  const int heads = a.n_heads - h0 < QH ? a.n_heads - h0 : QH;
  const bf16_t* src = a.qkv + (size_t)t * a.ld + (size_t)h0 * a.hd;
  bf16_t* dst = a.q_out + (size_t)t * a.ldq + (size_t)h0 * a.hd;
  const int half = a.rot / 2, pos = a.positions[t];
  const size_t at = (size_t)(pos < 0 ? 0 : (pos < a.table_rows ? pos : a.table_rows - 1)) * half;
  if constexpr (PIECES) {
    const bool far = unit < u.far;
    const int d0 = far ? unit * 8 : 16 * u.far + (unit - u.far) * 8, d1 = far ? d0 + half : d0;
    uint4 lo[QH], hi[QH];
    if constexpr (!SUMS) {
#pragma unroll
      for (int h = 0; h < QH; ++h) {                     // a head past the last: the last again
        const bf16_t* p = src + (size_t)(h < heads ? h : heads - 1) * a.hd;
        lo[h] = *(const uint4*)(p + d0);
        hi[h] = *(const uint4*)(p + d1);
      }
    }
    const bool turns = a.cos_t && d0 < a.rot;
    float cs[8], sn[8];
    if (turns) {
      const size_t i0 = at + (far ? d0 : d0 / 2);
#pragma unroll
      for (int e = 0; e < 8; e += 4) {                   // interleaved pairs have four angles a piece
        *(float4*)(cs + e) = *(const float4*)(a.cos_t + i0 + (far ? e : 0));
        *(float4*)(sn + e) = *(const float4*)(a.sin_t + i0 + (far ? e : 0));
      }
    }
#pragma unroll
    for (int h = 0; h < QH; ++h) {
      if (h >= heads) break;
      float x[8], y[8];
      if constexpr (SUMS) {
        row8<true>(a, t, (h0 + h) * a.hd + d0, x);
        row8<true>(a, t, (h0 + h) * a.hd + d1, y);
      } else {
        load8((const bf16_t*)&lo[h], x);
        load8((const bf16_t*)&hi[h], y);
      }
      if (turns && far) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x0 = x[e], x1 = y[e];
          x[e] = rotated_lo(x0, x1, cs[e], sn[e]);
          y[e] = rotated_hi(x0, x1, cs[e], sn[e]);
        }
      } else if (turns) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x0 = x[2 * i], x1 = x[2 * i + 1];
          x[2 * i] = rotated_lo(x0, x1, cs[i], sn[i]);
          x[2 * i + 1] = rotated_hi(x0, x1, cs[i], sn[i]);
        }
      }
      store8(dst + (size_t)h * a.hd + d0, x);
      if (far) store8(dst + (size_t)h * a.hd + d1, y);
    }
  } else {      // widths that no model of a usual shape has: a thread takes whole heads, pair by pair
#pragma unroll 1
    for (int h = 0; h < heads; ++h) {
      const bf16_t* head = src + (size_t)h * a.hd;
      bf16_t* out = dst + (size_t)h * a.hd;
#pragma unroll 1
      for (int i = 0; i < half; ++i) {
        const int i0 = a.interleaved ? 2 * i : i, i1 = a.interleaved ? 2 * i + 1 : i + half;
        float x0 = bf16_to_f32(head[i0]), x1 = bf16_to_f32(head[i1]);
        if (a.cos_t) {
          const float c_ = a.cos_t[at + i], s_ = a.sin_t[at + i];
          const float y0 = rotated_lo(x0, x1, c_, s_), y1 = rotated_hi(x0, x1, c_, s_);
          x0 = y0;
          x1 = y1;
        }
        out[i0] = f32_to_bf16(x0);
        out[i1] = f32_to_bf16(x1);
      }
#pragma unroll 1
      for (int i = a.rot; i < a.hd; ++i) out[i] = head[i];
    }
  }
}

// `lanes` (a power of two, at least hd / (8 N)) neighbouring threads share a token's key and value of one head, N pieces of
// eight elements each: with N = 2 piece p and piece p + hd / 16, which are each other's partners where the whole head is
// rotated in halves (half the loads); with N = 1 piece p (a shorter way for a launch of few rows: 8 tokens 5.6 -> 4.5 us).
template <bool PIECES, bool SUMS, int N>
static __device__ __forceinline__ void key_and_value(const RopeQ8& a, int t, int kvh, int piece, int lanes, int pos, uint2* kb, uint2* vb,
                                                     int* ks, int* vs) {
  float k[N][8], v[N][8];
  uint32_t kt = 0, vt = 0;
  const int d0 = piece * 8, d1 = d0 + a.hd / 2;
  if (d0 < a.hd / N) {
    const int key = (a.n_heads + kvh) * a.hd, val = (a.n_heads + a.n_kv + kvh) * a.hd;
    if (N == 2 && PIECES && a.cos_t && !a.interleaved && a.rot == a.hd) {
      row8<SUMS>(a, t, key + d0, k[0]);
      row8<SUMS>(a, t, key + d1, k[N - 1]);
      row8<SUMS>(a, t, val + d0, v[0]);
      row8<SUMS>(a, t, val + d1, v[N - 1]);
      const size_t at = (size_t)(pos < 0 ? 0 : (pos < a.table_rows ? pos : a.table_rows - 1)) * (a.hd / 2) + d0;
      float c[8], s[8];
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        *(float4*)(c + e) = *(const float4*)(a.cos_t + at + e);
        *(float4*)(s + e) = *(const float4*)(a.sin_t + at + e);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x0 = k[0][e], x1 = k[N - 1][e];
        k[0][e] = rotated_lo(x0, x1, c[e], s[e]);
        k[N - 1][e] = rotated_hi(x0, x1, c[e], s[e]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        rotated8<PIECES, SUMS>(a, t, key, pos, i ? d1 : d0, k[i]);
        plain8<PIECES, SUMS>(a, t, val + (i ? d1 : d0), v[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t k1 = q8_top_bits(k[i]), v1 = q8_top_bits(v[i]);
      kt = k1 > kt ? k1 : kt;
      vt = v1 > vt ? v1 : vt;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) k[i][e] = v[i][e] = 0.f;
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    const uint32_t k2 = (uint32_t)__shfl_xor((int)kt, o, WAVE), v2 = (uint32_t)__shfl_xor((int)vt, o, WAVE);
    kt = k2 > kt ? k2 : kt;
    vt = v2 > vt ? v2 : vt;
  }
  const bool finite = kt < 0x7f800000u && vt < 0x7f800000u;
  const int ke = q8_power_for(kt), ve = q8_power_for(vt);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    kb[i] = finite ? q8_to_e4m3(k[i], ke) : make_uint2(0, 0);
    vb[i] = finite ? q8_to_e4m3(v[i], ve) : make_uint2(0, 0);
  }
  *ks = finite ? ke + 127 : Q8_NAN;
  *vs = finite ? ve + 127 : 127;
}

// Few rows: no two of them need lie in one page, so a thread stores what it has where it goes (values byte by byte).
template <bool PIECES, bool SUMS>
__global__ __launch_bounds__(256) void rope_kv_q8_rows_kernel(RopeQ8 a, int kv_blocks, int lanes) {
  if ((int)blockIdx.x >= kv_blocks) {
    queries<PIECES, SUMS>(a, (long long)((int)blockIdx.x - kv_blocks) * 256 + threadIdx.x);
    return;
  }
  const long long unit = ((long long)blockIdx.x * 256 + threadIdx.x) / lanes;
  const int piece = threadIdx.x % lanes;
  const long long units = (long long)a.n_tokens * a.n_kv;
  const bool real = unit < units;
  const int t = real ? (int)(unit / a.n_kv) : 0, kvh = real ? (int)(unit % a.n_kv) : 0;
  const int pos = a.positions[t];
  uint2 kb[1], vb[1];
  int ks, vs;
  const long long off = page_of(a, t, pos);
  key_and_value<PIECES, SUMS, 1>(a, t, kvh, piece, lanes, pos, kb, vb, &ks, &vs);
  if (!real || off < 0 || piece * 8 >= a.hd) return;
  uint8_t* head = a.cache + off + (size_t)kvh * q8_head_bytes(a.hd);
  const int in = pos % Q8_PAGE, t16 = in >> 4, i = in & 15, g = i >> 2, r = i & 3;
  *(uint2*)(head + (t16 * (a.hd / 16) + piece / 2) * 256 + i * 16 + (piece & 1) * 8) = kb[0];
  uint8_t* val = head + Q8_PAGE * a.hd + ((piece / 2 * 4 + g) * 16 + (piece & 1) * 8) * 16 + 4 * t16 + r;
#pragma unroll
  for (int e = 0; e < 8; ++e) val[e * 16] = (uint8_t)((e < 4 ? vb[0].x : vb[0].y) >> (8 * (e & 3)));
  if (piece == 0) {
    uint8_t* scales = head + 2 * Q8_PAGE * a.hd;
    scales[4 * i + t16] = (uint8_t)ks;
    scales[64 + 16 * g + 4 * t16 + r] = (uint8_t)vs;
  }
}

// Many rows: a block takes 64 consecutive rows of the step and one kv head, brings keys and values together in LDS, and
// stores with its lanes in the order of the page: 16 tokens of a keys' piece are 256 bytes in a row, and four tokens of a
// value's element one word, where four neighbouring rows are neighbouring tokens of a page (elsewhere byte by byte).
template <bool PIECES, bool SUMS>
__global__ __launch_bounds__(256) void rope_kv_q8_tiles_kernel(RopeQ8 a, int kv_blocks, int lanes) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  if ((int)blockIdx.x >= kv_blocks) {
    queries<PIECES, SUMS>(a, (long long)((int)blockIdx.x - kv_blocks) * 256 + threadIdx.x);
    return;
  }
  __shared__ long long at[64];        // each row's page in the cache, -1 where there is none
  __shared__ int in_page[64];
  __shared__ long long group[16];
  const int stride = a.hd + 16;       // rows 16 bytes apart in the banks
  uint8_t* kt = lds;
  uint8_t* vt = lds + 64 * stride;
  const int kvh = blockIdx.x % a.n_kv, t0 = (blockIdx.x / a.n_kv) * 64;
  const int n = a.n_tokens - t0 < 64 ? a.n_tokens - t0 : 64;
  if (threadIdx.x < 64) {
    const int t = t0 + ((int)threadIdx.x < n ? (int)threadIdx.x : n - 1);
    const int pos = a.positions[t];
    at[threadIdx.x] = (int)threadIdx.x < n ? page_of(a, t, pos) : -1;
    in_page[threadIdx.x] = pos & (Q8_PAGE - 1);
  }
  __syncthreads();
  // where the word of each group of four rows goes that are four tokens of one word (for element 0), -1 for the others
  const int lead = 3 & -in_page[0];
  if (threadIdx.x < 16) {
    const int j = lead + 4 * (int)threadIdx.x;
    const bool whole = j + 3 < n && at[j] >= 0 && (in_page[j] & 3) == 0 && at[j + 3] == at[j] && at[j + 1] == at[j] && at[j + 2] == at[j] &&
                       in_page[j + 1] == in_page[j] + 1 && in_page[j + 2] == in_page[j] + 2 && in_page[j + 3] == in_page[j] + 3;
    group[threadIdx.x] = whole ? at[j] + Q8_PAGE * a.hd + ((in_page[j] >> 2) & 3) * 256 + (in_page[j] >> 4) * 4 : -1;
  }
  const size_t head = (size_t)kvh * q8_head_bytes(a.hd);
  const int piece = threadIdx.x % lanes;
  for (int j0 = 0; j0 < 64; j0 += 256 / lanes) {        // whole waves take part in the shuffles
    const int j = j0 + threadIdx.x / lanes;
    const int t = t0 + (j < n ? j : n - 1);
    uint2 kb[2], vb[2];
    int ks, vs;
    key_and_value<PIECES, SUMS, 2>(a, t, kvh, piece, lanes, a.positions[t], kb, vb, &ks, &vs);
    if (j >= 64 || piece * 16 >= a.hd) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *(uint2*)(kt + j * stride + piece * 8 + h * (a.hd / 2)) = kb[h];
      *(uint2*)(vt + j * stride + piece * 8 + h * (a.hd / 2)) = vb[h];
    }
    if (piece == 0 && at[j] >= 0) {
      uint8_t* scales = a.cache + at[j] + head + 2 * Q8_PAGE * a.hd;
      const int in = in_page[j], t16 = in >> 4, i = in & 15;
      scales[4 * i + t16] = (uint8_t)ks;
      scales[64 + 16 * (i >> 2) + 4 * t16 + (i & 3)] = (uint8_t)vs;
    }
  }
  __syncthreads();
  {
    const int j = threadIdx.x & 63, pieces = a.hd / 16;
    if (at[j] >= 0) {
      uint8_t* page = a.cache + at[j] + head + (in_page[j] >> 4) * pieces * 256 + (in_page[j] & 15) * 16;
      for (int p = threadIdx.x >> 6; p < pieces; p += 4) *(uint4*)(page + p * 256) = *(const uint4*)(kt + j * stride + p * 16);
    }
  }
  // 16 groups of four rows from the first row on whose place in its page is a multiple of four; the rows left over at both
  // ends are the sixteenth.  A thread's groups are 16 rows apart from its neighbours', so that 64 lanes write 256 bytes in a row.
  const int q = threadIdx.x & 3;
  for (int g = 0; g < 4; ++g) {
    const int j = lead + 16 * q + 4 * g;
    const long long to = group[4 * q + g];
    if (to >= 0) {
      uint8_t* page = a.cache + to + head;
      for (int d = threadIdx.x >> 2; d < a.hd; d += 64) {
        const uint8_t* src = vt + d + j * stride;
        *(uint32_t*)(page + (d & ~15) * 64 + (d & 15) * 16) = src[0] | (src[stride] << 8) | (src[2 * stride] << 16) | ((uint32_t)src[3 * stride] << 24);
      }
      continue;
    }
    for (int m = 0; m < 4; ++m) {
      const int jm = (j + m) & 63;            // the last group's rows past the tile are the first ones, before `lead`
      if (jm >= n || at[jm] < 0) continue;
      const int in = in_page[jm];
      uint8_t* page = a.cache + at[jm] + head + Q8_PAGE * a.hd + ((in >> 2) & 3) * 256 + (in >> 4) * 4 + (in & 3);
      for (int d = threadIdx.x >> 2; d < a.hd; d += 64) page[(d & ~15) * 64 + (d & 15) * 16] = vt[d + jm * stride];
    }
  }
}

extern "C" const char* dlgo_rope_kv_q8(const void* qkv, int ld, void* q_out, int ldq, int n_tokens, int n_heads, int n_kv, int hd,
                                       int rot, int interleaved, const float* cos_t, const float* sin_t, int table_rows,
                                       const int32_t* positions, const int32_t* tok_seq, const int32_t* slots, int n_seq,
                                       const int32_t* page_table, int n_slots, int max_pages, void* cache, long long page_stride,
                                       int n_pages, int write_kv, const float* part, int n_parts, long long plane, int part_ld,
                                       hipStream_t stream) {
  DLGO_REQUIRE(n_tokens >= 0 && n_heads > 0 && n_kv >= 0 && hd >= 16 && hd % 16 == 0 && hd <= 256,
               "rope_kv_q8: %d rows, %d query and %d kv heads of size %d (head sizes come in steps of 16, up to 256)", n_tokens, n_heads, n_kv, hd);
  DLGO_REQUIRE(rot >= 0 && rot <= hd && rot % 2 == 0, "rope_kv_q8: rotated width %d must be even and at most the head size %d", rot, hd);
  DLGO_REQUIRE(ld >= (n_heads + (write_kv ? 2 * n_kv : 0)) * hd && ldq >= n_heads * hd, "rope_kv_q8: row strides %d and %d are shorter than the heads they hold", ld, ldq);
  DLGO_REQUIRE((cos_t == nullptr) == (sin_t == nullptr), "rope_kv_q8: cos and sin tables come together");
  DLGO_REQUIRE(cos_t == nullptr || table_rows > 0, "rope_kv_q8: empty rotation table");
  DLGO_REQUIRE(!write_kv || (n_kv > 0 && cache && page_table && slots && tok_seq && max_pages > 0 && n_slots > 0 && n_seq > 0 && n_pages > 0),
               "rope_kv_q8: cache arguments missing");
  DLGO_REQUIRE(!write_kv || (((uintptr_t)cache & 15) == 0 && page_stride % 16 == 0 && page_stride >= n_kv * q8_head_bytes(hd)),
               "rope_kv_q8: pages %lld bytes apart (16-byte aligned pages of at least %lld bytes are needed)", page_stride, n_kv * q8_head_bytes(hd));
  if (n_tokens == 0) return nullptr;
  RopeQ8 a = {(const bf16_t*)qkv, (bf16_t*)q_out, (uint8_t*)cache, cos_t, sin_t, positions, tok_seq, slots, page_table,
              page_stride, ld, ldq, n_tokens, n_heads, n_kv, hd, rot, interleaved, table_rows, n_seq, n_slots, max_pages, n_pages,
              part, plane, n_parts, part_ld};
  const bool pieces = rot % (interleaved ? 8 : 16) == 0 && (part || (ld % 8 == 0 && ((uintptr_t)qkv & 15) == 0)) && ldq % 8 == 0 && ((uintptr_t)q_out & 15) == 0 &&
                      (!cos_t || (((uintptr_t)cos_t & 15) == 0 && ((uintptr_t)sin_t & 15) == 0));
  DLGO_REQUIRE(!part || (pieces && n_parts > 0 && part_ld >= (n_heads + (write_kv ? 2 * n_kv : 0)) * hd && plane >= (long long)n_tokens * part_ld && part_ld % 4 == 0 && plane % 4 == 0 && ((uintptr_t)part & 15) == 0),
               "rope_kv_q8: unsummed rows need whole 16-byte pieces (rotated width %d, %d runs of rows %d apart)", rot, n_parts, part_ld);
  // The many-rows kernel stores whole lines where the other stores single bytes, but its blocks are long: it is faster from
  // 512 rows of a prompt on (32 heads of 64 over 8: 128 rows 4.9 against 4.8 us, 512 rows 5.1 against 5.6, 1,024 6.0
  // against 7.2, 17,408 rows of 24 heads of 128: 69 us).
  const bool tiles = n_tokens >= 512;
  int lanes = 1;
  while (lanes * (tiles ? 16 : 8) < hd) lanes *= 2;
  const long long kv_blocks = !write_kv ? 0 : tiles ? (long long)((n_tokens + 63) / 64) * n_kv : ((long long)n_tokens * n_kv * lanes + 255) / 256;
  const QueryUnits u = query_units(part ? 1 : 4, n_heads, hd, rot, pieces, cos_t != nullptr, interleaved != 0);
  const long long q_blocks = ((long long)n_tokens * u.groups * u.per_head + 255) / 256;
  DLGO_REQUIRE(kv_blocks + q_blocks < (1ll << 31), "rope_kv_q8: too many rows at once");
  const dim3 grid((unsigned)(kv_blocks + q_blocks));
  const int lds = 2 * 64 * (hd + 16);
  if (tiles) {
    if (part) hipLaunchKernelGGL((rope_kv_q8_tiles_kernel<true, true>), grid, dim3(256), lds, stream, a, (int)kv_blocks, lanes);
    else if (pieces) hipLaunchKernelGGL((rope_kv_q8_tiles_kernel<true, false>), grid, dim3(256), lds, stream, a, (int)kv_blocks, lanes);
    else hipLaunchKernelGGL((rope_kv_q8_tiles_kernel<false, false>), grid, dim3(256), lds, stream, a, (int)kv_blocks, lanes);
  } else {
    if (part) hipLaunchKernelGGL((rope_kv_q8_rows_kernel<true, true>), grid, dim3(256), 0, stream, a, (int)kv_blocks, lanes);
    else if (pieces) hipLaunchKernelGGL((rope_kv_q8_rows_kernel<true, false>), grid, dim3(256), 0, stream, a, (int)kv_blocks, lanes);
    else hipLaunchKernelGGL((rope_kv_q8_rows_kernel<false, false>), grid, dim3(256), 0, stream, a, (int)kv_blocks, lanes);
  }
  DLGO_LAUNCH_CHECK("rope_kv_q8");
  return nullptr;
}

#include "exact_end.h"
