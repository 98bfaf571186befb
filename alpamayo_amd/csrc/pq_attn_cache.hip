// Attention over the paged int8 cache, and the weights that it gives.
//
//   s_ij = scale * q_i . k_j,  o_i = sum_j p_ij v_j / sum_j p_ij,  p = exp(s - max)
//
// for the last n tokens of each sequence, token i seeing the keys up to its
// own place.  A key/value head's rows are its (token, query head) pairs: at
// one token and 4 query heads to a key/value head 4 rows, in a verify block
// of 16 tokens 64.
//
// Products run on the fp16 matrix instructions.  Codes are small whole
// numbers, exact in fp16; a page's scale multiplies the float32 results.  A
// row of q is scaled by a power of two so that its largest value lies in
// [2^14, 2^15): every bf16 or fp16 value within 2^28 of it is exact, and what
// lies below counts for less than a float32 sum can hold.  p is rounded to
// fp16 (half a step 2^-12 of values up to 1), sums and statistics are float32.
//
// Both products are taken transposed: S^T = K Q^T with tokens as the rows of
// the result, O^T = V^T P^T.  A lane then holds the scores of one row (column
// lane & 15), so that maxima and rescaling need no exchange but across the
// four groups of lanes, and the tokens of a page are dealt to the rows of S^T
// such that a lane's 16 scores are 16 neighbouring tokens: just the operand
// that the second product takes, and the 16 bytes of a V row next to it.
//
// Work: all pages of all (sequence, head, rows) units in one line, cut into
// equal shares for the workgroups whatever the lengths; the four waves of a
// workgroup take a segment's pages in turn and join at its end through LDS.
// A unit that spans workgroups leaves partial results (at most two for each
// workgroup), which the second kernel joins.
#include <algorithm>

#include "pq_attn.h"
#include "pq_device.h"

namespace {

using namespace pqa;

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kWorkers = 512;
#ifndef KRT
#define KRT 1
#endif
constexpr int kRT = KRT;

struct CacheArgs {
  const void* q;                      // [tokens, heads * group, d]
  const int8_t* kc;                   // [pages, heads, 64, d]
  const int8_t* vc;                   // [pages, heads, d, 64]
  const float* ks;                    // [pages, heads]
  const float* vs;
  const int* table;                   // [batch, width]
  const int* cu;                      // [batch + 1]
  const int* lens;                    // [batch]
  void* out;                          // [tokens, heads * group, d]
  float* lse;                         // [heads * group, tokens]
  float* part;                        // partial results, 2 for each workgroup
  float* weights;                     // weights kernel: [batch, heads, span]
  int64_t q_st, q_sh, span;
  int batch, width, tokens, heads, group, pages, workers;
  float scale_log2;
};

__device__ __forceinline__ int seq_len(const CacheArgs& a, int b) {
  return min(max(a.lens[b], 0), a.width * kPage);
}

// A unit: kRows rows of a sequence and head.  Units of a sequence are ordered by tile, then by head.
template <int ROWS>
struct Plan {
  // pages that sequence b's units read in all
  static __device__ __forceinline__ int64_t cost(const CacheArgs& a, int b) {
    const int64_t rows = static_cast<int64_t>(span_of(a.cu, b, a.tokens).count) * a.group;
    return (rows + ROWS - 1) / ROWS * a.heads * ((seq_len(a, b) + kPage - 1) / kPage);
  }
  // Workgroups that take part: each has work for its waves.
  static __device__ __forceinline__ int64_t workers(const CacheArgs& a, int64_t total) {
    const int64_t w = (total + kWaves - 1) / kWaves;
    return w < a.workers ? w : a.workers;
  }
  static __device__ __forceinline__ int64_t begin(int64_t w, int64_t total, int64_t n) { return w * total / n; }
  // The workgroup whose share holds page x.
  static __device__ __forceinline__ int64_t owner(int64_t x, int64_t total, int64_t n) {
    int64_t w = x * n / total;
    while (begin(w + 1, total, n) <= x) ++w;
    while (begin(w, total, n) > x) --w;
    return w;
  }
};

// Partial results of a unit: rows [ROWS][D], then maxima and sums.
template <int ROWS, int D>
constexpr int64_t part_floats() { return ROWS * (D + 2); }

__device__ __forceinline__ float q_to_f32(uint32_t raw, bool bf16) {
  return bf16 ? pq_bf16_to_f32(static_cast<uint16_t>(raw)) : pq_f16_to_f32(static_cast<uint16_t>(raw));
}

// 16 rows of q as the operand with a row for each lane & 15, scaled to fp16; the scores' factor goes to `mult`.
// In step s, lane group g holds channels 64 (s / 2) + 16 g + 8 (s & 1) .. + 7.
template <int D, bool BF16>
__device__ __forceinline__ void load_q(const CacheArgs& a, int first, int rows, int head, int row0, h8 (&qf)[D / 32],
                                       float& mult) {
  const int lane = lane_id(), g = lane >> 4, r = row0 + (lane & 15);
  float v[D / 32][8];
  uint32_t big = 0;
  const bool valid = r < rows;
  const int token = valid ? r / a.group : 0, h = valid ? r - token * a.group : 0;
  const uint16_t* p = static_cast<const uint16_t*>(a.q) + (first + token) * a.q_st +
                      (static_cast<int64_t>(head) * a.group + h) * a.q_sh;
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    u4 w = {0, 0, 0, 0};
    if (valid) w = *reinterpret_cast<const u4*>(p + (s >> 1) * 64 + g * 16 + (s & 1) * 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[s][j] = q_to_f32(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu, BF16);
      const uint32_t m = __float_as_uint(v[s][j]) & 0x7f800000u;
      big = m > big ? m : big;
    }
  }
  big = max(big, static_cast<uint32_t>(__shfl_xor(static_cast<int>(big), 16)));
  big = max(big, static_cast<uint32_t>(__shfl_xor(static_cast<int>(big), 32)));
  // exponents 15..254 keep both factors normal; infinities and NaN pass through
  const uint32_t e = min(max(big >> 23, 15u), 254u);
  const float up = __uint_as_float((268u - e) << 23), down = __uint_as_float((e - 14u) << 23);
#pragma unroll
  for (int s = 0; s < D / 32; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) qf[s][j] = static_cast<_Float16>(v[s][j] * up);
  mult = down * a.scale_log2;
}

// The K codes of a page: tile t's row r is token at(t, r), 2 x 16 bytes of it (d = 64: 1) for each lane.
template <int D, bool INTERLEAVED>
__device__ __forceinline__ void load_k(const int8_t* page, u4 (&kr)[4][D / 64]) {
  const int lane = lane_id(), g = lane >> 4, r = lane & 15;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int token = INTERLEAVED ? 16 * (r >> 2) + 4 * t + (r & 3) : 16 * t + r;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) kr[t][i] = *reinterpret_cast<const u4*>(page + token * D + i * 64 + g * 16);
  }
}

// RT row tiles of 16 for each wave, RW waves with rows of their own on the same pages.
template <int D, int RT, int RW, bool BF16>
__global__ __launch_bounds__(kThreads, RT == 4 ? 1 : 2) void attn_cache_kernel(CacheArgs a) {
  constexpr int kRows = 16 * RT * RW, kDt = D / 16, kStreams = kWaves / RW;
  constexpr int kPitch = D + 4;
  __shared__ __align__(16) float so[kWaves][16][kPitch];
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  using P = Plan<kRows>;
  const int t = threadIdx.x, lane = t & 63, g = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6), stream = wave / RW, part_of = wave % RW;

  const auto cost = [&](int b) { return P::cost(a, b); };
  const int64_t total = sum_seqs(a.batch, cost);
  const int64_t n = P::workers(a, total), w = blockIdx.x;
  if (w >= n) return;
  const int64_t from = P::begin(w, total, n), to = P::begin(w + 1, total, n);

  for (int64_t at = from; at < to;) {
    const Found f = find_seq(a.batch, at, cost);
    if (f.b < 0) break;
    const Span sp = span_of(a.cu, f.b, a.tokens);
    const int len = seq_len(a, f.b), npages = (len + kPage - 1) / kPage;
    const int rows = sp.count * a.group;
    const int unit = static_cast<int>(f.local / npages), p0 = static_cast<int>(f.local % npages);
    const int head = unit % a.heads, row0 = unit / a.heads * kRows;
    const int p1 = static_cast<int>(min(static_cast<int64_t>(npages), p0 + (to - at)));

    h8 qf[RT][D / 32];
    float mult[RT];
    int limit[RT];     // keys that the lane's row sees
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int first = row0 + 16 * (RT * part_of + i);
      load_q<D, BF16>(a, sp.first, rows, head, first, qf[i], mult[i]);
      limit[i] = min((first + col) / a.group + len - sp.count + 1, len);
    }
    const int sure = (row0 + 16 * RT * part_of) / a.group + len - sp.count + 1;   // keys that every row of the wave sees

    float m[RT], l[RT];
    f4 o[RT][kDt];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < kDt; ++k) o[i][k] = f4{0, 0, 0, 0};
    }

    // The next page's codes are asked for as soon as the registers of this one's are free: K behind the first product,
    // V behind the second; its number one page ahead of that.
    const int* table = a.table + static_cast<int64_t>(f.b) * a.width;
    u4 kr[4][D / 64], vr[kDt];
    float ks = 0.0f, vs = 0.0f, ks_next = 0.0f, vs_next = 0.0f;
    const auto load_v = [&](int64_t ph) {
      const int8_t* vp = a.vc + ph * (kPage * D);
#pragma unroll
      for (int k = 0; k < kDt; ++k) vr[k] = *reinterpret_cast<const u4*>(vp + (16 * k + col) * kPage + g * 16);
    };
    const auto number = [&](int p) { return scalar_load(table + p); };
    // page and head of place p; a number that is no page: page 0, with no token to see
    const auto page_head = [&](int id) { return static_cast<int64_t>(id < 0 || id >= a.pages ? 0 : id) * a.heads + head; };

    // seen: tokens of the cache that rows may see; masked: some row does not see some token of the page
    const auto step = [&](bool masked, int seen, int p, int64_t ph_next) {
      ks_next = scalar_load(a.ks + ph_next);
      vs_next = scalar_load(a.vs + ph_next);
      f4 s[RT][4];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) s[i][q] = f4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < D / 32; ++k)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const h8 kf = codes_f16(kr[q][k >> 1][2 * (k & 1)], kr[q][k >> 1][2 * (k & 1) + 1]);
#pragma unroll
          for (int i = 0; i < RT; ++i) s[i][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[i][k], s[i][q], 0, 0, 0);
        }
      load_k<D, true>(a.kc + ph_next * (kPage * D), kr);
      __builtin_amdgcn_sched_barrier(0);

      // the lane's tokens: 16 g + 4 q + e
      h8 pf[RT][2];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        // never 0: what is masked stays -inf, and scores of rows and pages of zeros stay as good as 0
        const float c = fmaxf(ks * mult[i], 1e-37f);
        float big = -INFINITY;
        if (masked) {
          const int see = min(limit[i], seen) - p * kPage - 16 * g;
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][q][e] = 4 * q + e >= see ? -INFINITY : s[i][q][e];
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) big = fmaxf(big, s[i][q][e]);
        // a row's maximum moves by more than 8 (in base 2) at a time, each row by itself
        big = max_xor32(max_xor16(big)) * c;
        const bool moves = big > m[i] + 8.0f;
        if (__any(moves)) {
          const float now = moves ? big : m[i];
          const float alpha = moves ? exp2_fast(m[i] - now) : 1.0f;
          m[i] = now;
          l[i] *= alpha;
#pragma unroll
          for (int k = 0; k < kDt; ++k) o[i][k] *= alpha;
        }
        const float base = m[i] == -INFINITY ? 0.0f : m[i];
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          u4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = exp2_fast(__builtin_fmaf(s[i][2 * q + (e >> 1)][2 * (e & 1)], c, -base));
            const float y = exp2_fast(__builtin_fmaf(s[i][2 * q + (e >> 1)][2 * (e & 1) + 1], c, -base));
            sum += x + y;
            w[e] = pqd::pk_f16(x, y);
          }
          pf[i][q] = __builtin_bit_cast(h8, w);
        }
        l[i] += sum;
      }
#pragma unroll
      for (int k = 0; k < kDt; ++k) {
        const h8 v0 = codes_f16(vr[k][0], vr[k][1]), v1 = codes_f16(vr[k][2], vr[k][3]);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          f4 x = {0, 0, 0, 0};
          x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[i][0], x, 0, 0, 0);
          x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[i][1], x, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][k][e] = __builtin_fmaf(x[e], vs, o[i][k][e]);
        }
      }
      load_v(ph_next);
      __builtin_amdgcn_sched_barrier(0);
    };

    int p = p0 + stream;
    if (p < p1) {
      int id = number(p), id_next = p + kStreams < p1 ? number(p + kStreams) : 0;
      const int64_t ph = page_head(id);
      ks = scalar_load(a.ks + ph);
      vs = scalar_load(a.vs + ph);
      load_k<D, true>(a.kc + ph * (kPage * D), kr);
      __builtin_amdgcn_sched_barrier(0);   // K before V, as in the loop: the wait for K then leaves V in flight
      load_v(ph);
      __builtin_amdgcn_sched_barrier(0);
      for (; p < p1; p += kStreams) {
        // behind the last page the loads, which the waits count on, go to that page again
        const bool there = id >= 0 && id < a.pages;
        id = p + kStreams < p1 ? id_next : id;
        const int64_t ph_next = page_head(id);
        if (p + 2 * kStreams < p1) id_next = number(p + 2 * kStreams);
        step(!there || (p + 1) * kPage > sure, there ? len : 0, p, ph_next);
        ks = ks_next;
        vs = vs_next;
      }
    }

    // the results of the segment, from the waves that went through its pages
    const bool whole = p0 == 0 && p1 == npages;
    float* part = a.part + (2 * w + (at == from ? 0 : 1)) * part_floats<kRows, D>();
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const float lt = sum_xor32(sum_xor16(l[i]));
      if (g == 0) {
        sm[wave][col] = m[i];
        sl[wave][col] = lt;
      }
#pragma unroll
      for (int k = 0; k < kDt; ++k) *reinterpret_cast<f4*>(&so[wave][col][16 * k + 4 * g]) = o[i][k];
      __syncthreads();
#pragma unroll
      for (int x = 0; x < RW; ++x) {
        const int r = t >> 4, local = 16 * (RT * x + i) + r, row = row0 + local;
        if (row >= rows) continue;
        float big = sm[x][r];
#pragma unroll
        for (int q = 1; q < kStreams; ++q) big = fmaxf(big, sm[RW * q + x][r]);
        const float base = big == -INFINITY ? 0.0f : big;
        float sum = 0.0f;
        f4 acc[D / 64];
#pragma unroll
        for (int k = 0; k < D / 64; ++k) acc[k] = f4{0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < kStreams; ++q) {
          const float y = exp2_fast(sm[RW * q + x][r] - base);
          sum += sl[RW * q + x][r] * y;
#pragma unroll
          for (int k = 0; k < D / 64; ++k) acc[k] += *reinterpret_cast<const f4*>(&so[RW * q + x][r][64 * k + 4 * (t & 15)]) * y;
        }
        if (whole) {
          const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;
          const int token = sp.first + row / a.group, h = head * a.group + row % a.group;
          uint16_t* op = static_cast<uint16_t*>(a.out) + (static_cast<int64_t>(token) * a.heads * a.group + h) * D;
#pragma unroll
          for (int k = 0; k < D / 64; ++k) {
            uint16_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = BF16 ? pq_f32_to_bf16(acc[k][e] * inv) : pq_f32_to_f16(acc[k][e] * inv);
            *reinterpret_cast<uint2*>(op + 64 * k + 4 * (t & 15)) =
                make_uint2(y[0] | static_cast<uint32_t>(y[1]) << 16, y[2] | static_cast<uint32_t>(y[3]) << 16);
          }
          if ((t & 15) == 0) a.lse[static_cast<int64_t>(h) * a.tokens + token] = (big + log2_fast(sum)) * kLn2;
        } else {
#pragma unroll
          for (int k = 0; k < D / 64; ++k) *reinterpret_cast<f4*>(part + local * D + 64 * k + 4 * (t & 15)) = acc[k];
          if ((t & 15) == 0) {
            part[kRows * D + local] = big;
            part[kRows * D + kRows + local] = sum;
          }
        }
      }
      __syncthreads();
    }
    at += p1 - p0;
  }
}

// Joins the partial results of the rows whose unit spans workgroups.  A workgroup takes four (query head, token) rows of a
// token: a wave each, or, where the parts are many, its waves together on one row after the other.  Rows outside of the
// sequences and rows of empty ones get zeros and lse = -inf.
template <int D, int RT, bool BF16>
__global__ __launch_bounds__(kThreads) void attn_cache_join_kernel(CacheArgs a) {
  constexpr int kRows = 16 * RT, kV = D / 64;
  __shared__ float so[kWaves][D], sl[kWaves], sm[kWaves];
  using P = Plan<kRows>;
  const int token = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int hq = a.heads * a.group;

  // the sequence that the token belongs to, and the pages of the units before it
  const auto cost = [&](int b) { return P::cost(a, b); };
  int b = -1;
  int64_t before = 0, total = 0;
  for (int base = 0; base < a.batch; base += 64) {
    const int own = base + lane;
    const bool there = own < a.batch;
    const Span sp = there ? span_of(a.cu, own, a.tokens) : Span{0, 0};
    const int64_t c = there ? cost(own) : 0;
    const uint64_t hit = __ballot(token >= sp.first && token < sp.first + sp.count);
    const int64_t incl = wave_scan(c);
    if (b < 0 && hit) {
      const int at = __builtin_ctzll(hit);
      b = base + at;
      before = total + read_lane(incl - c, at);
    }
    total += read_lane(incl, 63);
  }
  const int len = b < 0 ? 0 : seq_len(a, b);
  const auto out_row = [&](int h) { return static_cast<uint16_t*>(a.out) + (static_cast<int64_t>(token) * hq + h) * D; };
  const auto lse_of = [&](int h) { return a.lse + static_cast<int64_t>(h) * a.tokens + token; };
  if (len == 0) {
    const int h = blockIdx.y * kWaves + wave;
    if (h < hq) {
#pragma unroll
      for (int k = 0; k < kV; ++k) out_row(h)[lane * kV + k] = 0;
      if (lane == 0) *lse_of(h) = -INFINITY;
    }
    return;
  }
  const Span sp = span_of(a.cu, b, a.tokens);
  const int npages = (len + kPage - 1) / kPage;
  const int64_t n = P::workers(a, total);

  // parts w0 + first, w0 + first + step, ... of a row into m, l, o
  struct Parts { int64_t begin, w0, w1; int r; };
  const auto parts_of = [&](int h) {
    const int head = h / a.group, row = (token - sp.first) * a.group + h - head * a.group;
    Parts q;
    q.begin = before + (static_cast<int64_t>(row / kRows) * a.heads + head) * npages;
    q.w0 = P::owner(q.begin, total, n);
    q.w1 = P::owner(q.begin + npages - 1, total, n);
    q.r = row % kRows;
    return q;
  };
  const auto gather = [&](const Parts& q, int first, int step, float& m, float& l, float (&o)[kV]) {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int k = 0; k < kV; ++k) o[k] = 0.0f;
    constexpr int kAhead = 4;
    for (int64_t w = q.w0 + first; w <= q.w1; w += kAhead * step) {
      float pm[kAhead], pl[kAhead], po[kAhead][kV];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        pm[i] = -INFINITY;
        pl[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < kV; ++k) po[i][k] = 0.0f;
        const int64_t x = w + i * step;
        if (x <= q.w1) {
          const bool own = x > q.w0 || P::begin(x, total, n) == q.begin;
          const float* p = a.part + (2 * x + (own ? 0 : 1)) * part_floats<kRows, D>();
          pm[i] = p[kRows * D + q.r];
          pl[i] = p[kRows * D + kRows + q.r];
#pragma unroll
          for (int k = 0; k < kV; ++k) po[i][k] = p[q.r * D + lane * kV + k];
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float big = fmaxf(m, pm[i]), base = big == -INFINITY ? 0.0f : big;
        const float ca = exp2_fast(m - base), cb = exp2_fast(pm[i] - base);
        l = l * ca + pl[i] * cb;
#pragma unroll
        for (int k = 0; k < kV; ++k) o[k] = o[k] * ca + po[i][k] * cb;
        m = big;
      }
    }
  };
  const auto write = [&](int h, float m, float l, const float (&o)[kV]) {
    const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
#pragma unroll
    for (int k = 0; k < kV; ++k)
      out_row(h)[lane * kV + k] = BF16 ? pq_f32_to_bf16(o[k] * inv) : pq_f32_to_f16(o[k] * inv);
    if (lane == 0) *lse_of(h) = (m + log2_fast(l)) * kLn2;
  };

  // heads of a unit's rows share their parts but not their first one: whether they are many is the same for all of them
  if ((static_cast<int64_t>(npages) * n) / total <= 16) {
    const int h = blockIdx.y * kWaves + wave;
    if (h >= hq) return;
    const Parts q = parts_of(h);
    if (q.w0 == q.w1) return;   // written by the workgroup that had all of it
    float m, l, o[kV];
    gather(q, 0, 1, m, l, o);
    write(h, m, l, o);
    return;
  }
  for (int i = 0; i < kWaves; ++i) {
    const int h = blockIdx.y * kWaves + i;
    if (h >= hq) return;
    const Parts q = parts_of(h);
    float m, l, o[kV];
    gather(q, wave, kWaves, m, l, o);
    if (lane == 0) {
      sm[wave] = m;
      sl[wave] = l;
    }
#pragma unroll
    for (int k = 0; k < kV; ++k) so[wave][lane * kV + k] = o[k];
    __syncthreads();
    if (wave == 0) {
      float big = sm[0];
#pragma unroll
      for (int x = 1; x < kWaves; ++x) big = fmaxf(big, sm[x]);
      const float base = big == -INFINITY ? 0.0f : big;
      l = 0.0f;
#pragma unroll
      for (int k = 0; k < kV; ++k) o[k] = 0.0f;
#pragma unroll
      for (int x = 0; x < kWaves; ++x) {
        const float f = exp2_fast(sm[x] - base);
        l += sl[x] * f;
#pragma unroll
        for (int k = 0; k < kV; ++k) o[k] += so[x][lane * kV + k] * f;
      }
      write(h, big, l, o);
    }
    __syncthreads();
  }
}

// weights[b, head, j] += sum over the head's rows of exp(s_ij - lse_i).  A wave per page: its codes become matrix
// operands once, and the rows pass 16 at a time.  Here tokens are the columns of the scores, so that the rows' sum is
// over a lane's own values and the four groups of lanes.
template <int D, bool BF16>
__global__ __launch_bounds__(kThreads) void attn_weights_kernel(CacheArgs a) {
  const int lane = lane_id(), g = lane >> 4, col = lane & 15;
  const auto cost = [&](int b) -> int64_t {
    return span_of(a.cu, b, a.tokens).count > 0 ? static_cast<int64_t>(a.heads) * ((seq_len(a, b) + kPage - 1) / kPage) : 0;
  };
  const int64_t total = sum_seqs(a.batch, cost);
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  const int64_t workers = static_cast<int64_t>(gridDim.x) * kWaves;
  const int64_t from = w * total / workers, to = (w + 1) * total / workers;
  for (int64_t at = from; at < to; ++at) {
    const Found f = find_seq(a.batch, at, cost);
    if (f.b < 0) break;
    const Span sp = span_of(a.cu, f.b, a.tokens);
    const int len = seq_len(a, f.b), npages = (len + kPage - 1) / kPage;
    const int head = static_cast<int>(f.local / npages), p = static_cast<int>(f.local % npages);
    const int rows = sp.count * a.group;
    const int page = a.table[static_cast<int64_t>(f.b) * a.width + p];
    if (page < 0 || page >= a.pages) continue;
    const int64_t ph = static_cast<int64_t>(page) * a.heads + head;
    u4 kr[4][D / 64];
    load_k<D, false>(a.kc + ph * (kPage * D), kr);
    const float ks = a.ks[ph];
    h8 kf[4][D / 32];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int k = 0; k < D / 32; ++k) kf[q][k] = codes_f16(kr[q][k >> 1][2 * (k & 1)], kr[q][k >> 1][2 * (k & 1) + 1]);
    float sum[4] = {0, 0, 0, 0};
    // the first token that sees the page
    const int seen = max(0, p * kPage - (len - sp.count));
    for (int row0 = seen * a.group / 16 * 16; row0 < rows; row0 += 16) {
      h8 qf[D / 32];
      float mult;
      load_q<D, BF16>(a, sp.first, rows, head, row0, qf, mult);
      float c[4], z[4];
      int limit[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = row0 + 4 * g + e, token = r / a.group;
        c[e] = __shfl(mult, 4 * g + e) * ks;
        limit[e] = r < rows ? token + len - sp.count + 1 : 0;
        z[e] = 0.0f;
        if (r < rows) z[e] = a.lse[(static_cast<int64_t>(head) * a.group + r - token * a.group) * a.tokens + sp.first + token];
        if (z[e] == -INFINITY) limit[e] = 0;   // a row that sees nothing gives nothing
        z[e] *= kLog2e;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f4 s = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < D / 32; ++k) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[k], kf[q][k], s, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = exp2_fast(__builtin_fmaf(s[e], c[e], -z[e]));
          sum[q] += p * kPage + 16 * q + col < limit[e] ? x : 0.0f;
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) sum[q] = sum_xor32(sum_xor16(sum[q]));
    const float mine = g == 0 ? sum[0] : g == 1 ? sum[1] : g == 2 ? sum[2] : sum[3];
    const int64_t j = static_cast<int64_t>(p) * kPage + lane;
    if (j < len && j < a.span) a.weights[(static_cast<int64_t>(f.b) * a.heads + head) * a.span + j] += mine;
  }
}

// Row tiles of 16 that a unit carries: enough for the call's average rows, at most 4.
int row_tiles(int64_t batch, int64_t tokens, int64_t group) {
  const int64_t rows = (tokens * group + batch - 1) / batch;
  return rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
}

int check(const char* who, const void* q, int dtype, int64_t q_st, int64_t q_sh, const void* k_cache, const void* k_scale,
          const void* table, const void* cu, const void* lens, int64_t batch, int64_t width, int64_t tokens,
          int64_t heads, int64_t group, int64_t d, int64_t pages, float scale) {
  PQ_REQUIRE(dtype == PQ_F16 || dtype == PQ_BF16, PQ_ERR_UNSUPPORTED, "%s: dtype code %d (Half or BFloat16)", who, dtype);
  PQ_REQUIRE(d == 64 || d == 128, PQ_ERR_UNSUPPORTED, "%s: head_dim=%lld (supported: 64, 128)", who, (long long)d);
  PQ_REQUIRE(batch >= 0 && batch <= 0x7fffffffLL && width >= 0 && width <= 0x7fffffffLL / kPage, PQ_ERR_ARG,
             "%s: batch=%lld table_width=%lld", who, (long long)batch, (long long)width);
  PQ_REQUIRE(heads >= 1 && group >= 1 && heads * group <= 65535, PQ_ERR_ARG, "%s: kv_heads=%lld group=%lld", who,
             (long long)heads, (long long)group);
  PQ_REQUIRE(tokens >= 0 && tokens * group <= 0x7fffffffLL - 64 && pages >= 0 && pages <= 0x7fffffffLL, PQ_ERR_ARG,
             "%s: tokens=%lld pages=%lld", who, (long long)tokens, (long long)pages);
  PQ_REQUIRE(scale > 0.0f && scale < INFINITY, PQ_ERR_ARG, "%s: scale=%g must be positive and finite", who, scale);
  if (tokens == 0) return PQ_OK;
  PQ_REQUIRE(q != nullptr && pq::aligned_to(q, 16) && q_st % 8 == 0 && q_sh % 8 == 0, PQ_ERR_ARG,
             "%s: q must be 16-byte aligned, its strides multiples of 8 values", who);
  PQ_REQUIRE(batch == 0 || (cu && lens), PQ_ERR_ARG, "%s: null cu_seqlens or lens", who);
  PQ_REQUIRE(batch == 0 || width == 0 || table, PQ_ERR_ARG, "%s: null block_table", who);
  PQ_REQUIRE(pages == 0 || (k_cache && k_scale && pq::aligned_to(k_cache, 16)), PQ_ERR_ARG,
             "%s: null or unaligned cache", who);
  return PQ_OK;
}

}  // namespace

extern "C" size_t pq_attn_cache_i8_workspace_size(int64_t batch, int64_t tokens, int64_t group, int64_t head_dim) {
  if (batch <= 0 || tokens <= 0 || group <= 0 || head_dim <= 0) return 0;
  return static_cast<size_t>(2 * kWorkers) * (16 * row_tiles(batch, tokens, group)) * (head_dim + 2) * sizeof(float);
}

extern "C" int pq_attn_cache_i8(const void* q, int dtype, int64_t q_stride_token, int64_t q_stride_head,
                                const int8_t* k_cache, const int8_t* v_cache, const float* k_scale,
                                const float* v_scale, const int32_t* block_table, const int32_t* cu_seqlens,
                                const int32_t* lens, void* out, float* lse, int64_t batch, int64_t table_width,
                                int64_t tokens, int64_t kv_heads, int64_t group, int64_t head_dim, int64_t pages,
                                float scale, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "pq_attn_cache_i8";
  const int st = check(who, q, dtype, q_stride_token, q_stride_head, k_cache, k_scale, block_table, cu_seqlens, lens, batch,
                       table_width, tokens, kv_heads, group, head_dim, pages, scale);
  if (st != PQ_OK || tokens == 0) return st;
  PQ_REQUIRE(out && lse && pq::aligned_to(out, 16), PQ_ERR_ARG, "%s: null or unaligned output", who);
  PQ_REQUIRE(pages == 0 || (v_cache && v_scale && pq::aligned_to(v_cache, 16)), PQ_ERR_ARG,
             "%s: null or unaligned cache", who);
  const size_t need = pq_attn_cache_i8_workspace_size(batch, tokens, group, head_dim);
  PQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && pq::aligned_to(workspace, 16)), PQ_ERR_WORKSPACE,
             "%s: a 16-byte aligned workspace of %zu bytes is needed, got %zu", who, need,
             workspace ? workspace_bytes : (size_t)0);
  CacheArgs a = {};
  a.q = q; a.kc = k_cache; a.vc = v_cache; a.ks = k_scale; a.vs = v_scale; a.table = block_table; a.cu = cu_seqlens;
  a.lens = lens; a.out = out; a.lse = lse; a.part = static_cast<float*>(workspace);
  a.q_st = q_stride_token; a.q_sh = q_stride_head;
  a.batch = static_cast<int>(batch); a.width = pages > 0 ? static_cast<int>(table_width) : 0;
  a.tokens = static_cast<int>(tokens); a.heads = static_cast<int>(kv_heads); a.group = static_cast<int>(group);
  a.pages = static_cast<int>(pages); a.workers = kWorkers;
  a.scale_log2 = scale * kLog2e;
  const int rt = batch > 0 ? row_tiles(batch, tokens, group) : 1;
  const dim3 join(static_cast<unsigned>(tokens), static_cast<unsigned>((kv_heads * group + kWaves - 1) / kWaves));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define PQ_CACHE(D_, RT_, BF_)                                                    \
  do {                                                                            \
    if (a.batch > 0 && a.width > 0)                                               \
      attn_cache_kernel<D_, (RT_ == 1 ? 1 : kRT), (RT_ == 1 ? 1 : RT_ / kRT), BF_><<<a.workers, kThreads, 0, s>>>(a);           \
    attn_cache_join_kernel<D_, RT_, BF_><<<join, kThreads, 0, s>>>(a);            \
  } while (0)
#define PQ_CACHE_RT(D_, BF_)                 \
  do {                                       \
    if (rt == 1) PQ_CACHE(D_, 1, BF_);       \
    else if (rt == 2) PQ_CACHE(D_, 2, BF_);  \
    else PQ_CACHE(D_, 4, BF_);               \
  } while (0)
  if (head_dim == 64 && dtype == PQ_BF16) PQ_CACHE_RT(64, true);
  else if (head_dim == 64) PQ_CACHE_RT(64, false);
  else if (dtype == PQ_BF16) PQ_CACHE_RT(128, true);
  else PQ_CACHE_RT(128, false);
#undef PQ_CACHE_RT
#undef PQ_CACHE
  return pq::launch_status("pq_attn_cache_i8 launch");
}

extern "C" int pq_attn_cache_weights_i8(const void* q, int dtype, int64_t q_stride_token, int64_t q_stride_head,
                                        const int8_t* k_cache, const float* k_scale, const int32_t* block_table,
                                        const int32_t* cu_seqlens, const int32_t* lens, const float* lse,
                                        float* weights, int64_t batch, int64_t table_width, int64_t span,
                                        int64_t tokens, int64_t kv_heads, int64_t group, int64_t head_dim,
                                        int64_t pages, float scale, void* stream) {
  const char* who = "pq_attn_cache_weights_i8";
  const int st = check(who, q, dtype, q_stride_token, q_stride_head, k_cache, k_scale, block_table, cu_seqlens, lens, batch,
                       table_width, tokens, kv_heads, group, head_dim, pages, scale);
  if (st != PQ_OK) return st;
  PQ_REQUIRE(span >= 0 && span <= 0x7fffffffLL, PQ_ERR_ARG, "%s: span=%lld", who, (long long)span);
  if (tokens == 0 || batch == 0 || table_width == 0 || pages == 0 || span == 0) return PQ_OK;
  PQ_REQUIRE(lse && weights, PQ_ERR_ARG, "%s: null lse or weights", who);
  CacheArgs a = {};
  a.q = q; a.kc = k_cache; a.ks = k_scale; a.table = block_table; a.cu = cu_seqlens; a.lens = lens;
  a.lse = const_cast<float*>(lse); a.weights = weights; a.span = span;
  a.q_st = q_stride_token; a.q_sh = q_stride_head;
  a.batch = static_cast<int>(batch); a.width = static_cast<int>(table_width);
  a.tokens = static_cast<int>(tokens); a.heads = static_cast<int>(kv_heads); a.group = static_cast<int>(group);
  a.pages = static_cast<int>(pages);
  a.scale_log2 = scale * kLog2e;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t most = (batch * kv_heads * table_width + kWaves - 1) / kWaves;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(most, 2 * kWorkers));
  if (head_dim == 64 && dtype == PQ_BF16) attn_weights_kernel<64, true><<<grid, kThreads, 0, s>>>(a);
  else if (head_dim == 64) attn_weights_kernel<64, false><<<grid, kThreads, 0, s>>>(a);
  else if (dtype == PQ_BF16) attn_weights_kernel<128, true><<<grid, kThreads, 0, s>>>(a);
  else attn_weights_kernel<128, false><<<grid, kThreads, 0, s>>>(a);
  return pq::launch_status("pq_attn_cache_weights_i8 launch");
}
