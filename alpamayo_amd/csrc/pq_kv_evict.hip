// cache_evict_i8: each head of each sequence keeps its last `recent` tokens
// and, of those before them, the ones with the largest summed attention
// weights, `keep` in all; equal weights go to the earlier token.  What is
// kept moves, in order, to the front of new pages.
//
// Two kernels.  The first picks: one workgroup per sequence and head finds
// the smallest kept weight digit by digit (weights as unsigned keys of the
// same order, digits of 11, 11 and 10 bits, a histogram each), then walks the
// tokens once and writes the kept positions in order.  The second moves: one
// workgroup per new page, head and side gathers its 64 tokens and rounds them
// to the new page's scale, absmax / 127 of the values that they stand for.
#include "pq_attn.h"

namespace {

using namespace pqa;

constexpr int kPickThreads = 1024;
constexpr int kPickWaves = kPickThreads / 64;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;

// Unsigned keys in the order of the weights; NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct PickArgs {
  const float* weights;      // [batch, heads, span]
  const int* lens;           // [batch]
  float* weights_out;        // [batch, heads, span]
  int* lens_out;             // [batch]
  int* kept;                 // [batch, heads, keep]
  int heads, width, keep, recent;
  int64_t span;
};

__global__ __launch_bounds__(kPickThreads) void kv_pick_kernel(PickArgs a) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t above[kPickWaves];
  __shared__ uint32_t chosen, rest;
  const int b = blockIdx.y, head = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t row = static_cast<int64_t>(b) * a.heads + head;
  const float* w = a.weights + row * a.span;
  float* wo = a.weights_out + row * a.span;
  int* kept = a.kept + row * a.keep;

  int64_t most = static_cast<int64_t>(a.width) * kPage;
  most = most < a.span ? most : a.span;
  const int len = static_cast<int>(a.lens[b] < 0 ? 0 : a.lens[b] < most ? a.lens[b] : most);
  const int left = len < a.keep ? len : a.keep;
  const int fixed = len > a.recent ? len - a.recent : 0;   // tokens from here on stay
  int need = left - (len - fixed);                         // how many of those before them do

  // the smallest kept key, and how many tokens that have it are kept
  uint32_t key = 0, quota = 0;
  if (need > 0 && need < fixed) {
    uint32_t mask = 0, want = static_cast<uint32_t>(need);
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t bits = pass == 2 ? 1023u : 2047u;
      for (int i = t; i < kBins; i += kPickThreads) hist[i] = 0;
      __syncthreads();
      for (int i = t; i < fixed; i += kPickThreads) {
        const uint32_t u = weight_key(w[i]);
        if ((u & mask) == key) atomicAdd(&hist[(u >> shift) & bits], 1u);
      }
      __syncthreads();
      // bins from the top: thread t holds two, its wave's sum and those of the waves above tell how many lie over them
      const uint32_t hi = hist[kBins - 1 - 2 * t], lo = hist[kBins - 2 - 2 * t];
      uint32_t incl = hi + lo;
#pragma unroll
      for (int s = 1; s < 64; s <<= 1) {
        const uint32_t up = __shfl_up(incl, s);
        if (lane >= s) incl += up;
      }
      if (lane == 63) above[wave] = incl;
      __syncthreads();
      uint32_t over = incl - hi - lo;
      for (int i = 0; i < wave; ++i) over += above[i];
      if (over < want && over + hi >= want) { chosen = kBins - 1 - 2 * t; rest = want - over; }
      else if (over + hi < want && over + hi + lo >= want) { chosen = kBins - 2 - 2 * t; rest = want - over - hi; }
      __syncthreads();
      key |= chosen << shift;
      mask |= bits << shift;
      want = rest;
      __syncthreads();
    }
    quota = want;
  } else if (need > 0) {
    need = fixed;
    quota = static_cast<uint32_t>(fixed);   // all: every key is at least 0, and quota covers those that are 0
  }

  // the kept tokens in order
  uint32_t ties = 0, done = 0;
  for (int base = 0; base < len; base += kPickThreads) {
    const int i = base + t;
    const float x = i < len ? w[i] : 0.0f;
    const uint32_t u = weight_key(x);
    const bool tie = need > 0 && i < fixed && u == key;
    const uint64_t tm = __ballot(tie);
    const uint64_t below = (1ull << lane) - 1;
    if (lane == 0) above[wave] = static_cast<uint32_t>(__builtin_popcountll(tm));
    __syncthreads();
    uint32_t tb = ties, tsum = 0;
    for (int q = 0; q < kPickWaves; ++q) {
      const uint32_t c = above[q];
      if (q < wave) tb += c;
      tsum += c;
    }
    ties += tsum;
    tb += static_cast<uint32_t>(__builtin_popcountll(tm & below));
    const bool keep = i < len && (i >= fixed || (need > 0 && (u > key || (tie && tb < quota))));
    const uint64_t km = __ballot(keep);
    __syncthreads();
    if (lane == 0) above[wave] = static_cast<uint32_t>(__builtin_popcountll(km));
    __syncthreads();
    uint32_t at = done, ksum = 0;
    for (int q = 0; q < kPickWaves; ++q) {
      const uint32_t c = above[q];
      if (q < wave) at += c;
      ksum += c;
    }
    done += ksum;
    at += static_cast<uint32_t>(__builtin_popcountll(km & below));
    if (keep) {
      kept[at] = i;
      wo[at] = x;
    }
    __syncthreads();
  }
  for (int64_t i = left + t; i < a.keep; i += kPickThreads) kept[i] = -1;
  for (int64_t i = left + t; i < a.span; i += kPickThreads) wo[i] = 0.0f;
  if (t == 0 && head == 0) a.lens_out[b] = left;
}

struct MoveArgs {
  int8_t* cache[2];
  float* scale[2];
  const int* table;          // [batch, width]
  const int* new_table;      // [batch, new_width]
  const int* lens;           // [batch], what is kept
  const int* kept;           // [batch, heads, keep]
  int heads, width, new_width, keep, pages, new_pages;
};

template <int D>
__global__ __launch_bounds__(kMoveThreads) void kv_move_kernel(MoveArgs a) {
  __shared__ int64_t src[kPage];     // byte offset of each token's page side
  __shared__ int slot[kPage];
  __shared__ float mult[kPage];
  __shared__ uint32_t top[4];
  const int side = blockIdx.z, head = blockIdx.y, t = threadIdx.x;
  const int b = blockIdx.x / a.new_pages, j = blockIdx.x % a.new_pages;
  const int left = a.lens[b] - j * kPage;
  if (left <= 0 || j >= a.new_width) return;
  const int count = left < kPage ? left : kPage;
  const int page = a.new_table[static_cast<int64_t>(b) * a.new_width + j];
  if (page < 0 || page >= a.pages) return;
  if (t < kPage) {
    int64_t off = 0;
    int s = 0;
    float m = 0.0f;
    if (t < count) {
      const int pos = a.kept[(static_cast<int64_t>(b) * a.heads + head) * a.keep + j * kPage + t];
      const int from = a.table[static_cast<int64_t>(b) * a.width + pos / kPage];
      s = pos % kPage;
      if (from >= 0 && from < a.pages) {
        const int64_t ph = static_cast<int64_t>(from) * a.heads + head;
        off = ph * (kPage * D);
        m = a.scale[side][ph];
      }
    }
    src[t] = off;
    slot[t] = s;
    mult[t] = m;
  }
  __syncthreads();

  const int8_t* cache = a.cache[side];
  constexpr int kOwn = kPage * D / kMoveThreads;           // codes of a thread: 32 (d = 128) or 16
  float v[kOwn];
  uint32_t big = 0;
  // K: runs of 16 channels of a token; V: a token for each lane, channels wave by wave
  if (side == 0) {
#pragma unroll
    for (int r = 0; r < kOwn / 16; ++r) {
      const int q = t + r * kMoveThreads, tok = q / (D / 16), c = q % (D / 16);
      const u4 w = *reinterpret_cast<const u4*>(cache + src[tok] + slot[tok] * D + c * 16);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        v[r * 16 + e] = static_cast<float>(static_cast<int8_t>(w[e >> 2] >> (8 * (e & 3)))) * mult[tok];
    }
  } else {
    const int tok = t & 63, d0 = t >> 6;
    const int8_t* p = cache + src[tok] + slot[tok];
#pragma unroll
    for (int r = 0; r < kOwn; ++r) v[r] = static_cast<float>(p[(d0 + 4 * r) * kPage]) * mult[tok];
  }
#pragma unroll
  for (int r = 0; r < kOwn; ++r) {
    const uint32_t m = __float_as_uint(v[r]) & 0x7fffffffu;
    big = m < 0x7f800000u && m > big ? m : big;
  }
  big = pq_wave_umax(big);
  if ((t & 63) == 0) top[t >> 6] = big;
  __syncthreads();
  const float amax = __uint_as_float(max(max(top[0], top[1]), max(top[2], top[3])));
  const float now = amax < kTiny ? 0.0f : amax / 127.0f;
  const float inv = now > 0.0f ? 1.0f / now : 0.0f;
  const int64_t ph = static_cast<int64_t>(page) * a.heads + head;
  int8_t* out = a.cache[side] + ph * (kPage * D);
  if (side == 0) {
#pragma unroll
    for (int r = 0; r < kOwn / 16; ++r) {
      const int q = t + r * kMoveThreads, tok = q / (D / 16), c = q % (D / 16);
      if (tok >= count) continue;
      u4 w = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 16; ++e)
        w[e >> 2] |= (static_cast<uint32_t>(code_of(v[r * 16 + e], inv)) & 0xffu) << (8 * (e & 3));
      *reinterpret_cast<u4*>(out + tok * D + c * 16) = w;
    }
  } else {
    const int tok = t & 63, d0 = t >> 6;
    if (tok < count) {
#pragma unroll
      for (int r = 0; r < kOwn; ++r) out[(d0 + 4 * r) * kPage + tok] = static_cast<int8_t>(code_of(v[r], inv));
    }
  }
  if (t == 0) a.scale[side][ph] = now;
}

}  // namespace

extern "C" int pq_kv_evict_i8(int8_t* k_cache, int8_t* v_cache, float* k_scale, float* v_scale, const float* weights,
                              const int32_t* block_table, const int32_t* lens, const int32_t* new_table,
                              float* weights_out, int32_t* lens_out, int32_t* kept, int64_t batch, int64_t table_width,
                              int64_t new_width, int64_t span, int64_t heads, int64_t head_dim, int64_t pages,
                              int64_t keep, int64_t recent, void* stream) {
  const char* who = "pq_kv_evict_i8";
  PQ_REQUIRE(head_dim == 64 || head_dim == 128, PQ_ERR_UNSUPPORTED, "%s: head_dim=%lld (supported: 64, 128)", who,
             (long long)head_dim);
  PQ_REQUIRE(batch >= 0 && batch <= 65535 && heads >= 1 && heads <= 65535, PQ_ERR_ARG,
             "%s: batch=%lld heads=%lld (at most 65535)", who, (long long)batch, (long long)heads);
  PQ_REQUIRE(table_width >= 0 && table_width <= 0x7fffffffLL / kPage && new_width >= 0 &&
                 new_width <= 0x7fffffffLL / kPage && pages >= 0 && pages <= 0x7fffffffLL && span >= 0 &&
                 span <= 0x7fffffffLL, PQ_ERR_ARG,
             "%s: table_width=%lld new_width=%lld pages=%lld span=%lld", who, (long long)table_width,
             (long long)new_width, (long long)pages, (long long)span);
  PQ_REQUIRE(keep >= 1 && keep <= 0x7fffff00LL && recent >= 0 && recent <= keep, PQ_ERR_ARG,
             "%s: keep=%lld recent=%lld (keep at least 1, recent 0..keep)", who, (long long)keep, (long long)recent);
  const int64_t new_pages = (keep + kPage - 1) / kPage;
  PQ_REQUIRE(batch * new_pages <= 0x7fffffffLL, PQ_ERR_ARG, "%s: too many pages", who);
  if (batch == 0) return PQ_OK;
  PQ_REQUIRE(new_width >= new_pages || new_width * kPage >= table_width * kPage, PQ_ERR_ARG,
             "%s: new_table has room for %lld tokens, keep=%lld", who, (long long)(new_width * kPage), (long long)keep);
  PQ_REQUIRE(lens && lens_out && kept, PQ_ERR_ARG, "%s: null pointer", who);
  PQ_REQUIRE(span == 0 || (weights && weights_out), PQ_ERR_ARG, "%s: null weights", who);
  PQ_REQUIRE(table_width == 0 || (block_table && new_table), PQ_ERR_ARG, "%s: null table", who);
  PQ_REQUIRE(pages == 0 || (k_cache && v_cache && k_scale && v_scale), PQ_ERR_ARG, "%s: null cache", who);
  PQ_REQUIRE(pq::aligned_to(k_cache, 16) && pq::aligned_to(v_cache, 16), PQ_ERR_ARG,
             "%s: k_cache and v_cache must be 16-byte aligned", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  PickArgs p;
  p.weights = weights; p.lens = lens; p.weights_out = weights_out; p.lens_out = lens_out; p.kept = kept;
  p.heads = static_cast<int>(heads); p.width = static_cast<int>(table_width);
  p.keep = static_cast<int>(keep); p.recent = static_cast<int>(recent); p.span = span;
  kv_pick_kernel<<<dim3(static_cast<unsigned>(heads), static_cast<unsigned>(batch)), kPickThreads, 0, s>>>(p);
  if (pages > 0 && table_width > 0 && span > 0) {
    MoveArgs m;
    m.cache[0] = k_cache; m.cache[1] = v_cache; m.scale[0] = k_scale; m.scale[1] = v_scale;
    m.table = block_table; m.new_table = new_table; m.lens = lens_out; m.kept = kept;
    m.heads = static_cast<int>(heads); m.width = static_cast<int>(table_width);
    m.new_width = static_cast<int>(new_width); m.keep = static_cast<int>(keep);
    m.pages = static_cast<int>(pages);
    m.new_pages = static_cast<int>(new_pages < new_width ? new_pages : new_width);
    const dim3 grid(static_cast<unsigned>(batch * m.new_pages), static_cast<unsigned>(heads), 2);
    if (m.new_pages > 0) {
      if (head_dim == 64) kv_move_kernel<64><<<grid, kMoveThreads, 0, s>>>(m);
      else kv_move_kernel<128><<<grid, kMoveThreads, 0, s>>>(m);
    }
  }
  return pq::launch_status("pq_kv_evict_i8 launch");
}
