// The next token of each row from a given uniform number: temperature, top-k, top-p, min-p.
//
// w_i = exp((l_i - max l) / T) in 64 bits. In order of falling logits (equal ones by rising index) every filter keeps a beginning of the row, so the
// kept tokens are the first n, and the token drawn is the first whose cumulative weight exceeds u times theirs. A 16-bit logit has 65536 values:
// counting how often each occurs sorts the row, and what has to be computed in 64 bits is one exponential per value that occurs, not per token.
// Counts are whole numbers and the weights of a row are added in one order, so results do not depend on what arrives when.
//
// A row that one workgroup counts (sample_one_kernel: its counts, 16 bits a value, stay in LDS) takes one launch. Of a longer one workgroups count parts and write the runs of
// 1024 values that occur (sample_count_kernel), and a second launch has a workgroup add the parts' counts up (sample_pick_kernel). Either goes on with sample_token: weights of
// the segments of 64 values that occur, from the largest value down, then the value and which of the tokens that have it is drawn, then that token's place in the row.
#include <type_traits>

#include "common.cuh"

namespace mui {

constexpr int kCountThreads = 1024;
constexpr int kWaves = kCountThreads / kWave;
constexpr int kSegWords = 33;          // a segment's 64 counts in LDS, two in a word; a word further apart than they are long
constexpr int kRuns = 64;              // runs of 1024 values
constexpr int kMostPart = 65528;       // tokens of a part: their counts fit 16 bits
constexpr int kMostParts = 64;

struct SampleParams {
  const uint16_t* logits; long row_stride;
  int rows, vocab, parts, part_len;    // part_len a multiple of 8
  const float* u;
  const float* temperature; const int32_t* top_k; const float* top_p; const float* min_p;  // per row, or null: the one below
  float temperature1; int top_k1; float top_p1, min_p1;
  uint16_t* counts;                    // [rows][parts][65536]
  unsigned long long* runs;            // [rows][parts]: which runs of 1024 values occur
  int64_t* token;
  float* share;
};

// Place of a logit in falling order: 0 the largest (+inf). -0 and 0 are one; NaN and -inf have none (0xffffffff).
template <typename T>
__device__ __forceinline__ uint32_t place_of(uint32_t bits) {
  constexpr uint32_t kInf = T::kDtype == MUI_DTYPE_F16 ? 0x7c00u : 0x7f80u;
  if ((bits & 0x7fffu) > kInf || bits == (0x8000u | kInf)) return 0xffffffffu;
  if (bits == 0x8000u) bits = 0;
  return bits & 0x8000u ? bits : 0x7fffu - bits;
}
__device__ __forceinline__ uint32_t bits_of(uint32_t place) { return place & 0x8000u ? place : 0x7fffu - place; }

// A row's tokens begin .. end - 1 into counts that are 0: value k's in half k & 1 of word at(k >> 1).
template <typename T, typename At>
__device__ __forceinline__ void count_tokens(const uint16_t* x, int begin, int end, uint32_t* words, At at) {
  const int t = threadIdx.x;
  auto count = [&](uint32_t bits) {
    const uint32_t k = place_of<T>(bits);
    if (k != 0xffffffffu) atomicAdd(&words[at(k >> 1)], 1u << (16 * (k & 1)));
  };
  // (rows begin anywhere: 16 bytes at a time from the first place that is aligned)
  const int head = (int)(0u - (uint32_t)((uintptr_t)(x + begin) >> 1)) & 7;
  const int first = begin + head < end ? begin + head : end, whole = end > first ? (end - first) >> 3 : 0;
  constexpr int kAhead = 4;
  for (int c0 = t; c0 < whole; c0 += kAhead * kCountThreads) {
    u32x4 v[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) v[a] = ld16(x + first + 8 * (c0 + a * kCountThreads < whole ? c0 + a * kCountThreads : c0));
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (c0 + a * kCountThreads >= whole) break;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        count(v[a][j] & 0xffffu);
        count(v[a][j] >> 16);
      }
    }
  }
  if (begin + t < first) count(x[begin + t]);
  if (first + 8 * whole + t < end) count(x[first + 8 * whole + t]);
}

// One row of 128256 bf16 logits: 5.3 us here, 12.0 in sample_pick_kernel, of those 1.2 until the runs are known, 2.3 adding counts up, 2.1 weights, 2.2 the filters.
template <typename T>
__global__ void __launch_bounds__(kCountThreads) sample_count_kernel(const SampleParams p) {
  __shared__ u32x4 lds[8192];
  __shared__ unsigned long long mask_s;
  const int t = threadIdx.x, part = blockIdx.x, row = blockIdx.y;
  for (int i = t; i < 8192; i += kCountThreads) lds[i] = u32x4{0, 0, 0, 0};
  if (t == 0) mask_s = 0;
  __syncthreads();
  const int begin = part * p.part_len, end = begin + p.part_len < p.vocab ? begin + p.part_len : p.vocab;
  count_tokens<T>(p.logits + (long)row * p.row_stride, begin, end, (uint32_t*)lds, [](uint32_t w) { return w; });
  __syncthreads();
  // a wave per run of 1024 values = 2 KB
  uint16_t* out = p.counts + ((long)row * p.parts + part) * 65536;
  for (int r = t >> 6; r < kRuns; r += kWaves) {
    const int at = r * 128 + (t & 63);
    const u32x4 a = lds[at], b = lds[at + 64];
    if (__any((a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w) != 0)) {
      *(u32x4*)(out + 8 * at) = a;
      *(u32x4*)(out + 8 * at + 512) = b;
      if ((t & 63) == 0) atomicOr(&mask_s, 1ull << r);
    }
  }
  __syncthreads();
  if (t == 0) p.runs[(long)row * p.parts + part] = mask_s;
}

// What a workgroup of sample_token shares.
struct SampleShared {
  uint32_t seg_n[kRuns * 16];   // tokens in front of each segment that occurs (at first: of it)
  double seg_w[kRuns * 16];     // their weight
  uint16_t seg_id[kRuns * 16];  // which it is: its first place / 64
  uint16_t seg_at[kRuns * 16];  // where its counts lie: word kSegWords * seg_at
  uint32_t wave_n[kWaves];
  double wave_w[kWaves];
  uint32_t place, rank, first;
  int part;
  float share;
};

// The row's values are looked at in segments of 64 that occur: first every segment's sums, by four threads each, then, a wave and a lane per value, the few segments in
// which something ends. Neighbouring values of a segment lie equally far apart, so their weights are a geometric series: a thread takes an exponential for its 16
// and multiplies on (15 products of 2^-53 and as many of the quotient's own rounding: 4e-15).
// words: the counts in LDS; slots: segments there, number i's first place id(i) * 64 (rising); count_at: a value's count wherever it is, for counts beyond 16 bits (large); part_with:
// the part of the row that has the rank-th token of a place, the rank taken down to that part's own.
template <typename T, typename Id, typename CountAt, typename PartWith>
__device__ __forceinline__ void sample_token(const SampleParams& p, SampleShared& sh, const uint32_t* words, int slots, bool large, Id id, CountAt count_at, PartWith part_with) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, row = blockIdx.x;
  const float temperature = p.temperature ? p.temperature[row] : p.temperature1;
  const int top_k = p.top_k ? p.top_k[row] : p.top_k1;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p1;
  const float min_p = p.min_p ? p.min_p[row] : p.min_p1;
  const float u = p.u[row];
  // the segments that occur, in a row
  uint32_t some = 0, front = 0;  // front: the first value in it that does
  if (t < slots) {
#pragma unroll
    for (int j = 31; j >= 0; --j) {
      const uint32_t c = words[t * kSegWords + j];
      some |= c;
      front = c ? 2 * j + (c & 0xffffu ? 0 : 1) : front;
    }
  }
  const unsigned long long have = __ballot(some != 0);
  if (lane == 0) sh.wave_n[wave] = __popcll(have);
  __syncthreads();
  int n_seg = 0, mine = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i == wave) mine = n_seg;
    n_seg += sh.wave_n[i];
  }
  if (n_seg == 0) {  // nothing above -inf
    if (t == 0) {
      p.token[row] = 0;
      if (p.share) p.share[row] = 0.f;
    }
    return;
  }
  if (some) {
    mine += __popcll(have & ((1ull << lane) - 1ull));
    sh.seg_id[mine] = (uint16_t)id(t);
    sh.seg_at[mine] = (uint16_t)t;
    if (mine == 0) sh.first = id(t) * 64 + front;
  }
  __syncthreads();
  const uint32_t top = sh.first;
  auto logit = [](uint32_t place) { return (double)T::one((uint16_t)bits_of(place)); };
  const double most = logit(top);
  const bool greedy = !(temperature > 0.f);
  const double cold = 1.0 / (double)temperature;
  auto weight_of = [&](uint32_t place) -> double {
    if (place == top) return 1.0;
    if (greedy || most == INFINITY) return 0.0;
    return exp((logit(place) - most) * cold);
  };
  for (int i0 = 0; i0 < 4 * n_seg; i0 += kCountThreads) {
    const int i = i0 + t, seg = i < 4 * n_seg ? i >> 2 : 0, q = i & 3;
    const uint32_t place0 = sh.seg_id[seg] * 64u + 16 * q;
    const double l0 = logit(place0), step = logit(place0 + 1) - l0;
    const bool flat = greedy || most == INFINITY || !(fabs(l0) < INFINITY) || place0 + 15 < top;
    // (a series that begins in front of the largest logit only has to be finite there: what lies there does not occur, and the largest has its weight of 1 apart. Where
    // the bound on its beginning counts, what follows the largest weighs less than e^-40 of it.)
    const double ratio = flat ? 0.0 : exp(step * cold);
    double w = flat ? 0.0 : exp(fmin((l0 - most) * cold, 600.0)), sum = 0.0;
    uint32_t n = 0, n_top = 0;
    auto add = [&](int j, uint32_t m) {
      const uint32_t rest = place0 + j == top ? 0u : m;
      n += m;
      n_top += m - rest;
      sum = fma((double)rest, w, sum);
      w *= ratio;
    };
    if (!large) {
      const uint32_t* at = words + sh.seg_at[seg] * kSegWords + 8 * q;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t c = at[j];
        add(2 * j, c & 0xffffu);
        add(2 * j + 1, c >> 16);
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < 16; ++j) add(j, count_at(place0 + j));
    }
    sum += (double)n_top;
    n += __shfl_xor(n, 1);
    sum += __shfl_xor(sum, 1);
    n += __shfl_xor(n, 2);
    sum += __shfl_xor(sum, 2);
    if (q == 0 && i < 4 * n_seg) {
      sh.seg_n[seg] = n;
      sh.seg_w[seg] = sum;
    }
  }
  __syncthreads();
  // what is in front of each
  const int n_waves = (n_seg + kWave - 1) / kWave;
  uint32_t in_n = 0;
  double in_w = 0.0;
  if (wave < n_waves) {
    const uint32_t my_n = t < n_seg ? sh.seg_n[t] : 0u;
    const double my_w = t < n_seg ? sh.seg_w[t] : 0.0;
    in_n = wave_scan(my_n);
    in_w = wave_scan(my_w);
    if (lane == 63) {
      sh.wave_n[wave] = in_n;
      sh.wave_w[wave] = in_w;
    }
  }
  __syncthreads();
  uint32_t n_all = 0;
  double sum_w = 0.0;
  {
    uint32_t before_n = 0;
    double before_w = 0.0;
    for (int i = 0; i < n_waves; ++i) {
      if (i == wave) { before_n = n_all; before_w = sum_w; }
      n_all += sh.wave_n[i];
      sum_w += sh.wave_w[i];
    }
    if (wave < n_waves) {
      const uint32_t a = __shfl_up(in_n, 1);
      const double b = __shfl_up(in_w, 1);
      if (t < n_seg) {
        sh.seg_n[t] = before_n + (lane ? a : 0u);
        sh.seg_w[t] = before_w + (lane ? b : 0.0);
      }
    }
  }
  __syncthreads();
  if (wave == 0) {
    // one segment: this lane's value, how many tokens have it, its weight; tokens and weight up to and with it
    struct Seg { int s; uint32_t place, n, to_n; double one, to_w; };
    Seg g;
    g.s = -1;
    auto segment = [&](int s) {
      if (s == g.s) return;  // (often the one that was looked at last)
      g.s = s;
      g.place = sh.seg_id[s] * 64u + lane;
      g.n = large ? count_at(g.place) : words[sh.seg_at[s] * kSegWords + (lane >> 1)] >> (16 * (lane & 1)) & 0xffffu;
      g.one = g.n ? weight_of(g.place) : 0.0;
      g.to_n = sh.seg_n[s] + wave_scan(g.n);
      g.to_w = sh.seg_w[s] + wave_scan(g.n * g.one);
    };
    // the last segment for which `in` holds (it holds of a beginning of them, and of the first): of the segments 0, 64, 128 .., then of the 64 from there on
    auto last_of = [&](auto in) {
      int from = 0;
      if (n_waves > 1) from = 64 * (63 - __clzll((long long)__ballot(lane < n_waves && in(lane < n_waves ? 64 * lane : 0))));
      return from + 63 - __clzll((long long)__ballot(from + lane < n_seg && in(from + lane < n_seg ? from + lane : 0)));
    };
    // the weight of the first n > 0 tokens, and the place of the last of them
    uint32_t last = 0xffffffffu;
    auto weight_of_first = [&](uint32_t n) {
      if (n >= n_all) return sum_w;
      segment(last_of([&](int s) { return sh.seg_n[s] < n; }));
      const int l = __ffsll((long long)__ballot(g.to_n >= n)) - 1;
      last = (uint32_t)__shfl((int)g.place, l);
      return __shfl(g.to_w - (double)(g.to_n - n) * g.one, l);
    };
    uint32_t kept = greedy ? 1u : n_all;
    if (top_k > 0 && (uint32_t)top_k < kept) kept = (uint32_t)top_k;
    if (top_p < 1.f) {
      const double limit = (double)top_p * weight_of_first(kept);
      segment(last_of([&](int s) { return s == 0 || sh.seg_w[s] < limit; }));
      const unsigned long long reached = __ballot(g.to_w >= limit);
      uint32_t n = __shfl(g.to_n, 63);
      if (reached) {  // of the value that reaches the limit: the tokens in front of which less lies
        const double in_front = g.to_w - g.n * g.one;
        const double some_n = g.one > 0 ? ceil((limit - in_front) / g.one) : 0.0;
        const uint32_t upto = g.to_n - g.n + (some_n < 0 ? 0u : some_n < (double)g.n ? (uint32_t)some_n : g.n);
        n = __shfl(upto, __ffsll((long long)reached) - 1);
      }
      if (n < kept) kept = n;
    }
    if (kept < 1 || min_p > 1.f) kept = 1;  // (no weight reaches a min_p above 1)
    double all = weight_of_first(kept);
    if (min_p > 0.f && kept > 1) {  // (weights and logits fall together)
      const double least = log((double)min_p);
      auto enough = [&](uint32_t place) { return place <= top || (logit(place) - most) * cold >= least; };
      if (kept >= n_all || !enough(last)) {
        segment(last_of([&](int s) { return s == 0 || enough(sh.seg_id[s] * 64u); }));
        const uint32_t n = __shfl(g.to_n, 63 - __clzll((long long)__ballot(enough(g.place))));
        if (n < kept) {
          kept = n;
          all = weight_of_first(kept);
        }
      }
    }
    const double target = (u > 0.f ? (double)u : 0.0) * all;
    segment(last_of([&](int s) { return s == 0 || (sh.seg_n[s] < kept && sh.seg_w[s] <= target); }));
    const unsigned long long over = __ballot(g.n && (g.to_w > target || g.to_n >= kept));
    // (no lane: the segment's sum, added in another order, stops short of the target by a rounding: its last value)
    const int l = over ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)__ballot(g.n != 0));
    const uint32_t first_n = g.to_n - g.n, here = g.n < kept - first_n ? g.n : kept - first_n;
    const double r = g.one > 0 ? floor((target - (g.to_w - g.n * g.one)) / g.one) : 0.0;
    const uint32_t rank = r < 0 ? 0u : r < (double)here ? (uint32_t)r : here - 1u;
    const uint32_t place = (uint32_t)__shfl((int)g.place, l);
    uint32_t left = (uint32_t)__shfl((int)rank, l);
    const double one = __shfl(g.one, l);
    const int part = part_with(place, left);
    if (lane == 0) {
      sh.place = place;
      sh.rank = left;
      sh.part = part;
      sh.share = (float)(one / all);
    }
  }
  __syncthreads();
  // the rank-th token of that value in its part: 8 in a row per lane and step, which ones have it kept in a bit each
  const uint32_t bits = bits_of(sh.place), or_bits = bits ? bits : 0x8000u;
  uint32_t rank = sh.rank;
  const int part = sh.part;
  const uint16_t* x = p.logits + (long)row * p.row_stride;
  const int begin = part * p.part_len, end = begin + p.part_len < p.vocab ? begin + p.part_len : p.vocab;
  const int per = ((p.part_len + 7) / 8 + kWaves) / kWaves * 8;  // tokens of a wave, at most 4096; one chunk of 8 more where the part begins within one
  const int wb = begin - (int)((uintptr_t)(x + begin) >> 1 & 7) + wave * per, we = wb + per < end ? wb + per : end;
  unsigned long long found = 0;
#pragma unroll 4
  for (int s = 0; s < 8; ++s) {
    const int i = wb + 512 * s + 8 * lane;
    if (i >= we) break;
    uint32_t m = 0;
    if (i >= begin && i + 8 <= we) {
      const u32x4 v = ld16(x + i);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        m |= ((v[j] & 0xffffu) == bits || (v[j] & 0xffffu) == or_bits ? 1u : 0u) << (2 * j) | (v[j] >> 16 == bits || v[j] >> 16 == or_bits ? 2u : 0u) << (2 * j);
    } else {
      for (int j = 0; j < 8; ++j)
        if (i + j >= begin && i + j < we) m |= (x[i + j] == bits || x[i + j] == or_bits ? 1u : 0u) << j;
    }
    found |= (unsigned long long)m << (8 * s);
  }
  uint32_t hits = __popcll(found);
  for (int off = 32; off; off >>= 1) hits += __shfl_xor(hits, off);
  if (lane == 0) sh.wave_n[wave] = hits;
  __syncthreads();
  for (int w = 0; w < wave; ++w) rank -= sh.wave_n[w];  // (below zero: it wraps, and is no token of this wave)
  if (rank >= sh.wave_n[wave]) return;
  for (int s = 0; s < 8; ++s) {
    const uint32_t here = (uint32_t)(found >> (8 * s)) & 0xffu;
    const uint32_t n = __popc(here), to = wave_scan(n), total = __shfl(to, 63);
    if (rank < total) {
      if (rank >= to - n && rank < to) {
        uint32_t left = rank - (to - n), b = here;
        while (left--) b &= b - 1;
        p.token[row] = wb + 512 * s + 8 * lane + __ffs((int)b) - 1;
        if (p.share) p.share[row] = sh.share;
      }
      return;
    }
    rank -= total;
  }
}

// 256 rows of 32000 fp16 logits 17.3 us, 4.3 of them counting, 2.6 looking for the segments that occur, 4.1 their weights, 1.4 the token's place; one row of 4000 bf16 ones 10.8, mostly
// steps that wait for one another.
template <typename T>
__global__ void __launch_bounds__(kCountThreads) sample_one_kernel(const SampleParams p) {
  __shared__ SampleShared sh;
  __shared__ u32x4 words[kRuns * 16 * kSegWords / 4];
  const int t = threadIdx.x;
  for (int i = t; i < kRuns * 16 * kSegWords / 4; i += kCountThreads) words[i] = u32x4{0, 0, 0, 0};
  __syncthreads();
  count_tokens<T>(p.logits + (long)blockIdx.x * p.row_stride, 0, p.vocab, (uint32_t*)words, [](uint32_t w) { return w + (w >> 5); });
  __syncthreads();
  sample_token<T>(p, sh, (const uint32_t*)words, kRuns * 16, false, [](int i) { return (uint32_t)i; }, [](uint32_t) { return 0u; }, [](uint32_t, uint32_t&) { return 0; });
}

template <typename T>
__global__ void __launch_bounds__(kCountThreads) sample_pick_kernel(const SampleParams p) {
  __shared__ SampleShared sh;
  __shared__ uint32_t held[kRuns * 16 * kSegWords];  // the parts' counts together, of the runs that occur
  __shared__ int large_s;                            // a count that does not fit 16 bits: the row's are then taken from memory
  __shared__ unsigned long long masks[kMostParts];
  __shared__ int list[kRuns];
  const int t = threadIdx.x, lane = t & 63, row = blockIdx.x;
  const uint16_t* counts = p.counts + (long)row * p.parts * 65536;
  const int parts = p.parts;
  unsigned long long all_runs = lane < parts ? p.runs[(long)row * parts + lane] : 0ull;
  if (t < kMostParts) masks[t] = all_runs;
  for (int off = 1; off < kMostParts; off <<= 1) all_runs |= __shfl_xor(all_runs, off);
  const int n_runs = __popcll(all_runs);
  if (t == 0) large_s = 0;
  if (t < kRuns && (all_runs >> t & 1ull)) list[__popcll(all_runs & ((1ull << t) - 1ull))] = t;
  __syncthreads();
  // (counts are read whether their part has the run or not, so that no load waits for another: what a part has not written does not count)
  constexpr int kAhead = 4;
  auto count_at = [&](uint32_t place) {
    uint32_t n = 0;
    for (int i0 = 0; i0 < parts; i0 += kAhead) {
      uint16_t c[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) c[i] = counts[(long)(i0 + i < parts ? i0 + i : i0) * 65536 + place];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) n += i0 + i < parts && (masks[i0 + i < parts ? i0 + i : i0] >> (place >> 10) & 1ull) ? c[i] : 0;
    }
    return n;
  };
  // the parts' counts together, 8 values of a run per thread; 8 loads in flight, of as many parts as there are
  auto add_up = [&](auto at_once) {
    constexpr int PB = decltype(at_once)::value, CB = 8 / PB;
    for (int c0 = t; c0 < n_runs * 128; c0 += CB * kCountThreads) {
      uint32_t n[CB][8] = {};
      int run[CB];
#pragma unroll
      for (int k = 0; k < CB; ++k) run[k] = __builtin_amdgcn_readfirstlane(list[(c0 + k * kCountThreads < n_runs * 128 ? c0 + k * kCountThreads : c0) >> 7]);
      for (int i0 = 0; i0 < parts; i0 += PB) {
        u32x4 v[CB][PB];
#pragma unroll
        for (int k = 0; k < CB; ++k)
#pragma unroll
          for (int i = 0; i < PB; ++i) v[k][i] = ld16(counts + (long)(i0 + i < parts ? i0 + i : i0) * 65536 + run[k] * 1024 + (t & 127) * 8);
#pragma unroll
        for (int k = 0; k < CB; ++k)
#pragma unroll
          for (int i = 0; i < PB; ++i) {
            if (i0 + i >= parts || !(masks[i0 + i] >> run[k] & 1ull)) continue;  // (the same for the wave)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              n[k][2 * j] += v[k][i][j] & 0xffffu;
              n[k][2 * j + 1] += v[k][i][j] >> 16;
            }
          }
      }
#pragma unroll
      for (int k = 0; k < CB; ++k) {
        const int c = c0 + k * kCountThreads;
        if (c >= n_runs * 128) break;
        uint32_t* to = held + (c >> 3) * kSegWords + (c & 7) * 4;
        uint32_t high = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a = n[k][2 * j], b = n[k][2 * j + 1];
          to[j] = (a < 0xffffu ? a : 0xffffu) | (b < 0xffffu ? b : 0xffffu) << 16;
          high |= a | b;
        }
        if (high >> 16) large_s = 1;
      }
    }
  };
  if (parts == 2) add_up(std::integral_constant<int, 2>()); else add_up(std::integral_constant<int, 8>());
  __syncthreads();
  auto part_with = [&](uint32_t place, uint32_t& left) {
    uint32_t c = 0;
    if (lane < parts && (masks[lane < parts ? lane : 0] >> (place >> 10) & 1ull)) c = counts[(long)lane * 65536 + place];
    const uint32_t to = wave_scan(c);
    const unsigned long long has = __ballot(to > left);
    const int part = has ? __ffsll((long long)has) - 1 : 0;
    left -= __shfl(to - c, part);
    return part;
  };
  sample_token<T>(p, sh, held, n_runs * 16, large_s != 0, [&](int i) { return (uint32_t)list[i >> 4] * 16u + (i & 15); }, count_at, part_with);
}

struct SamplePlan { int parts, part_len; bool one; };
static SamplePlan sample_plan(int rows, int vocab, int dtype) {
  SamplePlan r;
  // One workgroup a row, or several and a second launch. us, one / several: one row of 32000 bf16 logits 15.1 / 17.2, of 50000 18.9 / 17.5; 64 rows of 50000 20.4 / 20.4,
  // 256 rows of 32000 17.3 / 23.0, of 65000 24.7 / 29.6; fp16, one row of 50000 20.8 / 21.3, 16 rows 22.1 / 24.1.
  r.one = vocab <= (rows < 64 && dtype == MUI_DTYPE_BF16 ? 40000 : kMostPart);
  // Parts of 16384 tokens or more, no more workgroups than there are CUs (one's counts fill its LDS); of 32768 for fp16, whose counts of usual logits are 72 KB a part to add up
  // (bf16's 10). us, 16384 / 32768: one row of 128256 bf16 logits 19.0 / 20.9, fp16 26.2 / 25.1, 16 rows of 200000 fp16 37.2 / 32.1.
  int parts = (vocab + kMostPart - 1) / kMostPart;
  const int least = dtype == MUI_DTYPE_F16 ? 32768 : 16384;
  const int want = rows < 256 ? 256 / rows : 1, most = (vocab + least - 1) / least;
  const int more = r.one ? 1 : want < most ? want : most;
  parts = parts > more ? parts : more;
  parts = parts < kMostParts ? parts : kMostParts;
  r.part_len = ((vocab + parts - 1) / parts + 7) / 8 * 8;
  r.parts = (vocab + r.part_len - 1) / r.part_len;
  return r;
}

}  // namespace mui

using namespace mui;

extern "C" size_t mui_sample_filtered_workspace_bytes(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  const SamplePlan plan = sample_plan(rows, vocab, MUI_DTYPE_BF16);  // (the most parts)
  return plan.one ? 0 : (size_t)rows * plan.parts * (131072 + 8);
}

extern "C" int mui_sample_filtered(mui_stream_t stream, const mui_sample_filtered_args_t* args) {
  MUI_CHECK_ARG(args);
  const mui_sample_filtered_args_t& a = *args;
  MUI_CHECK_ARG(a.logits && a.random_numbers && a.out_token && a.rows > 0 && a.vocab > 0 && a.row_stride >= a.vocab);
  if (a.dtype != MUI_DTYPE_F16 && a.dtype != MUI_DTYPE_BF16) return MUI_ERR_INVALID_ARG;
  if (a.rows > 65535 || a.vocab > kMostParts * kMostPart) return MUI_ERR_UNSUPPORTED;
  if ((uintptr_t)a.workspace & 15u) return MUI_ERR_ALIGNMENT;
  const SamplePlan plan = sample_plan(a.rows, a.vocab, a.dtype);
  if (!plan.one && (!a.workspace || a.workspace_bytes < mui_sample_filtered_workspace_bytes(a.rows, a.vocab))) return MUI_ERR_INVALID_ARG;
  SampleParams p = {};
  p.logits = (const uint16_t*)a.logits; p.row_stride = a.row_stride; p.rows = a.rows; p.vocab = a.vocab; p.parts = plan.parts; p.part_len = plan.part_len;
  p.u = a.random_numbers;
  p.temperature = a.temperatures; p.top_k = a.top_ks; p.top_p = a.top_ps; p.min_p = a.min_ps;
  p.temperature1 = a.temperature; p.top_k1 = a.top_k; p.top_p1 = a.top_p; p.min_p1 = a.min_p;
  p.counts = (uint16_t*)a.workspace;
  p.runs = (unsigned long long*)((char*)a.workspace + (size_t)a.rows * plan.parts * 131072);
  p.token = a.out_token; p.share = a.out_probability;
  hipStream_t s = (hipStream_t)stream;
#define MUI_SAMPLE_GO(TT)                                                                                          \
  do {                                                                                                              \
    if (plan.one) {                                                                                                 \
      hipLaunchKernelGGL((sample_one_kernel<TT>), dim3(a.rows), dim3(kCountThreads), 0, s, p);                      \
    } else {                                                                                                        \
      hipLaunchKernelGGL((sample_count_kernel<TT>), dim3(plan.parts, a.rows), dim3(kCountThreads), 0, s, p);        \
      hipLaunchKernelGGL((sample_pick_kernel<TT>), dim3(a.rows), dim3(kCountThreads), 0, s, p);                     \
    }                                                                                                               \
  } while (0)
  if (a.dtype == MUI_DTYPE_F16) MUI_SAMPLE_GO(F16); else MUI_SAMPLE_GO(BF16);
  return launch_status();
}
