// The next token of each row from a given uniform number: temperature, top-k, top-p, min-p.
//
// w_i = exp((l_i - max l) / T) in 64 bits. In order of falling logits (equal ones by rising index) every filter keeps a beginning of the row, so the
// kept tokens are the first n, and the token drawn is the first whose cumulative weight exceeds u times theirs. A 16-bit logit has 65536 values:
// counting how often each occurs sorts the row, and what has to be computed in 64 bits is one exponential per value that occurs, not per token.
// Counts are whole numbers and the weights of a row are added in one order, so results do not depend on what arrives when.
//
// First kernel: workgroups count parts of a row in LDS (16 bits a value, 128 KB) and write the runs of 1024 values that occur. Second: a workgroup per row adds
// the parts' counts up from the largest value down, finds the value and which of the tokens that have it is drawn, and looks for that token in its part.
#include <type_traits>

#include "common.cuh"

namespace mui {

constexpr int kCountThreads = 1024;
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
  uint32_t* first;                     // [rows][parts]: the first place that does
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

template <typename T>
__global__ void __launch_bounds__(kCountThreads) sample_count_kernel(const SampleParams p) {
  __shared__ u32x4 lds[8192];
  __shared__ unsigned long long mask_s;
  __shared__ uint32_t first_s;
  uint32_t* words = (uint32_t*)lds;
  const int t = threadIdx.x, part = blockIdx.x, row = blockIdx.y;
  for (int i = t; i < 8192; i += kCountThreads) lds[i] = u32x4{0, 0, 0, 0};
  if (t == 0) {
    mask_s = 0;
    first_s = 0xffffffffu;
  }
  __syncthreads();
  const uint16_t* x = p.logits + (long)row * p.row_stride;
  const int begin = part * p.part_len, end = begin + p.part_len < p.vocab ? begin + p.part_len : p.vocab;
  auto count = [&](uint32_t bits) {
    const uint32_t k = place_of<T>(bits);
    if (k != 0xffffffffu) atomicAdd(&words[k >> 1], 1u << (16 * (k & 1)));
  };
  const bool vec = ((uintptr_t)(x + begin) & 15u) == 0;
  const int whole = vec && end > begin ? (end - begin) >> 3 : 0;
  constexpr int kAhead = 4;
  for (int c0 = t; c0 < whole; c0 += kAhead * kCountThreads) {
    u32x4 v[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) v[a] = ld16(x + begin + 8 * (c0 + a * kCountThreads < whole ? c0 + a * kCountThreads : c0));
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
  for (int i = begin + 8 * whole + t; i < end; i += kCountThreads) count(x[i]);
  __syncthreads();
  // a wave per run of 1024 values = 2 KB
  uint16_t* out = p.counts + ((long)row * p.parts + part) * 65536;
  for (int r = t >> 6; r < kRuns; r += kCountThreads / kWave) {
    const int at = r * 128 + (t & 63);
    const u32x4 a = lds[at], b = lds[at + 64];
    const unsigned long long in_a = __ballot((a.x | a.y | a.z | a.w) != 0), in_b = __ballot((b.x | b.y | b.z | b.w) != 0);
    if (in_a | in_b) {
      *(u32x4*)(out + 8 * at) = a;
      *(u32x4*)(out + 8 * at + 512) = b;
      const u32x4 f = in_a ? a : b;
      const int j = f.x ? 0 : f.y ? 1 : f.z ? 2 : 3;
      const uint32_t mine = (uint32_t)(8 * at + (in_a ? 0 : 512) + 2 * j + ((f[j] & 0xffffu) ? 0 : 1));
      if ((t & 63) == __ffsll((long long)(in_a ? in_a : in_b)) - 1) {
        atomicOr(&mask_s, 1ull << r);
        atomicMin(&first_s, mine);
      }
    }
  }
  __syncthreads();
  if (t == 0) {
    p.runs[(long)row * p.parts + part] = mask_s;
    p.first[(long)row * p.parts + part] = first_s;
  }
}

// Inclusive sums over a wave, always in the same order: rows of 16 lanes by shifts, then the last lane of one to the rows behind it, in the vector ALU.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t n) { return n + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)n, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double w) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, w);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return w + __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
template <typename V>
__device__ __forceinline__ V wave_scan(V x) {
  x = dpp_add<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // row_bcast 15: rows 1, 3
  return dpp_add<0x143, 0xc>(x);  // row_bcast 31: rows 2, 3
}

// The row's values are looked at in segments of 64: first every segment's sums, by a thread each, then, a wave and a lane per value, the few segments in
// which something ends. Neighbouring values of a segment lie equally far apart, so their weights are a geometric series: a thread takes an exponential at every 16th
// and multiplies on (15 products of 2^-53 and as many of the quotient's own rounding: 4e-15). An exponential per value and sums across lanes took 26 us for a row of
// 32000 fp16 logits, which have 36 runs.
template <typename T>
__global__ void __launch_bounds__(kCountThreads) sample_pick_kernel(const SampleParams p) {
  constexpr int kWaves = kCountThreads / kWave, kSegs = 16;  // segments of a run
  __shared__ uint32_t seg_n[kRuns * kSegs], seg_m[kRuns * kSegs];  // tokens (then: those in front); tokens of min_p's weight
  __shared__ double seg_w[kRuns * kSegs];
  __shared__ uint32_t held[kRuns * kSegs * 33];  // the row's counts, two in a word; segments a word further apart than they are long
  __shared__ int large_s;                        // a count that does not fit: the row's are then taken from memory
  __shared__ unsigned long long masks[kMostParts];
  __shared__ int list[kRuns];
  __shared__ uint32_t wave_n[kWaves], place_s, rank_s;
  __shared__ double wave_w[kWaves];
  __shared__ int part_s;
  __shared__ float share_s;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, row = blockIdx.x;
  const uint16_t* counts = p.counts + (long)row * p.parts * 65536;
  const int parts = p.parts;
  unsigned long long all_runs = 0;
  uint32_t top = 0xffffffffu;
  for (int i = 0; i < parts; ++i) {
    const unsigned long long m = p.runs[(long)row * parts + i];
    const uint32_t f = p.first[(long)row * parts + i];
    all_runs |= m;
    top = f < top ? f : top;
    if (t == i) masks[i] = m;
  }
  if (all_runs == 0) {  // nothing above -inf
    if (t == 0) {
      p.token[row] = 0;
      if (p.share) p.share[row] = 0.f;
    }
    return;
  }
  const int n_runs = __popcll(all_runs);
  if (t == 0) large_s = 0;
  if (t < kRuns && (all_runs >> t & 1ull)) list[__popcll(all_runs & ((1ull << t) - 1ull))] = t;
  __syncthreads();
  const double most = (double)T::one((uint16_t)bits_of(top));
  const float temperature = p.temperature ? p.temperature[row] : p.temperature1;
  const int top_k = p.top_k ? p.top_k[row] : p.top_k1;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p1;
  const float min_p = p.min_p ? p.min_p[row] : p.min_p1;
  const float u = p.u[row];
  const bool greedy = !(temperature > 0.f);
  const double cold = 1.0 / (double)temperature;
  // (counts are read whether their part has the run or not, so that no load waits for another: what a part has not written does not count)
  constexpr int kAhead = 4;
  auto weight_of = [&](uint32_t place) -> double {
    if (place == top) return 1.0;
    if (greedy || most == INFINITY) return 0.0;
    return exp(((double)T::one((uint16_t)bits_of(place)) - most) * cold);
  };
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
        uint32_t* to = held + (c >> 3) * 33 + (c & 7) * 4;
        uint32_t high = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          to[j] = n[k][2 * j] | n[k][2 * j + 1] << 16;
          high |= n[k][2 * j] | n[k][2 * j + 1];
        }
        if (high >> 16) large_s = 1;
      }
    }
  };
  if (parts == 1) add_up(std::integral_constant<int, 1>()); else if (parts == 2) add_up(std::integral_constant<int, 2>());
  else if (parts <= 4) add_up(std::integral_constant<int, 4>()); else add_up(std::integral_constant<int, 8>());
  __syncthreads();
  const bool large = large_s;
  const int n_seg = n_runs * kSegs;
  if (t < n_seg) {
    const uint32_t place0 = list[t / kSegs] * 1024 + (t % kSegs) * 64;
    const double l0 = (double)T::one((uint16_t)bits_of(place0)), step = ((double)T::one((uint16_t)bits_of(place0 + 1)) - l0);
    const bool flat = greedy || most == INFINITY || !(fabs(l0) < INFINITY);
    const double ratio = flat ? 0.0 : exp(step * cold);
    uint32_t n = 0, m = 0, n_top = 0;
    double w[4], sum[4] = {};
    // (a series that begins in front of the largest logit only has to be finite there: what lies there is not counted, and the largest has its weight of 1 apart. Where
    // the bound on its beginning counts, what follows the largest weighs less than e^-40 of it.)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      w[q] = flat || place0 + 16 * q + 15 < top ? 0.0 : exp(fmin(((double)T::one((uint16_t)bits_of(place0 + 16 * q)) - most) * cold, 600.0));
    auto add_one = [&](int q, int j, uint32_t c) {
      const uint32_t rest = place0 + j == top ? 0u : c;
      n += c;
      n_top += c - rest;
      if (min_p > 0.f) m += w[q] < (double)min_p ? 0u : rest;
      sum[q] += (double)rest * w[q];
      w[q] *= ratio;
    };
    if (!large) {
      const uint32_t* at = held + t * 33;
#pragma unroll 2
      for (int j = 0; j < 8; ++j) {
        uint32_t c[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) c[q] = at[8 * q + j];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          add_one(q, 16 * q + 2 * j, c[q] & 0xffffu);
          add_one(q, 16 * q + 2 * j + 1, c[q] >> 16);
        }
      }
    } else {
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) add_one(q, 16 * q + j, count_at(place0 + 16 * q + j));
    }
    m = min_p > 0.f ? m + n_top : n;
    sum[0] += (double)n_top;
    seg_n[t] = n;
    seg_m[t] = m;
    seg_w[t] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }
  __syncthreads();
  // what is in front of each
  const uint32_t my_n = t < n_seg ? seg_n[t] : 0u;
  const double my_w = t < n_seg ? seg_w[t] : 0.0;
  uint32_t my_m = t < n_seg ? seg_m[t] : 0u;
  const uint32_t in_n = wave_scan(my_n);
  const double in_w = wave_scan(my_w);
  for (int off = 32; off; off >>= 1) my_m += __shfl_xor(my_m, off);
  __syncthreads();
  if (lane == 63) { wave_n[wave] = in_n; wave_w[wave] = in_w; seg_m[wave] = my_m; }
  __syncthreads();
  uint32_t n_all = 0, m_all = 0, before_n = 0;
  double before_w = 0.0, sum_w = 0.0;
  for (int i = 0; i < kWaves; ++i) {
    if (i == wave) { before_n = n_all; before_w = sum_w; }
    n_all += wave_n[i];
    sum_w += wave_w[i];
    m_all += seg_m[i];
  }
  {
    const uint32_t a = __shfl_up(in_n, 1);
    const double b = __shfl_up(in_w, 1);
    if (t < n_seg) {
      seg_n[t] = before_n + (lane ? a : 0u);
      seg_w[t] = before_w + (lane ? b : 0.0);
    }
  }
  __syncthreads();
  if (wave == 0) {
    // one segment: this lane's value, how many tokens have it, its weight; tokens and weight up to and with it
    struct Seg { uint32_t place, n, to_n; double one, to_w; };
    auto segment = [&](int s) {
      Seg g;
      g.place = list[s / kSegs] * 1024 + (s % kSegs) * 64 + lane;
      g.n = large ? count_at(g.place) : held[s * 33 + (lane >> 1)] >> (16 * (lane & 1)) & 0xffffu;
      g.one = g.n ? weight_of(g.place) : 0.0;
      g.to_n = seg_n[s] + wave_scan(g.n);
      g.to_w = seg_w[s] + wave_scan(g.n * g.one);
      return g;
    };
    // the last segment for which `in` holds of what is in front of it (it holds of a beginning of them, and of the first)
    auto last_of = [&](auto in) {
      int s = 0;
      for (int i = 0; i < n_seg; i += 64) {
        const unsigned long long b = __ballot(i + lane < n_seg && in(seg_n[i + lane < n_seg ? i + lane : 0], seg_w[i + lane < n_seg ? i + lane : 0]));
        if (!b) break;
        s = i + 63 - __clzll((long long)b);
      }
      return s;
    };
    // the weight of the first n tokens
    auto weight_of_first = [&](uint32_t n) {
      if (n >= n_all) return sum_w;
      const Seg g = segment(last_of([&](uint32_t bn, double) { return bn < n; }));
      const int l = __ffsll((long long)__ballot(g.to_n >= n)) - 1;
      return __shfl(g.to_w - (double)(g.to_n - n) * g.one, l);
    };
    uint32_t kept = greedy ? 1u : n_all;
    if (top_k > 0 && (uint32_t)top_k < kept) kept = (uint32_t)top_k;
    if (top_p < 1.f) {
      const double limit = (double)top_p * weight_of_first(kept);
      const Seg g = segment(last_of([&](uint32_t, double bw) { return bw < limit; }));
      const unsigned long long reached = __ballot(g.to_w >= limit);
      uint32_t n = __shfl(g.to_n, 63);
      if (reached) {  // of the value that reaches the limit: the tokens in front of which less lies
        const double in_front = g.to_w - g.n * g.one;
        const double some = g.one > 0 ? ceil((limit - in_front) / g.one) : 0.0;
        const uint32_t mine = g.to_n - g.n + (some < 0 ? 0u : some < (double)g.n ? (uint32_t)some : g.n);
        n = __shfl(mine, __ffsll((long long)reached) - 1);
      }
      if (n < kept) kept = n;
    }
    if (m_all < kept) kept = m_all;
    if (kept < 1) kept = 1;
    const double all = weight_of_first(kept);
    const double target = (u > 0.f ? (double)u : 0.0) * all;
    const Seg g = segment(last_of([&](uint32_t bn, double bw) { return bn < kept && bw <= target; }));
    const unsigned long long over = __ballot(g.n && (g.to_w > target || g.to_n >= kept));
    // (no lane: the segment's sum, added in another order, stops short of the target by a rounding: its last value)
    const unsigned long long there = over ? over & (0ull - over) : 0ull;
    const unsigned long long some = __ballot(g.n != 0);
    const int l = there ? __ffsll((long long)there) - 1 : 63 - __clzll((long long)some);
    const uint32_t first_n = g.to_n - g.n, here = g.n < kept - first_n ? g.n : kept - first_n;
    const double r = g.one > 0 ? floor((target - (g.to_w - g.n * g.one)) / g.one) : 0.0;
    const uint32_t rank = r < 0 ? 0u : r < (double)here ? (uint32_t)r : here - 1u;
    const uint32_t place = (uint32_t)__shfl((int)g.place, l);
    uint32_t left = (uint32_t)__shfl((int)rank, l);
    const double one = __shfl(g.one, l);
    // the part that holds that token
    uint32_t c = 0;
    if (lane < parts && (masks[lane < parts ? lane : 0] >> (place >> 10) & 1ull)) c = counts[(long)lane * 65536 + place];
    const uint32_t to = wave_scan(c);
    const unsigned long long has = __ballot(to > left);
    const int part = has ? __ffsll((long long)has) - 1 : 0;
    left -= __shfl(to - c, part);
    if (lane == 0) {
      place_s = place;
      rank_s = left;
      part_s = part;
      share_s = (float)(one / all);
    }
  }
  __syncthreads();
  // the rank-th token of that value in its part: 8 in a row per lane and step, which ones have it kept in a bit each
  const uint32_t bits = bits_of(place_s), or_bits = bits ? bits : 0x8000u;
  uint32_t rank = rank_s;
  const int part = part_s;
  const uint16_t* x = p.logits + (long)row * p.row_stride;
  const int begin = part * p.part_len, end = begin + p.part_len < p.vocab ? begin + p.part_len : p.vocab;
  const int per = ((p.part_len >> 3) + kWaves - 1) / kWaves * 8;  // tokens of a wave, at most 4096
  const int wb = begin + wave * per, we = wb + per < end ? wb + per : end;
  const bool vec = ((uintptr_t)(x + wb) & 15u) == 0;
  unsigned long long found = 0;
#pragma unroll 4
  for (int s = 0; s < 8; ++s) {
    const int i = wb + 512 * s + 8 * lane;
    if (i >= we) break;
    uint32_t m = 0;
    if (i + 8 <= we && vec) {
      const u32x4 v = ld16(x + i);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        m |= ((v[j] & 0xffffu) == bits || (v[j] & 0xffffu) == or_bits ? 1u : 0u) << (2 * j) | (v[j] >> 16 == bits || v[j] >> 16 == or_bits ? 2u : 0u) << (2 * j);
    } else {
      for (int j = 0; j < 8; ++j)
        if (i + j < we) m |= (x[i + j] == bits || x[i + j] == or_bits ? 1u : 0u) << j;
    }
    found |= (unsigned long long)m << (8 * s);
  }
  uint32_t mine = __popcll(found);
  for (int off = 32; off; off >>= 1) mine += __shfl_xor(mine, off);
  if (lane == 0) wave_n[wave] = mine;
  __syncthreads();
  for (int w = 0; w < wave; ++w) rank -= wave_n[w];  // (below zero: it wraps, and is no token of this wave)
  if (rank >= wave_n[wave]) return;
  for (int s = 0; s < 8; ++s) {
    const uint32_t here = (uint32_t)(found >> (8 * s)) & 0xffu;
    const uint32_t n = __popc(here), to = wave_scan(n), total = __shfl(to, 63);
    if (rank < total) {
      if (rank >= to - n && rank < to) {
        uint32_t left = rank - (to - n), b = here;
        while (left--) b &= b - 1;
        p.token[row] = wb + 512 * s + 8 * lane + __ffs((int)b) - 1;
        if (p.share) p.share[row] = share_s;
      }
      return;
    }
    rank -= total;
  }
}

struct SamplePlan { int parts, part_len; };
static SamplePlan sample_plan(int rows, int vocab) {
  int parts = (vocab + kMostPart - 1) / kMostPart;
  const int want = (256 + rows - 1) / rows, most = (vocab + 16383) / 16384;
  const int more = want < most ? want : most;
  parts = parts > more ? parts : more;
  parts = parts < kMostParts ? parts : kMostParts;
  SamplePlan r;
  r.part_len = ((vocab + parts - 1) / parts + 7) / 8 * 8;
  r.parts = (vocab + r.part_len - 1) / r.part_len;
  return r;
}

}  // namespace mui

using namespace mui;

extern "C" size_t mui_sample_filtered_workspace_bytes(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  const SamplePlan plan = sample_plan(rows, vocab);
  return (size_t)rows * plan.parts * (131072 + 16);
}

extern "C" int mui_sample_filtered(mui_stream_t stream, const mui_sample_filtered_args_t* args) {
  MUI_CHECK_ARG(args);
  const mui_sample_filtered_args_t& a = *args;
  MUI_CHECK_ARG(a.logits && a.random_numbers && a.out_token && a.workspace && a.rows > 0 && a.vocab > 0 && a.row_stride >= a.vocab);
  if (a.dtype != MUI_DTYPE_F16 && a.dtype != MUI_DTYPE_BF16) return MUI_ERR_INVALID_ARG;
  if (a.rows > 65535 || a.vocab > kMostParts * kMostPart) return MUI_ERR_UNSUPPORTED;
  if ((uintptr_t)a.workspace & 15u) return MUI_ERR_ALIGNMENT;
  if (a.workspace_bytes < mui_sample_filtered_workspace_bytes(a.rows, a.vocab)) return MUI_ERR_INVALID_ARG;
  const SamplePlan plan = sample_plan(a.rows, a.vocab);
  SampleParams p = {};
  p.logits = (const uint16_t*)a.logits; p.row_stride = a.row_stride; p.rows = a.rows; p.vocab = a.vocab; p.parts = plan.parts; p.part_len = plan.part_len;
  p.u = a.random_numbers;
  p.temperature = a.temperatures; p.top_k = a.top_ks; p.top_p = a.top_ps; p.min_p = a.min_ps;
  p.temperature1 = a.temperature; p.top_k1 = a.top_k; p.top_p1 = a.top_p; p.min_p1 = a.min_p;
  p.counts = (uint16_t*)a.workspace;
  p.runs = (unsigned long long*)((char*)a.workspace + (size_t)a.rows * plan.parts * 131072);
  p.first = (uint32_t*)(p.runs + (size_t)a.rows * plan.parts);
  p.token = a.out_token; p.share = a.out_probability;
  hipStream_t s = (hipStream_t)stream;
  if (a.dtype == MUI_DTYPE_F16) {
    hipLaunchKernelGGL((sample_count_kernel<F16>), dim3(plan.parts, a.rows), dim3(kCountThreads), 0, s, p);
    hipLaunchKernelGGL((sample_pick_kernel<F16>), dim3(a.rows), dim3(kCountThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL((sample_count_kernel<BF16>), dim3(plan.parts, a.rows), dim3(kCountThreads), 0, s, p);
    hipLaunchKernelGGL((sample_pick_kernel<BF16>), dim3(a.rows), dim3(kCountThreads), 0, s, p);
  }
  return launch_status();
}
