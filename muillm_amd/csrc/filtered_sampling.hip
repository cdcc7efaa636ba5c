// The next token of each row from a given uniform number: temperature, top-k, top-p, min-p.
//
// w_i = exp((l_i - max l) / T) in 64 bits. In order of falling logits (equal ones by rising index) every filter keeps a beginning of the row, so the
// kept tokens are the first n, and the token drawn is the first whose cumulative weight exceeds u times theirs. A 16-bit logit has 65536 values:
// counting how often each occurs sorts the row, and what has to be computed in 64 bits is one exponential per value that occurs, not per token.
// Counts are whole numbers and the weights of a row are added in one order, so results do not depend on what arrives when.
//
// First kernel: workgroups count parts of a row in LDS (16 bits a value, 128 KB) and write the runs of 1024 values that occur. Second: a workgroup per row adds
// the parts' counts up from the largest value down, finds the value and which of the tokens that have it is drawn, and looks for that token in its part.
#include "common.cuh"

namespace mui {

constexpr int kCountThreads = 1024;
constexpr int kRuns = 64;              // runs of 1024 values
constexpr int kMostPart = 65528;       // tokens of a part: their counts fit 16 bits

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

template <typename T>
__global__ void __launch_bounds__(kCountThreads) sample_count_kernel(const SampleParams p) {
  __shared__ u32x4 lds[8192];
  __shared__ unsigned long long mask_s;
  uint32_t* words = (uint32_t*)lds;
  const int t = threadIdx.x, part = blockIdx.x, row = blockIdx.y;
  for (int i = t; i < 8192; i += kCountThreads) lds[i] = u32x4{0, 0, 0, 0};
  if (t == 0) mask_s = 0;
  __syncthreads();
  const uint16_t* x = p.logits + (long)row * p.row_stride;
  const int begin = part * p.part_len, end = begin + p.part_len < p.vocab ? begin + p.part_len : p.vocab;
  auto count = [&](uint32_t bits) {
    const uint32_t k = place_of<T>(bits);
    if (k != 0xffffffffu) atomicAdd(&words[k >> 1], 1u << (16 * (k & 1)));
  };
  const bool vec = ((uintptr_t)(x + begin) & 15u) == 0;
  const int whole = vec && end > begin ? (end - begin) >> 3 : 0;
  for (int c = t; c < whole; c += kCountThreads) {
    const u32x4 v = ld16(x + begin + 8 * c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      count(v[j] & 0xffffu);
      count(v[j] >> 16);
    }
  }
  for (int i = begin + 8 * whole + t; i < end; i += kCountThreads) count(x[i]);
  __syncthreads();
  // a wave per run of 1024 values = 2 KB
  uint16_t* out = p.counts + ((long)row * p.parts + part) * 65536;
  for (int r = t >> 6; r < kRuns; r += kCountThreads / kWave) {
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

// exclusive sums over the workgroup in one fixed order; totals in `n_all`, `w_all`
__device__ __forceinline__ void scan_all(uint32_t n, double w, uint32_t& n_before, double& w_before, uint32_t& n_all, double& w_all, uint32_t* sn, double* sw) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t an = n;
  double aw = w;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t on = __shfl_up(an, off);
    const double ow = __shfl_up(aw, off);
    if (lane >= off) { an += on; aw += ow; }
  }
  if (lane == 63) { sn[wave] = an; sw[wave] = aw; }
  __syncthreads();
  uint32_t bn = 0;
  double bw = 0;
  n_all = 0;
  w_all = 0;
  for (int i = 0; i < kCountThreads / kWave; ++i) {
    if (i == wave) { bn = n_all; bw = w_all; }
    n_all += sn[i];
    w_all += sw[i];
  }
  const uint32_t en = __shfl_up(an, 1);
  const double ew = __shfl_up(aw, 1);
  n_before = bn + (lane ? en : 0);
  w_before = bw + (lane ? ew : 0);
}

template <typename T>
__global__ void __launch_bounds__(kCountThreads) sample_pick_kernel(const SampleParams p) {
  __shared__ uint32_t sn[16];
  __shared__ double sw[16];
  __shared__ int list[kRuns];
  __shared__ int n_list, who;
  __shared__ uint32_t n_kept_s, first_place, rank_s, place_s;
  __shared__ double weight_s, pick_w;
  __shared__ uint32_t wave_n[16];
  const int t = threadIdx.x, row = blockIdx.x;
  const uint16_t* counts = p.counts + (long)row * p.parts * 65536;
  const unsigned long long* runs = p.runs + (long)row * p.parts;
  if (t == 0) {
    unsigned long long m = 0;
    for (int i = 0; i < p.parts; ++i) m |= runs[i];
    int n = 0;
    while (m) {
      list[n++] = __ffsll((long long)m) - 1;
      m &= m - 1;
    }
    n_list = n;
    who = -1;
    first_place = 0xffffffffu;
    n_kept_s = 0;
    rank_s = 0;
    pick_w = 1.0;
  }
  __syncthreads();
  const int n_runs = n_list;
  if (n_runs == 0) {  // nothing above -inf
    if (t == 0) {
      p.token[row] = 0;
      if (p.share) p.share[row] = 0.f;
    }
    return;
  }
  // this thread's values: n_runs places in a row of the listed runs put together
  auto place_at = [&](int j) { const int i = t * n_runs + j; return (uint32_t)(list[i >> 10] * 1024 + (i & 1023)); };
  auto count_at = [&](uint32_t place) {
    uint32_t n = 0;
    for (int i = 0; i < p.parts; ++i)
      if (runs[i] >> (place >> 10) & 1ull) n += counts[(long)i * 65536 + place];
    return n;
  };
  for (int j = 0; j < n_runs; ++j) {
    const uint32_t k = place_at(j);
    if (count_at(k)) { atomicMin(&first_place, k); break; }
  }
  __syncthreads();
  const uint32_t top = first_place;
  if (t == 0) place_s = top;
  const double most = (double)T::one((uint16_t)bits_of(top));
  const float temperature = p.temperature ? p.temperature[row] : p.temperature1;
  const bool greedy = !(temperature > 0.f);
  const double cold = 1.0 / (double)temperature;
  auto weight_of = [&](uint32_t place) -> double {
    if (place == top) return 1.0;
    if (greedy || most == INFINITY) return 0.0;
    return exp(((double)T::one((uint16_t)bits_of(place)) - most) * cold);
  };
  const float min_p = p.min_p ? p.min_p[row] : p.min_p1;
  uint32_t n_mine = 0, n_min = 0;
  double w_mine = 0;
  for (int j = 0; j < n_runs; ++j) {
    const uint32_t k = place_at(j), n = count_at(k);
    if (n) {
      const double w = weight_of(k);
      n_mine += n;
      w_mine += n * w;
      if (!(w < (double)min_p)) n_min += n;
    }
  }
  uint32_t n_before, n_all, m_before, m_all;
  double w_before, w_all, dummy, dummy_all;
  scan_all(n_mine, w_mine, n_before, w_before, n_all, w_all, sn, sw);
  __syncthreads();
  scan_all(n_min, 0.0, m_before, dummy, m_all, dummy_all, sn, sw);
  __syncthreads();
  // the weight of the first n tokens: by the thread whose values hold the n-th
  auto weight_of_first = [&](uint32_t n) -> double {
    if (n_before < n && n <= n_before + n_mine) {
      uint32_t left = n - n_before;
      double w = w_before;
      for (int j = 0; j < n_runs && left; ++j) {
        const uint32_t k = place_at(j), c = count_at(k);
        if (!c) continue;
        const uint32_t take = left < c ? left : c;
        w += take * weight_of(k);
        left -= take;
      }
      weight_s = w;
    }
    __syncthreads();
    const double w = weight_s;
    __syncthreads();
    return w;
  };
  const int top_k = p.top_k ? p.top_k[row] : p.top_k1;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p1;
  uint32_t kept = greedy ? 1u : n_all;
  if (top_k > 0 && (uint32_t)top_k < kept) kept = (uint32_t)top_k;
  // the last thread with kept values in front of which less than `limit` lies
  auto last_below = [&](double limit, bool or_equal) {
    if (n_mine && n_before < kept && (w_before < limit || (or_equal && w_before == limit))) atomicMax(&who, t);
    __syncthreads();
    const int w = who;
    __syncthreads();
    if (t == 0) who = -1;
    return w;
  };
  if (top_p < 1.f) {
    const double limit = (double)top_p * weight_of_first(kept);
    if (t == last_below(limit, false)) {  // tokens in front of which less than the limit lies
      uint32_t n = n_before;
      double w = w_before;
      for (int j = 0; j < n_runs && w < limit; ++j) {
        const uint32_t k = place_at(j), c = count_at(k);
        if (!c) continue;
        const double one = weight_of(k);
        const double most_n = one > 0 ? ceil((limit - w) / one) : (double)c;
        n += most_n < (double)c ? (uint32_t)most_n : c;
        w += c * one;
      }
      n_kept_s = n;
    }
    __syncthreads();
    if (n_kept_s < kept) kept = n_kept_s;
    __syncthreads();
  }
  if (m_all < kept) kept = m_all;
  if (kept < 1) kept = 1;
  const double all = weight_of_first(kept);
  const float u = p.u[row];
  const double target = (u > 0.f ? (double)u : 0.0) * all;
  if (t == last_below(target, true)) {
    uint32_t n = n_before, place = top, rank = 0;
    double w = w_before, picked = 1.0;
    for (int j = 0; j < n_runs; ++j) {
      const uint32_t k = place_at(j), c = count_at(k);
      if (!c || n >= kept) continue;
      const double one = weight_of(k);
      const uint32_t here = c < kept - n ? c : kept - n;  // of this value, kept
      place = k;
      picked = one;
      if (target < w + here * one || n + here >= kept) {
        const double r = one > 0 ? floor((target - w) / one) : 0.0;
        rank = r < (double)here ? (uint32_t)(r < 0 ? 0 : r) : here - 1;
        break;
      }
      rank = here - 1;
      n += here;
      w += here * one;
    }
    place_s = place;
    rank_s = rank;
    pick_w = picked;
  }
  __syncthreads();
  // the part that holds the rank-th token of that value, and the token
  const uint32_t place = place_s;
  uint32_t rank = rank_s;
  int part = 0;
  for (; part < p.parts - 1; ++part) {
    const uint32_t c = runs[part] >> (place >> 10) & 1ull ? counts[(long)part * 65536 + place] : 0;
    if (rank < c) break;
    rank -= c;
  }
  const uint16_t* x = p.logits + (long)row * p.row_stride;
  const int begin = part * p.part_len, end = begin + p.part_len < p.vocab ? begin + p.part_len : p.vocab;
  const int lane = t & 63, wave = t >> 6;
  const int per = ((p.part_len >> 3) + 15) / 16 * 8;  // tokens of a wave
  const int wb = begin + wave * per, we = wb + per < end ? wb + per : end;
  const bool vec = ((uintptr_t)(x + wb) & 15u) == 0;
  auto matches = [&](int i) -> uint32_t {  // of the 8 tokens from i on, a bit each
    uint32_t m = 0;
    if (i + 8 <= we && vec) {
      const u32x4 v = ld16(x + i);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        m |= (place_of<T>(v[j] & 0xffffu) == place ? 1u : 0u) << (2 * j) | (place_of<T>(v[j] >> 16) == place ? 1u : 0u) << (2 * j + 1);
    } else {
      for (int j = 0; j < 8; ++j)
        if (i + j < we) m |= (place_of<T>(x[i + j]) == place ? 1u : 0u) << j;
    }
    return m;
  };
  uint32_t mine = 0;
  for (int i = wb + 8 * lane; i < we; i += 512) mine += __popc(matches(i));
  for (int off = 32; off; off >>= 1) mine += __shfl_xor(mine, off);
  if (lane == 0) wave_n[wave] = mine;
  __syncthreads();
  int w = 0;
  for (; w < 15; ++w) {
    if (rank < wave_n[w]) break;
    rank -= wave_n[w];
  }
  if (wave != w) return;
  for (int i0 = wb; i0 < we; i0 += 512) {
    const int i = i0 + 8 * lane;
    const uint32_t m = i < we ? matches(i) : 0u;
    uint32_t n = __popc(m), before = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t o = __shfl_up(before, off);
      if (lane >= off) before += o;
    }
    const uint32_t total = __shfl(before, 63);
    before -= n;
    if (rank < total) {
      if (rank >= before && rank < before + n) {
        uint32_t left = rank - before, bits = m;
        while (left--) bits &= bits - 1;
        p.token[row] = i + __ffs((int)bits) - 1;
        if (p.share) p.share[row] = (float)(pick_w / all);
      }
      return;
    }
    rank -= total;
  }
}

struct SamplePlan { int parts, part_len; };
static SamplePlan sample_plan(int rows, int vocab) {
  int parts = (vocab + kMostPart - 1) / kMostPart;
  const int want = (256 + rows - 1) / rows, most = (vocab + 8191) / 8192;
  const int more = want < most ? want : most;
  parts = parts > more ? parts : more;
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
  return (size_t)rows * plan.parts * (131072 + 8);
}

extern "C" int mui_sample_filtered(mui_stream_t stream, int dtype, const void* logits, long row_stride, int rows, int vocab, const float* random_numbers,
                                   const float* temperatures, float temperature, const int32_t* top_ks, int top_k, const float* top_ps, float top_p,
                                   const float* min_ps, float min_p, int64_t* out_token, float* out_probability, void* workspace, size_t workspace_bytes) {
  MUI_CHECK_ARG(logits && random_numbers && out_token && workspace && rows > 0 && vocab > 0 && row_stride >= vocab);
  if (dtype != MUI_DTYPE_F16 && dtype != MUI_DTYPE_BF16) return MUI_ERR_INVALID_ARG;
  if (rows > 65535 || vocab > (1 << 30)) return MUI_ERR_UNSUPPORTED;
  if ((uintptr_t)workspace & 15u) return MUI_ERR_ALIGNMENT;
  if (workspace_bytes < mui_sample_filtered_workspace_bytes(rows, vocab)) return MUI_ERR_INVALID_ARG;
  const SamplePlan plan = sample_plan(rows, vocab);
  SampleParams p = {};
  p.logits = (const uint16_t*)logits; p.row_stride = row_stride; p.rows = rows; p.vocab = vocab; p.parts = plan.parts; p.part_len = plan.part_len;
  p.u = random_numbers;
  p.temperature = temperatures; p.top_k = top_ks; p.top_p = top_ps; p.min_p = min_ps;
  p.temperature1 = temperature; p.top_k1 = top_k; p.top_p1 = top_p; p.min_p1 = min_p;
  p.counts = (uint16_t*)workspace;
  p.runs = (unsigned long long*)((char*)workspace + (size_t)rows * plan.parts * 131072);
  p.token = out_token; p.share = out_probability;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MUI_DTYPE_F16) {
    hipLaunchKernelGGL((sample_count_kernel<F16>), dim3(plan.parts, rows), dim3(kCountThreads), 0, s, p);
    hipLaunchKernelGGL((sample_pick_kernel<F16>), dim3(rows), dim3(kCountThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL((sample_count_kernel<BF16>), dim3(plan.parts, rows), dim3(kCountThreads), 0, s, p);
    hipLaunchKernelGGL((sample_pick_kernel<BF16>), dim3(rows), dim3(kCountThreads), 0, s, p);
  }
  return launch_status();
}
