// Queries and keys rotated by their positions, keys and values appended to a paged e4m3 cache (paged.cuh has its layout).
//
// Rotation of the first `rot` dimensions, in 32 bits: a' = a c - b s, b' = b c + a s for the pairs (i, i + rot / 2) or (2 i, 2 i + 1), c and s the
// cosine and sine (times rope_scale) of position * inv_freq[i], the angle's whole turns dropped in 64 bits. Queries are rounded once, to their own
// type; keys and values once, to codes x / scale. The scale of a page and head is the smallest power of two with which the largest new
// value fits 448, but not below what stands there for the page's earlier tokens; where it grows their codes follow.
//
// A thread works on units of two chunks of 8 dimensions, which hold their pairs whole: pairs of halves lie rot / 2 apart, and so do the chunks; of interleaved pairs and of
// dimensions that do not turn unit u has chunks u and u + half of them, so that neighbours' loads are neighbours too.
#include "paged.cuh"

namespace mui {

struct AppendParams {
  const uint16_t* q; long q_tok, q_head;
  const uint16_t* k; long k_tok, k_head;
  const uint16_t* v; long v_tok, v_head;
  uint8_t* kp; uint8_t* vp;
  float* ks; float* vs;
  const int64_t* positions;
  const double* inv_freq;
  uint16_t* q_out;
  PagedTable t;
  float rope_scale;
  int rot, interleaved, heads, kv_heads, dim;
  int q_blocks, at_once;  // at_once: KV heads of a workgroup
};

// A unit: first dimensions of its chunks, and which of them turn.
struct Unit { int d0, d1; bool turns0, turns1; };
__device__ __forceinline__ Unit unit_of(const AppendParams& p, int u) {
  const int units = p.dim >> 4, turned = p.rot >> 4;
  if (p.interleaved) return {8 * u, 8 * (u + units), 8 * u < p.rot, 8 * (u + units) < p.rot};
  if (u < turned) return {8 * u, 8 * u + (p.rot >> 1), true, true};
  return {p.rot + 8 * (u - turned), p.rot + 8 * (u - turned + units - turned), false, false};
}

// The angles of its eight pairs: halves 8 u .. 8 u + 7; interleaved four of either chunk. Those of a chunk that does not turn are not used.
__device__ __forceinline__ void unit_angles(const AppendParams& p, const Unit& n, double pos, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!(i < 4 ? n.turns0 : n.turns1)) continue;
    const int pair = !p.interleaved ? n.d0 + i : i < 4 ? (n.d0 >> 1) + i : (n.d1 >> 1) + i - 4;
    // the turns left over in 32 bits, and what that rounding took from them (it is 3 of the last places of a sine: enough to move a code in a few thousand)
    double a = pos * p.inv_freq[pair] * 0.15915494309189533576888376337251;
    a = 2.0 * (a - rint(a));
    const float f = (float)a, r = 3.14159265f * (float)(a - (double)f);
    float cf, sf;
    sincospif(f, &sf, &cf);
    c[i] = p.rope_scale * fmaf(-r, sf, cf);
    s[i] = p.rope_scale * fmaf(r, cf, sf);
  }
}

// x: the values of the two chunks
__device__ __forceinline__ void unit_turn(const AppendParams& p, const Unit& n, const float (&c)[8], const float (&s)[8], float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!(i < 4 ? n.turns0 : n.turns1)) continue;
    if (p.interleaved) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * c[i] - b * s[i];
      x[2 * i + 1] = b * c[i] + a * s[i];
    } else {
      const float a = x[i], b = x[i + 8];
      x[i] = a * c[i] - b * s[i];
      x[i + 8] = b * c[i] + a * s[i];
    }
  }
}

template <typename T>
__device__ __forceinline__ void unpack_unit(const u32x4 v, const u32x4 w, float (&x)[16]) {
  float a[8], b[8];
  unpack8<T>(v, a);
  unpack8<T>(w, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) { x[i] = a[i]; x[8 + i] = b[i]; }
}
template <typename T>
__device__ __forceinline__ void load_unit(const uint16_t* row, int d0, int d1, float (&x)[16]) {
  unpack_unit<T>(ld16(row + d0), ld16(row + d1), x);
}
template <typename T>
__device__ __forceinline__ void store_unit(uint16_t* row, int d0, int d1, const float (&x)[16]) {
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { a[i] = x[i]; b[i] = x[8 + i]; }
  *(u32x4*)(row + d0) = pack8<T>(a);
  *(u32x4*)(row + d1) = pack8<T>(b);
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// byte of a page and head that holds dimension d of token `at` of the page
__device__ __forceinline__ int k_at(int dim, int at, int d) { return (at >> 6) * 64 * dim + (d >> 6) * 4096 + (at & 63) * 64 + (d & 63); }
__device__ __forceinline__ int v_at(int dim, int at, int d) {
  const int r = at & 63;
  return (at >> 6) * 64 * dim + d * 64 + ((r >> 2) & 3) * 16 + (r >> 4) * 4 + (r & 3);
}

// The codes of the first `old` tokens of a page and head times `ratio`, by `n` threads. Sixteen bytes at a time; of values only the bytes of those tokens.
__device__ __forceinline__ void move_codes(uint8_t* base, int dim, int old, float ratio, bool values, int tid, int n) {
  const int chunks = ((old + 63) >> 6) * 4 * dim;  // of the tiles that hold them
  for (int c = tid; c < chunks; c += n) {
    const int tile = c / (4 * dim), in = c - tile * 4 * dim;
    const int left = old - tile * 64;  // > 0
    u32x4* at = (u32x4*)(base + (long)c * 16);
    if (!values) {
      if (((in >> 2) & 63) >= left) continue;
      u32x4 w = *at;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = e4m3x4_times(w[j], ratio);
      *at = w;
    } else {
      const int g = in & 3;
      if (4 * g >= left) continue;
      u32x4 w = *at;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int mine = left - (16 * t + 4 * g);
        const uint32_t m = mine >= 4 ? 0xffffffffu : (mine <= 0 ? 0u : (1u << (8 * mine)) - 1u);
        w[t] = (w[t] & ~m) | (e4m3x4_times(w[t], ratio) & m);
      }
      *at = w;
    }
  }
}

// ---------------------------------------------------------------------------------------
// One new token per request: dim / 16 lanes work on one head of one token (queries, keys, values), with 16 of its values each, so a head's largest is found by shuffles and
// nothing meets in LDS. The time is that of three loads that wait for one another (a request's length, its page, the page's scale): 4.5 us for one request of 32 query and 8 KV heads
// of 128 dimensions, 6.0 for 64 (1.4 MB). A page whose scale rises is gone over by the lanes of its head alone: 128 dimensions and 64 tokens are 64 loads of 16 bytes
// for each of 8 lanes, seldom, since a scale that has risen stays.
// ---------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) append_step_kernel(const AppendParams p) {
  const int units = p.dim >> 4;
  const int all = p.heads + 2 * p.kv_heads;
  const long item = (long)blockIdx.x * 256 + threadIdx.x;
  const int u = (int)(item % units);
  const long unit_row = item / units;
  const int b = (int)(unit_row / all);
  int h = (int)(unit_row - (long)b * all);
  if (b >= p.t.n_requests) return;  // (whole groups of `units` lanes)
  const PagedSpan sp = paged_span(p.t, b);
  if (sp.count < 1) return;
  const int kind = h < p.heads ? 0 : (h < p.heads + p.kv_heads ? 1 : 2);
  h -= kind == 0 ? 0 : (kind == 1 ? p.heads : p.heads + p.kv_heads);
  const uint16_t* row = kind == 0 ? p.q + (long)sp.row0 * p.q_tok + (long)h * p.q_head
                        : kind == 1 ? p.k + (long)sp.row0 * p.k_tok + (long)h * p.k_head : p.v + (long)sp.row0 * p.v_tok + (long)h * p.v_head;
  const Unit n = unit_of(p, u);
  const int d0 = n.d0, d1 = n.d1;
  float x[16];
  load_unit<T>(row, d0, d1, x);
  if (kind != 2 && n.turns0) {  // (the second chunk turns only where the first does)
    float c[8], s[8];
    unit_angles(p, n, (double)(p.positions ? p.positions[sp.row0] : sp.start), c, s);
    unit_turn(p, n, c, s, x);
  }
  if (kind == 0) {
    store_unit<T>(p.q_out + ((long)sp.row0 * p.heads + h) * p.dim, d0, d1, x);
    return;
  }
  if (sp.start < 0 || sp.start >= sp.length) return;
  const int page = paged_page(p.t, b, (int)(sp.start >> p.t.page_shift));
  if (page < 0) return;
  const int at = (int)(sp.start & ((1L << p.t.page_shift) - 1));
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) most = fmaxf(most, finite_abs(x[i]));
  for (int off = 1; off < units; off <<= 1) most = fmaxf(most, __shfl_xor(most, off));
  const long ph = (long)page * p.kv_heads + h;
  uint8_t* base = (kind == 1 ? p.kp : p.vp) + ph * ((long)p.dim << p.t.page_shift);
  float* scale = (kind == 1 ? p.ks : p.vs) + ph;
  int e = e4m3_exponent(most);
  if (at > 0) {
    const int before = scale_exponent(*scale);
    if (e > before) {
      const int down = before - e;
      move_codes(base, p.dim, at, exp2i(down < -126 ? -126 : down), kind == 2, u, units);
      __threadfence_block();  // (a new value's byte may lie between moved ones)
    } else {
      e = before;
    }
  }
  if (u == 0) *scale = exp2i(e);
  const float inv = exp2i(-e);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = to_e4m3x4(x[4 * j] * inv, x[4 * j + 1] * inv, x[4 * j + 2] * inv, x[4 * j + 3] * inv);
  if (kind == 1) {
    *(u32x2*)(base + k_at(p.dim, at, d0)) = u32x2{w[0], w[1]};
    *(u32x2*)(base + k_at(p.dim, at, d1)) = u32x2{w[2], w[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) base[v_at(p.dim, at, (i < 8 ? d0 : d1 - 8) + i)] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}

// ---------------------------------------------------------------------------------------
// prompts: workgroups of queries, then one per page, head and kind
// ---------------------------------------------------------------------------------------
constexpr int kQueryHeads = 8;  // of a workgroup: its angles serve that many, four loads at a time

template <typename T>
__device__ __forceinline__ void append_queries(const AppendParams& p, int block) {
  const int units = p.dim >> 4, per = (int)blockDim.x / units;  // tokens of a workgroup
  const int groups = (p.heads + kQueryHeads - 1) / kQueryHeads;
  const int h0 = block % groups * kQueryHeads, h1 = h0 + kQueryHeads < p.heads ? h0 + kQueryHeads : p.heads;
  const int u = threadIdx.x % units;
  const int row = block / groups * per + threadIdx.x / units;
  if (row >= p.t.n_rows) return;
  const Unit n = unit_of(p, u);
  constexpr int kAhead = 4;
  u32x4 raw[kAhead][2];
  auto request = [&](int h) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint16_t* from = p.q + (long)row * p.q_tok + (long)(h + k < h1 ? h + k : h1 - 1) * p.q_head;
      raw[k][0] = ld16(from + n.d0);
      raw[k][1] = ld16(from + n.d1);
    }
  };
  request(h0);  // (on their way while the row's place is looked up)
  const int b = request_of(p.t, row);
  if (b >= p.t.n_requests) return;
  const PagedSpan sp = paged_span(p.t, b);
  if (row < sp.row0 || row >= sp.row0 + sp.count) return;  // behind the last request: left as it is
  float c[8], s[8];
  if (n.turns0) unit_angles(p, n, (double)(p.positions ? p.positions[row] : sp.start + (row - sp.row0)), c, s);
  for (int h = h0; h < h1; h += kAhead) {
    float x[kAhead][16];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) unpack_unit<T>(raw[k][0], raw[k][1], x[k]);
    if (h + kAhead < h1) request(h + kAhead);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (h + k >= h1) break;
      if (n.turns0) unit_turn(p, n, c, s, x[k]);
      store_unit<T>(p.q_out + ((long)row * p.heads + h + k) * p.dim, n.d0, n.d1, x[k]);
    }
  }
}

// the largest of `most` over the workgroup
__device__ __forceinline__ float block_most(float most, float* red) {
  most = wave_max(most);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
  __syncthreads();
  for (int w = 0; w < (int)blockDim.x / kWave; ++w) most = fmaxf(most, red[w]);
  return most;
}

// The new exponent of a page and head that holds `old` earlier tokens, whose codes follow where it rises.
__device__ __forceinline__ int page_exponent(const AppendParams& p, float most, uint8_t* base, float* scale, float before_s, int old, bool values) {
  int e = e4m3_exponent(most);
  if (old > 0) {
    const int before = scale_exponent(before_s);
    if (e > before) {
      const int down = before - e;
      move_codes(base, p.dim, old, exp2i(down < -126 ? -126 : down), values, threadIdx.x, blockDim.x);
      __syncthreads();  // (a new value's bytes may lie between moved ones)
    } else {
      e = before;
    }
  }
  if (threadIdx.x == 0) *scale = exp2i(e);
  return e;
}

// A page of a head is 32 IT values a thread, which it holds between finding the largest and writing the codes. Keys: units of a token, as queries. Values: 8 dimensions of four tokens
// 4 q .. 4 q + 3, whose codes are a dword of each dimension's row. Where larger pages are filled as a rule a workgroup has 1024 threads (256 tokens of 256 dimensions: 512, and IT is 4);
// few tokens in one of them are the work of 512 for that part of the page (several parts are read twice, for the largest and for the codes). us, 128 dimensions, pages of 256, the whole
// page held / parts: 64 requests' 5 new tokens 28 / 19, 100 63 / 42; 8 requests' 1000 50 / 54; 256 dimensions, 8 requests' 500 52 / 76.
// Bytes bound it: every query, key and value is read once and written once. 11500 tokens of 32 + 8 + 8 heads of 128 bf16 dimensions (213 MB) 48.8 us, 4.4 TB/s; a copy of 2 GiB reaches 4.95.
// In the same launch queries fill the time in which pages wait for their largest value.
template <typename T, int IT>
__global__ void __launch_bounds__(IT == 1 ? 1024 : 512) append_rows_kernel(const AppendParams p) {
  __shared__ float red[16];
  if ((int)blockIdx.x < p.q_blocks) {
    append_queries<T>(p, blockIdx.x);
    return;
  }
  int i = blockIdx.x - p.q_blocks;
  const int groups = (p.kv_heads + p.at_once - 1) / p.at_once;
  const bool values = i % (2 * groups) >= groups;
  const int h0 = i % groups * p.at_once, h1 = h0 + p.at_once < p.kv_heads ? h0 + p.at_once : p.kv_heads;
  i /= 2 * groups;
  const int P = 1 << p.t.page_shift, units = p.dim >> 4, threads = blockDim.x;
  // the i-th page that takes new tokens: every wave adds the requests' pages up, 64 at a time
  int b = -1;
  long slot = 0;
  for (int r0 = 0; r0 < p.t.n_requests && b < 0; r0 += kWave) {
    const int r = r0 + (threadIdx.x & 63);
    int pages = 0;
    long from = 0;
    if (r < p.t.n_requests) {
      const PagedSpan s = paged_span(p.t, r);
      from = (s.start < 0 ? 0 : s.start) >> p.t.page_shift;
      if (s.count > 0 && s.length > 0 && ((s.length - 1) >> p.t.page_shift) >= from) pages = (int)(((s.length - 1) >> p.t.page_shift) - from) + 1;
    }
    int to = pages;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(to, off);
      if ((int)(threadIdx.x & 63) >= off) to += o;
    }
    const unsigned long long in = __ballot(to > i);
    if (in) {
      const int l = __ffsll((long long)in) - 1;
      b = uniform(r0 + l);
      slot = uniform(__shfl((int)from, l) + i - __shfl(to - pages, l));
    } else {
      i -= __shfl(to, 63);
    }
  }
  if (b < 0) return;
  const PagedSpan sp = uniform(paged_span(p.t, b));
  const long first = sp.start < 0 ? 0 : sp.start;
  const int page = paged_page(p.t, b, (int)slot);
  if (page < 0) return;
  const long low = first > slot * P ? first : slot * P;
  const long end = sp.length < (slot + 1) * P ? sp.length : (slot + 1) * P;
  const int at0 = (int)(low - slot * P), at1 = (int)(end - slot * P);
  if (at1 <= at0) return;
  const int row0 = sp.row0 + (int)(low - sp.start) - at0;  // of the page's first place
  const int part_tokens = IT == 1 ? 2 * threads / units : P, part0 = IT == 1 ? at0 / part_tokens : 0, part1 = IT == 1 ? (at1 - 1) / part_tokens : 0;
  constexpr int kHeads = 2;  // at_once, at most
  const long head_bytes = (long)p.dim << p.t.page_shift;
  if (!values) {
    // this thread's units of a part: the cosines and sines of their tokens (of more than two there are too many to hold), then, turned, a head's
    float c[2][8], s[2][8];
    auto angles = [&](int part) {
#pragma unroll
      for (int k = 0; k < (IT == 1 ? 2 : 0); ++k) {
        const int j = threadIdx.x + k * threads, at = part * part_tokens + j / units;
        const Unit n = unit_of(p, j % units);
        if (at >= at0 && at < at1 && n.turns0) unit_angles(p, n, (double)(p.positions ? p.positions[row0 + at] : slot * P + at), c[k], s[k]);
      }
    };
    float x[2 * IT][16];
    auto take = [&](int part, int h) {
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 2 * IT; ++k) {
        const int j = threadIdx.x + k * threads, at = part * part_tokens + j / units;
        if (at >= at0 && at < at1) {
          const Unit n = unit_of(p, j % units);
          load_unit<T>(p.k + (long)(row0 + at) * p.k_tok + (long)h * p.k_head, n.d0, n.d1, x[k]);
          if constexpr (IT > 1) {
            if (n.turns0) unit_angles(p, n, (double)(p.positions ? p.positions[row0 + at] : slot * P + at), c[0], s[0]);
          }
          if (n.turns0) unit_turn(p, n, c[IT == 1 ? k : 0], s[IT == 1 ? k : 0], x[k]);
#pragma unroll
          for (int m = 0; m < 16; ++m) most = fmaxf(most, finite_abs(x[k][m]));
        }
      }
      return most;
    };
    auto put = [&](int part, uint8_t* base, float inv) {
#pragma unroll
      for (int k = 0; k < 2 * IT; ++k) {
        const int j = threadIdx.x + k * threads, at = part * part_tokens + j / units;
        if (at >= at0 && at < at1) {
          const Unit n = unit_of(p, j % units);
          uint32_t w[4];
#pragma unroll
          for (int m = 0; m < 4; ++m) w[m] = to_e4m3x4(x[k][4 * m] * inv, x[k][4 * m + 1] * inv, x[k][4 * m + 2] * inv, x[k][4 * m + 3] * inv);
          *(u32x2*)(base + k_at(p.dim, at, n.d0)) = u32x2{w[0], w[1]};
          *(u32x2*)(base + k_at(p.dim, at, n.d1)) = u32x2{w[2], w[3]};
        }
      }
    };
    auto scaled = [&](int h, float most, float before_s) {
      const long ph = (long)page * p.kv_heads + h;
      __syncthreads();  // (red)
      return exp2i(-page_exponent(p, block_most(most, red), p.kp + ph * head_bytes, p.ks + ph, before_s, at0, false));
    };
    if (IT > 1 || part0 == part1) {
      angles(part0);
      for (int h = h0; h < h1; ++h) {
        const long ph = (long)page * p.kv_heads + h;
        const float before_s = p.ks[ph], most = take(part0, h);
        put(part0, p.kp + ph * head_bytes, scaled(h, most, before_s));
      }
      return;
    }
    float most[kHeads] = {}, inv[kHeads];
    for (int part = part0; part <= part1; ++part) {
      angles(part);
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (h0 + i < h1) most[i] = fmaxf(most[i], take(part, h0 + i));
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (h0 + i < h1) inv[i] = scaled(h0 + i, most[i], p.ks[(long)page * p.kv_heads + h0 + i]);
    for (int part = part0; part <= part1; ++part) {
      angles(part);
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (h0 + i < h1) {
          take(part, h0 + i);
          put(part, p.kp + ((long)page * p.kv_heads + h0 + i) * head_bytes, inv[i]);
        }
    }
    return;
  }
  u32x4 raw[IT][4];
  auto d_of = [&](int j) { return (j & 7) * 8 + j / (2 * part_tokens) * 64; };
  auto at_of = [&](int part, int j) { return part * part_tokens + 4 * (j / 8 % (part_tokens / 4)); };
  auto take = [&](int part, int h) {
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int j = threadIdx.x + k * threads;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int at = at_of(part, j) + m;
        raw[k][m] = u32x4{0, 0, 0, 0};
        if (at >= at0 && at < at1) raw[k][m] = ld16(p.v + (long)(row0 + at) * p.v_tok + (long)h * p.v_head + d_of(j));
      }
    }
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < IT; ++k)
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        float x[8];
        unpack8<T>(raw[k][m], x);
#pragma unroll
        for (int d = 0; d < 8; ++d) most = fmaxf(most, finite_abs(x[d]));
      }
    return most;
  };
  auto put = [&](int part, uint8_t* base, float inv) {
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int j = threadIdx.x + k * threads, at = at_of(part, j);
      const int before = at0 - at, behind = at + 4 - at1;  // places of the four that stay as they are
      if (before >= 4 || behind >= 4) continue;
      float x[4][8];
#pragma unroll
      for (int m = 0; m < 4; ++m) unpack8<T>(raw[k][m], x[m]);
      const uint32_t keep = (before > 0 ? (1u << (8 * before)) - 1u : 0u) | (behind > 0 ? ~(0xffffffffu >> (8 * behind)) : 0u);
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        uint32_t* to = (uint32_t*)(base + v_at(p.dim, at, d_of(j) + d));
        uint32_t w = to_e4m3x4(x[0][d] * inv, x[1][d] * inv, x[2][d] * inv, x[3][d] * inv);
        if (keep) w = (w & ~keep) | (*to & keep);
        *to = w;
      }
    }
  };
  for (int h = h0; h < h1; ++h) {
    const long ph = (long)page * p.kv_heads + h;
    uint8_t* base = p.vp + ph * head_bytes;
    const float before_s = p.vs[ph];
    float most = take(part0, h);
    for (int part = part0 + 1; part <= part1; ++part) most = fmaxf(most, take(part, h));
    __syncthreads();  // (red)
    const float inv = exp2i(-page_exponent(p, block_most(most, red), base, p.vs + ph, before_s, at0, true));
    put(part1, base, inv);  // (the one that was read last)
    for (int part = part0; part < part1; ++part) {
      take(part, h);
      put(part, base, inv);
    }
  }
}

}  // namespace mui

using namespace mui;

extern "C" int mui_paged_append(mui_stream_t stream, const mui_paged_append_args_t* args) {
  MUI_CHECK_ARG(args);
  const mui_paged_append_args_t& a = *args;
  MUI_CHECK_ARG(a.k && a.v && a.k_pages && a.v_pages && a.k_scale && a.v_scale && a.table && a.lengths && (!a.q || a.q_out));
  MUI_CHECK_ARG(a.n_pages > 0 && a.table_pages > 0 && a.table_stride >= a.table_pages && a.n_rows > 0 && a.n_requests > 0 && a.max_tokens > 0 && a.n_kv_heads > 0);
  MUI_CHECK_ARG(!a.q || a.n_q_heads > 0);
  MUI_CHECK_ARG(a.rot_dim >= 0 && a.rot_dim <= a.head_dim && (a.rot_dim == 0 || a.inv_freq));
  MUI_CHECK_ARG(a.offsets || a.n_rows == a.n_requests);
  if (a.dtype != MUI_DTYPE_F16 && a.dtype != MUI_DTYPE_BF16) return MUI_ERR_INVALID_ARG;
  if (a.page_tokens != 64 && a.page_tokens != 128 && a.page_tokens != 256) return MUI_ERR_UNSUPPORTED;
  if ((a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) || a.rot_dim % 16) return MUI_ERR_UNSUPPORTED;
  if (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.k_pages | (uintptr_t)a.v_pages | (uintptr_t)a.q_out) & 15u) return MUI_ERR_ALIGNMENT;
  if ((a.k_token_stride | a.k_head_stride | a.v_token_stride | a.v_head_stride) & 7) return MUI_ERR_ALIGNMENT;
  if (a.q && ((a.q_token_stride | a.q_head_stride) & 7)) return MUI_ERR_ALIGNMENT;
  if ((long)a.table_pages * a.page_tokens > 0x7fffffffL) return MUI_ERR_UNSUPPORTED;
  AppendParams p = {};
  p.q = (const uint16_t*)a.q; p.q_tok = a.q_token_stride; p.q_head = a.q_head_stride;
  p.k = (const uint16_t*)a.k; p.k_tok = a.k_token_stride; p.k_head = a.k_head_stride;
  p.v = (const uint16_t*)a.v; p.v_tok = a.v_token_stride; p.v_head = a.v_head_stride;
  p.kp = (uint8_t*)a.k_pages; p.vp = (uint8_t*)a.v_pages; p.ks = a.k_scale; p.vs = a.v_scale;
  p.positions = a.positions; p.inv_freq = a.inv_freq; p.q_out = (uint16_t*)a.q_out;
  p.t = {a.table, a.table_stride, a.table_pages, a.lengths, a.offsets, a.n_requests, a.n_rows, a.n_pages, a.page_tokens == 64 ? 6 : a.page_tokens == 128 ? 7 : 8};
  p.rope_scale = a.rope_scale; p.rot = a.rot_dim; p.interleaved = a.interleaved ? 1 : 0;
  p.heads = a.q ? a.n_q_heads : 0; p.kv_heads = a.n_kv_heads; p.dim = a.head_dim;
  hipStream_t s = (hipStream_t)stream;
  const int units = a.head_dim / 16;
  if (a.max_tokens == 1) {
    const long blocks = ((long)a.n_requests * (p.heads + 2 * a.n_kv_heads) * units + 255) / 256;
    if (blocks > 0x7fffffffL) return MUI_ERR_UNSUPPORTED;
    if (a.dtype == MUI_DTYPE_F16)
      hipLaunchKernelGGL((append_step_kernel<F16>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((append_step_kernel<BF16>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    return launch_status();
  }
  const bool full = a.n_rows > (long)a.n_requests * a.page_tokens;  // pages are filled, as a rule
  const int values = a.page_tokens * a.head_dim / 32, threads = values < 512 ? values : full && values == 1024 ? 1024 : 512;
  const long rows_per = threads / units;
  const long q_blocks = a.q ? (a.n_rows + rows_per - 1) / rows_per * ((a.n_q_heads + kQueryHeads - 1) / kQueryHeads) : 0;
  const long pages = (long)a.n_rows / a.page_tokens + 2 * (long)a.n_requests;  // that new tokens can lie in
  // A workgroup takes two heads where there are many pages: workgroups begin no faster than about 130 a microsecond, and the keys' angles serve both. Those 11500 tokens with one,
  // two, four heads: 53.3, 50.5, 51.9 us; with few pages one head each has more CUs at work.
  p.at_once = pages * 2 * a.n_kv_heads > 1024 ? 2 : 1;
  const long blocks = q_blocks + pages * 2 * ((a.n_kv_heads + p.at_once - 1) / p.at_once);
  if (blocks > 0x7fffffffL) return MUI_ERR_UNSUPPORTED;
  p.q_blocks = (int)q_blocks;
  const dim3 grid((unsigned)blocks), block(threads);
#define MUI_APPEND_GO(TT)                                                                                     \
  do {                                                                                                        \
    if (values <= 1024 || !full) hipLaunchKernelGGL((append_rows_kernel<TT, 1>), grid, block, 0, s, p);       \
    else hipLaunchKernelGGL((append_rows_kernel<TT, 4>), grid, block, 0, s, p);                               \
  } while (0)
  if (a.dtype == MUI_DTYPE_F16) MUI_APPEND_GO(F16); else MUI_APPEND_GO(BF16);
  return launch_status();
}
