// Queries and keys rotated by their positions, keys and values appended to a paged e4m3 cache (paged.cuh has its layout).
//
// Rotation of the first `rot` dimensions, in 32 bits: a' = a c - b s, b' = b c + a s for the pairs (i, i + rot / 2) or (2 i, 2 i + 1), c and s the
// cosine and sine (times rope_scale) of position * inv_freq[i], the angle's whole turns dropped in 64 bits. Queries are rounded once, to their own
// type; keys and values once, to codes x / scale. The scale of a page and head is the smallest power of two with which the largest new
// value fits 448, but not below what stands there for the page's earlier tokens; where it grows their codes follow.
//
// A thread works on units of 16 dimensions, which hold their pairs whole: 8 + 8 at a distance of rot / 2, or 16 in a row.
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
  int q_blocks, spans;
};

// dimension of the first value of either half of a unit
__device__ __forceinline__ void unit_dims(const AppendParams& p, int u, bool turned, int& d0, int& d1) {
  if (turned && !p.interleaved) {
    d0 = 8 * u;
    d1 = d0 + (p.rot >> 1);
  } else {
    d0 = 16 * u;
    d1 = d0 + 8;
  }
}

__device__ __forceinline__ void unit_angles(const AppendParams& p, int u, double pos, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    rope_angle(pos, p.inv_freq[8 * u + i], c[i], s[i]);
    c[i] *= p.rope_scale;
    s[i] *= p.rope_scale;
  }
}

// x: 16 values of a unit in the order of its two halves
__device__ __forceinline__ void unit_turn(bool interleaved, const float (&c)[8], const float (&s)[8], float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int ia = interleaved ? 2 * i : i, ib = interleaved ? 2 * i + 1 : i + 8;
    const float a = x[ia], b = x[ib];
    x[ia] = a * c[i] - b * s[i];
    x[ib] = b * c[i] + a * s[i];
  }
}

template <typename T>
__device__ __forceinline__ void load_unit(const uint16_t* row, int d0, int d1, float (&x)[16]) {
  float a[8], b[8];
  unpack8<T>(ld16(row + d0), a);
  unpack8<T>(ld16(row + d1), b);
#pragma unroll
  for (int i = 0; i < 8; ++i) { x[i] = a[i]; x[8 + i] = b[i]; }
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
// one new token per request: dim / 16 lanes work on one head of one token (queries, keys, values)
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
  const bool turned = kind != 2 && 16 * u < p.rot;
  int d0, d1;
  unit_dims(p, u, turned, d0, d1);
  float x[16];
  load_unit<T>(row, d0, d1, x);
  if (turned) {
    float c[8], s[8];
    unit_angles(p, u, (double)(p.positions ? p.positions[sp.row0] : sp.start), c, s);
    unit_turn(p.interleaved, c, s, x);
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
// prompts: workgroups of queries (16 tokens each), then one workgroup per page, head and kind
// ---------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) append_rows_kernel(const AppendParams p) {
  const int units = p.dim >> 4;
  __shared__ float red[4];
  if ((int)blockIdx.x < p.q_blocks) {
    const int per = 256 / units;  // tokens of a workgroup
    const int u = threadIdx.x % units;
    const int row = blockIdx.x * per + threadIdx.x / units;
    if (row >= p.t.n_rows) return;
    int b = row;
    if (p.t.offsets) {  // the last request that starts at or before the row
      int lo = 0, hi = p.t.n_requests;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.t.offsets[mid] <= row) lo = mid; else hi = mid;
      }
      b = lo;
    }
    if (b >= p.t.n_requests) return;
    const PagedSpan sp = paged_span(p.t, b);
    if (row < sp.row0 || row >= sp.row0 + sp.count) return;  // behind the last request: left as it is
    const bool turned = 16 * u < p.rot;
    int d0, d1;
    unit_dims(p, u, turned, d0, d1);
    float c[8], s[8];
    if (turned) unit_angles(p, u, (double)(p.positions ? p.positions[row] : sp.start + (row - sp.row0)), c, s);
    for (int h = 0; h < p.heads; ++h) {
      float x[16];
      load_unit<T>(p.q + (long)row * p.q_tok + (long)h * p.q_head, d0, d1, x);
      if (turned) unit_turn(p.interleaved, c, s, x);
      store_unit<T>(p.q_out + ((long)row * p.heads + h) * p.dim, d0, d1, x);
    }
    return;
  }
  int i = blockIdx.x - p.q_blocks;
  const int hk = i % (2 * p.kv_heads);
  i /= 2 * p.kv_heads;
  const int span = i % p.spans, b = i / p.spans;
  const bool values = hk >= p.kv_heads;
  const int h = values ? hk - p.kv_heads : hk;
  const PagedSpan sp = paged_span(p.t, b);
  const int P = 1 << p.t.page_shift;
  const long first = sp.start < 0 ? 0 : sp.start;
  for (long slot = (first >> p.t.page_shift) + span; slot * P < sp.length; slot += p.spans) {
    const int page = paged_page(p.t, b, (int)slot);
    if (page < 0) continue;
    const long low = first > slot * P ? first : slot * P;
    const long end = sp.length < (slot + 1) * P ? sp.length : (slot + 1) * P;
    const int n = (int)(end - low), at0 = (int)(low - slot * P);
    if (n <= 0) continue;
    const int row0 = sp.row0 + (int)(low - sp.start);
    const long ph = (long)page * p.kv_heads + h;
    uint8_t* base = (values ? p.vp : p.kp) + ph * ((long)p.dim << p.t.page_shift);
    float* scale = (values ? p.vs : p.ks) + ph;
    const float before_s = *scale;
    float most = 0.f;
    float inv = 0.f;
    for (int pass = 0; pass < 2; ++pass) {  // the largest value, then the codes
      for (int j = threadIdx.x; j < n * units; j += 256) {
        const int u = j % units, row = row0 + j / units, at = at0 + j / units;
        const bool turned = !values && 16 * u < p.rot;
        int d0, d1;
        unit_dims(p, u, turned, d0, d1);
        float x[16];
        load_unit<T>(values ? p.v + (long)row * p.v_tok + (long)h * p.v_head : p.k + (long)row * p.k_tok + (long)h * p.k_head, d0, d1, x);
        if (turned) {
          float c[8], s[8];
          unit_angles(p, u, (double)(p.positions ? p.positions[row] : sp.start + (row - sp.row0)), c, s);
          unit_turn(p.interleaved, c, s, x);
        }
        if (pass == 0) {
#pragma unroll
          for (int k = 0; k < 16; ++k) most = fmaxf(most, finite_abs(x[k]));
        } else {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = to_e4m3x4(x[4 * k] * inv, x[4 * k + 1] * inv, x[4 * k + 2] * inv, x[4 * k + 3] * inv);
          if (!values) {
            *(u32x2*)(base + k_at(p.dim, at, d0)) = u32x2{w[0], w[1]};
            *(u32x2*)(base + k_at(p.dim, at, d1)) = u32x2{w[2], w[3]};
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) base[v_at(p.dim, at, (k < 8 ? d0 : d1 - 8) + k)] = (uint8_t)(w[k >> 2] >> (8 * (k & 3)));
          }
        }
      }
      if (pass) break;
      most = wave_max(most);
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
      __syncthreads();
      most = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      int e = e4m3_exponent(most);
      if (at0 > 0) {
        const int before = scale_exponent(before_s);
        if (e > before) {
          const int down = before - e;
          move_codes(base, p.dim, at0, exp2i(down < -126 ? -126 : down), values, threadIdx.x, 256);
          __syncthreads();  // (a new value's byte may lie between moved ones)
        } else {
          e = before;
        }
      }
      if (threadIdx.x == 0) *scale = exp2i(e);
      inv = exp2i(-e);
    }
  }
}

}  // namespace mui

using namespace mui;

extern "C" int mui_paged_append(mui_stream_t stream, int dtype, const void* q, long q_token_stride, long q_head_stride, const void* k, long k_token_stride,
                                long k_head_stride, const void* v, long v_token_stride, long v_head_stride, void* k_pages, void* v_pages, float* k_scale,
                                float* v_scale, int n_pages, int page_tokens, const int32_t* table, long table_stride, int table_pages, const int64_t* lengths,
                                const int64_t* offsets, const int64_t* positions, const double* inv_freq, int rot_dim, int interleaved, float rope_scale,
                                void* q_out, int n_rows, int n_requests, int max_tokens, int n_q_heads, int n_kv_heads, int head_dim) {
  MUI_CHECK_ARG(k && v && k_pages && v_pages && k_scale && v_scale && table && lengths && (!q || q_out));
  MUI_CHECK_ARG(n_pages > 0 && table_pages > 0 && table_stride >= table_pages && n_rows > 0 && n_requests > 0 && max_tokens > 0 && n_kv_heads > 0);
  MUI_CHECK_ARG(!q || n_q_heads > 0);
  MUI_CHECK_ARG(rot_dim >= 0 && rot_dim <= head_dim && (rot_dim == 0 || inv_freq));
  MUI_CHECK_ARG(offsets || n_rows == n_requests);
  if (dtype != MUI_DTYPE_F16 && dtype != MUI_DTYPE_BF16) return MUI_ERR_INVALID_ARG;
  if (page_tokens != 64 && page_tokens != 128 && page_tokens != 256) return MUI_ERR_UNSUPPORTED;
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || rot_dim % 16) return MUI_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)q_out) & 15u) return MUI_ERR_ALIGNMENT;
  if ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) return MUI_ERR_ALIGNMENT;
  if (q && ((q_token_stride | q_head_stride) & 7)) return MUI_ERR_ALIGNMENT;
  AppendParams p = {};
  p.q = (const uint16_t*)q; p.q_tok = q_token_stride; p.q_head = q_head_stride;
  p.k = (const uint16_t*)k; p.k_tok = k_token_stride; p.k_head = k_head_stride;
  p.v = (const uint16_t*)v; p.v_tok = v_token_stride; p.v_head = v_head_stride;
  p.kp = (uint8_t*)k_pages; p.vp = (uint8_t*)v_pages; p.ks = k_scale; p.vs = v_scale;
  p.positions = positions; p.inv_freq = inv_freq; p.q_out = (uint16_t*)q_out;
  p.t = {table, table_stride, table_pages, lengths, offsets, n_requests, n_rows, n_pages, page_tokens == 64 ? 6 : page_tokens == 128 ? 7 : 8};
  p.rope_scale = rope_scale; p.rot = rot_dim; p.interleaved = interleaved ? 1 : 0;
  p.heads = q ? n_q_heads : 0; p.kv_heads = n_kv_heads; p.dim = head_dim;
  hipStream_t s = (hipStream_t)stream;
  const int units = head_dim / 16;
  if (max_tokens == 1) {
    const long blocks = ((long)n_requests * (p.heads + 2 * n_kv_heads) * units + 255) / 256;
    if (blocks > 0x7fffffffL) return MUI_ERR_UNSUPPORTED;
    if (dtype == MUI_DTYPE_F16)
      hipLaunchKernelGGL((append_step_kernel<F16>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((append_step_kernel<BF16>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    return launch_status();
  }
  p.q_blocks = q ? (n_rows + 256 / units - 1) / (256 / units) : 0;
  p.spans = (max_tokens + page_tokens - 2) / page_tokens + 1;
  const long blocks = p.q_blocks + (long)n_requests * p.spans * 2 * n_kv_heads;
  if (blocks > 0x7fffffffL) return MUI_ERR_UNSUPPORTED;
  if (dtype == MUI_DTYPE_F16)
    hipLaunchKernelGGL((append_rows_kernel<F16>), dim3((unsigned)blocks), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((append_rows_kernel<BF16>), dim3((unsigned)blocks), dim3(256), 0, s, p);
  return launch_status();
}
