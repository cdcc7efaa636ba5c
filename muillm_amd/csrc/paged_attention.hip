// Attention over a paged e4m3 cache (paged.cuh has its layout).
//
// The matrix cores take the codes as they lie in memory: v_mfma_scale_f32_16x16x128_f8f6f4, whose block exponents carry the pages' scales. What
// meets them is split into pieces of e4m3 so that nothing is lost by it: a query into two (bf16: 8 bits are two pieces of 4) or three (fp16), each 2^5 below
// the one before; a probability into two, of 8 bits together, relative to the largest of its query's 64 in the tile (2^-18 of it at least), which goes
// with the product as its block exponent -- so a tile whose keys weigh little is as exact as one whose weigh much, however long the cache.
// Sums and the running maximum are 32 bits; the maximum is rounded up to a whole power of two, so moving to a new one is exact.
//
// Score products are K Q^T (rows keys, columns queries), value products V^T P^T: scores leave the first as the second wants them, in registers.
#include "paged.cuh"

namespace mui {

struct PagedAttnParams {
  const uint16_t* q; long q_tok, q_head;
  const uint8_t* kp; const uint8_t* vp;
  const float* ks; const float* vs;
  PagedTable t;
  float scale;          // of the scores, times log2(e)
  int window, keep;
  int heads, kv_heads, group;
  int col_tiles;        // tiles of 16 columns (new token, head of the group) of a request at most
  int split_tiles;      // tiles of 64 keys per workgroup
  int splits;           // at most
  float* part;          // [splits][n_rows * heads][dim + 2], or null: one split
  uint16_t* out;
};

constexpr float kNoMax = -1e30f;

// The tiles of 64 keys that queries at positions first .. last see: `kept` from the beginning, then those from `from` to `end`.
struct TileRange { int kept, from, end; __device__ int count() const { return kept + (end > from ? end - from : 0); }
  __device__ int at(int i) const { return i < kept ? i : from + i - kept; } };
__device__ __forceinline__ TileRange tile_range(const PagedAttnParams& p, long first, long last, long length) {
  TileRange r;
  const long most = last + 1 < length ? last + 1 : length;
  r.end = most > 0 ? (int)((most + 63) >> 6) : 0;
  r.from = 0;
  r.kept = 0;
  if (p.window > 0) {
    const long low = first - p.window + 1;
    r.from = low > 0 ? (int)(low >> 6) : 0;
    r.from = r.from < r.end ? r.from : r.end;
    r.kept = (int)((p.keep + 63L) >> 6);
    r.kept = r.kept < r.from ? r.kept : r.from;
  }
  return r;
}

__device__ __forceinline__ i32x8 pair8(u32x4 a, u32x4 b) { return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w}; }

__device__ __forceinline__ f32x4 mfma_e4m3(i32x8 a, i32x8 b, f32x4 c, int scale_a, int scale_b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, scale_a, 0, scale_b);
}

// 16 columns of queries as the score products want them: lane (column l % 16, g = l / 16) has of every 64 dimensions the 16 from 16 g on.
template <int DC, int PIECES>
struct QueryTile {
  static constexpr int M = (DC + 1) / 2;
  i32x8 piece[PIECES][M];
  float unit;  // what the products are multiplied by, the score scale included
};
template <typename T, int DC, int PIECES>
__device__ __forceinline__ void load_queries(QueryTile<DC, PIECES>& t, const uint16_t* row, bool there, float score_scale, int g) {
  float x[DC][16];
  float most = 0.f;
#pragma unroll
  for (int c = 0; c < DC; ++c) {
    const u32x4 zero = {0, 0, 0, 0};
    float a[8], b[8];
    unpack8<T>(there ? ld16(row + c * 64 + g * 16) : zero, a);
    unpack8<T>(there ? ld16(row + c * 64 + g * 16 + 8) : zero, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[c][i] = a[i];
      x[c][8 + i] = b[i];
      most = fmaxf(most, fmaxf(fabsf(a[i]), fabsf(b[i])));
    }
  }
  most = rows_max(most);
  int e = (int)((__float_as_uint(most) >> 23) & 0xff) - 126 - 8;  // |x| 2^-e < 2^8
  e = e < -110 ? -110 : (e > 119 ? 119 : e);
  t.unit = exp2i(e) * score_scale;
  const float inv = exp2i(-e);
  uint32_t w[PIECES][2 * QueryTile<DC, PIECES>::M][4];
#pragma unroll
  for (int c = 0; c < 2 * QueryTile<DC, PIECES>::M; ++c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = c < DC ? x[c < DC ? c : 0][4 * j + i] * inv : 0.f;
#pragma unroll
      for (int s = 0; s < PIECES; ++s) {
        const uint32_t v = to_e4m3x4(r[0], r[1], r[2], r[3]);
        w[s][c][j] = v;
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true);
        r[0] = (r[0] - a[0]) * 32.f; r[1] = (r[1] - a[1]) * 32.f; r[2] = (r[2] - b[0]) * 32.f; r[3] = (r[3] - b[1]) * 32.f;
      }
    }
  }
#pragma unroll
  for (int s = 0; s < PIECES; ++s)
#pragma unroll
    for (int m = 0; m < QueryTile<DC, PIECES>::M; ++m)
      t.piece[s][m] = pair8(u32x4{w[s][2 * m][0], w[s][2 * m][1], w[s][2 * m][2], w[s][2 * m][3]},
                            u32x4{w[s][2 * m + 1][0], w[s][2 * m + 1][1], w[s][2 * m + 1][2], w[s][2 * m + 1][3]});
}

// one tile of 64 keys, as a wave holds it: 1 KB per register of 16 bytes
template <int DC>
struct KvTile { u32x4 k[4 * DC]; u32x4 v[4 * DC]; };
template <int DC>
__device__ __forceinline__ void load_tile(KvTile<DC>& t, const uint8_t* k, const uint8_t* v, int lane) {
  // lane (row l % 16, g): chunk g of row's 64 bytes
  const int at = (lane & 15) * 64 + (lane >> 4) * 16;
#pragma unroll
  for (int i = 0; i < 4 * DC; ++i) t.k[i] = ld16_stream(k + i * 1024 + at);
#pragma unroll
  for (int i = 0; i < 4 * DC; ++i) t.v[i] = ld16_stream(v + i * 1024 + at);
}

// 0xff in the bytes of a dword of codes that are NaN
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t a = (w & 0x7f7f7f7fu) + 0x01010101u;  // 0x80 where the code is NaN
  return ((a & 0x80808080u) >> 7) * 0xffu;
}

template <int DC>
struct Columns {
  f32x4 o[4 * DC];  // lane (column, g), dimensions 16 i + 4 g + r
  float m, l;       // the maximum, a whole number of powers of two; this lane's part of the sum
};

// The tile's scores and values into the running result of 16 columns. pos: the lane's column's position (-1: no column); first_key: key 0 of the tile;
// whole: every column sees all 64 keys. `ks`, `vs`: the page's scales.
template <typename T, int DC, int PIECES>
__device__ __forceinline__ void attend_tile(Columns<DC>& c, const QueryTile<DC, PIECES>& q, const KvTile<DC>& t, float ks, float vs, bool whole, long first_key,
                                            long pos, long length, int window, int keep, int g) {
  constexpr int M = (DC + 1) / 2;
  const u32x4 zero = {0, 0, 0, 0};
  f32x4 s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const i32x8 kk = pair8(t.k[8 * m + i], 2 * m + 1 < DC ? t.k[8 * m + 4 + i < 4 * DC ? 8 * m + 4 + i : 0] : zero);
#pragma unroll
      for (int j = 0; j < PIECES; ++j) a = mfma_e4m3(kk, q.piece[j][m], a, 127, 127 - 5 * j);
    }
    s[i] = a;
  }
  const float unit = q.unit * ks;
  uint32_t hidden = 0;  // keys 16 i + 4 g + r that the column does not see, bit 4 i + r
  if (!whole) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const long key = first_key + 16 * i + 4 * g + r;
        const bool see = key <= pos && key < length && (window <= 0 || key > pos - window || key < keep);
        hidden |= see ? 0u : 1u << (4 * i + r);
      }
  }
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (!whole && (hidden >> (4 * i + r) & 1u)) s[i][r] = -INFINITY;
      most = fmaxf(most, s[i][r]);
    }
  most = rows_max(most) * unit;  // (unit > 0)
  const float mt = fmaxf(ceilf(fminf(most, 1e30f)), kNoMax);
  if (__any(mt > c.m)) {
    const float to = fmaxf(c.m, mt), f = __builtin_amdgcn_exp2f(c.m - to);
    c.m = to;
    c.l *= f;
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) c.o[i] *= f;
  }
  // probabilities of the tile, its largest in (2^7, 2^8]
  const float base = fabsf(mt) < 1e8f ? mt - 8.f : mt;  // (beyond, the difference would be rounded)
  uint32_t hi[4], lo[4];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float e[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      e[r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], unit, -base));
      sum += e[r];
    }
    hi[i] = to_e4m3x4(e[0], e[1], e[2], e[3]);
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi[i], true);
    lo[i] = to_e4m3x4(e[0] - a[0], e[1] - a[1], e[2] - b[0], e[3] - b[1]);
  }
  const float up = fmaxf(base - c.m, -127.f);
  c.l += sum * __builtin_amdgcn_exp2f(up);
  const int sb = 127 + (int)up, sa = 127 + scale_exponent(vs);
  const i32x8 pp = i32x8{(int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3], (int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3]};
  if (whole) {
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) c.o[i] = mfma_e4m3(pair8(t.v[i], t.v[i]), pp, c.o[i], sa, sb);
    return;
  }
  // Part of the tile is hidden: what stands there may be anything, and 0 * NaN is NaN. A NaN code counts as zero, and a column that sees it gets a NaN.
  uint32_t found = 0;
#pragma unroll
  for (int i = 0; i < 4 * DC; ++i) {
    u32x4 v = t.v[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t n = nan_bytes(v[j]);
      found |= n;
      v[j] &= ~n;
    }
    c.o[i] = mfma_e4m3(pair8(v, v), pp, c.o[i], sa, sb);
  }
  if (__any(found != 0)) {
    i32x8 ones;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) w |= (hidden >> (4 * i + r) & 1u) ? 0u : 0x38u << (8 * r);
      ones[i] = (int)w;
      ones[4 + i] = 0;
    }
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) {
      u32x4 v = t.v[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = nan_bytes(v[j]) & 0x38383838u;
      const f32x4 seen = mfma_e4m3(pair8(v, zero), ones, f32x4{0.f, 0.f, 0.f, 0.f}, 127, 127);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (seen[r] > 0.f) c.o[i][r] = __builtin_nanf("");
    }
  }
}

// Single tokens, and several: a workgroup takes 16 columns (new token, head of the group) of one KV head and `split_tiles` tiles of 64 keys, its waves
// every fourth tile each; their results meet in LDS.
template <typename T, int DC, int PIECES>
__global__ void __launch_bounds__(256) paged_columns_kernel(const PagedAttnParams p) {
  constexpr int D = DC * 64, W = 4;
  __shared__ float so[W][16][D + 4];
  __shared__ float sm[W][16], sl[W][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.z, h = blockIdx.y % p.kv_heads, ct = blockIdx.y / p.kv_heads;
  const PagedSpan sp = paged_span(p.t, b);
  const long n_cols = (long)sp.count * p.group;
  if (16L * ct >= n_cols) return;
  const int g = lane >> 4;
  const long col = 16L * ct + (lane & 15);
  const bool there = col < n_cols;
  const int token = (int)((there ? col : n_cols - 1) / p.group), head = h * p.group + (int)((there ? col : n_cols - 1) % p.group);
  const long pos = there ? sp.start + token : -1;
  const int token0 = (int)(16L * ct / p.group), token1 = (int)((16L * ct + 15 < n_cols ? 16L * ct + 15 : n_cols - 1) / p.group);
  const TileRange range = tile_range(p, sp.start + token0, sp.start + token1, sp.length);
  const int begin = blockIdx.x * p.split_tiles;
  const int n_tiles = range.count();
  if (begin >= n_tiles && begin > 0) return;
  const int end = begin + p.split_tiles < n_tiles ? begin + p.split_tiles : n_tiles;

  QueryTile<DC, PIECES> q;
  load_queries<T, DC, PIECES>(q, p.q + (long)(sp.row0 + token) * p.q_tok + (long)head * p.q_head, there, p.scale, g);
  Columns<DC> c;
  c.m = kNoMax;
  c.l = 0.f;
#pragma unroll
  for (int i = 0; i < 4 * DC; ++i) c.o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int per_page = p.t.page_shift - 6;
  for (int i = begin + wave; i < end; i += W) {
    const int tile = range.at(i);
    const int page = paged_page(p.t, b, tile >> per_page);
    if (page < 0) continue;
    const long ph = (long)page * p.kv_heads + h;
    const long at = (ph << per_page) + (tile & ((1 << per_page) - 1));
    KvTile<DC> t;
    load_tile<DC>(t, p.kp + at * (64 * D), p.vp + at * (64 * D), lane);
    const long k0 = 64L * tile;
    const bool whole = k0 + 63 <= sp.start + token0 && k0 + 64 <= sp.length &&
                       (p.window <= 0 || k0 > sp.start + token1 - p.window || k0 + 64 <= p.keep);
    attend_tile<T, DC, PIECES>(c, q, t, p.ks[ph], p.vs[ph], whole, k0, pos, sp.length, p.window, p.keep, g);
  }
  const float l = rows_sum(c.l);
#pragma unroll
  for (int i = 0; i < 4 * DC; ++i) *(f32x4*)&so[wave][lane & 15][16 * i + 4 * g] = c.o[i];
  if (g == 0) { sm[wave][lane & 15] = c.m; sl[wave][lane & 15] = l; }
  __syncthreads();
  // 16 threads per column
  const int cc = threadIdx.x >> 4;
  const long my = 16L * ct + cc;
  if (my >= n_cols) return;
  const int my_token = (int)(my / p.group), my_head = h * p.group + (int)(my % p.group);
  float m = sm[0][cc];
#pragma unroll
  for (int w = 1; w < W; ++w) m = fmaxf(m, sm[w][cc]);
  float f[W], sum = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    f[w] = __builtin_amdgcn_exp2f(sm[w][cc] - m);
    sum += f[w] * sl[w][cc];
  }
  const long row = (long)(sp.row0 + my_token) * p.heads + my_head;
  const float inv = p.part ? 1.f : (sum > 0.f || sum != sum ? 1.f / sum : 0.f);
  float* part = p.part ? p.part + ((long)blockIdx.x * p.t.n_rows * p.heads + row) * (D + 4) : nullptr;
  for (int d = 4 * (threadIdx.x & 15); d < D; d += 64) {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) o += f[w] * *(const f32x4*)&so[w][cc][d];
    o *= inv;
    if (part) {
      *(f32x4*)(part + d) = o;
    } else {
      *(u32x2*)(p.out + row * D + d) = u32x2{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])};
    }
  }
  if (part && (threadIdx.x & 15) == 0) { part[D] = m; part[D + 1] = sum; }
}

// The splits of a row and head together: a wave each.
template <typename T, int DC>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedAttnParams p) {
  constexpr int D = DC * 64;
  const int lane = threadIdx.x & 63;
  const long n = (long)p.t.n_rows * p.heads;
  const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= n) return;
  const int row = (int)(item / p.heads), head = (int)(item % p.heads);
  int b = row;
  if (p.t.offsets) {
    int lo = 0, hi = p.t.n_requests;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.t.offsets[mid] <= row) lo = mid; else hi = mid;
    }
    b = lo;
  }
  const PagedSpan sp = paged_span(p.t, b);
  if (row < sp.row0 || row >= sp.row0 + sp.count) return;
  // the tiles of the row's column tile, as the kernel above has them
  const int token = row - sp.row0;
  const long ct = ((long)token * p.group + head % p.group) / 16;
  const long n_cols = (long)sp.count * p.group;
  const int token0 = (int)(16L * ct / p.group), token1 = (int)((16L * ct + 15 < n_cols ? 16L * ct + 15 : n_cols - 1) / p.group);
  const int n_tiles = tile_range(p, sp.start + token0, sp.start + token1, sp.length).count();
  int splits = n_tiles > 0 ? (n_tiles + p.split_tiles - 1) / p.split_tiles : 1;
  splits = splits < p.splits ? splits : p.splits;
  const float* part = p.part + item * (D + 4);
  const long step = n * (D + 4);
  float m = kNoMax;
  for (int i = 0; i < splits; ++i) m = fmaxf(m, part[i * step + D]);
  float sum = 0.f, o[DC] = {};
  for (int i = 0; i < splits; ++i) {
    const float f = __builtin_amdgcn_exp2f(part[i * step + D] - m);
    sum += f * part[i * step + D + 1];
#pragma unroll
    for (int j = 0; j < DC; ++j) o[j] += f * part[i * step + 64 * j + lane];
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
  for (int j = 0; j < DC; ++j) p.out[item * D + 64 * j + lane] = T::pack(o[j] * inv);
}

struct PagedPlan { int col_tiles, split_tiles, splits; };
static PagedPlan paged_plan(int n_requests, int max_tokens, int max_length, int window, int keep, int n_q_heads, int n_kv_heads) {
  PagedPlan r;
  const long group = n_q_heads / n_kv_heads;
  r.col_tiles = (int)((max_tokens * group + 15) / 16);
  long tiles = ((long)max_length + 63) / 64;
  if (window > 0) {
    const long seen = ((long)window + max_tokens + 62) / 64 + 1 + ((long)keep + 63) / 64;
    tiles = tiles < seen ? tiles : seen;
  }
  if (tiles < 1) tiles = 1;
  const long work = (long)n_requests * n_kv_heads * r.col_tiles;
  long splits = (1024 + work - 1) / work;
  if (splits > (tiles + 7) / 8) splits = (tiles + 7) / 8;
  if (splits < 1) splits = 1;
  r.split_tiles = (int)((tiles + splits - 1) / splits);
  r.splits = (int)((tiles + r.split_tiles - 1) / r.split_tiles);
  return r;
}

}  // namespace mui

using namespace mui;

static bool paged_attention_sizes(int n_rows, int n_requests, int max_tokens, int max_length, int window, int keep_first, int n_q_heads, int n_kv_heads, int head_dim) {
  return n_rows > 0 && n_requests > 0 && max_tokens > 0 && max_length > 0 && window >= 0 && keep_first >= 0 && n_kv_heads > 0 && n_q_heads > 0 &&
         n_q_heads % n_kv_heads == 0 && head_dim > 0;
}

extern "C" size_t mui_paged_attention_scratch_bytes(int n_rows, int n_requests, int max_tokens, int max_length, int window, int keep_first, int n_q_heads,
                                                    int n_kv_heads, int head_dim) {
  if (!paged_attention_sizes(n_rows, n_requests, max_tokens, max_length, window, keep_first, n_q_heads, n_kv_heads, head_dim)) return 0;
  const PagedPlan plan = paged_plan(n_requests, max_tokens, max_length, window, keep_first, n_q_heads, n_kv_heads);
  return plan.splits > 1 ? (size_t)plan.splits * n_rows * n_q_heads * (head_dim + 4) * 4 : 0;
}

extern "C" int mui_paged_attention(mui_stream_t stream, int dtype, const void* q, long q_token_stride, long q_head_stride, const void* k_pages,
                                   const void* v_pages, const float* k_scale, const float* v_scale, int n_pages, int page_tokens, const int32_t* table,
                                   long table_stride, int table_pages, const int64_t* lengths, const int64_t* offsets, float scale, int window, int keep_first,
                                   int max_tokens, int max_length, void* scratch, size_t scratch_bytes, void* out, int n_rows, int n_requests, int n_q_heads,
                                   int n_kv_heads, int head_dim) {
  MUI_CHECK_ARG(q && k_pages && v_pages && k_scale && v_scale && table && lengths && out);
  MUI_CHECK_ARG(paged_attention_sizes(n_rows, n_requests, max_tokens, max_length, window, keep_first, n_q_heads, n_kv_heads, head_dim));
  MUI_CHECK_ARG(n_pages > 0 && table_pages > 0 && table_stride >= table_pages && (offsets || n_rows == n_requests) && scale > 0.f);
  if (dtype != MUI_DTYPE_F16 && dtype != MUI_DTYPE_BF16) return MUI_ERR_INVALID_ARG;
  if (page_tokens != 64 && page_tokens != 128 && page_tokens != 256) return MUI_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return MUI_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out | (uintptr_t)scratch) & 15u) return MUI_ERR_ALIGNMENT;
  if ((q_token_stride | q_head_stride) & 7) return MUI_ERR_ALIGNMENT;
  const long cap = (long)table_pages * page_tokens;
  if (max_length > cap) max_length = (int)cap;
  const PagedPlan plan = paged_plan(n_requests, max_tokens, max_length, window, keep_first, n_q_heads, n_kv_heads);
  if (plan.splits > 1 && (!scratch || scratch_bytes < (size_t)plan.splits * n_rows * n_q_heads * (head_dim + 4) * 4)) return MUI_ERR_INVALID_ARG;
  if ((long)plan.col_tiles * n_kv_heads > 65535 || n_requests > 65535) return MUI_ERR_UNSUPPORTED;
  PagedAttnParams p = {};
  p.q = (const uint16_t*)q; p.q_tok = q_token_stride; p.q_head = q_head_stride;
  p.kp = (const uint8_t*)k_pages; p.vp = (const uint8_t*)v_pages; p.ks = k_scale; p.vs = v_scale;
  p.t = {table, table_stride, table_pages, lengths, offsets, n_requests, n_rows, n_pages, page_tokens == 64 ? 6 : page_tokens == 128 ? 7 : 8};
  p.scale = scale * 1.4426950408889634f;
  p.window = window; p.keep = window > 0 ? keep_first : 0;
  p.heads = n_q_heads; p.kv_heads = n_kv_heads; p.group = n_q_heads / n_kv_heads;
  p.col_tiles = plan.col_tiles; p.split_tiles = plan.split_tiles; p.splits = plan.splits;
  p.part = plan.splits > 1 ? (float*)scratch : nullptr;
  p.out = (uint16_t*)out;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid(plan.splits, plan.col_tiles * n_kv_heads, n_requests);
  const dim3 join((unsigned)(((long)n_rows * n_q_heads + 3) / 4));
#define MUI_PAGED_GO(TT, DC, PIECES)                                                                     \
  do {                                                                                                   \
    hipLaunchKernelGGL((paged_columns_kernel<TT, DC, PIECES>), grid, dim3(256), 0, s, p);                \
    if (plan.splits > 1) hipLaunchKernelGGL((paged_join_kernel<TT, DC>), join, dim3(256), 0, s, p);      \
  } while (0)
#define MUI_PAGED_TYPES(DC) \
  do { if (dtype == MUI_DTYPE_F16) MUI_PAGED_GO(F16, DC, 3); else MUI_PAGED_GO(BF16, DC, 2); } while (0)
  if (head_dim == 64) MUI_PAGED_TYPES(1); else if (head_dim == 128) MUI_PAGED_TYPES(2); else MUI_PAGED_TYPES(4);
  return launch_status();
}
