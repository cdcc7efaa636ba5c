// Attention over a paged e4m3 cache (paged.cuh has its layout).
//
// Codes are widened to 16 bits, which hold them whole, and meet the queries in the queries' own type: scores are sums of exact products in 32 bits. (The matrix cores' 8-bit
// instructions take codes as they lie, but keep 13 bits below the largest of a lane's products: keys that have a channel in common, as trained models' do, lost all that tells
// them apart.) Probabilities meet the values in fp16: relative to the largest of a query's 64 in a tile (single tokens, two pieces of 11 bits each) or to a running reference
// (prompts: one piece for bf16 outputs, whose own rounding is 8 times as coarse, two for fp16).
// Sums and the running maximum are 32 bits; the maximum is rounded up to a whole power of two, so moving to a new one is exact.
//
// Score products are K Q^T (rows keys, columns queries), value products V^T P^T: scores leave the first as the second wants them, in registers.
#include <type_traits>

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
  int block_cols;       // columns (new token, head of the group) of a workgroup
  int col_tiles;        // such blocks of a request at most
  int split_tiles;      // tiles of 64 keys per workgroup
  int splits;           // at most
  float* part;          // partial results, or null: none. Single tokens: [workgroups][2][16][dim + 4], prompts [splits][n_rows * heads][dim + 4]; dim values, maximum, sum
  int* before;          // [n_requests + 1], single tokens: see paged_columns_kernel
  uint16_t* out;
};

constexpr float kNoMax = -0x1.fffffep127f;  // below every score
constexpr int kDealtRequests = 1024;  // requests whose tiles are dealt out (more give a workgroup each anyway)

// tiles of a workgroup's share, at least one a wave
__device__ __forceinline__ int share_of(int total, int workgroups, int waves) {
  const int s = (total + workgroups - 1) / workgroups;
  return s > waves ? s : waves;
}

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

// (counts; not for sums: within an instruction the matrix cores keep 13 bits below the largest of a lane's products)
__device__ __forceinline__ f32x4 mfma_e4m3(i32x8 a, i32x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 127, 0, 127);
}

// Two of four codes in 16 bits, which hold every e4m3 number.
template <typename T>
__device__ __forceinline__ uint32_t widen2(uint32_t w, bool high) {
  if constexpr (T::kDtype == MUI_DTYPE_F16)
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)) : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
  else
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)) : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
}
template <typename T>
__device__ __forceinline__ u32x4 widen8(uint32_t a, uint32_t b) { return u32x4{widen2<T>(a, false), widen2<T>(a, true), widen2<T>(b, false), widen2<T>(b, true)}; }

// the same in fp16 times a power of two
__device__ __forceinline__ uint32_t scaled2(uint32_t w, float s, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true)) : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false));
}

// 16 columns of queries as the score products want them: lane (column l % 16, g = l / 16) has of every 64 dimensions the 16 from 16 g on, 8 for each of two products.
template <int DC>
struct QueryTile {
  u32x4 v[DC][2];
  float unit;  // what the products are multiplied by, the score scale included
};
template <int DC>
struct QueryRow { u32x4 v[DC][2]; };
template <int DC>
__device__ __forceinline__ QueryRow<DC> request_queries(const uint16_t* row, int g) {
  QueryRow<DC> r;
#pragma unroll
  for (int c = 0; c < DC; ++c) {
    r.v[c][0] = ld16(row + c * 64 + g * 16);
    r.v[c][1] = ld16(row + c * 64 + g * 16 + 8);
  }
  return r;
}
// fp16 queries go in as they are; of bf16 ones the row's largest is brought below 2^8 by a power of two, so that no sum of their products with codes overflows
template <typename T, int DC>
__device__ __forceinline__ void take_queries(QueryTile<DC>& t, const QueryRow<DC>& row, bool there, float score_scale) {
  t.unit = score_scale;
  const u32x4 zero = {0, 0, 0, 0};
#pragma unroll
  for (int c = 0; c < DC; ++c)
#pragma unroll
    for (int j = 0; j < 2; ++j) t.v[c][j] = there ? row.v[c][j] : zero;
  if constexpr (T::kDtype == MUI_DTYPE_BF16) {
    float most = 0.f;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x[8];
        unpack8<T>(t.v[c][j], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[i]));
      }
    most = rows_max(most);
    int e = (int)((__float_as_uint(most) >> 23) & 0xff) - 126 - 8;  // |x| 2^-e < 2^8
    e = e < -110 ? -110 : (e > 119 ? 119 : e);
    t.unit = exp2i(e) * score_scale;
    const float inv = exp2i(-e);
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x[8];
        unpack8<T>(t.v[c][j], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= inv;
        t.v[c][j] = pack8<T>(x);
      }
  }
}

// One tile of 64 keys. A chunk of 1 KB is one operand of a wave: lane (row l % 16, g) has chunk g of the row's 64 bytes.
template <int DC>
struct KvRegs {
  u32x4 kr[4 * DC], vr[4 * DC];
  __device__ __forceinline__ void load(const uint8_t* kp, const uint8_t* vp, int lane) {
    const int at = (lane & 15) * 64 + (lane >> 4) * 16;
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) kr[i] = ld16_stream(kp + i * 1024 + at);
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) vr[i] = ld16_stream(vp + i * 1024 + at);
  }
};
// 0xff in the bytes of a dword of codes that are NaN
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t a = (w & 0x7f7f7f7fu) + 0x01010101u;  // 0x80 where the code is NaN
  return ((a & 0x80808080u) >> 7) * 0xffu;
}

// Which of a tile's keys first_key .. + 63 a query at `pos` sees, a bit each; from key 4 g on.
__device__ __forceinline__ unsigned long long seen_keys(long first_key, long pos, long length, int window, int keep, int g) {
  auto below = [](long n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; };  // keys first_key .. + n - 1
  unsigned long long m = below((pos + 1 < length ? pos + 1 : length) - first_key);
  if (window > 0) m &= ~below(pos - window + 1 - first_key) | below(keep - first_key);
  return m >> (4 * g);
}

// keys 16 i + 4 g + r of a tile that a query sees: bit 4 i + r
__device__ __forceinline__ uint32_t seen_bits(long first_key, long pos, long length, int window, int keep, int g) {
  const unsigned long long m = seen_keys(first_key, pos, length, window, keep, g);
  return (uint32_t)(m & 0xf) | (uint32_t)(m >> 16 & 0xf) << 4 | (uint32_t)(m >> 32 & 0xf) << 8 | (uint32_t)(m >> 48 & 0xf) << 12;
}

// x *= f where it stands: a multiplication behind a branch would have the compiler copy every result on the other way round it. What it does not see into it does not
// space from others either, so between_matrix() stands in front of such products, behind the instructions that make f, and behind them: 24 waits cover a matrix
// instruction that writes x (16 passes: 19) and the exponential that gives f (1).
__device__ __forceinline__ void between_matrix() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void times_here(f32x4& x, float f) {
  float a = x[0], b = x[1], c = x[2], d = x[3];
  asm volatile("v_mul_f32 %0, %4, %0\n\tv_mul_f32 %1, %4, %1\n\tv_mul_f32 %2, %4, %2\n\tv_mul_f32 %3, %4, %3" : "+v"(a), "+v"(b), "+v"(c), "+v"(d) : "v"(f));
  x = f32x4{a, b, c, d};
}

// What a tile's score products are multiplied by. Not 0, which a query and keys of zeros would make it (2^-120 is a page's scale then): a hidden key's score is -inf. Nor
// infinite, which products of 0 would make NaN.
__device__ __forceinline__ float score_unit(float query, float keys) { return __builtin_amdgcn_fmed3f(query * keys, 0x1p-126f, -kNoMax); }

// Scores so far from zero that what a fused product keeps and a maximum has rounded away counts in an exponential: they are rounded first.
__device__ __forceinline__ bool is_far(float most) { return fabsf(most) >= 0x1p22f && most > kNoMax; }

// The running result of 16 columns: lane (column, g) has dimensions 16 i + 4 g + r.
template <int DC>
struct Columns {
  f32x4 o[4 * DC];
  f32x4 l;  // the sum of the probabilities, as they went into the products: four times the same
  float m;  // the maximum, a whole number of powers of two
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    l = f32x4{0.f, 0.f, 0.f, 0.f};
    m = kNoMax;
  }
};

// The tile's scores and values into the results of 16 columns. pos: the lane's column's position (-1: no column); first_key: key 0 of the tile;
// whole: every column sees all 64 keys. `ks`, `vs`: the page's scales.
template <typename T, int DC>
__device__ __forceinline__ void attend_tile(Columns<DC>& c, const QueryTile<DC>& q, const KvRegs<DC>& kv, float ks, float vs, bool whole, long first_key, long pos,
                                            long length, int window, int keep, int g) {
  f32x4 s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int cc = 0; cc < DC; ++cc) {
      const u32x4 k = kv.kr[4 * cc + i];
      s[i] = mfma16x16x32<T>(widen8<T>(k.x, k.y), q.v[cc][0], s[i]);
      s[i] = mfma16x16x32<T>(widen8<T>(k.z, k.w), q.v[cc][1], s[i]);
    }
  }
  uint32_t seen = 0xffffu;
  if (!whole) {
    seen = seen_bits(first_key, pos, length, window, keep, g);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[i][r] = seen >> (4 * i + r) & 1u ? s[i][r] : -INFINITY;
  }
  float unit = score_unit(q.unit, ks);
  float most = s[0][0];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) most = fmaxf(most, s[i][r]);
  most = rows_max(most) * unit;
  const float mt = fmaxf(ceilf(most), kNoMax);
  if (__any(is_far(mt))) {
#pragma unroll
    for (int i = 0; i < 4; ++i) times_here(s[i], unit);
    unit = 1.f;
  }
  if (__any(mt > c.m)) {
    const float to = fmaxf(c.m, mt), f = __builtin_amdgcn_exp2f(c.m - to);
    c.m = to;
    c.l *= f;
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) c.o[i] *= f;
  }
  // probabilities of the tile, its largest in (2^13, 2^14]
  const float base = fabsf(mt) < 0x1p24f ? mt - 14.f : mt;  // (beyond, the difference would be rounded)
  u32x4 hi[2], lo[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float e[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], unit, -base));
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      const uint32_t w = F16::pack2(e[r], e[r + 1]);
      hi[i >> 1][2 * (i & 1) + r / 2] = w;
      lo[i >> 1][2 * (i & 1) + r / 2] = F16::pack2(e[r] - F16::lo(w), e[r + 1] - F16::hi(w));
    }
  }
  const int down = (int)fmaxf(base - c.m, -300.f);
  const float f = __builtin_amdgcn_ldexpf(vs, down);
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const u32x4 ones = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
  auto product = [&](u32x4 v0, u32x4 v1) {
    f32x4 t = mfma16x16x32<F16>(v0, lo[0], zero);
    t = mfma16x16x32<F16>(v1, lo[1], t);
    t = mfma16x16x32<F16>(v0, hi[0], t);
    return mfma16x16x32<F16>(v1, hi[1], t);
  };
  c.l += product(ones, ones) * __builtin_amdgcn_ldexpf(1.f, down);
  // Where part of the tile is hidden, what stands there may be anything, and 0 * NaN is NaN.
  bool nan = false;
  if (!whole) {
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) {
      const u32x4 v = kv.vr[i];
      found |= nan_bytes(v.x) | nan_bytes(v.y) | nan_bytes(v.z) | nan_bytes(v.w);
      __builtin_amdgcn_sched_barrier(0);  // (one chunk at a time here and below: kept apart, these rare steps cost the others no registers)
    }
    nan = __any(found != 0);
  }
  if (!nan) {
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) c.o[i] += product(widen8<F16>(kv.vr[i].x, kv.vr[i].y), widen8<F16>(kv.vr[i].z, kv.vr[i].w)) * f;
    return;
  }
  // A NaN code counts as zero, and a column that sees it gets a NaN.
  const u32x4 none = {0, 0, 0, 0};
  u32x4 mine;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) w |= seen >> (4 * i + r) & 1u ? 0x38u << (8 * r) : 0u;
    mine[i] = w;
  }
#pragma unroll
  for (int i = 0; i < 4 * DC; ++i) {
    __builtin_amdgcn_sched_barrier(0);
    u32x4 v = kv.vr[i], x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = nan_bytes(v[j]);
      v[j] &= ~x[j];
      x[j] &= 0x38383838u;
    }
    c.o[i] += product(widen8<F16>(v.x, v.y), widen8<F16>(v.z, v.w)) * f;
    const f32x4 sees = mfma_e4m3(pair8(x, none), pair8(mine, none), zero);
#pragma unroll
    for (int r = 0; r < 4; ++r) c.o[i][r] = sees[r] > 0.f ? __builtin_nanf("") : c.o[i][r];
  }
  __builtin_amdgcn_sched_barrier(0);
}

// The columns of a block: new tokens times heads of a KV head's group, `per` from number `block * per` on.
struct ColumnBlock {
  int first, end;        // columns
  long pos0, pos1;       // positions of the first and the last
  TileRange range;
};
__device__ __forceinline__ ColumnBlock column_block(const PagedAttnParams& p, const PagedSpan& sp, int block, int per) {
  ColumnBlock b;
  const int n_cols = sp.count * p.group;  // (at most n_rows times heads, which fits)
  b.first = block * per;
  b.end = n_cols - b.first > per ? b.first + per : n_cols;
  b.pos0 = sp.start + (unsigned)b.first / (unsigned)p.group;
  b.pos1 = sp.start + (unsigned)(b.end - 1) / (unsigned)p.group;
  b.range = tile_range(p, b.pos0, b.pos1, sp.length);
  return b;
}

// where a tile lies, and its page's scales
struct TilePlace { long at; float ks, vs; };
__device__ __forceinline__ TilePlace tile_place(const PagedAttnParams& p, int page, int tile, int h) {
  if (page < 0) return {0, 1.f, 1.f};
  const int per_page = p.t.page_shift - 6;
  const long ph = (long)page * p.kv_heads + h;
  return {(ph << per_page) + (tile & ((1 << per_page) - 1)), p.ks[ph], p.vs[ph]};
}
__device__ __forceinline__ bool sees_whole(const PagedAttnParams& p, long k0, long pos0, long pos1, long length) {
  return k0 + 63 <= pos0 && k0 + 64 <= length && (p.window <= 0 || k0 > pos1 - p.window || k0 + 64 <= p.keep);
}

// A request's tiles of 64 keys that any of its new tokens sees (at least one, so that a token without keys gets its zeros) and its blocks of 16 columns; not
// more than the host has been told, so that the sums over all requests fit.
struct RequestWork { int tiles, blocks; };
__device__ __forceinline__ RequestWork request_work(const PagedAttnParams& p, const PagedSpan& sp) {
  RequestWork w = {0, (sp.count * p.group + 15) / 16};
  if (sp.count > 0) w.tiles = tile_range(p, sp.start, sp.start + sp.count - 1, sp.length).count();
  w.tiles = w.tiles < 1 ? 1 : w.tiles < p.split_tiles ? w.tiles : p.split_tiles;
  w.blocks = w.blocks < p.col_tiles ? w.blocks : p.col_tiles;
  return w;
}

// lane l's, in scalar registers
__device__ __forceinline__ PagedSpan span_of_lane(const PagedSpan& s, int l) {
  auto of = [l](int x) { return __builtin_amdgcn_readlane(x, l); };
  auto of_long = [&](long x) { return (long)((unsigned long long)(uint32_t)of((int)(x >> 32)) << 32 | (uint32_t)of((int)(x & 0xffffffffL))); };
  return {of(s.row0), of(s.count), of_long(s.start), of_long(s.length)};
}

// Single tokens, and several. A unit is 16 columns of one KV head and request. All tiles of all units, one after another, are dealt out to the workgroups in
// equal shares, whatever the requests' lengths: the units that a share cuts are joined by a second launch. (Short caches: a workgroup per unit, nothing to join.) The waves of
// a workgroup take every W-th tile each and meet in LDS. Two waves on a SIMD keep the memory busy, 16 KB on the way for each (128 dimensions): with the next tile requested
// while one is worked on as well their registers do not suffice (64 requests of 4096 to 16384 tokens 204 instead of 187 us).
// The cache's bytes bound it where there are many: those 64 requests, 8 KV heads of 128 dimensions (1.17 GB), 186 us, 6.2 TB/s; 32 requests of 200 to 4096 (90 MB) 27.8. With few it is the loads that
// wait for one another (length, page, keys and values, again for each tile of a wave): 700 keys 9.0 us.
template <typename T, int DC, int W>
__global__ void __launch_bounds__(64 * W, DC == 4 ? W / 4 : 2) paged_columns_kernel(const PagedAttnParams p) {
  constexpr int D = DC * 64, kThreads = 64 * W;
  __shared__ float so[W][16][D + 4];
  __shared__ float sm[W][16], sl[W][16];
  __shared__ int before[kDealtRequests + 1];  // tiles of the units of the requests in front of each
  __shared__ int wave_sum[W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  int b, unit = 0, tile0 = 0, share_begin = 0, share_end = 0, share = 0;
  if (p.part) {
    int to = 0;
    const bool few = p.t.n_requests <= kWave;  // a request a lane, and every wave for itself
    if (few) {
      if (lane < p.t.n_requests) {
        const RequestWork w = request_work(p, paged_span(p.t, lane));
        to = w.tiles * w.blocks * p.kv_heads;
      }
      to = (int)wave_scan((uint32_t)to);
      if (lane < p.t.n_requests) before[lane + 1] = to;  // (the same from all waves)
    } else {
      int mine[kDealtRequests / kThreads], sum = 0;
#pragma unroll
      for (int k = 0; k < kDealtRequests / kThreads; ++k) {
        const int r = threadIdx.x * (kDealtRequests / kThreads) + k;
        if (r < p.t.n_requests) {
          const RequestWork w = request_work(p, paged_span(p.t, r));
          sum += w.tiles * w.blocks * p.kv_heads;
        }
        mine[k] = sum;
      }
      to = (int)wave_scan((uint32_t)sum);
      if (lane == 63) wave_sum[wave] = to;
      __syncthreads();
      int base = to - sum;
      for (int w = 0; w < wave; ++w) base += wave_sum[w];
#pragma unroll
      for (int k = 0; k < kDealtRequests / kThreads; ++k) before[threadIdx.x * (kDealtRequests / kThreads) + k + 1] = base + mine[k];
      __syncthreads();
    }
    if (lane == 0) before[0] = 0;  // (of every wave, too)
    const int total = uniform(before[p.t.n_requests]);
    share = uniform(share_of(total, gridDim.x, W));
    if (blockIdx.x == 0)  // for the joining launch (of few requests by every wave, which has them all)
      for (int i = few ? lane : threadIdx.x; i <= p.t.n_requests; i += few ? kWave : kThreads) p.before[i] = before[i];
    share_begin = (int)blockIdx.x * share;  // (share * workgroups < total + workgroups, which the host has checked)
    share_end = total - share_begin < share ? total : share_begin + share;
    if (share_begin >= total) return;
    // the last request that begins at or before the share
    if (few) {
      b = __ffsll((long long)__ballot(to > share_begin)) - 1;
    } else {
      int lo = 0, hi = p.t.n_requests;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= share_begin) lo = mid; else hi = mid;
      }
      b = uniform(lo);
    }
    unit = share_begin - uniform(before[b]);
  } else {
    unit = blockIdx.x % (p.kv_heads * p.col_tiles);
    b = blockIdx.x / (p.kv_heads * p.col_tiles);
  }
  PagedSpan sp = uniform(paged_span(p.t, b));
  RequestWork work = request_work(p, sp);
  int done = share_begin;
  if (p.part) {
    const int in = unit;
    unit = uniform(in / work.tiles);
    tile0 = in - unit * work.tiles;
  } else if (unit >= work.blocks * p.kv_heads) {
    return;
  }
  const int per_page = p.t.page_shift - 6;
  while (true) {
    // the unit's tiles tile0 .. tile0 + n - 1
    const int n = p.part && share_end - done < work.tiles - tile0 ? share_end - done : work.tiles - tile0;
    const bool all = n == work.tiles;
    const int h = unit % p.kv_heads;
    const ColumnBlock cb = column_block(p, sp, unit / p.kv_heads, 16);
    const TileRange range = tile_range(p, sp.start, sp.start + sp.count - 1, sp.length);  // of the request
    const int end = tile0 + n < range.count() ? tile0 + n : range.count();
    const int col = cb.first + (lane & 15);
    const bool there = col < cb.end;
    const int token = (unsigned)(there ? col : cb.end - 1) / (unsigned)p.group, head = h * p.group + (there ? col : cb.end - 1) - token * p.group;
    const long pos = there ? sp.start + token : -1;
    const QueryRow<DC> query = request_queries<DC>(p.q + (long)(sp.row0 + token) * p.q_tok + (long)head * p.q_head, g);
    Columns<DC> c;
    c.clear();
    auto page_of = [&](int i) { return i < end ? paged_page(p.t, b, range.at(i) >> per_page) : -1; };
    KvRegs<DC> t;
    int page = page_of(tile0 + wave);
    TilePlace at = tile_place(p, page, range.at(tile0 + wave), h);
    if (page >= 0) t.load(p.kp + at.at * (64 * D), p.vp + at.at * (64 * D), lane);
    QueryTile<DC> q;
    take_queries<T, DC>(q, query, there, p.scale);
    for (int i = tile0 + wave; i < end; i += W) {
      const int page1 = page_of(i + W);
      if (page >= 0) {
        const long k0 = 64L * range.at(i);
        attend_tile<T, DC>(c, q, t, at.ks, at.vs, sees_whole(p, k0, cb.pos0, cb.pos1, sp.length), k0, pos, sp.length, p.window, p.keep, g);
      }
      page = page1;
      at = tile_place(p, page, range.at(i + W), h);
      if (page >= 0) t.load(p.kp + at.at * (64 * D), p.vp + at.at * (64 * D), lane);
    }
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) *(f32x4*)&so[wave][lane & 15][16 * i + 4 * g] = c.o[i];
    if (g == 0) { sm[wave][lane & 15] = c.m; sl[wave][lane & 15] = c.l[0]; }
    __syncthreads();
    const int cc = threadIdx.x / (4 * W), in = threadIdx.x % (4 * W), my = cb.first + cc;  // 4 W threads per column
    if (my < cb.end) {
      float m = sm[0][cc];
#pragma unroll
      for (int w = 1; w < W; ++w) m = fmaxf(m, sm[w][cc]);
      float f[W], sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        f[w] = __builtin_amdgcn_exp2f(sm[w][cc] - m);
        sum += f[w] * sl[w][cc];
      }
      const int my_token = (unsigned)my / (unsigned)p.group, my_head = h * p.group + my - my_token * p.group;
      const long row = (long)(sp.row0 + my_token) * p.heads + my_head;
      const float inv = !all ? 1.f : (sum > 0.f || sum != sum ? 1.f / sum : 0.f);
      // (a share cuts two units at most: the one it begins with and the one it ends with)
      float* part = all ? nullptr : p.part + (((long)blockIdx.x * 2 + (done == share_begin ? 0 : 1)) * 16 + cc) * (D + 4);
      for (int d = 4 * in; d < D; d += 16 * W) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) o += f[w] * *(const f32x4*)&so[w][cc][d];
        o *= inv;
        if (all) *(u32x2*)(p.out + row * D + d) = u32x2{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])};
        else *(f32x4*)(part + d) = o;
      }
      if (!all && in == 0) { part[D] = m; part[D + 1] = sum; }
    }
    done += n;
    if (!p.part || done >= share_end) return;
    __syncthreads();
    tile0 = 0;
    if (++unit == work.blocks * p.kv_heads) {
      unit = 0;
      do ++b; while (uniform(before[b + 1]) <= done);  // (requests without new tokens)
      sp = uniform(paged_span(p.t, b));
      work = request_work(p, sp);
    }
  }
}

// The units that shares have cut: a wave per row and head adds its parts up (4 us: where its parts begin, the parts, and the launch).
template <typename T, int DC>
__global__ void __launch_bounds__(256) paged_join_units_kernel(const PagedAttnParams p, int workgroups, int waves) {
  constexpr int D = DC * 64;
  const int lane = threadIdx.x & 63;
  const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (long)p.t.n_rows * p.heads) return;
  const int row = (int)(item / p.heads), head = (int)(item % p.heads);
  const int b = request_of_wave(p.t, row);
  const PagedSpan sp = paged_span(p.t, b);
  if (row < sp.row0 || row >= sp.row0 + sp.count) return;
  const int col = (row - sp.row0) * p.group + head % p.group;
  int blocks = (sp.count * p.group + 15) / 16;
  blocks = blocks < p.col_tiles ? blocks : p.col_tiles;
  if (col >= 16 * blocks) return;
  const int first = p.before[b], tiles = (p.before[b + 1] - first) / (blocks * p.kv_heads);
  const int begin = first + (col / 16 * p.kv_heads + head / p.group) * tiles;
  const int share = share_of(p.before[p.t.n_requests], workgroups, waves);
  const int w0 = begin / share, w1 = (begin + tiles - 1) / share;
  if (w0 == w1) return;  // done by one
  float m = kNoMax, sum = 0.f, o[DC] = {};
  constexpr int kAtOnce = 4;
  for (int w = w0; w <= w1; w += kAtOnce) {
    float pm[kAtOnce], ps[kAtOnce], po[kAtOnce][DC];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int x = w + k <= w1 ? w + k : w1;
      const float* part = p.part + (((long)x * 2 + (x * share >= begin ? 0 : 1)) * 16 + col % 16) * (D + 4);
      pm[k] = part[D];
      ps[k] = part[D + 1];
#pragma unroll
      for (int j = 0; j < DC; ++j) po[k][j] = part[64 * j + lane];
    }
    float to = m;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) to = fmaxf(to, pm[k]);
    const float f0 = __builtin_amdgcn_exp2f(m - to);
    m = to;
    sum *= f0;
#pragma unroll
    for (int j = 0; j < DC; ++j) o[j] *= f0;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const float f = w + k <= w1 ? __builtin_amdgcn_exp2f(pm[k] - m) : 0.f;
      sum += f * ps[k];
#pragma unroll
      for (int j = 0; j < DC; ++j) o[j] += w + k <= w1 ? f * po[k][j] : 0.f;
    }
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
  for (int j = 0; j < DC; ++j) p.out[item * D + 64 * j + lane] = T::pack(o[j] * inv);
}

// ---------------------------------------------------------------------------------------
// prompts
// ---------------------------------------------------------------------------------------
// Codes are widened once for the workgroup, on their way to LDS: keys to the queries' type, values to fp16 (keys widened by every
// wave behind LDS, 8 KB less of it to read per tile, took 6 % longer). A probability is taken relative to a power of two that moves only if a maximum passes it by kRoom, so that the largest are 2^7 to
// 2^15; what is 2^-21 of the largest still has all its bits in one piece.
constexpr float kBias = 7.f, kRoom = 8.f;

template <int DC>
struct PromptColumns {
  f32x4 o[4 * DC];
  f32x4 l;      // the sum of the probabilities, as they went into the products: four times the same
  float m, to;  // what probabilities are relative to: 2^m; kBias - m
};

// a tile in LDS as a wave's lanes have its operands: keys in the queries' type (chunk i: 16 keys and 64 dimensions, in halves), values in fp16 (16 dimensions, 32 keys)
struct PromptTile {
  const u32x4* kp; const u32x4* vp;
  __device__ __forceinline__ u32x4 k(int i, int half) const { return kp[(2 * i + half) * 64]; }
  __device__ __forceinline__ u32x4 v(int i, int half) const { return vp[(2 * i + half) * 64]; }
};

// scores of a tile
template <typename T, int DC, int NT>
__device__ __forceinline__ void prompt_scores(f32x4 (&s)[NT][4], const QueryTile<DC> (&q)[NT], const PromptTile& t) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {  // (two chunks' products between one product and the next on its result)
#pragma unroll
    for (int c = 0; c < DC; ++c) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        u32x4 kk[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) kk[x] = t.k(4 * c + i + x, j);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int n = 0; n < NT; ++n) s[n][i + x] = mfma16x16x32<T>(kk[x], q[n].v[c][j], c || j ? s[n][i + x] : f32x4{0.f, 0.f, 0.f, 0.f});
      }
    }
  }
}

// The reference of the probabilities moves where the tile's largest score (of this lane's keys) passes it by kRoom.
template <int DC, int NT>
__device__ __forceinline__ void prompt_move(PromptColumns<DC> (&c)[NT], const float (&most)[NT], f32x4 (&s)[NT][4], float (&unit)[NT]) {
  bool moves = false, far = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    moves |= most[n] > c[n].m + kRoom;
    far |= is_far(most[n]);
  }
  if (__any(far)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) times_here(s[n][i], unit[n]);
      unit[n] = 1.f;
    }
  }
  if (__any(moves)) {
    float f[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {  // (a column's four lanes move together)
      const float mt = fmaxf(ceilf(rows_max(most[n])), kNoMax), to = mt > c[n].m + kRoom ? mt : c[n].m;
      f[n] = __builtin_amdgcn_exp2f(c[n].m - to);
      c[n].m = to;
      c[n].to = fabsf(to) < 0x1p24f ? kBias - to : -to;  // (beyond, the sum would be rounded)
    }
    between_matrix();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      times_here(c[n].l, f[n]);
#pragma unroll
      for (int i = 0; i < 4 * DC; ++i) times_here(c[n].o[i], f[n]);
    }
    between_matrix();
  }
}

template <int NT>
__device__ __forceinline__ void prompt_most(float (&most)[NT], const f32x4 (&s)[NT][4]) {
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    most[n] = s[n][0][0];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) most[n] = fmaxf(most[n], s[n][i][r]);
  }
}

// probabilities of a tile, in `PIECES` pieces: unit = what its scores are multiplied by
template <int DC, int PIECES, int NT>
__device__ __forceinline__ void prompt_exp(u32x4 (&pp)[NT][PIECES][2], const f32x4 (&s)[NT][4], const PromptColumns<DC> (&c)[NT], const float (&unit)[NT]) {
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float e[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[n][i][r], unit[n], c[n].to));
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const uint32_t w = F16::pack2(e[r], e[r + 1]);
        pp[n][0][i >> 1][2 * (i & 1) + r / 2] = w;
        if constexpr (PIECES == 2) pp[n][1][i >> 1][2 * (i & 1) + r / 2] = F16::pack2(e[r] - F16::lo(w), e[r + 1] - F16::hi(w));
      }
    }
}

template <int DC, int PIECES, int NT>
__device__ __forceinline__ void prompt_values(PromptColumns<DC> (&c)[NT], const u32x4 (&pp)[NT][PIECES][2], const PromptTile& t) {
  const u32x4 ones = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n) c[n].l = mfma16x16x32<F16>(ones, pp[n][k][half], c[n].l);
#pragma unroll
  for (int i = 0; i < 4 * DC; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const u32x4 v = t.v(i, half);
#pragma unroll
      for (int k = 0; k < PIECES; ++k)
#pragma unroll
        for (int n = 0; n < NT; ++n) c[n].o[i] = mfma16x16x32<F16>(v, pp[n][k][half], c[n].o[i]);
    }
}

// Where part of a tile is hidden its NaN codes have gone into the products as zeros, since 0 * NaN is NaN: here the columns that see one get a NaN. v: the tile's values.
template <int DC, int NT>
__device__ __forceinline__ void prompt_nans(PromptColumns<DC> (&c)[NT], const uint8_t* v, const uint32_t (&seen)[NT]) {
  const u32x4 zero = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 4 * DC; ++i) {
    __builtin_amdgcn_sched_barrier(0);  // (one chunk at a time: kept apart, these rare steps cost the others no registers)
    u32x4 x = ld16(v + i * 1024);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = nan_bytes(x[j]) & 0x38383838u;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      u32x4 mine;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t w = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) w |= seen[n] >> (4 * k + r) & 1u ? 0x38u << (8 * r) : 0u;
        mine[k] = w;
      }
      const f32x4 sees = mfma_e4m3(pair8(x, zero), pair8(mine, zero), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int r = 0; r < 4; ++r) c[n].o[i][r] = sees[r] > 0.f ? __builtin_nanf("") : c[n].o[i][r];
    }
  }
  __builtin_amdgcn_sched_barrier(0);
}

// The requests' blocks of PER columns, those first whose last column stands furthest behind (it sees most keys; of 64 requests at a time): the n-th one's request, number and
// the request's rows. Every wave looks for itself, a request a lane. A block's place is counted in blocks too: the request's tokens times heads, and down from there. A request that
// has more blocks than the host has been told keeps its first ones: the others' are all found among those that were launched.
template <int PER>
__device__ __forceinline__ bool nth_block(const PagedAttnParams& p, int n, int& b, int& block, PagedSpan& sp) {
  const int lane = threadIdx.x & 63;
  auto of = [](int x, int l) { return __builtin_amdgcn_readlane(x, l); };
  for (int r0 = 0; r0 < p.t.n_requests; r0 += kWave) {
    PagedSpan s = {};
    int blocks = 0, top = 0;
    if (r0 + lane < p.t.n_requests) {
      s = paged_span(p.t, r0 + lane);
      blocks = (s.count * p.group + PER - 1) / PER;
      const long last = s.length * p.group / PER;
      top = last < (1 << 30) ? (int)last : 1 << 30;
      const int over = blocks - p.col_tiles;
      if (over > 0) {
        top -= over;
        blocks = p.col_tiles;
      }
    }
    const int here = p.t.n_requests - r0 < kWave ? p.t.n_requests - r0 : kWave;
    int total = 0, high = 0, low = 1 << 30;  // the places there are
    for (int r = 0; r < here; ++r) {
      const int t = of(top, r), m = of(blocks, r);
      total += m;
      high = t > high ? t : high;
      low = m && t - m + 1 < low ? t - m + 1 : low;
    }
    if (n >= total) {
      n -= total;
      continue;
    }
    // the last place from which on there are more than n blocks, a place a lane
    int step, front = 0;  // front: blocks behind it
    do {
      step = (high - low) / kWave + 1;
      const int place = low + lane * step;
      int from = 0, behind = 0;
      for (int r = 0; r < here; ++r) {
        const int mine = of(top, r) - place + 1, m = of(blocks, r);
        from += mine < 0 ? 0 : mine < m ? mine : m;
        behind += mine < 1 ? 0 : mine - 1 < m ? mine - 1 : m;
      }
      const int last = 63 - __clzll((long long)__ballot(from > n));
      front = of(behind, last);
      low += last * step;
      high = low + step - 1;
    } while (step > 1);
    n -= front;
    const int down = top - low;
    const unsigned long long at = __ballot(down >= 0 && down < blocks);
    const int l = __ffsll((long long)__ballot((at >> lane & 1ull) && __popcll(at & ((1ull << lane) - 1ull)) == n)) - 1;
    b = r0 + l;
    block = of(blocks - 1 - down, l);
    sp = span_of_lane(s, l);
    return true;
  }
  return false;
}

// A workgroup of four waves takes 64 NT columns of one KV head (16 NT a wave) and `split_tiles` tiles, which its waves share through LDS: two tiles' room, the
// next ones on their way to registers while the waves work on one, one barrier a tile. Two such workgroups on a CU (one of 256 dimensions).
// 2048 tokens behind 6144, 32 query and 8 KV heads of 128 bf16 dimensions (240 GFLOP): 255 us, 0.94 PFLOP/s. The matrix instructions alone (1088 cycles of a SIMD for a
// wave's 32 columns and a tile) take half of that at the clock that the card keeps under them; the rest is the tile's way through LDS (32 KB for each wave), exponentials and maxima.
template <typename T, int DC, int NT>
__global__ void __launch_bounds__(256, DC == 4 ? 1 : 2) paged_tiles_kernel(const PagedAttnParams p) {
  constexpr int D = DC * 64, kCols = 64 * NT;
  constexpr int kPieces = T::kDtype == MUI_DTYPE_F16 ? 2 : 1;
  __shared__ u32x4 keys[2][64 * D / 8], values[2][64 * D / 8];
  __shared__ int nan_tile[2];  // number of the tile + 1 where its values hold a NaN (looked for, and taken out, where not every column sees all of it)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x % p.kv_heads;  // (neighbours go to different XCDs: of eight heads each XCD has one, whose keys stay in its L2)
  int b, ct;
  PagedSpan sp;
  if (!nth_block<kCols>(p, blockIdx.x / p.kv_heads, b, ct, sp)) return;
  const ColumnBlock cb = column_block(p, sp, ct, kCols);
  const int n_tiles = cb.range.count();
  const int begin = blockIdx.y * p.split_tiles;
  if (begin >= n_tiles && begin > 0) return;
  const int end = begin + p.split_tiles < n_tiles ? begin + p.split_tiles : n_tiles;
  const int g = lane >> 4;
  if (threadIdx.x < 2) nan_tile[threadIdx.x] = 0;
  QueryTile<DC> q[NT];
  PromptColumns<DC> c[NT];
  int token[NT];  // of the request's new ones, the lane's columns'; -1: no column
  const int wave_col = cb.first + wave * (16 * NT);
  const bool mine = wave_col < cb.end;
  const int wave_end = wave_col + 16 * NT < cb.end ? wave_col + 16 * NT : cb.end;
  const long my_pos1 = sp.start + (unsigned)(mine ? wave_end - 1 : cb.end - 1) / (unsigned)p.group;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = wave_col + 16 * n + (lane & 15);
    const bool there = col < cb.end;
    const unsigned at = there ? col : cb.end - 1, tok = at / (unsigned)p.group, head = at - tok * p.group;
    token[n] = there ? (int)tok : -1;
    take_queries<T, DC>(q[n], request_queries<DC>(p.q + (long)(sp.row0 + (int)tok) * p.q_tok + (long)(h * p.group + (int)head) * p.q_head, g), there, p.scale);
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) c[n].o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    c[n].l = f32x4{0.f, 0.f, 0.f, 0.f};
    c[n].m = kNoMax;
    c[n].to = -kNoMax;
  }
  const int per_page = p.t.page_shift - 6;
  const int lane_at = (lane & 15) * 64 + (lane >> 4) * 16;
  // a tile's page is loaded a tile before it is looked at: what follows would wait for it
  auto entry_of = [&](int i) { return i < end ? paged_entry(p.t, b, cb.range.at(i) >> per_page) : -1; };
  auto page_of = [&](int entry) { return uniform(page_of_entry(p.t, entry)); };
  u32x4 rawk[DC];
  auto fetch_keys = [&](const TilePlace& at) {
#pragma unroll
    for (int i = 0; i < DC; ++i) rawk[i] = ld16(p.kp + at.at * (64 * D) + (wave * DC + i) * 1024 + lane_at);
  };
  auto put_keys = [&](int slot) {
#pragma unroll
    for (int i = 0; i < DC; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) keys[slot][((wave * DC + i) * 2 + half) * 64 + lane] = widen8<T>(rawk[i][2 * half], rawk[i][2 * half + 1]);
  };
  u32x4 raw[DC];
  auto fetch_values = [&](const TilePlace& at) {
#pragma unroll
    for (int i = 0; i < DC; ++i) raw[i] = ld16(p.vp + at.at * (64 * D) + (wave * DC + i) * 1024 + lane_at);
  };
  // tiles that all columns see: in front of the first's end and, with a window, in it for the last, or among the first keys
  const long whole_end = cb.pos0 + 1 < sp.length ? (cb.pos0 + 1) >> 6 : sp.length >> 6;
  const int seen_end = whole_end < 0 ? 0 : (int)whole_end, seen_kept = p.keep >> 6;
  const int seen_from = p.window > 0 ? (int)((cb.pos1 - p.window) >> 6) + 1 : 0;
  auto all_seen = [&](int tile_no) {
    const int t = cb.range.at(tile_no);
    return t < seen_end && (t >= seen_from || t < seen_kept);
  };
  // The sums of values are relative to 2^level, and fp16 holds a page's values times 2^(7 - level): all codes exactly down to 2^22 below the level, which follows louder pages at once and
  // quieter ones where they would lose bits, but not further than 2^60 below the loudest (what has been added up fits 2^62 relative to that). It begins where 2^(level - 7) is still normal.
  int level = -119, loudest = -119;
  auto put_values = [&](const TilePlace& at, int slot, int tile_no, auto whole) {
    if (!decltype(whole)::value && !all_seen(tile_no)) {
      uint32_t found = 0;
#pragma unroll
      for (int i = 0; i < DC; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t n = nan_bytes(raw[i][j]);
          found |= n;
          raw[i][j] &= ~n;
        }
      if (__any(found != 0) && lane == 0) nan_tile[slot] = tile_no + 1;
    }
    const int e = scale_exponent(at.vs);
    if (e > level || e < level - 22) {
      loudest = e > loudest ? e : loudest;
      const int least = loudest - 60 > -119 ? loudest - 60 : -119, to = e > least ? e : least;
      if (to != level) {
        const float f = exp2i(level - to < -126 ? -126 : level - to);
        between_matrix();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4 * DC; ++i) times_here(c[n].o[i], f);
        between_matrix();
        level = to;
      }
    }
    const float s = exp2i(e - level + 7 < -126 ? -126 : e - level + 7);
#pragma unroll
    for (int i = 0; i < DC; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t a = raw[i][2 * half], d = raw[i][2 * half + 1];
        values[slot][((wave * DC + i) * 2 + half) * 64 + lane] = u32x4{scaled2(a, s, false), scaled2(a, s, true), scaled2(d, s, false), scaled2(d, s, true)};
      }
  };
  // Tile i's probabilities and value products go with tile i + 1's scores: while the vector ALU takes exponentials the matrix cores have products that wait for nothing.
  // A step begins with tile i's scores in registers, its values in LDS or about to be, tile i + 1's keys on their way to LDS.
  int page = page_of(entry_of(begin)), page1 = page_of(entry_of(begin + 1)), entry2 = entry_of(begin + 2);
  TilePlace at = tile_place(p, page, cb.range.at(begin), h), at1 = tile_place(p, page1, cb.range.at(begin + 1), h);
  f32x4 s[NT][4];
  float most[NT], unit[NT];
  __syncthreads();  // (nan_tile)
  if (page >= 0) {
    fetch_keys(at);
    fetch_values(at);
    put_keys(0);
    put_values(at, 0, begin, std::false_type());
  }
  __syncthreads();
  if (page1 >= 0) {
    fetch_keys(at1);
    put_keys(1);
  }
  // scores that may be hidden: tile number, its place in LDS, whether it has a page
  auto masked_scores = [&](int tile_no, int slot, bool there) {
    const long k0 = 64L * cb.range.at(tile_no);
    if (there && mine && k0 <= my_pos1) prompt_scores<T, DC, NT>(s, q, PromptTile{&keys[slot][lane], nullptr});
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint32_t seen = there && mine ? seen_bits(k0, token[n] < 0 ? -1 : sp.start + token[n], sp.length, p.window, p.keep, g) : 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[n][i][r] = seen >> (4 * i + r) & 1u ? s[n][i][r] : -INFINITY;
    }
  };
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (begin < end) {
    masked_scores(begin, 0, page >= 0);
    prompt_most<NT>(most, s);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      unit[n] = score_unit(q[n].unit, at.ks);
      most[n] *= unit[n];
    }
    prompt_move<DC, NT>(c, most, s, unit);
  }
  int i = begin;
  auto step = [&](auto whole) {
    constexpr bool kWhole = decltype(whole)::value;  // all columns see all of tiles i and i + 1
    const int slot = (i - begin) & 1;
    __syncthreads();  // tile i's values and tile i + 1's keys are there, for all; the other rooms' readers are done
    asm volatile("" : "+v"(entry2));  // (not looked at earlier: it would be waited for)
    const int page2 = page_of(entry2);
    entry2 = entry_of(i + 3);
    const TilePlace at2 = tile_place(p, page2, cb.range.at(i + 2), h);
    if (page2 >= 0) fetch_keys(at2);
    if (kWhole || page1 >= 0) fetch_values(at1);
    u32x4 pp[NT][kPieces][2];
    const PromptTile here = {nullptr, &values[slot][lane]}, ahead = {&keys[slot ^ 1][lane], nullptr};
    prompt_exp<DC, kPieces, NT>(pp, s, c, unit);
    if constexpr (kWhole) {
      prompt_scores<T, DC, NT>(s, q, ahead);
      prompt_values<DC, kPieces, NT>(c, pp, here);
    } else {
      if (i + 1 < end) masked_scores(i + 1, slot ^ 1, page1 >= 0);
      const long k0 = 64L * cb.range.at(i);
      if (page >= 0 && mine && k0 <= my_pos1) {
        prompt_values<DC, kPieces, NT>(c, pp, here);
        if (nan_tile[slot] == i + 1) {
          uint32_t seen[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) seen[n] = seen_bits(k0, token[n] < 0 ? -1 : sp.start + token[n], sp.length, p.window, p.keep, g);
          prompt_nans<DC, NT>(c, p.vp + tile_place(p, page, cb.range.at(i), h).at * (64 * D) + lane_at, seen);
        }
      }
    }
    prompt_most<NT>(most, s);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      unit[n] = score_unit(q[n].unit, at1.ks);
      most[n] *= unit[n];
    }
    if (kWhole || page1 >= 0) put_values(at1, slot ^ 1, i + 1, whole);
    if (page2 >= 0) put_keys(slot);
    if (kWhole || i + 1 < end) prompt_move<DC, NT>(c, most, s, unit);
    at1 = at2;
    page = page1;
    page1 = page2;
    ++i;
  };
  // (a loop for tiles that all columns see and one for others: with both in one the compiler copied the results between their registers at every tile)
  auto whole_now = [&]() { return i + 1 < end && page >= 0 && page1 >= 0 && all_seen(i) && all_seen(i + 1); };
  while (i < end) {
    while (whole_now()) step(std::true_type());
    while (i < end && !whole_now()) step(std::false_type());
  }
  const float loud = exp2i(level - 7);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = wave_col + 16 * n + (lane & 15);
    if (col >= cb.end) continue;
    const unsigned token = (unsigned)col / (unsigned)p.group;
    const long row = (long)(sp.row0 + (int)token) * p.heads + h * p.group + (col - (int)token * p.group);
    const float sum = c[n].l[0], inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    if (p.part) {
      float* part = p.part + ((long)blockIdx.y * p.t.n_rows * p.heads + row) * (D + 4);
#pragma unroll
      for (int i = 0; i < 4 * DC; ++i) *(f32x4*)(part + 16 * i + 4 * g) = c[n].o[i] * inv * loud;
      if (g == 0) { part[D] = -c[n].to; part[D + 1] = sum; }
    } else {
#pragma unroll
      for (int i = 0; i < 4 * DC; ++i) {
        const f32x4 o = c[n].o[i] * inv * loud;
        *(u32x2*)(p.out + row * D + 16 * i + 4 * g) = u32x2{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])};
      }
    }
  }
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
  const int b = request_of_wave(p.t, row);
  const PagedSpan sp = paged_span(p.t, b);
  if (row < sp.row0 || row >= sp.row0 + sp.count) return;
  const int col = (row - sp.row0) * p.group + head % p.group;
  if (col / p.block_cols >= p.col_tiles) return;  // (beyond what the host has been told: nobody's work)
  const int n_tiles = column_block(p, sp, col / p.block_cols, p.block_cols).range.count();
  int splits = n_tiles > 0 ? (n_tiles + p.split_tiles - 1) / p.split_tiles : 1;
  splits = splits < p.splits ? splits : p.splits;
  const float* part = p.part + item * (D + 4);
  const long step = n * (D + 4);
  float m = kNoMax;
  for (int i = 0; i < splits; ++i) m = fmaxf(m, part[i * step + D]);
  float sum = 0.f, o[DC] = {};
  for (int i = 0; i < splits; ++i) {
    const float f = __builtin_amdgcn_exp2f(part[i * step + D] - m) * part[i * step + D + 1];
    sum += f;
#pragma unroll
    for (int j = 0; j < DC; ++j) o[j] += f * part[i * step + 64 * j + lane];
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
  for (int j = 0; j < DC; ++j) p.out[item * D + 64 * j + lane] = T::pack(o[j] * inv);
}

struct PagedPlan { int block_cols, col_tiles, split_tiles, splits, waves, workgroups; long blocks; size_t scratch; };
static PagedPlan paged_plan(int n_rows, int n_requests, int max_tokens, int max_length, int window, int keep, int n_q_heads, int n_kv_heads, int head_dim) {
  PagedPlan r = {};
  if (max_tokens > n_rows) max_tokens = n_rows;
  const long group = n_q_heads / n_kv_heads;
  long tiles = ((long)max_length + 63) / 64;
  if (window > 0) {
    const long seen = ((long)window + max_tokens + 62) / 64 + 1 + ((long)keep + 63) / 64;
    tiles = tiles < seen ? tiles : seen;
  }
  if (tiles < 1) tiles = 1;
  // Blocks of `per` columns of a request at most, and of all requests: no more than the rows fill, and one of each request that is not full.
  auto each = [&](int per) { return (max_tokens * group + per - 1) / per; };
  auto all = [&](int per) {
    const long filled = (long)n_rows * group / per + n_requests, most = n_requests * each(per);
    return filled < most ? filled : most;
  };
  const int wide = head_dim == 256 ? 64 : 128;  // (256 dimensions: results of 32 columns a wave do not fit its registers)
  // The kernel for single tokens takes 2.2 ns for a block of 16 columns and a tile, the one for prompts 5 to 6 for a block of 128, and 6 us more to begin with and to join. us, the one / the
  // other, 32 heads, 8 KV heads, 128 bf16 dimensions: one request of 1000 keys and 32 new tokens 12 / 26; of 8000 and 16 24 / 31, 32 33 / 32; 16 requests of 1000 and 16 23 / 34, 32 42 / 39;
  // of 8000 and 4 54 / 92, 8 93 / 96 (fp16 93 / 114, 64 dimensions 41 / 74, 256 138 / 179), 32 281 / 119.
  // A workgroup per unit needs no scan and no joining launch. us, a unit each / dealt out, 8 KV heads, requests of equal lengths, which suit it best: 64 dimensions, 8 requests of 1400 keys
  // 10.6 / 13.6; 128 dimensions, one of 1400 13.4 / 14.7, 30 17.9 / 22.0, one of 2000 15.6 / 12.1, 30 23.7 / 30.7; 256 dimensions, 30 of 800 25.7 / 28.2, 8 of 1400 29.4 / 22.6.
  // Workgroups without work take 8 ns each: a thousand of them are as long as dealing out (16 requests of up to 60 new tokens, 764 of 1728 workgroups with work, 25 / 30).
  const bool sparse = ((long)n_requests * each(16) - all(16)) * n_kv_heads > 1024;
  const bool unit = !sparse && (tiles <= (head_dim == 256 ? 16 : 24) || n_requests > kDealtRequests);
  const bool dealt = !unit && n_requests <= kDealtRequests && (long)n_requests * each(16) <= 0x3fffffffL / tiles / n_kv_heads;
  // Units of short caches, several a request, go to the prompts' kernel from the third round of them on (dealt out: the second) where they fill its blocks. us, units / there: 4 KV heads of
  // 128 dimensions, 28 heads, 64 requests of 200 keys and 20 new tokens (4.5 units to a block) 57 / 31, 200 and up to 8 (2.9) 75 / 58, 200 and up to 3 (1.9) 41 / 57; 8 and 32, 200 of 1500
  // and 8 (2) 198 / 314; 11 requests of up to 238 keys and 155 new tokens, 28 heads, dealt out 47 / 19.
  const bool rounds = each(16) > 1 && tiles <= 24 && all(16) * n_kv_heads > (unit ? 512 : 256) && 2 * all(16) > 5 * all(wide);
  const bool prompt = !(unit || dealt) || rounds || (2 * all(16) - 5 * all(wide)) * n_kv_heads >= (12000 + tiles - 1) / tiles;
  r.block_cols = prompt ? wide : 16;
  r.col_tiles = (int)each(r.block_cols);
  const long units = n_kv_heads * all(r.block_cols);
  r.blocks = prompt ? units : (long)n_kv_heads * n_requests * r.col_tiles;
  r.splits = 1;
  r.split_tiles = (int)tiles;
  if (prompt) {
    // Keys divided among the workgroups that the card has room for at once, 8 tiles each at least, where that ends earlier: a workgroup takes 1.4 us a tile, two on a CU 2.2 (256
    // dimensions, one on a CU: 2.5), joining 10. us undivided / in two / in four: 1000 tokens of one request 39 / 47 / 52, 100 of 4 requests of 8000 keys 228 / 134 / 99, two of 1477,
    // 4 heads on one, 51 / 41 / 36; 256 dimensions, 500 behind 1000 61 / 80 / 97 (more than there is room for), 64 behind 8000 260 / 145 / 85 (in eight 54).
    const long room = head_dim == 256 ? 256 : 512;
    long splits = 1, least = 0;
    for (long n = 1; n == 1 || (n <= tiles / 8 && n * units <= room); n += 1 + n / 16) {
      const long ns = (head_dim == 256 ? 2500 : n * units <= 256 ? 1400 : 2200) * ((tiles + n - 1) / n) + (n > 1 ? 10000 : 0);
      if (n == 1 || ns < least) {
        least = ns;
        splits = n;
      }
    }
    r.split_tiles = (int)((tiles + splits - 1) / splits);
    r.splits = (int)((tiles + r.split_tiles - 1) / r.split_tiles);
    r.scratch = r.splits > 1 ? (size_t)r.splits * n_rows * n_q_heads * (head_dim + 4) * 4 : 0;
    return r;
  }
  // Eight waves to a workgroup and one workgroup to a CU, or four and two: eight cut fewer units, four have more of them at work where the shares are small. us, four / eight:
  // 64 heads x 64 dimensions, 16 requests of 4096 keys 27.7 / 22.0; 8 KV heads of 128 dimensions, 32 requests of 200 to 4096 keys 44 / 53, 64 76 / 98, 100 of 2000 79 / 77, 128 of 500 to
  // 8000 194 / 196, 16 of 30000 160 / 156, 64 of 4096 to 16384 223 / 219. 256 dimensions: a wave's registers are all of a SIMD's.
  r.waves = head_dim == 256 ? 4 : head_dim == 64 || unit || units * tiles >= 192 * 256 ? 8 : 4;
  if (unit) return r;
  const long wanted = (units * tiles + r.waves - 1) / r.waves, most = head_dim == 256 || r.waves == 8 ? 256 : 512;
  r.workgroups = (int)(wanted < most ? wanted : most);
  r.scratch = (((size_t)n_requests + 1) * 4 + 255) / 256 * 256 + (size_t)r.workgroups * 2 * 16 * (head_dim + 4) * 4;
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
  return paged_plan(n_rows, n_requests, max_tokens, max_length, window, keep_first, n_q_heads, n_kv_heads, head_dim).scratch;
}

extern "C" int mui_paged_attention(mui_stream_t stream, const mui_paged_attention_args_t* args) {
  MUI_CHECK_ARG(args);
  const mui_paged_attention_args_t& a = *args;
  MUI_CHECK_ARG(a.q && a.k_pages && a.v_pages && a.k_scale && a.v_scale && a.table && a.lengths && a.out);
  MUI_CHECK_ARG(paged_attention_sizes(a.n_rows, a.n_requests, a.max_tokens, a.max_length, a.window, a.keep_first, a.n_q_heads, a.n_kv_heads, a.head_dim));
  MUI_CHECK_ARG(a.n_pages > 0 && a.table_pages > 0 && a.table_stride >= a.table_pages && (a.offsets || a.n_rows == a.n_requests) && a.scale > 0.f);
  if (a.dtype != MUI_DTYPE_F16 && a.dtype != MUI_DTYPE_BF16) return MUI_ERR_INVALID_ARG;
  if (a.page_tokens != 64 && a.page_tokens != 128 && a.page_tokens != 256) return MUI_ERR_UNSUPPORTED;
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return MUI_ERR_UNSUPPORTED;
  if (((uintptr_t)a.q | (uintptr_t)a.k_pages | (uintptr_t)a.v_pages | (uintptr_t)a.out | (uintptr_t)a.scratch) & 15u) return MUI_ERR_ALIGNMENT;
  if ((a.q_token_stride | a.q_head_stride) & 7) return MUI_ERR_ALIGNMENT;
  const long cap = (long)a.table_pages * a.page_tokens;
  if (cap > 0x7fffffffL) return MUI_ERR_UNSUPPORTED;
  const PagedPlan plan = paged_plan(a.n_rows, a.n_requests, a.max_tokens, a.max_length < cap ? a.max_length : (int)cap, a.window, a.keep_first, a.n_q_heads, a.n_kv_heads, a.head_dim);
  if (plan.scratch && (!a.scratch || a.scratch_bytes < plan.scratch)) return MUI_ERR_INVALID_ARG;
  if ((long)a.n_rows * a.n_q_heads > 0x7fffffffL - 256) return MUI_ERR_UNSUPPORTED;
  const bool prompt = plan.block_cols > 16;
  const long blocks = plan.blocks;
  if (blocks > 0x7fffffffL || plan.splits > 65535 || a.n_requests > 65535) return MUI_ERR_UNSUPPORTED;
  PagedAttnParams p = {};
  p.q = (const uint16_t*)a.q; p.q_tok = a.q_token_stride; p.q_head = a.q_head_stride;
  p.kp = (const uint8_t*)a.k_pages; p.vp = (const uint8_t*)a.v_pages; p.ks = a.k_scale; p.vs = a.v_scale;
  p.t = {a.table, a.table_stride, a.table_pages, a.lengths, a.offsets, a.n_requests, a.n_rows, a.n_pages, a.page_tokens == 64 ? 6 : a.page_tokens == 128 ? 7 : 8};
  p.scale = a.scale * 1.4426950408889634f;
  p.window = a.window; p.keep = a.window > 0 ? a.keep_first : 0;
  p.heads = a.n_q_heads; p.kv_heads = a.n_kv_heads; p.group = a.n_q_heads / a.n_kv_heads;
  p.block_cols = plan.block_cols; p.col_tiles = plan.col_tiles; p.split_tiles = plan.split_tiles; p.splits = plan.splits;
  if (plan.scratch && prompt) p.part = (float*)a.scratch;
  if (plan.scratch && !prompt) {
    p.before = (int*)a.scratch;
    p.part = (float*)((char*)a.scratch + (((size_t)a.n_requests + 1) * 4 + 255) / 256 * 256);
  }
  p.out = (uint16_t*)a.out;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(plan.workgroups ? plan.workgroups : blocks));
  const dim3 join((unsigned)(((long)a.n_rows * a.n_q_heads + 3) / 4));
#define MUI_PAGED_GO(TT, DC)                                                                                                               \
  do {                                                                                                                                     \
    if (prompt) {                                                                                                                          \
      hipLaunchKernelGGL((paged_tiles_kernel<TT, DC, DC == 4 ? 1 : 2>), dim3((unsigned)blocks, plan.splits), dim3(256), 0, s, p); \
      if (p.part) hipLaunchKernelGGL((paged_join_kernel<TT, DC>), join, dim3(256), 0, s, p);                                               \
    } else {                                                                                                                               \
      if constexpr (DC < 4) {                                                                                                              \
        if (plan.waves == 8)                                                                                                               \
          hipLaunchKernelGGL((paged_columns_kernel<TT, DC, 8>), grid, dim3(512), 0, s, p);                                         \
      }                                                                                                                                    \
      if constexpr (DC > 1) {                                                                                                              \
        if (plan.waves == 4)                                                                                                               \
          hipLaunchKernelGGL((paged_columns_kernel<TT, DC, 4>), grid, dim3(256), 0, s, p);                                         \
      }                                                                                                                                    \
      if (p.part) hipLaunchKernelGGL((paged_join_units_kernel<TT, DC>), join, dim3(256), 0, s, p, plan.workgroups, plan.waves);            \
    }                                                                                                                                      \
  } while (0)
#define MUI_PAGED_TYPES(DC) \
  do { if (a.dtype == MUI_DTYPE_F16) MUI_PAGED_GO(F16, DC); else MUI_PAGED_GO(BF16, DC); } while (0)
  if (a.head_dim == 64) MUI_PAGED_TYPES(1); else if (a.head_dim == 128) MUI_PAGED_TYPES(2); else MUI_PAGED_TYPES(4);
  return launch_status();
}
