// Rotary embedding of packed rows, and their append to a paged cache with that
// rotation on the way (fa_rotary_rows, fa_paged_append; no counterpart in the
// reference, whose rotation and append take [batch, new tokens] rows and one
// position axis, flash_attn_mps/_cache.py:99-155).
//
// Pair (a, b) of a head at angle t becomes (a cos t - b sin t, b cos t + a sin
// t) in fp32, rounded once: to the rows' type, to the cache's type, or to E4M3
// under a scale.  Everything here moves each element once, so HBM bounds large
// calls and the chain row -> request -> position -> cos/sin and page bounds
// small ones.
//
// A unit is W pairs of a row (W = 16 bytes of elements, or one pair where
// strides, dims or alignment, of the tables too, forbid vectors): two pieces of W
// elements, next to each other for interleaved pairs, half_rot apart otherwise;
// dims that do not rotate are copied two pieces a unit.  A lane keeps its unit over all the
// heads it takes, so cos and sin are loaded once per token and lane.  A wave
// works on one token, or on one block of one head: what follows from those
// (request, position, page) is scalar.
//
// Block-scaled caches: a workgroup owns a block of tokens of as many heads of K or
// V as a wave holds of a row, its waves the rows in turn, so a block's largest
// magnitude (a maximum in LDS), its scale and its rows need no one else, and the
// result does not depend on any order.  The rows stay in registers until the scale
// is known, and are turned a second time (16 registers a row would hold them
// turned, 8 do as they came).
//
// Kernel times: 9001 tokens of 16 + 16 heads d80 on two axes, 94 MB: 26.6 us, 3.5
// TB/s; 4095 rows of 16 + 4 + 4 heads d256 to a 16-bit cache, 103 MB: 23.6 us, 4.4
// TB/s; 43K rows of 16 + 8 + 8 heads d128 to a block-scaled one, 619 MB: 149 us, 4.2
// TB/s (a large copy: 4.8); one token: 4.0 us, with its append 5.9.
#include "attn_common.h"

namespace {

constexpr int THREADS = 256, MOST_THREADS = 1024;

// What an append writes: nothing, rows of the input's type, E4M3 with a scale
// per head, E4M3 with a scale per block.
enum { CACHE_NONE, CACHE_SAME, CACHE_E4M3, CACHE_BLOCK };

struct AppendRows {
  const void* x;
  void* out;                 // contiguous rows, or the cache
  const float* scale;        // CACHE_E4M3
  int64_t xs[3], os[4];      // os: page, row, head, element (rows: 0, token, head, element)
  int64_t scale_stride;
  int32_t heads, dim, half, units;
};

struct AppendParams {
  AppendRows part[3];        // q, k, v (rotary alone: both sets of rows as parts 0 and 1)
  fa_rotation rot;
  uint8_t* block_scale[2];
  int64_t block_stride[2][3];
  const int32_t *cu, *used, *table;
  int64_t cu_stride, used_stride, bt_stride[2];
  int64_t tokens, num_pages, table_cols;
  int32_t batch, page_size, block;   // page_size: clipped to 32 bits, as positions are
  int32_t lanes, per;                // units of a row handled at once, rows (64 / lanes)
  uint32_t lane_part;                // 2^16 / lanes, rounded up: lane / lanes = lane * lane_part >> 16
  int32_t passes[3];                 // passes of 64 / lanes heads over each part's rows (0: not as rows)
  uint32_t token_waves;              // waves of a token
  int32_t head_sets;                 // sets of `per` heads
  uint32_t block_groups;             // workgroups that own blocks, before those of the tokens
  uint32_t threads;
};

// The largest i < n with key(i) <= target (key nondecreasing), -1 if none: 64
// candidates a round.
template <typename F>
FA_DEV int last_at_most(int n, int64_t target, int lane, F key) {
  int lo = -1, end = n - 1;
  while (lo < end) {
    const int step = (end - lo + 63) / 64;
    const int64_t at = lo + (int64_t)(lane + 1) * step;
    const bool hit = at <= end && key((int)at) <= target;
    const int count = __builtin_popcountll(__ballot(hit));
    lo += count * step;
    end = min(end, lo + step - 1);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

FA_DEV int cu_at(const AppendParams& p, int b) { return p.cu[b * p.cu_stride]; }
FA_DEV int cu_of(const AppendParams& p, int b) { return load_invariant_i32(p.cu, b * p.cu_stride); }   // uniform b

// Where position `pos` of request b lies; page -1: nowhere.
struct Place {
  int64_t page;
  int row;
};

// (Without a branch past the first: the table's load need not be waited for
// where the place is not yet used.)
FA_DEV Place place_of(const AppendParams& p, int b, int64_t pos) {
  if (p.table_cols == 0) return Place{-1, 0};
  const uint32_t size = (uint32_t)p.page_size, at = pos < 0 || pos > INT32_MAX ? 0u : (uint32_t)pos, column = at / size;
  const bool in = at == pos && (int64_t)column < p.table_cols;
  const int64_t page = load_invariant_i32(p.table, b * p.bt_stride[0] + (in ? (int64_t)column : 0) * p.bt_stride[1]);
  return Place{in && page >= 0 && page < p.num_pages ? page : -1, (int)(at - column * size)};
}

FA_DEV uint32_t pair_axes(const AppendParams& p, int i) {
  uint64_t w = p.rot.pair_axis[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) w = i >> 5 == k ? p.rot.pair_axis[k] : w;
  return (uint32_t)(w >> (2 * (i & 31)));
}

FA_DEV int64_t position_of(const AppendParams& p, int64_t t, int axis) {
  const int64_t at = axis * p.rot.position_stride[0] + t * p.rot.position_stride[1];
  return p.rot.position_dtype == FA_I64 ? ((const int64_t*)p.rot.positions)[at] : ((const int32_t*)p.rot.positions)[at];
}

// W elements as they are stored: 16 bytes, or one element's bits.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int W> struct PieceOf { using type = u32x4; };
template <> struct PieceOf<1> { using type = uint32_t; };
template <int W> using Piece = typename PieceOf<W>::type;

template <int BYTES> struct LoadOf { using type = u32x4; };
template <> struct LoadOf<8> { using type = u32x2; };

template <typename XT>
FA_DEV float value_of_bits(uint32_t bits) {
  if constexpr (XT::id == FA_F32) return __uint_as_float(bits);
  else if constexpr (XT::id == FA_BF16) return bf16_bits_to_f32(bits);
  else return f16_bits_to_f32(bits);
}

// Element j of a vector of T.
template <typename T, typename V>
FA_DEV float value_at(V v, int j) {
  return value_of_bits<T>(T::bytes == 4 ? v[j] : v[j / 2] >> (16 * (j & 1)) & 0xffffu);
}

// What a position without a table row reads: NaN in every type.
#define FA_NAN4 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u
#define FA_NAN32 FA_NAN4, FA_NAN4, FA_NAN4, FA_NAN4, FA_NAN4, FA_NAN4, FA_NAN4, FA_NAN4
static __device__ const __align__(16) uint32_t nan_row[256] = {FA_NAN32, FA_NAN32, FA_NAN32, FA_NAN32,
                                                               FA_NAN32, FA_NAN32, FA_NAN32, FA_NAN32};

// cos and sin of pairs i .. i + W - 1 at row `row` of the tables (W > 1: aligned
// pieces of contiguous rows of TT).  Without a branch, so that the loads of
// several rows are in flight together.
template <typename TT, int W>
FA_DEV void load_row(const AppendParams& p, int64_t row, int i, float (&c)[W], float (&s)[W]) {
  const bool in = row >= 0 && row < p.rot.table_rows;
  if constexpr (W == 1) {
    c[0] = s[0] = __builtin_nanf("");
    if (!in) return;
    c[0] = load_any(p.rot.cos_table, row * p.rot.cos_stride[0] + i * p.rot.cos_stride[1], p.rot.trig_dtype);
    s[0] = load_any(p.rot.sin_table, row * p.rot.sin_stride[0] + i * p.rot.sin_stride[1], p.rot.trig_dtype);
  } else {
    using S = typename TT::storage;
    const S* const ct = in ? (const S*)p.rot.cos_table + row * p.rot.cos_stride[0] : (const S*)nan_row;
    const S* const st = in ? (const S*)p.rot.sin_table + row * p.rot.sin_stride[0] : (const S*)nan_row;
    constexpr int N = 16 / TT::bytes < W ? 16 / TT::bytes : W;   // values of a load
    using V = typename LoadOf<N * TT::bytes>::type;
#pragma unroll
    for (int j = 0; j < W; j += N) {
      const V x = *(const V*)(ct + (uint32_t)(i + j)), y = *(const V*)(st + (uint32_t)(i + j));
#pragma unroll
      for (int k = 0; k < N; ++k) {
        c[j + k] = value_at<TT>(x, k);
        s[j + k] = value_at<TT>(y, k);
      }
    }
  }
}

// cos and sin of pairs i .. i + W - 1 (i a multiple of W) of token t: at its
// cache position, or (POS) at the positions of the pairs' axes.
template <typename TT, bool POS, int W>
FA_DEV void load_trig(const AppendParams& p, int64_t t, int64_t cache_pos, int i, float (&c)[W], float (&s)[W]) {
  if constexpr (!POS) {
    load_row<TT, W>(p, cache_pos, i, c, s);
  } else {
    constexpr uint32_t MASK = (1u << (2 * W)) - 1, ONES = MASK / 3;
    const uint32_t axes = p.rot.axes > 1 ? pair_axes(p, i) & MASK : 0;
    load_row<TT, W>(p, position_of(p, t, axes & 3), i, c, s);
    if (W == 1 || axes == (axes & 3) * ONES) return;
    // Axes that alternate within a unit: the others' rows.
    for (uint32_t axis = 0; axis < (uint32_t)p.rot.axes; ++axis) {
      float ca[W], sa[W];
      load_row<TT, W>(p, position_of(p, t, axis), i, ca, sa);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const bool own = (axes >> (2 * j) & 3) == axis;
        c[j] = own ? ca[j] : c[j];
        s[j] = own ? sa[j] : s[j];
      }
    }
  }
}

// The elements at which unit u's two pieces start; the second is -1 where the
// row ends before it.
struct Unit {
  int lo, hi;
  bool turns;
};

template <int W>
FA_DEV Unit unit_of(const AppendRows& r, bool interleaved, int u) {
  const int rotated = r.half / W;
  Unit x;
  x.turns = u < rotated;
  if (x.turns) {
    x.lo = interleaved ? 2 * u * W : u * W;
    x.hi = interleaved ? x.lo + W : r.half + x.lo;
  } else {
    x.lo = 2 * r.half + (u - rotated) * 2 * W;
    x.hi = x.lo + W < r.dim ? x.lo + W : -1;
  }
  return x;
}

template <typename XT, int W>
FA_DEV Piece<W> load_piece(const void* x, int64_t at) {
  using S = typename XT::storage;
  if constexpr (W > 1) {
    static_assert(W * sizeof(S) == 16, "vector pieces");
    return *(const u32x4*)((const S*)x + at);
  } else if constexpr (sizeof(S) == 4) {
    return ((const uint32_t*)x)[at];
  } else {
    return ((const S*)x)[at];
  }
}

template <typename XT, int W>
FA_DEV void store_piece(void* x, int64_t at, Piece<W> v) {
  using S = typename XT::storage;
  if constexpr (W > 1) *(u32x4*)((S*)x + at) = v;
  else if constexpr (sizeof(S) == 4) ((uint32_t*)x)[at] = v;
  else ((S*)x)[at] = (S)v;
}

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

// Two values rounded to XT's 16 bits, in one word.
template <typename XT>
FA_DEV uint32_t pack2(float lo, float hi) {
  if constexpr (XT::id == FA_BF16) return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi});
  else return __builtin_bit_cast(uint32_t, f16x2{(_Float16)lo, (_Float16)hi});
}

template <typename XT, int W>
FA_DEV void widen(Piece<W> v, float (&f)[W]) {
  if constexpr (W == 1) {
    f[0] = value_of_bits<XT>(v);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) f[j] = value_at<XT>(v, j);
  }
}

template <typename XT, int W>
FA_DEV Piece<W> narrow(const float (&f)[W]) {
  if constexpr (W == 1) {
    return XT::bytes == 4 ? __float_as_uint(f[0]) : pack2<XT>(f[0], 0.0f) & 0xffffu;
  } else {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = XT::bytes == 4 ? __float_as_uint(f[j % W]) : pack2<XT>(f[2 * j % W], f[(2 * j + 1) % W]);
    return v;
  }
}

// a x - b y.  TIES: the rounding of b y goes back in (bounded to either side: where
// b y is infinite there is none, and the difference stays infinite), since ties
// between E4M3 codes are where rounding twice shows: of 20M rotated values 14 codes
// off the 64-bit ones, 20 without it and 32 with each product rounded.
template <bool TIES>
FA_DEV float turned_by(float a, float x, float b, float y) {
  const float by = b * y, v = fmaf(a, x, -by);
  return TIES ? v + __builtin_amdgcn_fmed3f(fmaf(-b, y, by), -3e38f, 3e38f) : v;
}

// The W pairs of a unit turned; lo and hi are its pieces.
template <bool TIES, int W>
FA_DEV void turn(float (&lo)[W], float (&hi)[W], const float (&c)[W], const float (&s)[W], bool interleaved) {
  if (W > 1 && interleaved) {
#pragma unroll
    for (int j = 0; j < W; j += 2) {
      const float a = lo[j], b = lo[j + 1], x = hi[j], y = hi[j + 1];
      const int m = j / 2, n = (W + j) / 2;
      lo[j] = turned_by<TIES>(a, c[m], b, s[m]);
      lo[j + 1] = turned_by<TIES>(b, c[m], -a, s[m]);
      hi[j] = turned_by<TIES>(x, c[n], y, s[n]);
      hi[j + 1] = turned_by<TIES>(y, c[n], -x, s[n]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float a = lo[j], b = hi[j];
      lo[j] = turned_by<TIES>(a, c[j], b, s[j]);
      hi[j] = turned_by<TIES>(b, c[j], -a, s[j]);
    }
  }
}

// W values as contiguous E4M3 codes: the hardware conversion of values clamped
// to 448, which gives e4m3_code's byte for all but NaN.
template <int W>
FA_DEV void store_codes(uint8_t* out, const float (&f)[W]) {
  if constexpr (W == 1) {
    out[0] = f32_to_e4m3(f[0]);
  } else {
    uint32_t w[W / 4];
    float probe = 0.0f;   // 0 unless a value is NaN or infinite
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      float x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = __builtin_amdgcn_fmed3f(f[j + k], -448.0f, 448.0f);
        probe = fmaf(f[j + k], 0.0f, probe);
      }
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
      w[j / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
    }
    if (__builtin_expect(probe != 0.0f, 0)) {
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (f[j] != f[j]) w[j / 4] = (w[j / 4] & ~(0xffu << (8 * (j % 4)))) | (e4m3_code(f[j]) & 0xffu) << (8 * (j % 4));
    }
    if constexpr (W == 8) *(uint2*)out = make_uint2(w[0], w[1]);
    else *(uint32_t*)out = w[0];
  }
}

template <int W>
FA_DEV void load_codes(const uint8_t* in, float (&f)[W]) {
  if constexpr (W == 1) {
    f[0] = e4m3_to_f32(in[0]);
  } else {
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      const uint32_t w = *(const uint32_t*)(in + j);
#pragma unroll
      for (int k = 0; k < 4; ++k) f[j + k] = e4m3_to_f32(w >> (8 * k) & 0xffu);
    }
  }
}

// ------------------------------------------------------------ rows of a token

// A lane's offset of element e of head h within a row: 32 bits for vectors (the
// host checks that a row fits), 64 for single elements.
template <int W>
FA_DEV auto lane_offset(int h, int64_t head_stride, int e, int64_t stride) {
  if constexpr (W > 1) return (uint32_t)h * (uint32_t)head_stride + (uint32_t)e;
  else return h * head_stride + e * stride;
}

// Passes of a wave over a token's rows whose loads are all issued before the
// first of them is used.  GPU us with 1 / 2 / 3 / 4 / 6 / 8: 9001 tokens of 16 + 16
// heads d80, two axes (94 MB) 32.4 / 31.5 / 30.4 / 28.8 / 32.7 / 33.2; 4100 rows of
// 16 + 4 + 4 heads d256 to a 16-bit cache (103 MB) 26.4 / 26.6 / 26.9 / 26.4 / 25.3 /
// 25.4 (registers, and so waves, are what more of them cost).
constexpr int BATCH = 4;

template <typename XT, typename TT, int CACHE, bool POS, int W>
FA_DEV void token_rows(const AppendParams& p, uint32_t w, int lane) {
  const bool keeps = CACHE == CACHE_SAME || CACHE == CACHE_E4M3;   // k and v of this token go to the cache as rows
  const int64_t t = p.token_waves == 1 ? w : w / p.token_waves;
  if (t >= p.tokens) return;
  const int per = p.per, sub = (int)(lane * p.lane_part >> 16), u0 = lane - sub * p.lanes;
  const int pass0 = (int)(w - (uint32_t)t * p.token_waves);
  const int total = p.passes[0] + p.passes[1] + p.passes[2];
  const bool inter = p.rot.interleaved;
  int b = -1;
  int64_t pos = -1;
  Place at{-1, 0};
  bool located = CACHE == CACHE_NONE || (!keeps && POS);   // (nothing here depends on the request)
  auto locate = [&]() {
    located = true;
    b = last_at_most(p.batch + 1, t, lane, [&](int i) { return (int64_t)cu_at(p, i); });
    if (b >= p.batch) b = -1;
    if (b < 0) return;
    pos = (int64_t)load_invariant_i32(p.used, b * p.used_stride) - cu_of(p, b + 1) + t;
    if (keeps) at = place_of(p, b, pos);
  };
  for (int u = u0; u < 256; u += 64) {   // (one round but for pieces of one element)
    float c[W], s[W];
    bool have = false;
    for (int s0 = pass0; s0 < total; s0 += BATCH * (int)p.token_waves) {
      Piece<W> a[BATCH], z[BATCH];
      bool on[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int pass = s0 + k * (int)p.token_waves;
        const int which = pass < p.passes[0] ? 0 : pass < p.passes[0] + p.passes[1] ? 1 : 2;
        const int h = (pass - (which > 0 ? p.passes[0] : 0) - (which > 1 ? p.passes[1] : 0)) * per + sub;
        const AppendRows& r = p.part[which];
        on[k] = pass < total && sub < per && h < r.heads && u < r.units;
        if (!on[k]) continue;
        const Unit x = unit_of<W>(r, inter, u);
        const void* const src = (const typename XT::storage*)r.x + t * r.xs[0];
        a[k] = load_piece<XT, W>(src, lane_offset<W>(h, r.xs[1], x.lo, r.xs[2]));
        z[k] = x.hi >= 0 ? load_piece<XT, W>(src, lane_offset<W>(h, r.xs[1], x.hi, r.xs[2])) : a[k];
      }
      if (!located) locate();   // behind the first rows' loads, which need not wait for it
      // (Parts that do not turn come last, so a batch that turns starts with one that does.)
      if (!have && u * W < p.part[s0 < p.passes[0] ? 0 : 1].half && s0 < p.passes[0] + p.passes[1]) {
        load_trig<TT, POS, W>(p, t, pos, u * W, c, s);
        have = true;
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        if (!on[k]) continue;
        const int pass = s0 + k * (int)p.token_waves;
        const int which = pass < p.passes[0] ? 0 : pass < p.passes[0] + p.passes[1] ? 1 : 2;
        const int h = (pass - (which > 0 ? p.passes[0] : 0) - (which > 1 ? p.passes[1] : 0)) * per + sub;
        const AppendRows& r = p.part[which];
        const Unit x = unit_of<W>(r, inter, u);
        const bool cached = CACHE != CACHE_NONE && which > 0;
        if (cached && at.page < 0) continue;
        const bool turns = x.turns && (cached || CACHE == CACHE_NONE || POS || b >= 0);
        const int64_t dst = cached ? at.page * r.os[0] + at.row * r.os[1] : t * r.os[1];
        const auto lo = lane_offset<W>(h, r.os[2], x.lo, r.os[3]), hi = lane_offset<W>(h, r.os[2], x.hi, r.os[3]);
        const bool codes = CACHE == CACHE_E4M3 && cached;
        void* const out = (typename XT::storage*)r.out + (codes ? 0 : dst);
        if (!turns && !codes) {
          store_piece<XT, W>(out, lo, a[k]);
          if (x.hi >= 0) store_piece<XT, W>(out, hi, z[k]);
          continue;
        }
        float f[W], g[W];
        widen<XT, W>(a[k], f);
        widen<XT, W>(z[k], g);
        if (turns) turn<CACHE == CACHE_E4M3>(f, g, c, s, inter);
        if (codes) {
          const float scale = r.scale[h * r.scale_stride];
#pragma unroll
          for (int j = 0; j < W; ++j) f[j] /= scale, g[j] /= scale;
          store_codes<W>((uint8_t*)r.out + dst + lo, f);
          if (x.hi >= 0) store_codes<W>((uint8_t*)r.out + dst + hi, g);
        } else {
          store_piece<XT, W>(out, lo, narrow<XT, W>(f));
          if (x.hi >= 0) store_piece<XT, W>(out, hi, narrow<XT, W>(g));
        }
      }
    }
    if (u + 64 >= 256 || p.lanes < 64) break;
  }
}

// ------------------------------------------------------------ blocks

// log2 of the smallest power of two >= 2^-100 under which `most` (finite) is at
// most 448 = 1.75 * 2^8.
FA_DEV int block_exponent(float most) {
  const uint32_t bits = __float_as_uint(most);
  if (bits < 0x00800000u) return -100;   // zero and fp32 subnormals
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, -100);
}

// Rows a lane holds between a block's largest magnitude and its codes.  GPU us with
// 2 / 4 / 8: 43K rows, blocks of 32, 157.4 / 147.4 / 146.3; 64 requests of one row,
// blocks of 16, 5.7 / 5.7 / 6.3.
constexpr int HOLD = 4;

template <typename XT, typename TT, bool POS, int W>
FA_DEV void own_block(const AppendParams& p, uint32_t group, int lane, uint32_t* most_of) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  const int per = p.per, sub = (int)(lane * p.lane_part >> 16), u0 = lane - sub * p.lanes;
  const uint32_t heads = (uint32_t)p.part[1].heads, sets = (uint32_t)p.head_sets;
  const int h = (int)(group % sets) * per + sub, which = (int)(group / sets) & 1;
  const int id = (int)(group / (2 * sets)), block = p.block;
  // A request of n rows touches at most n / block + 2 blocks: request b has the
  // ids from cu[b] / block + 2 b on.
  const int b = last_at_most(p.batch, id, lane, [&](int i) { return (int64_t)(cu_at(p, i) / block) + 2 * (int64_t)i; });
  if (b < 0) return;
  const int t0 = cu_of(p, b);
  const int64_t n = (int64_t)cu_of(p, b + 1) - t0;
  const int64_t end = load_invariant_i32(p.used, b * p.used_stride), start = end - n, from = max(start, (int64_t)0);
  if (t0 < 0 || n <= 0 || end <= 0) return;
  const int64_t base = ((uint32_t)from / (uint32_t)block + (int64_t)(id - t0 / block - 2 * b)) * block;   // its first position
  if (base >= end || base - start >= p.tokens - t0) return;
  const Place place = place_of(p, b, base);   // (used behind the rows' loads)
  // The block's new rows (none past the last row there is).
  const int first = (int)(max(base, from) - base);
  const int last = (int)(min(min(base + block, end), start + p.tokens - t0) - base);
  const AppendRows& r = p.part[1 + which];
  const bool inter = p.rot.interleaved;
  const bool on = sub < per && h < (int)heads && u0 < r.units;
  const int64_t token = t0 + base - start;   // row 0's
  const typename XT::storage* const x0 = (const typename XT::storage*)r.x + token * r.xs[0];
  // The pieces of a unit of row `row`, and their values turned.
  auto load = [&](int row, const Unit& x, Piece<W>& a, Piece<W>& z) {
    const typename XT::storage* const src = x0 + row * r.xs[0];
    a = load_piece<XT, W>(src, lane_offset<W>(h, r.xs[1], x.lo, r.xs[2]));
    z = x.hi >= 0 ? load_piece<XT, W>(src, lane_offset<W>(h, r.xs[1], x.hi, r.xs[2])) : Piece<W>{};
  };
  auto turned = [&](auto ties, int row, int u, const Unit& x, Piece<W> a, Piece<W> z, float (&f)[W], float (&g)[W]) {
    widen<XT, W>(a, f);
    widen<XT, W>(z, g);
    if (!x.turns) return;
    float c[W], s[W];
    load_trig<TT, POS, W>(p, token + row, base + row, u * W, c, s);
    turn<decltype(ties)::value>(f, g, c, s, inter);
  };
  // The largest finite magnitude (a maximum leaves NaN out; infinities are rare).
  auto largest = [&](float most, const float (&f)[W], const float (&g)[W]) {
    float all = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) all = fmaxf(all, fmaxf(fabsf(f[j]), fabsf(g[j])));
    if (__builtin_expect(all == INFINITY, 0)) {
      all = 0.0f;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float a = fabsf(f[j]), z = fabsf(g[j]);
        all = fmaxf(all, fmaxf(a < INFINITY ? a : 0.0f, z < INFINITY ? z : 0.0f));
      }
    }
    return fmaxf(most, all);
  };
  // This wave's rows: first + wave, and every `waves` on.
  const bool held = W > 1 && block <= HOLD * waves;
  Piece<W> a[HOLD], z[HOLD];
  float f[W], g[W], most = 0.0f;
  const Unit x = unit_of<W>(r, inter, u0);
  if (held) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (on && first + wave + i * waves < last) load(first + wave + i * waves, x, a[i], z[i]);
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      const int row = first + wave + i * waves;
      if (!on || row >= last) continue;
      turned(std::false_type{}, row, u0, x, a[i], z[i], f, g);
      most = largest(most, f, g);
    }
  } else if (on) {
    for (int row = first + wave; row < last; row += waves)
      for (int u = u0; u < r.units; u += p.lanes) {
        const Unit y = unit_of<W>(r, inter, u);
        load(row, y, a[0], z[0]);
        turned(std::false_type{}, row, u, y, a[0], z[0], f, g);
        most = largest(most, f, g);
      }
  }
  if (place.page < 0) return;   // (like the returns before it, the same for the whole workgroup)
  uint8_t* const o0 = (uint8_t*)r.out + place.page * r.os[0] + place.row * r.os[1];
  uint8_t* const sp = p.block_scale[which] + place.page * p.block_stride[which][0] +
                      (uint32_t)place.row / (uint32_t)block * p.block_stride[which][1] + h * p.block_stride[which][2];
  const int old = on && first > 0 ? (int)sp[0] - 127 : 0;
  auto code_at = [&](int row, int e) { return o0 + row * r.os[1] + lane_offset<W>(h, r.os[2], e, r.os[3]); };
  auto store = [&](int row, const Unit& x, float (&f)[W], float (&g)[W], float inverse) {
#pragma unroll
    for (int j = 0; j < W; ++j) f[j] *= inverse, g[j] *= inverse;   // exact where E4M3 tells it from zero
    store_codes<W>(code_at(row, x.lo), f);
    if (x.hi >= 0) store_codes<W>(code_at(row, x.hi), g);
  };
  // A head's largest magnitude, from its lanes in all the waves (the bits of
  // positive floats are in their order).
  if ((int)threadIdx.x < per) most_of[threadIdx.x] = 0;
  __syncthreads();
  if (on) atomicMax(&most_of[sub], __float_as_uint(most));
  __syncthreads();
  if (!on) return;
  // The block's scale; rows of the request before the new ones are coded again
  // where it grows.
  int e = block_exponent(__uint_as_float(most_of[sub]));
  if (first > 0 && old >= e) {
    e = old;
  } else if (first > 0) {
    for (int row = wave; row < first; row += waves)
      for (int u = u0; u < r.units; u += p.lanes) {
        const Unit y = unit_of<W>(r, inter, u);
        for (int at = y.lo;; at = y.hi) {
          float v[W];
          load_codes<W>(code_at(row, at), v);
#pragma unroll
          for (int j = 0; j < W; ++j) v[j] = ldexpf(v[j], old - e);
          store_codes<W>(code_at(row, at), v);
          if (at == y.hi || y.hi < 0) break;
        }
      }
  }
  const float inverse = ldexpf(1.0f, -e);
  if (held) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      const int row = first + wave + i * waves;
      if (row >= last) continue;
      turned(std::true_type{}, row, u0, x, a[i], z[i], f, g);
      store(row, x, f, g, inverse);
    }
  } else {
    for (int row = first + wave; row < last; row += waves)
      for (int u = u0; u < r.units; u += p.lanes) {
        const Unit y = unit_of<W>(r, inter, u);
        load(row, y, a[0], z[0]);
        turned(std::true_type{}, row, u, y, a[0], z[0], f, g);
        store(row, y, f, g, inverse);
      }
  }
  if (wave == 0 && u0 == 0) sp[0] = (uint8_t)(e + 127);
}

template <typename XT, typename TT, int CACHE, bool POS, int W>
__global__ __launch_bounds__(CACHE == CACHE_BLOCK ? MOST_THREADS : THREADS) void append_kernel(const AppendParams p) {
  const int lane = threadIdx.x & 63;
  uint32_t group = blockIdx.x;
  if constexpr (CACHE == CACHE_BLOCK) {
    __shared__ uint32_t most[64];
    if (group < p.block_groups) {
      own_block<XT, TT, POS, W>(p, group, lane, most);
      return;
    }
    group -= p.block_groups;
  }
  token_rows<XT, TT, CACHE, POS, W>(p, group * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane);
}

// ------------------------------------------------------------ host

bool input_type(int t) { return t == FA_F16 || t == FA_BF16 || t == FA_F32; }

int check_rotation(const fa_rotation& r, bool needs_positions, const char* who) {
  FA_REQUIRE(!r.cos_table == !r.sin_table, "%s: cos and sin come together", who);
  if (!r.cos_table) return FA_OK;
  FA_REQUIRE(input_type(r.trig_dtype), "%s: cos/sin dtype must be f16/bf16/f32", who);
  FA_REQUIRE(r.half_rot >= 0 && r.half_rot <= 256 && r.table_rows >= 0, "%s: bad cos/sin tables", who);
  FA_REQUIRE(r.positions || !needs_positions, "%s: null positions", who);
  FA_REQUIRE(!r.positions || (r.axes >= 1 && r.axes <= 4 && (r.position_dtype == FA_I32 || r.position_dtype == FA_I64)),
             "%s: positions are int32/int64 on 1 to 4 axes", who);
  if (r.positions)
    for (int i = 0; i < r.half_rot; ++i)
      FA_REQUIRE((int)(r.pair_axis[i >> 5] >> (2 * (i & 31)) & 3) < r.axes, "%s: pair %d has no axis", who, i);
  return FA_OK;
}

int check_rows(const fa_rows& r, const fa_rotation& rot, const char* who) {
  FA_REQUIRE(r.out && r.heads >= 1 && r.heads <= 65535 && r.dim >= 1 && r.dim <= 512, "%s: bad rows", who);
  FA_REQUIRE(!rot.cos_table || 2 * rot.half_rot <= r.dim, "%s: rotary dim exceeds head dim", who);
  return FA_OK;
}

AppendRows to_part(const fa_rows& r) {
  AppendRows p = {};
  p.x = r.x, p.out = r.out;
  p.heads = (int32_t)r.heads, p.dim = (int32_t)r.dim;
  for (int i = 0; i < 3; ++i) p.xs[i] = r.x_stride[i];
  p.os[1] = r.heads * r.dim, p.os[2] = r.dim, p.os[3] = 1;
  return p;
}

AppendRows to_part(const fa_store_desc& d) {
  AppendRows p = {};
  p.x = d.x, p.out = d.cache, p.scale = d.scale, p.scale_stride = d.scale_stride;
  p.heads = (int32_t)d.heads, p.dim = (int32_t)d.dim;
  for (int i = 0; i < 3; ++i) p.xs[i] = d.x_stride[i];
  for (int i = 0; i < 4; ++i) p.os[i] = d.cache_stride[i];
  return p;
}

// Whether every piece of W elements starts on 16 bytes of input and W elements
// of output.
bool pieces_aligned(const AppendRows& p, int esz, int osz) {
  const int w = 16 / esz;
  if (!p.heads) return true;
  if (p.dim % w || p.half % w || p.xs[2] != 1 || p.os[3] != 1) return false;
  if ((uintptr_t)p.x % 16 || (uintptr_t)p.out % (uintptr_t)(w * osz)) return false;
  for (int i = 0; i < 2; ++i)
    if ((p.xs[i] * esz) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (p.os[i] % w) return false;
  // Offsets within a row stay below 2^29 elements.
  const int64_t most = (int64_t)1 << 29;
  return p.heads * p.xs[1] + p.dim < most && p.heads * p.os[2] + p.dim < most && p.xs[1] >= 0 && p.os[2] >= 0;
}

// Whether cos and sin come in aligned pieces wherever a unit's start in their rows.
bool trig_aligned(const fa_rotation& r) {
  const int esz = r.trig_dtype == FA_F32 ? 4 : 2;
  return r.cos_stride[1] == 1 && r.sin_stride[1] == 1 && (uintptr_t)r.cos_table % 16 == 0 &&
         (uintptr_t)r.sin_table % 16 == 0 && (r.cos_stride[0] * esz) % 16 == 0 && (r.sin_stride[0] * esz) % 16 == 0;
}

template <typename XT, typename TT, bool POS, int W>
void launch_append(int cache, const AppendParams& p, uint32_t groups, hipStream_t s) {
  const dim3 grid(groups), block(p.threads);
  switch (cache) {
    case CACHE_NONE:   // (always by positions)
      if constexpr (POS) hipLaunchKernelGGL((append_kernel<XT, TT, CACHE_NONE, POS, W>), grid, block, 0, s, p);
      break;
    case CACHE_SAME: hipLaunchKernelGGL((append_kernel<XT, TT, CACHE_SAME, POS, W>), grid, block, 0, s, p); break;
    case CACHE_E4M3: hipLaunchKernelGGL((append_kernel<XT, TT, CACHE_E4M3, POS, W>), grid, block, 0, s, p); break;
    default: hipLaunchKernelGGL((append_kernel<XT, TT, CACHE_BLOCK, POS, W>), grid, block, 0, s, p); break;
  }
}

// Vectors with fp32 tables or tables of the rows' type; single elements else.
template <typename XT, bool POS>
void launch_typed(int cache, bool vec, const AppendParams& p, uint32_t groups, hipStream_t s) {
  if (!vec) launch_append<XT, F32T, POS, 1>(cache, p, groups, s);
  else if (XT::id == FA_F32 || (p.rot.cos_table && p.rot.trig_dtype == XT::id)) launch_append<XT, XT, POS, 16 / XT::bytes>(cache, p, groups, s);
  else launch_append<XT, F32T, POS, 16 / XT::bytes>(cache, p, groups, s);
}

template <typename XT>
void launch_rows(int cache, bool vec, const AppendParams& p, uint32_t groups, hipStream_t s) {
  if (p.rot.positions) launch_typed<XT, true>(cache, vec, p, groups, s);
  else launch_typed<XT, false>(cache, vec, p, groups, s);
}

// Fills in what the parts have in common and launches.
int run_append(AppendParams& p, int dtype, int cache, void* stream, const char* who) {
  const int esz = dtype == FA_F32 ? 4 : 2;
  bool vec = !p.rot.cos_table || (trig_aligned(p.rot) && (p.rot.trig_dtype == FA_F32 || p.rot.trig_dtype == dtype));
  for (int i = 0; i < 3; ++i) {
    AppendRows& r = p.part[i];
    const bool cached = cache != CACHE_NONE && i > 0;
    r.half = p.rot.cos_table && !(cached && i == 2) && r.heads ? (int32_t)p.rot.half_rot : 0;
    vec = vec && pieces_aligned(r, esz, cached && cache >= CACHE_E4M3 ? 1 : esz);
  }
  const int w = vec ? 16 / esz : 1;
  int units = 1;
  for (int i = 0; i < 3; ++i) {
    AppendRows& r = p.part[i];
    r.units = r.heads ? r.half / w + (int)fa_ceil_div(r.dim - 2 * r.half, 2 * w) : 0;
    units = r.units > units ? r.units : units;
  }
  p.lanes = units < 64 ? units : 64;
  p.per = 64 / p.lanes;
  p.lane_part = (65536u + (uint32_t)p.lanes - 1) / (uint32_t)p.lanes;
  int64_t passes = 0;
  for (int i = 0; i < 3; ++i) {
    p.passes[i] = cache == CACHE_BLOCK && i > 0 ? 0 : (int)fa_ceil_div(p.part[i].heads, p.per);
    passes += p.passes[i];
  }
  // A few tokens: every pass over a token's rows on a wave of its own, for the
  // shortest chain.  Many: a wave a token, which finds its request, position and
  // cos/sin once.  GPU us, a wave each / a wave a token: one token of 32 + 8 heads
  // d128 3.5 / 5.8; 9001 tokens of 16 + 16 heads d80 39.7 / 26.8; up to 32768 waves
  // neither side gains.
  p.token_waves = (uint32_t)(passes > 0 && p.tokens * passes <= 4096 ? passes : 1);
  FA_REQUIRE(p.tokens * p.token_waves <= INT32_MAX, "%s: too many rows", who);
  p.threads = THREADS;
  int64_t groups = 0;
  if (cache == CACHE_BLOCK) {
    // As many waves as hold a block's rows in HOLD rounds, so that they are read
    // once (blocks past that, and single elements: twice).
    while (p.threads < MOST_THREADS && p.block > HOLD * (int)(p.threads / 64)) p.threads *= 2;
    p.head_sets = (int32_t)fa_ceil_div(p.part[1].heads, p.per);
    groups = (p.tokens / p.block + 2 * (int64_t)p.batch) * 2 * p.head_sets;
    FA_REQUIRE(groups <= INT32_MAX, "%s: too many blocks", who);
    p.block_groups = (uint32_t)groups;
  }
  if (passes) groups += fa_ceil_div(p.tokens * p.token_waves, p.threads / 64);
  FA_REQUIRE(groups * p.threads < 1ll << 32, "%s: too many rows", who);   // 2^32 threads a launch
  if (groups == 0) return FA_OK;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case FA_F16: launch_rows<F16T>(cache, vec, p, (uint32_t)groups, s); break;
    case FA_BF16: launch_rows<BF16T>(cache, vec, p, (uint32_t)groups, s); break;
    default: launch_rows<F32T>(cache, vec, p, (uint32_t)groups, s); break;
  }
  return fa_check_launch(who);
}

}  // namespace

extern "C" int fa_rotary_rows(const fa_rotary_rows_args* a, void* stream) {
  const char* who = "fa_rotary_rows";
  FA_REQUIRE(a && a->size == (int64_t)sizeof(fa_rotary_rows_args), "%s: null or mismatched arguments", who);
  FA_REQUIRE(input_type(a->dtype) && a->tokens >= 0, "%s: bad dtype or rows", who);
  FA_REQUIRE(a->rot.cos_table, "%s: null tables", who);
  int rc = check_rotation(a->rot, true, who);
  if (rc) return rc;
  AppendParams p = {};
  for (int i = 0; i < 2; ++i) {
    if (!a->rows[i].x && (i == 1 || a->tokens == 0)) continue;
    FA_REQUIRE(a->rows[i].x, "%s: null rows", who);
    rc = check_rows(a->rows[i], a->rot, who);
    if (rc) return rc;
    p.part[i] = to_part(a->rows[i]);
  }
  p.rot = a->rot;
  p.tokens = a->tokens;
  return run_append(p, a->dtype, CACHE_NONE, stream, who);
}

extern "C" int fa_paged_append(const fa_paged_append_args* a, void* stream) {
  const char* who = "fa_paged_append";
  FA_REQUIRE(a && a->size == (int64_t)sizeof(fa_paged_append_args), "%s: null or mismatched arguments", who);
  FA_REQUIRE(a->tokens >= 0 && a->batch >= 0 && a->batch < INT32_MAX && a->page_size >= 1 && a->num_pages >= 0 &&
                 a->table_cols >= 0 && a->block >= 0,
             "%s: bad sizes", who);
  if (a->tokens == 0) return FA_OK;
  FA_REQUIRE(a->cu_seqlens_q && (a->batch == 0 || a->seqused_k), "%s: null lengths", who);
  FA_REQUIRE(a->batch == 0 || a->table_cols == 0 || a->block_table, "%s: null block table", who);
  const int xdt = a->kv[0].x_dtype, cdt = a->kv[0].cache_dtype;
  FA_REQUIRE(input_type(xdt), "%s: input dtype must be f16/bf16/f32", who);
  FA_REQUIRE(cdt == xdt || cdt == FA_E4M3, "%s: cache dtype must match input or be E4M3", who);
  FA_REQUIRE(a->block == 0 || (cdt == FA_E4M3 && a->page_size <= INT32_MAX && a->block <= a->page_size && a->page_size % a->block == 0),
             "%s: block scales go with an E4M3 cache whose pages they divide", who);
  int rc = check_rotation(a->rot, false, who);
  if (rc) return rc;
  AppendParams p = {};
  for (int i = 0; i < 2; ++i) {
    const fa_store_desc& d = a->kv[i];
    FA_REQUIRE(d.x && (d.cache || a->num_pages == 0), "%s: null tensor %d", who, i);
    FA_REQUIRE(d.x_dtype == xdt && d.cache_dtype == cdt, "%s: K and V must share dtypes", who);
    FA_REQUIRE(d.heads == a->kv[0].heads && d.heads >= 1 && d.heads <= 65535 && d.dim >= 1 && d.dim <= 512,
               "%s: bad heads or dims", who);
    if (a->block) FA_REQUIRE(a->block_scale[i] || a->num_pages == 0, "%s: null block scales", who);
    else FA_REQUIRE(cdt != FA_E4M3 || d.scale, "%s: an E4M3 cache needs a scale", who);
    p.part[1 + i] = to_part(d);
    p.block_scale[i] = a->block_scale[i];
    for (int j = 0; j < 3; ++j) p.block_stride[i][j] = a->block_stride[i][j];
  }
  FA_REQUIRE(!a->rot.cos_table || 2 * a->rot.half_rot <= a->kv[0].dim, "%s: rotary dim exceeds head dim", who);
  if (a->q.x) {
    rc = check_rows(a->q, a->rot, who);
    if (rc) return rc;
    p.part[0] = to_part(a->q);
  }
  p.rot = a->rot;
  p.cu = a->cu_seqlens_q, p.cu_stride = a->cu_q_stride;
  p.used = a->seqused_k, p.used_stride = a->used_k_stride;
  p.table = a->block_table;
  for (int i = 0; i < 2; ++i) p.bt_stride[i] = a->bt_stride[i];
  p.tokens = a->tokens, p.batch = (int32_t)a->batch;
  p.page_size = (int32_t)(a->page_size < INT32_MAX ? a->page_size : INT32_MAX);
  p.num_pages = a->num_pages, p.table_cols = a->table_cols;
  p.block = (int32_t)a->block;
  return run_append(p, xdt, a->block ? CACHE_BLOCK : cdt == FA_E4M3 ? CACHE_E4M3 : CACHE_SAME, stream, who);
}
