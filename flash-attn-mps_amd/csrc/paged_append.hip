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
// strides, dims or alignment forbid vectors): two pieces of W elements, next to
// each other for interleaved pairs, half_rot apart otherwise; dims that do not
// rotate are copied two pieces a unit.  A lane keeps its unit over all the
// heads it takes, so cos and sin are loaded once per token and lane.
//
// Block-scaled caches: one wave owns a (block of tokens, head) of K or V, so
// the block's largest magnitude, its scale and its rows need no other wave, and
// the result does not depend on any order.
#include "attn_common.h"

namespace {

constexpr int THREADS = 256, WAVES = 4;

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
  int64_t tokens, page_size, num_pages, table_cols;
  int32_t batch, block, lanes;   // lanes: units of a row handled at once
  int32_t row_heads;             // heads of a token that run as rows (parts in order)
  uint32_t block_waves;          // workgroups 0 .. ceil(block_waves / 4) - 1 own blocks
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
  return lo;
}

FA_DEV int64_t cu_at(const AppendParams& p, int b) { return p.cu[b * p.cu_stride]; }

// One page of the cache that position `pos` of request b lies in; -1: none.
FA_DEV int64_t page_of(const AppendParams& p, int b, int64_t pos) {
  if (pos < 0) return -1;
  const int64_t column = pos / p.page_size;
  if (column >= p.table_cols) return -1;
  const int64_t page = p.table[b * p.bt_stride[0] + column * p.bt_stride[1]];
  return page >= 0 && page < p.num_pages ? page : -1;
}

// The row of the cos/sin tables for pair i of token t; -1: none.
FA_DEV int64_t trig_row(const AppendParams& p, int64_t t, int64_t cache_pos, int i) {
  int64_t pos = cache_pos;
  if (p.rot.positions) {
    const int axis = (int)(p.rot.pair_axis[i >> 5] >> (2 * (i & 31))) & 3;
    const int64_t at = axis * p.rot.position_stride[0] + t * p.rot.position_stride[1];
    pos = p.rot.position_dtype == FA_I64 ? ((const int64_t*)p.rot.positions)[at] : ((const int32_t*)p.rot.positions)[at];
  }
  return pos >= 0 && pos < p.rot.table_rows ? pos : -1;
}

// cos and sin of pairs i .. i + W - 1 of token t.
template <int W>
FA_DEV void load_trig(const AppendParams& p, int64_t t, int64_t cache_pos, int i, float (&c)[W], float (&s)[W]) {
#pragma unroll
  for (int j = 0; j < W; ++j) {
    const int64_t row = trig_row(p, t, cache_pos, i + j);
    c[j] = s[j] = __builtin_nanf("");
    if (row >= 0) {
      c[j] = load_any(p.rot.cos_table, row * p.rot.cos_stride[0] + (i + j) * p.rot.cos_stride[1], p.rot.trig_dtype);
      s[j] = load_any(p.rot.sin_table, row * p.rot.sin_stride[0] + (i + j) * p.rot.sin_stride[1], p.rot.trig_dtype);
    }
  }
}

// The elements at which unit u's two pieces start; the second is -1 where the
// row ends before it.
template <int W>
FA_DEV void unit_places(const AppendRows& r, bool interleaved, int u, int& lo, int& hi, bool& turns) {
  const int rotated = r.half / W;
  turns = u < rotated;
  if (turns) {
    lo = interleaved ? 2 * u * W : u * W;
    hi = interleaved ? lo + W : r.half + lo;
  } else {
    lo = 2 * r.half + (u - rotated) * 2 * W;
    hi = lo + W < r.dim ? lo + W : -1;
  }
}

template <typename XT, int W> struct Piece { typename XT::storage e[W]; };

template <typename XT, int W>
FA_DEV Piece<XT, W> load_piece(const void* x, int64_t at, int64_t stride) {
  using S = typename XT::storage;
  Piece<XT, W> r;
  if constexpr (W > 1) {
    static_assert(W * sizeof(S) == 16, "vector pieces");
    r = __builtin_bit_cast(Piece<XT, W>, *(const uint4*)((const S*)x + at));
  } else {
    r.e[0] = ((const S*)x)[at];
  }
  return r;
}

template <typename XT, int W>
FA_DEV void store_piece(void* x, int64_t at, const Piece<XT, W>& v) {
  using S = typename XT::storage;
  if constexpr (W > 1) *(uint4*)((S*)x + at) = __builtin_bit_cast(uint4, v);
  else ((S*)x)[at] = v.e[0];
}

template <typename XT, int W>
FA_DEV void widen(const Piece<XT, W>& v, float (&f)[W]) {
#pragma unroll
  for (int j = 0; j < W; ++j) f[j] = load_elem<XT>(v.e, j);
}

template <typename XT, int W>
FA_DEV Piece<XT, W> narrow(const float (&f)[W]) {
  Piece<XT, W> v;
#pragma unroll
  for (int j = 0; j < W; ++j) store_elem<XT>(v.e, j, f[j]);
  return v;
}

// The W pairs of a unit turned; lo and hi are its pieces.
template <int W>
FA_DEV void turn(float (&lo)[W], float (&hi)[W], const float (&c)[W], const float (&s)[W], bool interleaved) {
  if (W > 1 && interleaved) {
#pragma unroll
    for (int j = 0; j < W; j += 2) {
      const float a = lo[j], b = lo[j + 1], x = hi[j], y = hi[j + 1];
      const int m = j / 2, n = (W + j) / 2;
      lo[j] = fmaf(a, c[m], -(b * s[m]));
      lo[j + 1] = fmaf(b, c[m], a * s[m]);
      hi[j] = fmaf(x, c[n], -(y * s[n]));
      hi[j + 1] = fmaf(y, c[n], x * s[n]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float a = lo[j], b = hi[j];
      lo[j] = fmaf(a, c[j], -(b * s[j]));
      hi[j] = fmaf(b, c[j], a * s[j]);
    }
  }
}

// W values as E4M3 codes at element `at` (16-byte pieces: W contiguous codes).
template <int W>
FA_DEV void store_codes(uint8_t* out, const float (&f)[W]) {
  if constexpr (W == 1) {
    out[0] = f32_to_e4m3(f[0]);
  } else {
    uint32_t w[W / 4];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint32_t code = e4m3_code(f[j]) & 0xffu;
      if (j % 4 == 0) w[j / 4] = code;
      else w[j / 4] |= code << (8 * (j % 4));
    }
    if constexpr (W == 8) *(uint2*)out = make_uint2(w[0], w[1]);
    else *(uint32_t*)out = w[0];
  }
}

// ------------------------------------------------------------ rows of a token

template <typename XT, int CACHE, int W>
FA_DEV void token_rows(const AppendParams& p, int64_t t, int wave, int lane) {
  const bool keeps = CACHE == CACHE_SAME || CACHE == CACHE_E4M3;   // k and v of this token go to the cache as rows
  int b = -1;
  int64_t pos = -1, page = -1;
  if (CACHE != CACHE_NONE && (keeps || !p.rot.positions)) {
    b = last_at_most(p.batch + 1, t, lane, [&](int i) { return cu_at(p, i); });
    if (b >= p.batch) b = -1;
    if (b >= 0) {
      pos = (int64_t)p.used[b * p.used_stride] - cu_at(p, b + 1) + t;
      if (keeps) page = page_of(p, b, pos);
    }
  }
  const bool q_turns = CACHE == CACHE_NONE || p.rot.positions || b >= 0;
  const bool inter = p.rot.interleaved;
  const int per = 64 / p.lanes;   // heads of a wave at once
  if (lane >= per * p.lanes) return;
  for (int u = lane % p.lanes; u < 256; u += p.lanes) {
    if (u >= max(max(p.part[0].units, p.part[1].units), p.part[2].units)) break;
    float c[W], s[W];
    bool have = false;
    for (int g = wave * per + lane / p.lanes; g < p.row_heads; g += WAVES * per) {
      int h = g, which = 0;
      if (h >= p.part[0].heads) h -= p.part[0].heads, which = 1;
      if (which == 1 && h >= p.part[1].heads) h -= p.part[1].heads, which = 2;
      const AppendRows& r = p.part[which];
      if (u >= r.units) continue;
      const bool cached = CACHE != CACHE_NONE && which > 0;
      if (cached && page < 0) continue;
      int lo, hi;
      bool turns;
      unit_places<W>(r, inter, u, lo, hi, turns);
      const int64_t src = t * r.xs[0] + h * r.xs[1];
      const Piece<XT, W> a = load_piece<XT, W>(r.x, src + lo * r.xs[2], r.xs[2]);
      Piece<XT, W> z = a;
      if (hi >= 0) z = load_piece<XT, W>(r.x, src + hi * r.xs[2], r.xs[2]);
      turns = turns && (cached || q_turns);
      if (turns && !have) {
        load_trig<W>(p, t, pos, u * W, c, s);
        have = true;
      }
      const int64_t row = cached ? pos % p.page_size : t;
      const int64_t dst = (cached ? page : 0) * r.os[0] + row * r.os[1] + h * r.os[2];
      const bool codes = CACHE == CACHE_E4M3 && cached;
      if (!turns && !codes) {
        store_piece<XT, W>(r.out, dst + lo * r.os[3], a);
        if (hi >= 0) store_piece<XT, W>(r.out, dst + hi * r.os[3], z);
        continue;
      }
      float x[W], y[W];
      widen<XT, W>(a, x);
      widen<XT, W>(z, y);
      if (turns) turn<W>(x, y, c, s, inter);
      if (codes) {
        const float scale = r.scale[h * r.scale_stride];
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] /= scale, y[j] /= scale;
        store_codes<W>((uint8_t*)r.out + dst + lo * r.os[3], x);
        if (hi >= 0) store_codes<W>((uint8_t*)r.out + dst + hi * r.os[3], y);
      } else {
        store_piece<XT, W>(r.out, dst + lo * r.os[3], narrow<XT, W>(x));
        if (hi >= 0) store_piece<XT, W>(r.out, dst + hi * r.os[3], narrow<XT, W>(y));
      }
    }
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

// x * 2^-e, exact (e in -127 .. 127, any fp32 x whose result E4M3 tells from zero).
FA_DEV float unscale(float x, int e) { return ldexpf(x, -e); }

template <typename XT, int W>
FA_DEV void own_block(const AppendParams& p, uint32_t w, int lane) {
  const int heads = p.part[1].heads;
  const int h = (int)(w % (uint32_t)heads), which = (int)(w / (uint32_t)heads) & 1;
  const int64_t id = w / (2u * (uint32_t)heads);
  const int64_t block = p.block;
  // A request of n rows touches at most n / block + 2 blocks: request b has the
  // ids from cu[b] / block + 2 b on.
  const int b = last_at_most(p.batch, id, lane, [&](int i) { return cu_at(p, i) / block + 2 * i; });
  if (b < 0) return;
  const int64_t t0 = cu_at(p, b), n = cu_at(p, b + 1) - t0;
  const int64_t end = p.used[b * p.used_stride], start = end - n;
  if (t0 < 0 || n <= 0 || end <= 0) return;
  const int64_t from = max(start, (int64_t)0);
  const int64_t base = (from / block + (id - t0 / block - 2 * b)) * block;   // the block's first position
  if (base >= end || base - start >= p.tokens - t0) return;
  const int64_t page = page_of(p, b, base);
  if (page < 0) return;
  // The block's new rows (none past the last row there is).
  const int first = (int)(max(base, from) - base), last = (int)(min(min(base + block, end), start + p.tokens - t0) - base);
  const AppendRows& r = p.part[1 + which];
  const int64_t row0 = base % p.page_size;
  const int64_t x0 = (t0 + base - start) * r.xs[0] + h * r.xs[1];
  const int64_t o0 = page * r.os[0] + row0 * r.os[1] + h * r.os[2];
  const bool inter = p.rot.interleaved;
  const int per = 64 / p.lanes, rl = lane / p.lanes;
  const bool on = rl < per;
  uint8_t* const sp = p.block_scale[which] + page * p.block_stride[which][0] + row0 / block * p.block_stride[which][1] +
                      h * p.block_stride[which][2];
  // f(row, lo, hi, values of the pieces) over this lane's units of the new rows.
  auto each = [&](auto f) {
    for (int row = first + rl; row < last; row += per) {
      for (int u = lane % p.lanes; u < r.units; u += p.lanes) {
        int lo, hi;
        bool turns;
        unit_places<W>(r, inter, u, lo, hi, turns);
        const int64_t src = x0 + row * r.xs[0];
        float x[W], y[W];
        widen<XT, W>(load_piece<XT, W>(r.x, src + lo * r.xs[2], r.xs[2]), x);
        if (hi >= 0) widen<XT, W>(load_piece<XT, W>(r.x, src + hi * r.xs[2], r.xs[2]), y);
        else
#pragma unroll
          for (int j = 0; j < W; ++j) y[j] = 0.0f;
        if (turns) {
          float c[W], s[W];
          load_trig<W>(p, t0 + base + row - start, base + row, u * W, c, s);
          turn<W>(x, y, c, s, inter);
        }
        f(row, lo, hi, x, y);
      }
    }
  };
  float most = 0.0f;
  if (on)
    each([&](int, int, int, float (&x)[W], float (&y)[W]) {
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float a = fabsf(x[j]), z = fabsf(y[j]);
        most = fmaxf(most, a < INFINITY ? a : 0.0f);
        most = fmaxf(most, z < INFINITY ? z : 0.0f);
      }
    });
  int e = block_exponent(wave_max(most));
  if (first > 0) {
    const int old = (int)sp[0] - 127;
    if (old >= e) {
      e = old;
    } else if (on) {
      // Rows of the request before the new ones, under the larger scale.
      for (int row = rl; row < first; row += per) {
        for (int u = lane % p.lanes; u < r.units; u += p.lanes) {
          int place[2];
          bool turns;
          unit_places<W>(r, inter, u, place[0], place[1], turns);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (place[i] < 0) continue;
            uint8_t* const at = (uint8_t*)r.out + o0 + row * r.os[1] + place[i] * r.os[3];
            float f[W];
#pragma unroll
            for (int j = 0; j < W; ++j) f[j] = unscale(e4m3_to_f32(at[j]), e - old);
            store_codes<W>(at, f);
          }
        }
      }
    }
  }
  if (on)
    each([&](int row, int lo, int hi, float (&x)[W], float (&y)[W]) {
#pragma unroll
      for (int j = 0; j < W; ++j) x[j] = unscale(x[j], e), y[j] = unscale(y[j], e);
      uint8_t* const at = (uint8_t*)r.out + o0 + row * r.os[1];
      store_codes<W>(at + lo * r.os[3], x);
      if (hi >= 0) store_codes<W>(at + hi * r.os[3], y);
    });
  if (lane == 0) sp[0] = (uint8_t)(e + 127);
}

template <typename XT, int CACHE, int W>
__global__ __launch_bounds__(THREADS) void append_kernel(const AppendParams p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t group = blockIdx.x;
  if constexpr (CACHE == CACHE_BLOCK) {
    const uint32_t groups = (p.block_waves + WAVES - 1) / WAVES;
    if (group < groups) {
      const uint32_t w = group * WAVES + wave;
      if (w < p.block_waves) own_block<XT, W>(p, w, lane);
      return;
    }
    group -= groups;
  }
  token_rows<XT, CACHE, W>(p, group, wave, lane);
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
  return true;
}

template <typename XT, int W>
void launch_append(int cache, const AppendParams& p, uint32_t groups, hipStream_t s) {
  const dim3 grid(groups), block(THREADS);
  switch (cache) {
    case CACHE_NONE: hipLaunchKernelGGL((append_kernel<XT, CACHE_NONE, W>), grid, block, 0, s, p); break;
    case CACHE_SAME: hipLaunchKernelGGL((append_kernel<XT, CACHE_SAME, W>), grid, block, 0, s, p); break;
    case CACHE_E4M3: hipLaunchKernelGGL((append_kernel<XT, CACHE_E4M3, W>), grid, block, 0, s, p); break;
    default: hipLaunchKernelGGL((append_kernel<XT, CACHE_BLOCK, W>), grid, block, 0, s, p); break;
  }
}

// Fills in what the parts have in common and launches.
int run_append(AppendParams& p, int dtype, int cache, void* stream, const char* who) {
  const int esz = dtype == FA_F32 ? 4 : 2;
  bool vec = true;
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
  p.row_heads = p.part[0].heads + (cache == CACHE_BLOCK ? 0 : p.part[1].heads + p.part[2].heads);
  int64_t groups = p.row_heads ? p.tokens : 0;
  if (cache == CACHE_BLOCK) {
    const int64_t waves = (p.tokens / p.block + 2 * (int64_t)p.batch) * 2 * p.part[1].heads;
    FA_REQUIRE(waves <= 0x7fffffffll, "%s: too many blocks", who);
    p.block_waves = (uint32_t)waves;
    groups += fa_ceil_div(waves, WAVES);
  }
  FA_REQUIRE(groups < 1ll << 24, "%s: too many rows", who);   // 2^32 threads a launch
  if (groups == 0) return FA_OK;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case FA_F16: vec ? launch_append<F16T, 8>(cache, p, groups, s) : launch_append<F16T, 1>(cache, p, groups, s); break;
    case FA_BF16: vec ? launch_append<BF16T, 8>(cache, p, groups, s) : launch_append<BF16T, 1>(cache, p, groups, s); break;
    default: vec ? launch_append<F32T, 4>(cache, p, groups, s) : launch_append<F32T, 1>(cache, p, groups, s); break;
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
  p.tokens = a->tokens, p.batch = (int32_t)a->batch, p.page_size = a->page_size;
  p.num_pages = a->num_pages, p.table_cols = a->table_cols;
  p.block = (int32_t)a->block;
  return run_append(p, xdt, a->block ? CACHE_BLOCK : cdt == FA_E4M3 ? CACHE_E4M3 : CACHE_SAME, stream, who);
}
