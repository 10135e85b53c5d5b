// Prefill over a block-scaled cache by way of 16-bit rows: one pass widens the
// keys and values that the batch sees to the queries' type in a workspace, the
// 16-bit prefill kernels run on that, and rows that met a value that is not
// finite run again by block_row.
//
// Sums past fp32: the prefill adds p v up before it divides by the sum of p, so
// finite values of bf16's topmost scales may leave fp32's range where their mean
// does not.  With n keys, p <= 2^8 (a running maximum moves in steps of 2^8) and
// codes below 2^9, |sum p v| < 2^(17 + log2 n + e - 127): tiles with larger scales
// than 2^128 allows are flagged too, and K's likewise (a score's sum over 256 dims
// stays below 2^128 while |q| <= n).
//
// A value times its power of two is exact in bf16, and in fp16 to fp16's own
// range; blocks past a type's range count as NaN (scale_for).  The E4M3 tiles widen
// every key tile again for each block of query rows; with many rows a key that
// costs more than this pass, which HBM bounds: 3 bytes a value, 43K keys of 8 heads
// x 128, K and V, 264 MB: 56 us, 4.7 TB/s.  That prefill of 16 prompts (16/8 heads,
// 542 GFLOP): 669 us in all, 901 on the tiles, 614 on a 16-bit cache.
#include "block_row.h"

namespace {

constexpr int TILE = 64;   // keys of a workgroup
// Codes of a thread's piece: 8 are read at once, 16 bytes written next to its
// neighbour's.  (16 codes, whose two writes interleave with the neighbours': 16
// prompts of 256..4096, 16/8 heads d128 653 us in all against 642, a chunk over 16K
// keys 317 against 309.)
constexpr int CODES = 8;

struct WideParams {
  fa_block_attn a;
  uint16_t* out[2];       // [batch, capacity, heads, dim], K and V
  int32_t* flags;         // [batch, tiles, 2]: whether rows over a tile may hold sums that are not finite
  int32_t* lengths;       // [batch]: keys of a request in the workspace
  int64_t capacity;
  int32_t tiles;
  int32_t chunks[2];      // pieces of a head's row
  uint32_t top_scale;     // the largest scale byte that cannot overflow a sum
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

// Four codes -> four 16-bit values times `scale`.
template <bool BF16>
FA_DEV u32x2 widen4(uint32_t w, float scale) {
  if constexpr (BF16)
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))};
  else
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true))};
}

// Request b with its length at most max_seqlen_k: the workspace holds no key past
// that, and every part of the call has to place the rows alike.
FA_DEV RequestInfo bounded_request(const fa_attn_args& a, int64_t b) {
  RequestInfo r = load_request(a, b);
  r.k_len = (int)min((int64_t)r.k_len, a.max_seqlen_k);
  return r;
}

// The first key of request r that some query row sees.
FA_DEV int first_key(const fa_attn_args& a, const RequestInfo& r) {
  if (a.mask_kind != 0 || a.window_left < 0) return 0;
  return max(r.k_len - r.q_len - a.window_left, 0);
}

FA_DEV bool runs_here(const fa_attn_args& a, const RequestInfo& r) {
  return r.q_len > 1 || (r.q_len == 1 && !(a.flags & FA_FLAG_SKIP_SINGLE_QUERY));
}

// One workgroup per (tile, request, K or V).
template <bool BF16>
__global__ __launch_bounds__(256) void widen_kernel(const WideParams p) {
  using T = std::conditional_t<BF16, BF16T, F16T>;
  __shared__ int64_t code_at[TILE], scale_at[TILE];
  const fa_block_attn& a = p.a;
  const int tile = blockIdx.x, which = blockIdx.z;
  const int64_t b = blockIdx.y;
  const RequestInfo r = bounded_request(a, b);
  const int heads = (int)a.heads_k, chunks = p.chunks[which], per_key = heads * chunks;
  const int64_t* const st = which ? a.v_stride : a.k_stride;
  const uint8_t* const in = (const uint8_t*)(which ? a.v : a.k);
  const int begin = tile * TILE, end = min(begin + TILE, r.k_len);
  bool odd = false;
  // The prefill reads whole tiles of up to 128 keys: the first one's keys that no
  // row sees are zeros here, and their pages are not read.
  const int first = first_key(a, r);
  if (runs_here(a, r) && begin >= (first & ~127) && begin < end) {
    // Where each key's row and scales start, once for all its pieces.
    const int keys = end - begin;
    if ((int)threadIdx.x < keys && begin + (int)threadIdx.x >= first) {
      const uint32_t size = (uint32_t)a.page_size, pos = (uint32_t)begin + threadIdx.x, column = pos / size, row = pos - column * size;
      const int64_t page = a.block_table[b * a.bt_stride[0] + (int64_t)column * a.bt_stride[1]];
      const int64_t* const ss = a.scale_stride[which];
      code_at[threadIdx.x] = page * st[0] + (int64_t)row * st[1];
      scale_at[threadIdx.x] = page * ss[0] + (int64_t)(row / (uint32_t)a.block) * ss[1];
    }
    __syncthreads();
    // A thread keeps its piece (head h, chunk c) over the keys.
    const int span = per_key < 256 ? per_key : 256, step = 256 / span;   // threads of a key, keys at once
    const int key0 = (int)threadIdx.x / span, mine = key0 < step ? (int)threadIdx.x - key0 * span : per_key;
    uint16_t* const out = p.out[which] + (b * p.capacity + begin) * per_key * CODES;
    const int64_t head_codes = st[2], head_scales = a.scale_stride[which][2];
    for (int piece = mine; piece < per_key; piece += 256) {
      const int h = piece / chunks;
      const uint8_t* const codes = in + h * head_codes + (piece - h * chunks) * CODES;
      const uint8_t* const scales = a.scale[which] + h * head_scales;
      // Keys of a thread in flight (2 / 4 / 8 / 16: 350 / 334 / 329 / 329 us for 8 prompts
      // of 256-dim heads in all, 328 / 323 / 324 / 330 for a chunk over 16K keys).
      constexpr int N = 8;
      for (int k0 = key0; k0 < keys; k0 += N * step) {
        u32x2 w[N];
        uint32_t e[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int key = k0 + n * step;
          w[n] = u32x2{0, 0};
          e[n] = 127;
          if (key >= keys || begin + key < first) continue;
          const uint8_t* const src = codes + code_at[key];
          w[n] = *(const u32x2*)src;
          e[n] = scales[scale_at[key]];
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int key = k0 + n * step;
          if (key >= keys) continue;
          const uint32_t byte = scale_for<T>(e[n]);   // (here: the loads above are in flight together)
          const float scale = e8m0_to_f32(byte);
          odd |= byte > p.top_scale;   // (255, NaN, among them)
          const u32x2 x = widen4<BF16>(w[n][0], scale), y = widen4<BF16>(w[n][1], scale);
          *(u32x4*)(out + ((int64_t)key * per_key + piece) * CODES) = u32x4{x[0], x[1], y[0], y[1]};
          // NaN codes: 0x7f without the sign.
          odd |= ((((w[n][0] & 0x7f7f7f7fu) + 0x01010101u) | ((w[n][1] & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u) != 0;
        }
      }
    }
  }
  const int any = __syncthreads_or(odd);
  if (threadIdx.x != 0) return;
  p.flags[(b * p.tiles + tile) * 2 + which] = any;
  if (tile == 0 && which == 0) p.lengths[b] = r.k_len;
}

// Rows whose output is not finite, where some tile was flagged: a few workgroups
// that stop after the flags in every usual call.
template <bool BF16>
__global__ __launch_bounds__(256) void again_kernel(const WideParams p) {
  const fa_block_attn& a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  bool odd = false;
  for (int64_t i = threadIdx.x; i < a.batch * p.tiles * 2; i += 256) odd |= p.flags[i] != 0;
  if (!__syncthreads_or(odd)) return;
  const int Dv = (int)a.head_dim_v;
  for (int64_t b = 0; b < a.batch; ++b) {
    const RequestInfo r = bounded_request(a, b);
    if (!runs_here(a, r)) continue;
    for (int64_t i = (int64_t)blockIdx.x * 4 + wave; i < (int64_t)r.q_len * a.heads_q; i += (int64_t)gridDim.x * 4) {
      const int row = (int)(i / a.heads_q), h = (int)(i - (int64_t)row * a.heads_q);
      const int64_t tq = (int64_t)r.q_begin + row;
      uint16_t* const out = (uint16_t*)a.out + tq * a.out_stride[0] + (int64_t)h * a.out_stride[1];
      const uint32_t top = BF16 ? 0x7f80u : 0x7c00u;
      bool bad = false;
      for (int d = lane; d < Dv; d += 64) bad |= (out[d] & top) == top;
      if (!__any(bad)) continue;
      const float lse = block_row<4>(
          a, b, r, h / (int)(a.heads_q / a.heads_k), h, 0, tq, row + r.k_len - r.q_len, 0, r.k_len, lane,
          [&](int d) {
            const uint32_t w = ((const uint16_t*)a.q)[tq * a.q_stride[0] + (int64_t)h * a.q_stride[1] + d];
            return BF16 ? bf16_bits_to_f32(w) : f16_bits_to_f32(w);
          },
          [&](int d, float x) {
            if constexpr (BF16) store_elem<BF16T>(out, d, x);
            else store_elem<F16T>(out, d, x);
          });
      if (lane == 0) a.lse[(int64_t)h * a.lse_stride[0] + tq * a.lse_stride[1]] = lse != lse ? -INFINITY : lse;
    }
  }
}

// Whether the rows come in aligned pieces.
bool pieces_aligned(const fa_attn_args& a) {
  bool ok = a.head_dim_qk % CODES == 0 && a.head_dim_v % CODES == 0 && a.k_stride[3] == 1 && a.v_stride[3] == 1 &&
            (uintptr_t)a.k % CODES == 0 && (uintptr_t)a.v % CODES == 0;
  for (int i = 0; i < 3; ++i) ok = ok && a.k_stride[i] % CODES == 0 && a.v_stride[i] % CODES == 0;
  return ok;
}

// The 16-bit call on the workspace: request b's keys are page b of pages of
// `capacity` rows.
fa_attn_args wide_attn(const fa_block_wide_args& w) {
  fa_attn_args a = w.block.attn;
  const int64_t heads = a.heads_k;
  a.k = w.k_wide, a.v = w.v_wide;
  a.k_dtype = a.v_dtype = a.q_dtype;
  a.page_size = w.capacity;
  const int64_t dims[2] = {a.head_dim_qk, a.head_dim_v};
  for (int i = 0; i < 2; ++i) {
    int64_t* const st = i ? a.v_stride : a.k_stride;
    st[0] = w.capacity * heads * dims[i], st[1] = heads * dims[i], st[2] = dims[i], st[3] = 1;
  }
  a.seqused_k = w.flags + a.batch * 2 * fa_ceil_div(a.max_seqlen_k, TILE);   // `lengths`
  a.used_k_stride = 1;
  a.block_table = w.rows;
  a.bt_stride[0] = 1, a.bt_stride[1] = 1;
  return a;
}

bool wide_ok(const fa_block_wide_args* w, fa_block_attn* a) {
  if (!w || w->size != (int64_t)sizeof(fa_block_wide_args) || !fa_block_arguments(&w->block, a)) return false;
  if ((a->q_dtype != FA_BF16 && a->q_dtype != FA_F16) || a->out_dtype != a->q_dtype) return false;
  if (a->head_dim_v > 256 || a->batch > 65535 || a->max_seqlen_k > w->capacity || w->capacity > INT32_MAX / 2) return false;
  if (w->capacity < 1 || !pieces_aligned(*a)) return false;
  // (Rows of a wave's output are read back as they were written.)
  if (a->out_stride[2] != 1) return false;
  const fa_attn_args wide = wide_attn(*w);
  return fa_prefill_supported(&wide);
}

}  // namespace

extern "C" int fa_block_wide_supported(const fa_block_wide_args* args) {
  fa_block_attn a;
  return wide_ok(args, &a);
}

extern "C" int fa_block_wide_fwd(const fa_block_wide_args* args, void* stream) {
  const char* who = "fa_block_wide_fwd";
  FA_REQUIRE(args && args->size == (int64_t)sizeof(fa_block_wide_args), "%s: null or mismatched arguments", who);
  WideParams p;
  const int rc = fa_validate_block(&args->block, &p.a, who);
  if (rc) return rc;
  FA_REQUIRE(args->k_wide && args->v_wide && args->rows && args->flags, "%s: null workspace", who);
  fa_block_attn checked;
  if (!wide_ok(args, &checked)) {
    fa_set_error("%s: combination not supported by the 16-bit prefill", who);
    return FA_ERR_UNSUPPORTED;
  }
  if (p.a.total_q == 0) return FA_OK;
  const bool bf16 = p.a.q_dtype == FA_BF16;
  p.out[0] = (uint16_t*)args->k_wide, p.out[1] = (uint16_t*)args->v_wide;
  p.flags = args->flags;
  p.capacity = args->capacity;
  p.lengths = p.flags + p.a.batch * 2 * fa_ceil_div(p.a.max_seqlen_k, TILE);
  FA_REQUIRE(p.a.max_seqlen_k >= 1, "%s: max_seqlen_k must be positive", who);
  p.tiles = (int32_t)fa_ceil_div(p.a.max_seqlen_k, TILE);
  p.top_scale = 127 + 128 - 17;
  for (int64_t n = 1; n < p.a.max_seqlen_k; n *= 2) --p.top_scale;
  p.chunks[0] = (int32_t)(p.a.head_dim_qk / CODES), p.chunks[1] = (int32_t)(p.a.head_dim_v / CODES);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)p.tiles, (unsigned)p.a.batch, 2);
  hipLaunchKernelGGL((bf16 ? widen_kernel<true> : widen_kernel<false>), grid, dim3(256), 0, s, p);
  const int launched = fa_check_launch(who);
  if (launched) return launched;
  const fa_attn_args wide = wide_attn(*args);
  const int ran = fa_prefill_fwd(&wide, stream);
  if (ran) return ran;
  hipLaunchKernelGGL((bf16 ? again_kernel<true> : again_kernel<false>), dim3(256), dim3(256), 0, s, p);
  return fa_check_launch(who);
}
