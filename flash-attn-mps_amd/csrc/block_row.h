// One query row over keys of a block-scaled cache, by one wave: the generic
// kernel's route, and what the matrix-core kernels run for rows whose sums are
// not finite.  A matrix product multiplies hidden values by probabilities of
// zero, so a NaN in a value that a row does not see reaches the row's sum; here
// a row reads only what it sees.  fp32 throughout; one key per lane for the
// scores, then lanes own output dims.
#pragma once

#include "attn_common.h"

// The arguments of a kernel whose first parameter they are, through an address
// that the compiler cannot see into: a rarely taken route then loads what it
// needs when it runs, where its uses of the parameter itself would keep two
// hundred scalars for the whole kernel.
FA_DEV const fa_block_attn& block_arguments() {
  auto p = (const fa_block_attn*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
}

// q(d): the query's element d.  emit(d, x): output element d, normalised.  The
// row sees keys of [begin, end) that key_allowed lets through; the sink joins
// split 0.  Returns the LSE: -inf without a key, NaN where the sum is.  Values
// enter the sum times 2^-16, so that 2^16 keys of the largest stay in fp32.
// Dv <= 64 * ACC.
template <int ACC, typename Q, typename E>
FA_DEV float block_row(const fa_block_attn& a, int64_t b, const RequestInfo& r, int kh, int h, int split, int64_t tq,
                       int q_abs, int begin, int end, int lane, Q q, E emit) {
  const float scale = a.softmax_scale * descale_of(a.q_descale, a.q_descale_stride, b, kh);
  const float slope = a.alibi ? a.alibi[b * a.alibi_stride[0] + (int64_t)h * a.alibi_stride[1]] : 0.0f;
  if (a.mask_kind == 0) {
    if (r.causal) end = min(end, q_abs + 1);
    if (a.window_left >= 0) begin = max(begin, q_abs - a.window_left);
    if (a.window_right >= 0) end = min(end, q_abs + a.window_right + 1);
  }
  // Page and row of key t, and the scale of its K or V.
  auto place = [&](int t, int64_t& page, int& row) {
    const uint32_t size = (uint32_t)a.page_size, column = (uint32_t)t / size;
    row = (int)((uint32_t)t - column * size);
    page = a.block_table[b * a.bt_stride[0] + (int64_t)column * a.bt_stride[1]];
  };
  auto offset = [&](const int64_t* st, int64_t page, int row) { return page * st[0] + row * st[1] + (int64_t)kh * st[2]; };
  float m = a.sinks && split == 0 ? a.sinks[(int64_t)h * a.sink_stride] : -INFINITY, l = m > -INFINITY ? 1.0f : 0.0f;
  float acc[ACC];
#pragma unroll
  for (int i = 0; i < ACC; ++i) acc[i] = 0.0f;
  const int Dq = (int)a.head_dim_qk, Dv = (int)a.head_dim_v;
  for (int t0 = begin; t0 < end; t0 += 64) {
    const int t = t0 + lane;
    const bool valid = t < end && key_allowed(a, b, t, q_abs, tq, r.causal);
    float s = -INFINITY;
    if (valid) {
      int64_t page;
      int row;
      place(t, page, row);
      const int64_t off = offset(a.k_stride, page, row);
      float dot = 0.0f;
      for (int d = 0; d < Dq; ++d) dot = fmaf(q(d), load_elem<E4M3T>(a.k, off + d * a.k_stride[3]), dot);
      s = dot * e8m0_to_f32(scale_byte(a, 0, page, row, kh)) * scale;
      if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
      s -= slope * (float)abs(q_abs - t);
    }
    const float m_new = fmaxf(m, wave_max(s)), ref = m_new == -INFINITY ? 0.0f : m_new;
    const float factor = expf(m - ref), p = valid ? expf(s - ref) : 0.0f;
    l = l * factor + wave_sum(p);
#pragma unroll
    for (int i = 0; i < ACC; ++i) acc[i] *= factor;
    for (uint64_t seen = __ballot(valid); seen; seen &= seen - 1) {
      const int j = __builtin_ctzll(seen);
      const float pj = readlane_f(p, j);
      int64_t page;
      int row;
      place(t0 + j, page, row);
      const int64_t off = offset(a.v_stride, page, row);
      const float vs = e8m0_to_f32(scale_byte(a, 1, page, row, kh)) * 0x1p-16f;
#pragma unroll
      for (int i = 0; i < ACC; ++i) {
        const int d = lane + 64 * i;
        if (d < Dv) acc[i] = fmaf(pj, load_elem<E4M3T>(a.v, off + d * a.v_stride[3]) * vs, acc[i]);
      }
    }
    m = m_new;
  }
  const float norm = l > 0.0f ? 1.0f / l : 0.0f;   // (a NaN sum has NaN in every acc)
#pragma unroll
  for (int i = 0; i < ACC; ++i) {
    const int d = lane + 64 * i;
    if (d < Dv) emit(d, l != l ? l : acc[i] * norm * 0x1p16f);
  }
  return l == 0.0f ? -INFINITY : m + logf(l);
}
