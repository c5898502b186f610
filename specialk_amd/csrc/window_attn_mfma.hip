// Attention within a sliding window, forward and backward, for bf16 heads on the matrix cores (v_mfma_f32_32x32x16_bf16).
// The mathematics stands in window_attn.hip; this is the path for 16-byte aligned heads of a multiple of 8 elements.  LDS
// rows are 64 or 128 columns (D), the arithmetic is done on the next multiple of 32 (W; elements beyond the head are zero).
//
// A wave owns 32 rows (queries; keys in the dK / dV kernel), a block 128, and sweeps the other side in tiles of 64 rows.
// All products are D[rho][c] = sum_k X[rho][k] Y[c][k] with X from LDS and the own rows Y in registers: lane c = lane & 31
// (+ 32 h) of the accumulator holds own row c, its 16 registers the other rows 8 (r / 4) + 4 h + r % 4.  The scores,
// turned into probabilities and rounded to bf16, are as they stand the Y operand of the next product when its X operand is
// taken in the same row order, which the transposing LDS read does.  So a softmax row is 32 registers and one exchange
// between the wave's halves, and nothing but operand tiles ever goes through LDS.
//
// Tiles come by buffer loads straight into LDS, one tile ahead of the arithmetic, their 16-byte chunks exchanged with the
// row number (applied to the source address) so that reads by rows and by columns spread over the banks.  A row that no
// query may use (padding, before the window, behind the text) gets an offset beyond the buffer: the load then writes
// zeros, and whatever the row holds never meets the arithmetic.  Tiles wholly visible to a wave skip the masks; tiles
// wholly invisible to it are skipped but for the barrier.
#include "window_attn.h"
#include <algorithm>
#include <type_traits>

using namespace skwin;

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((address_space(3))) void* lds_ptr;

constexpr int NT = 64;         // rows per LDS tile
constexpr int OWN = 128;       // own rows per block
constexpr int TOGETHER = 96;   // widest heads whose dK and dV come from one launch (see there)
constexpr float LOG2E = 1.44269504088896340736f;
constexpr uint32_t NOWHERE = 0x80000000u;   // offset beyond every buffer

__device__ __forceinline__ f32x16_t mfma(bf16x8_t x, bf16x8_t y, f32x16_t acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t zero16() {
  f32x16_t z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// Byte address of 16-byte chunk `chunk` of row `row` within a tile of D columns.  The banks' 256 bytes hold one row of 128
// columns or two of 64; the exchange sends the same chunk of 16 rows (reads by rows) to 16 different places, and four
// neighbouring chunks of 4 rows (reads by columns) too.
template <int D> __device__ __forceinline__ int mix(int row) {
  return D == 64 ? ((row & 2) << 1) | ((row & 4) >> 1) | ((row & 8) >> 3) : ((row & 3) << 2) | ((row & 12) >> 2);
}
template <int D> __device__ __forceinline__ int at(int row, int chunk) { return row * (2 * D) + ((chunk ^ mix<D>(row)) << 4); }
template <int D> constexpr int tile_bytes() { return NT * 2 * D; }

// rows row0 .. row0+31 as the X operand, columns 16 s + 8 h ..
template <int D> __device__ __forceinline__ bf16x8_t x_rows(const char* t, int row0, int s, int lane) {
  return *(const bf16x8_t*)(t + at<D>(row0 + (lane & 31), 2 * s + (lane >> 5)));
}
// columns col0 .. col0+31 as the X operand, rows row0 + 4 h .. + 3 and row0 + 8 + 4 h .. + 3
template <int D> __device__ __forceinline__ bf16x8_t x_cols(const char* t, int col0, int row0, int lane) {
  typedef __attribute__((address_space(3))) s16x4_t* lds_v4;
  const int row = row0 + 4 * (lane >> 5) + ((lane & 15) >> 2), col = col0 + (lane & 16) + 4 * (lane & 3);
  s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(t + at<D>(row, col >> 3) + (col & 7) * 2));
  s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(t + at<D>(row + 8, col >> 3) + (col & 7) * 2));
  s16x8_t f = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(bf16x8_t, f);
}

// Tile of 64 rows from `base` (row stride ld elements, d columns): rows whose bit in `ok` is clear become zero.
template <int D>
__device__ __forceinline__ void load_tile(char* t, const bf16_t* base, int64_t ld, int d, uint64_t ok, int wave, int lane) {
  constexpr int CH = D / 8, ROWS = 64 / CH;      // chunks per row, rows per instruction
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00027000);
  const uint32_t ldb = (uint32_t)ld * 2;
#pragma unroll
  for (int j = 0; j < NT / ROWS / 4; ++j) {
    const int idx = wave * (NT / ROWS / 4) + j, row = idx * ROWS + lane / CH, chunk = (lane % CH) ^ mix<D>(row);
    const bool use = ((ok >> row) & 1) && chunk * 8 < d;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(t + idx * 1024), 16, use ? row * ldb + chunk * 16 : NOWHERE, 0, 0, 0);
  }
}

// own row: y[s] = elements 16 s + 8 h .. + 7
template <int W>
__device__ __forceinline__ void load_own(bf16x8_t (&y)[W / 16], const bf16_t* row, int d, int h, bool ok) {
#pragma unroll
  for (int s = 0; s < W / 16; ++s) {
    const int c = 16 * s + 8 * h;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (ok && c < d) v = *(const uint4*)(row + c);
    y[s] = __builtin_bit_cast(bf16x8_t, v);
  }
}

__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {   // a's upper half <-> b's lower half
  auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
__device__ __forceinline__ float other_max(float v) {
  uint32_t a = __float_as_uint(v), b = a;
  swap_halves(a, b);
  return fmaxf(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float other_sum(float v) {
  uint32_t a = __float_as_uint(v), b = a;
  swap_halves(a, b);
  return __uint_as_float(a) + __uint_as_float(b);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
  bf16x2_t v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}
// registers 8 s .. 8 s + 7 of an accumulator as the Y operand of 16 rows
__device__ __forceinline__ bf16x8_t pack_y(const f32x16_t& a, int s) {
  uint4 v = make_uint4(pack2(a[8 * s], a[8 * s + 1]), pack2(a[8 * s + 2], a[8 * s + 3]), pack2(a[8 * s + 4], a[8 * s + 5]),
                       pack2(a[8 * s + 6], a[8 * s + 7]));
  return __builtin_bit_cast(bf16x8_t, v);
}

// Own row's output, columns 32 t + 8 (r / 4) + 4 h + r % 4: the halves exchange their 8-byte pieces so that each lane
// stores 16 bytes.
template <int W>
__device__ __forceinline__ void store_own(bf16_t* row, const f32x16_t (&o)[W / 32], float mul, int d, int h, bool ok) {
#pragma unroll
  for (int t = 0; t < W / 32; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t a0 = pack2(o[t][8 * u] * mul, o[t][8 * u + 1] * mul), a1 = pack2(o[t][8 * u + 2] * mul, o[t][8 * u + 3] * mul);
      uint32_t b0 = pack2(o[t][8 * u + 4] * mul, o[t][8 * u + 5] * mul), b1 = pack2(o[t][8 * u + 6] * mul, o[t][8 * u + 7] * mul);
      swap_halves(a0, b0);
      swap_halves(a1, b1);
      const int c = 32 * t + 16 * u + 8 * h;
      if (ok && c < d) *(uint4*)(row + c) = make_uint4(a0, a1, b0, b1);
    }
}

// the same in fp32, for partial sums
template <int W>
__device__ __forceinline__ void store_own_f32(float* row, const f32x16_t (&o)[W / 32], float mul, int d, int h) {
#pragma unroll
  for (int t = 0; t < W / 32; ++t)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = 32 * t + 8 * u + 4 * h;
      if (c < d) *(float4*)(row + c) = make_float4(o[t][4 * u] * mul, o[t][4 * u + 1] * mul, o[t][4 * u + 2] * mul, o[t][4 * u + 3] * mul);
    }
}

// All ones where register r's bit of the row mask is set, else 0: mk is the tile half's 32 bits, shifted by 4 h.
__device__ __forceinline__ uint32_t lane_bit(uint32_t mk, int r) { return (uint32_t)__builtin_amdgcn_sbfe((int)mk, 8 * (r >> 2) + (r & 3), 1); }
// (opaque(mk) inside a wave-uniform `if` keeps that a branch: hoisted and turned into selects, the masks of the few partly
// visible tiles would cost every tile three instructions a score)
__device__ __forceinline__ void opaque(uint32_t& mk) { asm volatile("" : "+v"(mk)); }
__device__ __forceinline__ float keep_or(float v, uint32_t m, uint32_t other) {
  return __uint_as_float((__float_as_uint(v) & m) | (other & ~m));
}

// ------------------------------------------------------------------------------ forward
// Bound by matrix and vector unit together: a 32 x 32 score tile costs 8 (d = 64) or 16 (d = 128) matrix instructions of 32
// cycles and some 100 vector instructions, 16 of them exponentials, and the two units' busy times add up to all of the
// kernel's (50 + 52 % at d = 128, 34 + 71 % at 64).  Dealing the matrix instructions out among the vector ones (scores of
// the next half tile beside the probabilities of this one) does not help: the chip, at 1.8 of 2.4 GHz in this kernel, is
// held by power as well (32771 tokens of 32 / 8 heads of 128, window 4096: 2.10 - 2.19 ms by box, 940 - 980 TFLOP/s; so dealt
// a twentieth to an eighth more; a product of two 8192 x 8192 matrices reaches 1214).  So the arithmetic itself is kept small: the scale goes into the exponent's
// multiply-add, and the accumulators are rescaled only when a row's maximum has grown by more than 2^8 since the last
// time: until then probabilities stay below 256, which bf16 holds as precisely as values below one.
// Small windows are bound by the rows' way from memory instead: 256 packed sentences of 3 - 400 tokens, 8 heads of 64,
// window 64 both ways: 61 us (3.4 TB/s of q, k, v, o), dQ 95 (3.4), dK and dV 98 (3.2), half of it waiting, at 2.2 waves a
// SIMD; a third tile buffer, a sentence's tiles closer together and earlier first loads changed nothing.
template <int D, int W>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void fwd_kernel(WinParams p, int qtiles) {
  __shared__ __attribute__((aligned(1024))) char lds[2][2 * tile_bytes<D>()];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, hf = lane >> 5;
  const Work work = work_of_block(p, qtiles * p.cuts, p.H / p.G, true);
  if (work.none) return;
  const int h = work.h, b = work.b, kh = h / (p.H / p.G), cut = work.tile % p.cuts;
  if (b == p.B) {
    zero_rest<bf16_t>((bf16_t*)p.Oout, p.ldo, (int64_t)h * p.d, p.d, p.q_off, p.B, p.Tq, work.tile, TAIL);
    return;
  }
  const Seq sq = seq_of(p, b);
  const int i0 = work.tile / p.cuts * OWN;
  if (i0 >= sq.Lq) return;
  const KeyTiles kt = KeyTiles::of<NT>(p, sq, i0, min(i0 + OWN, sq.Lq));
  const int w0 = i0 + 32 * wave, i = w0 + c, pos = i + sq.off;
  const int pmin = w0 + sq.off, pmax = min(w0 + 31, sq.Lq - 1) + sq.off;      // (pmax < pmin: no rows)
  const bf16_t* K = (const bf16_t*)p.K + sq.kbase * p.ldk + (int64_t)kh * p.d;
  const bf16_t* V = (const bf16_t*)p.V + sq.kbase * p.ldv + (int64_t)kh * p.d;
  const uint8_t* pad = p.key_pad ? p.key_pad + (int64_t)b * p.Lk : nullptr;
  const float cs = fabsf(p.scale) * LOG2E;
  bf16x8_t q[W / 16];
  load_own<W>(q, (const bf16_t*)p.Q + (sq.qbase + min(i, sq.Lq - 1)) * p.ldq + (int64_t)h * p.d, p.d, hf, i < sq.Lq);
  if (p.scale < 0.f) {   // the maximum is taken over unscaled scores
#pragma unroll
    for (int s = 0; s < W / 16; ++s) {
      uint4 v = __builtin_bit_cast(uint4, q[s]);
      v.x ^= 0x80008000u; v.y ^= 0x80008000u; v.z ^= 0x80008000u; v.w ^= 0x80008000u;
      q[s] = __builtin_bit_cast(bf16x8_t, v);
    }
  }
  f32x16_t o[W / 32];
#pragma unroll
  for (int t = 0; t < W / 32; ++t) o[t] = zero16();
  float m = -INFINITY, l = 0.f;

  // rows of tile t that may be used; the padding byte comes a round ahead, so that no wait for it waits for a tile too
  auto padding = [&](int t) -> int { return pad && t < kt.n ? pad[min(kt.start<NT>(t) + lane, sq.Lk - 1)] : 0; };
  auto usable = [&](int t, int gone) -> uint64_t { return __ballot(kt.holds(kt.start<NT>(t) + lane) && !gone); };
  auto fetch = [&](int t, uint64_t ok) {
    const int64_t j0 = kt.start<NT>(t);
    char* buf = lds[t & 1];
    load_tile<D>(buf, K + j0 * p.ldk, p.ldk, p.d, ok, wave, lane);
    load_tile<D>(buf + tile_bytes<D>(), V + j0 * p.ldv, p.ldv, p.d, ok, wave, lane);
  };
  const int n = max(0, kt.n), t_beg = (int)((int64_t)n * cut / p.cuts), t_end = (int)((int64_t)n * (cut + 1) / p.cuts);
  uint64_t ok = 0;
  int gone = padding(t_beg);
  if (t_beg < t_end) { ok = usable(t_beg, gone); fetch(t_beg, ok); }
  gone = padding(t_beg + 1);
  for (int t = t_beg; t < t_end; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();     // tile t is in LDS, and every wave is done with the other buffer
    const uint64_t use = ok;
    if (t + 1 < t_end) {
      ok = usable(t + 1, gone);
      fetch(t + 1, ok);
      gone = padding(t + 2);
    }
    const int j0 = kt.start<NT>(t);
    if (use == 0 || pmax < pmin || j0 > pmax + p.right || (j0 + NT - 1 < pmin - p.left && j0 >= p.sinks)) continue;   // wave-uniform
    const char* Ks = lds[t & 1];
    const char* Vs = Ks + tile_bytes<D>();
    f32x16_t sc[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      sc[k] = zero16();
#pragma unroll
      for (int s = 0; s < W / 16; ++s) sc[k] = mfma(x_rows<D>(Ks, 32 * k, s, lane), q[s], sc[k]);
    }
    const bool whole = use == ~0ull && j0 + NT - 1 <= pmin + p.right && (j0 >= pmax - p.left || j0 + NT <= p.sinks);
    if (!whole) {
      const uint64_t see = keys_seen(p, pos, j0, use);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t mk = (uint32_t)(see >> (32 * k)) >> (4 * hf);
        opaque(mk);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          sc[k][r] = keep_or(sc[k][r], lane_bit(mk, r), 0xff800000u);   // -inf
      }
    }
    float mx = sc[0][0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, sc[0][r]);
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[1][r]);
    mx = other_max(mx);
    if (__any((mx - m) * cs > 8.f)) {   // (also from -inf; both -inf: NaN, no)
      const float mn = m == -INFINITY || (mx - m) * cs > 8.f ? fmaxf(m, mx) : m;   // (a row's own scores decide, not its neighbours')
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * cs);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int x = 0; x < W / 32; ++x) o[x] *= alpha;
    }
    const float mc = m == -INFINITY ? 0.f : m * cs;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sc[k][r] = __builtin_amdgcn_exp2f(fmaf(sc[k][r], cs, -mc));
        sum += sc[k][r];
      }
    l += sum;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const bf16x8_t y = pack_y(sc[k], s);
#pragma unroll
        for (int x = 0; x < W / 32; ++x) o[x] = mfma(x_cols<D>(Vs, 32 * x, 32 * k + 16 * s, lane), y, o[x]);
      }
  }
  l = other_sum(l);   // the halves summed different keys
  if (p.cuts > 1) {
    if (i >= sq.Lq) return;
    const int64_t row = ((int64_t)cut * p.H + h) * p.Tq + sq.qbase + i;
    store_own_f32<W>(p.cut_o + row * p.d, o, 1.f, p.d, hf);
    if (hf == 0) { p.cut_ml[2 * row] = m * cs; p.cut_ml[2 * row + 1] = l; }
    return;
  }
  store_own<W>((bf16_t*)p.Oout + (sq.qbase + min(i, sq.Lq - 1)) * p.ldo + (int64_t)h * p.d, o, l > 0.f || l != l ? 1.f / l : 0.f, p.d, hf,
               i < sq.Lq);
  if (i < sq.Lq && hf == 0)
    p.LSE[(int64_t)h * p.Tq + sq.qbase + i] = l > 0.f ? m * fabsf(p.scale) + logf(l) : (l != l ? l : -INFINITY);
}

// ------------------------------------------------------------------------------ dQ, delta
// Also leaves the rows' -log-sum-exp / scale and -delta, delta = rowsum(dO O), for the dK / dV kernel.  dS is rounded to
// bf16 without the scale, which multiplies the fp32 sums at the end.
// O carries two roundings to 2^-8 (the probabilities', its own), and delta inherits them: against the rounding of dS
// itself that is 1 / sqrt(n) as much for a row that sees n keys alike.  Rows of at most FEW keys (the first rows of a text,
// rows behind it, small windows) take delta = sum_j P dP in fp32 from a sweep of its own: with four visible keys dQ and dK
// are then 1.4 instead of 1.65 times as far from the exact values as a result rounded once.  Waves without such rows
// sit that sweep out, and two tiles or fewer stay in LDS for the second (256 causal texts of 100 tokens, 8 heads of 64: dQ
// 47.5 -> 41.5 us).
template <int D, int W>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void dq_kernel(WinParams p, int qtiles) {
  __shared__ __attribute__((aligned(1024))) char lds[2][2 * tile_bytes<D>()];
  __shared__ int s_few[4][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, hf = lane >> 5;
  const Work work = work_of_block(p, qtiles * p.cuts, p.H / p.G, true);
  if (work.none) return;
  const int h = work.h, b = work.b, kh = h / (p.H / p.G), cut = work.tile % p.cuts;
  if (b == p.B) {
    zero_rest<bf16_t>((bf16_t*)p.dQ, p.lddq, (int64_t)h * p.d, p.d, p.q_off, p.B, p.Tq, work.tile, TAIL);
    return;
  }
  const Seq sq = seq_of(p, b);
  const int i0 = work.tile / p.cuts * OWN;
  if (i0 >= sq.Lq) return;
  const KeyTiles kt = KeyTiles::of<NT>(p, sq, i0, min(i0 + OWN, sq.Lq));
  const int w0 = i0 + 32 * wave, i = w0 + c, pos = i + sq.off;
  const int pmin = w0 + sq.off, pmax = min(w0 + 31, sq.Lq - 1) + sq.off;
  const int64_t row = sq.qbase + min(i, sq.Lq - 1), si = (int64_t)h * p.Tq + row;
  const bf16_t* K = (const bf16_t*)p.K + sq.kbase * p.ldk + (int64_t)kh * p.d;
  const bf16_t* V = (const bf16_t*)p.V + sq.kbase * p.ldv + (int64_t)kh * p.d;
  const uint8_t* pad = p.key_pad ? p.key_pad + (int64_t)b * p.Lk : nullptr;
  const float cs = p.scale * LOG2E;
  bf16x8_t q[W / 16], g[W / 16];
  load_own<W>(g, (const bf16_t*)p.dO + row * p.lddo + (int64_t)h * p.d, p.d, hf, i < sq.Lq);
  load_own<W>(q, (const bf16_t*)p.O + row * p.ldo + (int64_t)h * p.d, p.d, hf, i < sq.Lq);
  float dl = 0.f;
#pragma unroll
  for (int s = 0; s < W / 16; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) dl += (float)q[s][j] * (float)g[s][j];
  dl = other_sum(dl);
  load_own<W>(q, (const bf16_t*)p.Q + row * p.ldq + (int64_t)h * p.d, p.d, hf, i < sq.Lq);
  const float lse2 = p.LSE[si] * LOG2E;
  f32x16_t dq[W / 32];
#pragma unroll
  for (int t = 0; t < W / 32; ++t) dq[t] = zero16();

  // rows of tile t that may be used; the padding byte comes a round ahead, so that no wait for it waits for a tile too
  auto padding = [&](int t) -> int { return pad && t < kt.n ? pad[min(kt.start<NT>(t) + lane, sq.Lk - 1)] : 0; };
  auto usable = [&](int t, int gone) -> uint64_t { return __ballot(kt.holds(kt.start<NT>(t) + lane) && !gone); };
  auto fetch = [&](int t, uint64_t ok) {
    const int64_t j0 = kt.start<NT>(t);
    char* buf = lds[t & 1];
    load_tile<D>(buf, K + j0 * p.ldk, p.ldk, p.d, ok, wave, lane);
    load_tile<D>(buf + tile_bytes<D>(), V + j0 * p.ldv, p.ldv, p.d, ok, wave, lane);
  };
  const FewKeys fk = few_keys(p, kt, pos, i < sq.Lq, padding, usable);
  if (lane == 0) { s_few[wave][0] = fk.lo; s_few[wave][1] = fk.hi; }
  const bool few_row = fk.row, few_wave = __any(few_row), few = __syncthreads_or(few_row);
  // one half tile: scores and dP; then the half's part of delta, or dS and its product
  auto half_tile = [&](auto delta_only, bool whole, const char* Ks, const char* Vs, int k, uint32_t mk) {
    f32x16_t sc = zero16(), dp = zero16();
#pragma unroll
    for (int s = 0; s < W / 16; ++s) {
      sc = mfma(x_rows<D>(Ks, 32 * k, s, lane), q[s], sc);
      dp = mfma(x_rows<D>(Vs, 32 * k, s, lane), g[s], dp);
    }
    float part = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float pr = __builtin_amdgcn_exp2f(fmaf(sc[r], cs, -lse2));
      sc[r] = pr * (delta_only ? dp[r] : dp[r] - dl);
    }
    if (!whole) {
      opaque(mk);
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = keep_or(sc[r], lane_bit(mk, r), 0u);
    }
    if (delta_only) {
#pragma unroll
      for (int r = 0; r < 16; ++r) part += sc[r];
    }
    if constexpr (!delta_only) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const bf16x8_t y = pack_y(sc, s);
#pragma unroll
        for (int x = 0; x < W / 32; ++x) dq[x] = mfma(x_cols<D>(Ks, 32 * x, 32 * k + 16 * s, lane), y, dq[x]);
      }
    }
    return part;
  };
  auto sweep = [&](auto delta_only, bool resident, int t_beg, int t_end) {
    uint64_t ok = 0;
    int gone = padding(t_beg);
    float sum = 0.f;
    if (t_beg < t_end) ok = usable(t_beg, gone);
    if (t_beg < t_end && !resident) fetch(t_beg, ok);
    gone = padding(t_beg + 1);
    for (int t = t_beg; t < t_end; ++t) {
      if (!resident) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
      }
      const uint64_t use = ok;
      if (t + 1 < t_end) {
        ok = usable(t + 1, gone);
        if (!resident) fetch(t + 1, ok);
        gone = padding(t + 2);
      }
      if (delta_only && !few_wave) continue;
      const int j0 = kt.start<NT>(t);
      if (use == 0 || pmax < pmin || j0 > pmax + p.right || (j0 + NT - 1 < pmin - p.left && j0 >= p.sinks)) continue;
      const char* Ks = lds[t & 1];
      const char* Vs = Ks + tile_bytes<D>();
      const bool whole = use == ~0ull && j0 + NT - 1 <= pmin + p.right && (j0 >= pmax - p.left || j0 + NT <= p.sinks);
      const uint64_t see = whole ? 0 : keys_seen(p, pos, j0, use);
#pragma unroll
      for (int k = 0; k < 2; ++k) sum += half_tile(delta_only, whole, Ks, Vs, k, (uint32_t)(see >> (32 * k)) >> (4 * hf));
    }
    return sum;
  };
  const int n = max(0, kt.n);
  const bool both = few && n <= 2 && p.cuts == 1;   // (the tiles are then all in LDS when the first sweep ends)
  if (few) {
    const int lo = min(min(s_few[0][0], s_few[1][0]), min(s_few[2][0], s_few[3][0]));
    const int hi = max(max(s_few[0][1], s_few[1][1]), max(s_few[2][1], s_few[3][1]));
    const float exact = other_sum(sweep(std::true_type{}, false, both ? 0 : lo, both ? n : hi));
    dl = few_row ? exact : dl;
    if (!both) __syncthreads();   // every wave is done with the tiles
  }
  sweep(std::false_type{}, both, (int)((int64_t)n * cut / p.cuts), (int)((int64_t)n * (cut + 1) / p.cuts));
  if (i < sq.Lq && hf == 0 && cut == 0) {   // what the dK / dV kernel's accumulators start from
    p.delta[si] = -dl;
    p.delta[(int64_t)p.H * p.Tq + si] = -p.LSE[si] / p.scale;
  }
  if (p.cuts > 1) {
    if (i < sq.Lq) store_own_f32<W>(p.cut_o + (((int64_t)cut * p.H + h) * p.Tq + row) * p.d, dq, p.scale, p.d, hf);
    return;
  }
  store_own<W>((bf16_t*)p.dQ + row * p.lddq + (int64_t)h * p.d, dq, p.scale, p.d, hf, i < sq.Lq);
}

// ------------------------------------------------------------------------------ dK, dV
// Own rows are keys; the tiles hold 64 queries and their output gradients, head after head of the group that shares them.
// WHAT: 1 = dK, 2 = dV, 3 = both.  Up to a width of 96 one launch computes both (4 x 4096 tokens, 8 heads of 80, window 512,
// forward and backward: 240 us, apart 295).  At 128 the two sums and the own rows alone
// are 192 registers, and with them only one wave fits a SIMD: dK and dV as launches of their own cost the scores twice
// (10 instead of 8 products) but keep two (16384 tokens, causal, 16 heads: 3.73 ms together, 1.67 + 1.25 ms apart).
template <int D, int W, int WHAT>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void dkv_kernel(WinParams p, int ktiles) {
  constexpr bool DK = WHAT & 1, DV = WHAT & 2;
  // queries, output gradients, and their rows' -log-sum-exp / scale and -delta
  __shared__ __attribute__((aligned(1024))) char lds[2][2 * tile_bytes<D>() + 2 * NT * 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, hf = lane >> 5;
  const Work item = work_of_block(p, key_tiles_of_grid(p, ktiles), 1, p.nst > 0);
  if (item.none) return;
  const int work = item.tile, kh = item.h, b = item.b, rep = p.H / p.G;
  if (b == p.B) {
    if (DK) zero_rest<bf16_t>((bf16_t*)p.dK, p.lddk, (int64_t)kh * p.d, p.d, p.k_off, p.B, p.Tk, work, TAIL);
    if (DV) zero_rest<bf16_t>((bf16_t*)p.dV, p.lddv, (int64_t)kh * p.d, p.d, p.k_off, p.B, p.Tk, work, TAIL);
    return;
  }
  const Seq sq = seq_of(p, b);
  const KeyWork kw = key_work(p, ktiles, work);
  const int tile = kw.tile, chunk = kw.chunk;
  const int j0 = tile * OWN, j1 = min(j0 + OWN, sq.Lk);
  if (j0 >= sq.Lk) return;
  int i_lo, i_hi;
  query_range(p, sq, j0, j1, chunk, i_lo, i_hi);
  if (chunk >= 0 && i_lo >= i_hi) return;
  const int jw = j0 + 32 * wave, j = jw + c, jrow = min(j, sq.Lk - 1), jl = min(jw + 31, sq.Lk - 1);
  const bool alive = j < sq.Lk && !(p.key_pad && p.key_pad[(int64_t)b * p.Lk + jrow]);
  const bool all_alive = __all(alive), busy = jw < sq.Lk && (chunk < 0 || jw < p.sinks);   // wave-uniform
  bf16x8_t fk[W / 16], fv[W / 16];
  load_own<W>(fk, (const bf16_t*)p.K + (sq.kbase + jrow) * p.ldk + (int64_t)kh * p.d, p.d, hf, alive);
  if (DK) load_own<W>(fv, (const bf16_t*)p.V + (sq.kbase + jrow) * p.ldv + (int64_t)kh * p.d, p.d, hf, alive);
  const float cs = p.scale * LOG2E;
  f32x16_t dk[W / 32], dv[W / 32];
#pragma unroll
  for (int t = 0; t < W / 32; ++t) dk[t] = dv[t] = zero16();

  const int per = (i_hi - i_lo + NT - 1) / NT, n = per * rep;
  auto fetch = [&](int t, char* buf) {
    const int hh = t / per, r0 = i_lo + (t - hh * per) * NT, h = kh * rep + hh;
    const uint64_t ok = bits(0, i_hi - r0);
    load_tile<D>(buf, (const bf16_t*)p.Q + (sq.qbase + r0) * p.ldq + (int64_t)h * p.d, p.ldq, p.d, ok, wave, lane);
    load_tile<D>(buf + tile_bytes<D>(), (const bf16_t*)p.dO + (sq.qbase + r0) * p.lddo + (int64_t)h * p.d, p.lddo, p.d, ok, wave, lane);
    if (wave < 2) {
      const float* src = p.delta + (wave ? 0 : (int64_t)p.H * p.Tq) + (int64_t)h * p.Tq + sq.qbase + r0;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)src, 0, 0x7fffffff, 0x00027000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(buf + 2 * tile_bytes<D>() + wave * NT * 4), 4, r0 + lane < i_hi ? lane * 4 : NOWHERE, 0, 0, 0);
    }
  };
  auto half_tile = [&](bool whole, const char* Qs, int k, uint32_t mk) {
    const char* Gs = Qs + tile_bytes<D>();
    const float (*rv)[NT] = (const float (*)[NT])(Qs + 2 * tile_bytes<D>());
    // the sums start from the rows' -log-sum-exp / scale and -delta: no registers for them and no subtraction
    f32x16_t sc, dp;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float4 ls = *(const float4*)&rv[0][32 * k + 8 * u + 4 * hf], de = *(const float4*)&rv[1][32 * k + 8 * u + 4 * hf];
      sc[4 * u] = ls.x; sc[4 * u + 1] = ls.y; sc[4 * u + 2] = ls.z; sc[4 * u + 3] = ls.w;
      dp[4 * u] = de.x; dp[4 * u + 1] = de.y; dp[4 * u + 2] = de.z; dp[4 * u + 3] = de.w;
    }
#pragma unroll
    for (int s = 0; s < W / 16; ++s) {
      sc = mfma(x_rows<D>(Qs, 32 * k, s, lane), fk[s], sc);
      if (DK) dp = mfma(x_rows<D>(Gs, 32 * k, s, lane), fv[s], dp);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      sc[r] = __builtin_amdgcn_exp2f(sc[r] * cs);
      dp[r] *= sc[r];
    }
    if (!whole) {
      opaque(mk);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t m = lane_bit(mk, r);
        sc[r] = keep_or(sc[r], m, 0u);
        dp[r] = keep_or(dp[r], m, 0u);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bf16x8_t yp = pack_y(sc, s), ys = pack_y(dp, s);
#pragma unroll
      for (int x = 0; x < W / 32; ++x) {
        if (DV) dv[x] = mfma(x_cols<D>(Gs, 32 * x, 32 * k + 16 * s, lane), yp, dv[x]);
        if (DK) dk[x] = mfma(x_cols<D>(Qs, 32 * x, 32 * k + 16 * s, lane), ys, dk[x]);
      }
    }
  };
  const int t_beg = chunk < 0 ? (int)((int64_t)n * kw.part / p.parts) : 0, t_end = chunk < 0 ? (int)((int64_t)n * (kw.part + 1) / p.parts) : n;
  // (two restricted pointers: else the compiler waits for the tile on its way before it reads the one in use; 256 packed
  // sentences 103 -> 99 us.  Forward and dQ have vector work before those reads and gain nothing.)
  auto round = [&](int t, const char* __restrict Qs, char* __restrict next) {
    if (t + 1 < t_end) fetch(t + 1, next);
    const int r0 = i_lo + (t % per) * NT, p0 = r0 + sq.off, p1 = min(r0 + NT, i_hi) - 1 + sq.off;
    if (!busy || p1 < jw - p.right || (p0 > jl + p.left && jw >= p.sinks)) return;
    const bool whole = all_alive && r0 + NT <= i_hi && jl <= p0 + p.right && (jw >= p1 - p.left || jl < p.sinks);
    uint64_t see = 0;
    if (!whole && alive) see = queries_seeing(p, j, p0, i_hi - r0);
#pragma unroll(D == 64 ? 1 : 2)
    for (int k = 0; k < 2; ++k) half_tile(whole, Qs, k, (uint32_t)(see >> (32 * k)) >> (4 * hf));
  };
  if (t_beg < t_end) fetch(t_beg, lds[t_beg & 1]);
  for (int t = t_beg; t < t_end; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    round(t, lds[t & 1], lds[(t + 1) & 1]);
  }
  if (p.parts > 1 && chunk < 0) {
    if (j >= sq.Lk) return;
    if (DK) store_own_f32<W>(split_row(p, kw.part, 0, b, j, kh), dk, p.scale, p.d, hf);
    if (DV) store_own_f32<W>(split_row(p, kw.part, 1, b, j, kh), dv, 1.f, p.d, hf);
    return;
  }
  const bool sink = p.nst && j < p.sinks;   // (a sink's sum has further parts)
  if (sink && j < sq.Lk) {
    float* s = slab(p, b, kh, tile, 1 + chunk, OWN) + (int64_t)(j - j0) * p.d;
    if (DK) store_own_f32<W>(s, dk, p.scale, p.d, hf);
    if (DV) store_own_f32<W>(s + (int64_t)slab_rows(p, OWN) * p.d, dv, 1.f, p.d, hf);
  }
  if (chunk >= 0) return;
  if (DK) store_own<W>((bf16_t*)p.dK + (sq.kbase + jrow) * p.lddk + (int64_t)kh * p.d, dk, p.scale, p.d, hf, j < sq.Lk && !sink);
  if (DV) store_own<W>((bf16_t*)p.dV + (sq.kbase + jrow) * p.lddv + (int64_t)kh * p.d, dv, 1.f, p.d, hf, j < sq.Lk && !sink);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int D, int W>
void launch_fwd(const WinParams& p, hipStream_t stream) {
  const int qtiles = std::max(1, (p.Lq + OWN - 1) / OWN);
  const dim3 grid(work_blocks(p, qtiles * p.cuts, p.H / p.G));
  hipLaunchKernelGGL((fwd_kernel<D, W>), grid, dim3(256), 0, stream, p, qtiles);
}
template <int D, int W>
void launch_bwd(const WinParams& p, hipStream_t stream) {
  const int qtiles = std::max(1, (p.Lq + OWN - 1) / OWN), ktiles = std::max(1, (p.Lk + OWN - 1) / OWN);
  const dim3 gq(work_blocks(p, qtiles * p.cuts, p.H / p.G)), gk(work_blocks(p, key_tiles_of_grid(p, ktiles), 1));
  if (p.Tq) hipLaunchKernelGGL((dq_kernel<D, W>), gq, dim3(256), 0, stream, p, qtiles);
  if (!p.Tk) return;
  if constexpr (W <= TOGETHER) {
    hipLaunchKernelGGL((dkv_kernel<D, W, 3>), gk, dim3(256), 0, stream, p, ktiles);
  } else {
    hipLaunchKernelGGL((dkv_kernel<D, W, 1>), gk, dim3(256), 0, stream, p, ktiles);
    hipLaunchKernelGGL((dkv_kernel<D, W, 2>), gk, dim3(256), 0, stream, p, ktiles);
  }
}

}  // namespace

// Heads whose rows are whole 16-byte pieces; 32-bit offsets within a tile of 64 rows; a finite scale that is not zero or next
// to it: the maximum of the unscaled scores stands for that of the scaled ones, and the backward pass divides by it.
bool sk_window_mfma_supported(const WinParams& p, int dtype) {
  if (dtype != SK_BF16 || p.d % 8 || p.d > 128 || !(fabsf(p.scale) >= 1e-30f) || !(p.scale - p.scale == 0.f)) return false;
  const int64_t lds[] = {p.ldq, p.ldk, p.ldv, p.ldo, p.lddo, p.lddq, p.lddk, p.lddv};
  for (int64_t ld : lds)
    if (ld % 8 || ld > (1 << 23)) return false;
  const void* ptr[] = {p.Q, p.K, p.V, p.O, p.dO, p.Oout, p.dQ, p.dK, p.dV};
  for (const void* x : ptr)
    if (!aligned16(x)) return false;
  return true;
}

int sk_window_fwd_mfma(const WinParams& p, hipStream_t stream) {
  if (p.d <= 32) launch_fwd<64, 32>(p, stream);
  else if (p.d <= 64) launch_fwd<64, 64>(p, stream);
  else if (p.d <= 96) launch_fwd<128, 96>(p, stream);
  else launch_fwd<128, 128>(p, stream);
  SK_CHECK_LAUNCH("skhip_window_attn_fwd(mfma)");
  return SK_OK;
}

int sk_window_bwd_mfma(const WinParams& p, hipStream_t stream) {
  if (p.d <= 32) launch_bwd<64, 32>(p, stream);
  else if (p.d <= 64) launch_bwd<64, 64>(p, stream);
  else if (p.d <= 96) launch_bwd<128, 96>(p, stream);
  else launch_bwd<128, 128>(p, stream);
  SK_CHECK_LAUNCH("skhip_window_attn_bwd(mfma)");
  return SK_OK;
}
