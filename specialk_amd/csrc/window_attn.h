// Shared parameter block, visibility rule and tile lists of the windowed-attention kernels
// (window_attn.hip: fp32 arithmetic, any head size; window_attn_mfma.hip: bf16 matrix cores; window_step.hip: one query
// per sequence over a cache).
//
// Query i of a sequence with Lq queries and Lk keys stands at position p = i + Lk - Lq (the last query beside the last
// key).  It sees key j when  j <= p + right  and  (j >= p - left or j < sinks), and key j is not padding.  left and
// right are window - 1 (right = 0 in the causal form), clamped by the host to Lq + Lk.  A row that sees nothing has
// output 0, log-sum-exp -inf and no gradient.
#pragma once
#include "common.h"

namespace skwin {

struct WinParams {
  const void *Q, *K, *V, *O, *dO;
  void *Oout, *dQ, *dK, *dV;
  float* LSE;               // [H][Tq]
  float* delta;             // [H][Tq]; bf16 path: -delta, then -log-sum-exp / scale, [H][Tq] each
  float* slabs;             // partial dK, dV of the tiles that hold sinks (see below)
  const uint8_t* key_pad;   // [B][Lk]; padded batches only
  const int32_t* q_off;     // packed batches: rows of sequence b are q_off[b] .. q_off[b+1]-1; NULL: (B, Lq) rows
  const int32_t* k_off;
  int B, H, G, Lq, Lk, d;   // G key / value heads, head h reads h / (H / G); Lq, Lk: longest sequence when packed
  int64_t Tq, Tk;           // rows of Q resp. K
  int64_t ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
  float scale;
  int left, right, sinks;
  bool vec;                 // fp32 path: rows are read in pieces of 4 elements
  // Backward of the keys: queries beyond a key's window see it only if it is a sink, so the few key tiles that hold
  // sinks would sweep the whole sequence alone.  Their far queries are cut into nch chunks of ch rows, one block each;
  // window part and chunks leave fp32 partial sums in slabs, which a small kernel adds in a fixed order.
  int nst, nch, ch;
  // Few (sequence, key head, key tile)s, as where many query heads share a key head: what a block sweeps is cut into `parts`
  // blocks, each of which leaves fp32 sums in split, [parts][dK, dV][B * Lk][G * d], added in a fixed order as well.
  int parts;
  float* split;
  // Few query rows before many keys: a block's key tiles cut into `cuts` blocks, which leave unnormalised outputs (backward:
  // sums of dQ) [cuts][H][Tq][d] in cut_o and (maximum in powers of two, sum) [cuts][H][Tq][2] in cut_ml.
  int cuts;
  float *cut_o, *cut_ml;
};

constexpr int FEW = 32;   // bf16 rows that see no more keys: delta = rowsum(dO O) is not taken from the rounded O

struct Seq { int64_t qbase, kbase; int Lq, Lk, off; };

__device__ __forceinline__ Seq seq_of(const WinParams& p, int b) {
  Seq s;
  if (p.q_off) {   // offsets are device data: clamped to the tensors, lengths to what the grid covers
    const int64_t q0 = max((int64_t)0, min((int64_t)p.q_off[b], p.Tq)), q1 = max(q0, min((int64_t)p.q_off[b + 1], p.Tq));
    const int64_t k0 = max((int64_t)0, min((int64_t)p.k_off[b], p.Tk)), k1 = max(k0, min((int64_t)p.k_off[b + 1], p.Tk));
    s.qbase = q0; s.Lq = (int)min(q1 - q0, (int64_t)p.Lq);
    s.kbase = k0; s.Lk = (int)min(k1 - k0, (int64_t)p.Lk);
  } else {
    s.qbase = (int64_t)b * p.Lq; s.Lq = p.Lq;
    s.kbase = (int64_t)b * p.Lk; s.Lk = p.Lk;
  }
  s.off = s.Lk - s.Lq;
  return s;
}

// bits a .. b-1 of 64 (any a, b)
__device__ __forceinline__ uint64_t bits(int a, int b) {
  a = min(max(a, 0), 64);
  b = min(max(b, 0), 64);
  const uint64_t hi = b == 64 ? ~0ull : (1ull << b) - 1, lo = a == 64 ? ~0ull : (1ull << a) - 1;
  return hi & ~lo;
}

// Of keys j0 .. j0+63, those that a query at position pos sees; `use`: the ones that may be used at all.
__device__ __forceinline__ uint64_t keys_seen(const WinParams& p, int pos, int j0, uint64_t use) {
  const int end = pos + p.right + 1 - j0;
  return (bits(pos - p.left - j0, end) | bits(0, min(p.sinks - j0, end))) & use;
}
// Of queries at positions p0 .. p0+63, the first n of which exist, those that see key j.
__device__ __forceinline__ uint64_t queries_seeing(const WinParams& p, int j, int p0, int n) {
  return bits(j - p.right - p0, min(n, j < p.sinks ? 64 : j + p.left + 1 - p0));
}

// Keys that queries i0 .. i1-1 see: sinks [0, s_hi) where they lie before the window, and [lo, hi).  Tiles of N keys:
// the first nst cover the sinks, the others start at w0.
struct KeyTiles {
  int lo, hi, s_hi, nst, w0, n;
  template <int N>
  static __device__ __forceinline__ KeyTiles of(const WinParams& p, const Seq& sq, int i0, int i1) {
    KeyTiles t;
    t.hi = min(sq.Lk, i1 + sq.off + p.right);
    t.lo = max(0, i0 + sq.off - p.left);
    t.s_hi = max(0, min(min(p.sinks, t.lo), t.hi));
    t.nst = (t.s_hi + N - 1) / N;
    t.w0 = max(t.lo, t.nst * N);
    t.n = t.nst + max(0, (t.hi - t.w0 + N - 1) / N);
    return t;
  }
  template <int N> __device__ __forceinline__ int start(int t) const { return t < nst ? N * t : w0 + N * (t - nst); }
  __device__ __forceinline__ bool holds(int j) const { return j < hi && (j >= lo || j < s_hi); }
};

// Whether the row at position pos (on: it exists) sees few keys, and the tiles [lo, hi) in which such rows of the wave see any:
// the sweep for their delta, which every cut of the keys makes, needs no others (64 queries before 32768 keys, 8 heads of 128,
// all but 20 keys padding, forward and backward: 234 us, sweeping every tile for delta 545; nothing padded 172).
// padding(t), usable(t, padding): tile t's keys, lane by lane and as bits.
struct FewKeys { bool row; int lo, hi; };
template <typename Padding, typename Usable>
__device__ __forceinline__ FewKeys few_keys(const WinParams& p, const KeyTiles& kt, int pos, bool on, Padding padding, Usable usable) {
  FewKeys f = {false, 0, kt.n};
  int count = 0;
  auto enough = [&]() { return __all(count > FEW || !on); };
  if (!p.key_pad) {   // (the tiles are then those of the rows' windows, and few)
    for (int t = kt.n - 1; t >= 0; --t) {
      count += __popcll(keys_seen(p, pos, kt.start<64>(t), usable(t, 0)));
      if (enough()) break;
    }
    f.row = on && count <= FEW;
    return f;
  }
  constexpr int GROUP = 4;   // tiles whose padding is on its way at a time: where little is left the whole text is walked
  f.lo = kt.n;
  f.hi = 0;
  bool more = true;
  for (int t0 = kt.n - 1; more && t0 >= 0; t0 -= GROUP) {
    int gone[GROUP];
#pragma unroll
    for (int u = 0; u < GROUP; ++u) gone[u] = padding(max(t0 - u, 0));
#pragma unroll
    for (int u = 0; u < GROUP; ++u) {
      const int t = t0 - u;
      if (!more || t < 0) break;
      const uint64_t use = usable(t, gone[u]);
      if (!use) continue;
      const uint64_t see = keys_seen(p, pos, kt.start<64>(t), use);
      count += __popcll(see);
      if (__any(on && see)) {
        f.lo = t;
        f.hi = max(f.hi, t + 1);
      }
      more = !enough();
    }
  }
  f.row = on && count <= FEW;
  if (!__any(f.row)) f = {false, kt.n, 0};
  return f;
}

// Queries that see keys j0 .. j1-1 (rows [i_lo, i_hi)): chunk < 0: through the window, and beyond it if there are sinks among
// the keys and no chunks; else the given chunk of the queries beyond it, which see only the sinks among the keys.
__device__ __forceinline__ void query_range(const WinParams& p, const Seq& sq, int j0, int j1, int chunk, int& i_lo, int& i_hi) {
  const int far = max(0, min(sq.Lq, j1 + p.left - sq.off));
  if (chunk < 0) {
    i_lo = max(0, min(sq.Lq, j0 - p.right - sq.off));
    i_hi = !p.nst && j0 < p.sinks ? sq.Lq : far;
  } else {
    i_lo = min(sq.Lq, far + chunk * p.ch);
    i_hi = min(sq.Lq, i_lo + p.ch);
  }
}

// Slab of one (sequence, key head, sink tile, part): [2][sinks of a tile][d] floats; part 0 is the window, 1 + c chunk c.
__host__ __device__ inline int slab_rows(const WinParams& p, int tile_rows) { return p.sinks < tile_rows ? p.sinks : tile_rows; }
__device__ __forceinline__ float* slab(const WinParams& p, int b, int g, int st, int part, int tile_rows) {
  return p.slabs + ((((int64_t)b * p.G + g) * p.nst + st) * (1 + p.nch) + part) * 2 * slab_rows(p, tile_rows) * p.d;
}

// row j of sequence b, key head g in the partial sums of a part (which: 0 dK, 1 dV)
__device__ __forceinline__ float* split_row(const WinParams& p, int part, int which, int b, int j, int g) {
  return p.split + ((((int64_t)part * 2 + which) * p.B + b) * p.Lk + j) * ((int64_t)p.G * p.d) + (int64_t)g * p.d;
}

// The work of a block of the dK / dV kernels: a part of a key tile's window, or a chunk of a sink tile's far queries.
struct KeyWork { int tile, part, chunk; };
__device__ __forceinline__ KeyWork key_work(const WinParams& p, int ktiles, int work) {
  const int extra = work - ktiles * p.parts;
  if (extra < 0) return {work / p.parts, work % p.parts, -1};
  return {extra / p.nch, 0, extra % p.nch};
}
__host__ __device__ inline int key_tiles_of_grid(const WinParams& p, int ktiles) { return ktiles * p.parts + p.nst * p.nch; }

// The work of a block: tile `tile` of query head h (or key head, where `rep` is 1) of sequence b; the last blocks of a packed
// batch's grid (b == B) zero rows of no sequence, TAIL parts a head.
//  * A (sequence, key head) is a unit, whose keys and values its tiles and query heads share in the L2 of one XCD
//    (blockIdx mod 8).  Every row of 8 units gives each XCD one, turned by one from row to row: with 8 key heads an XCD
//    that kept the same head would read one 128-byte piece of every row, an eighth of its L2's channels (256 sequences of
//    200 tokens: dQ 96 us, turned 88).  Few units that do not fill rows are dealt tile by tile instead.
//  * Within an XCD the tile is the slowest index.  With the tiles of a sequence side by side, a batch where half of them
//    are empty repeats "two full, two empty", and the dispatcher, which deals blocks to 4 shader engines in turn, leaves
//    two engines without work (256 x 200 tokens given as at most 400: forward 81 instead of 55 us).
//  * Late tiles first where they are the long ones (queries of a causal text; the chunks of far queries behind the key
//    tiles), else early ones first (keys of a causal text).
struct Work { int tile, h, b; bool none; };
constexpr int TAIL = 8;
__host__ __device__ inline bool by_unit(int units) { return units % 8 == 0 || units >= 64; }
__host__ __device__ inline int main_blocks(int units, int tiles, int rep) {
  return by_unit(units) ? 8 * ((units + 7) / 8) * tiles * rep : units * tiles * rep;
}
__device__ __forceinline__ Work work_of_block(const WinParams& p, int tiles, int rep, bool late_first) {
  const int units = p.B * p.G, main = main_blocks(units, tiles, rep), i = blockIdx.x;
  Work w;
  w.none = false;
  if (i >= main) {
    w.b = p.B;
    w.tile = (i - main) / (p.G * rep);
    w.h = (i - main) - w.tile * (p.G * rep);
    return w;
  }
  int u, r;
  if (by_unit(units)) {
    const int rows = (units + 7) >> 3, x = i & 7, s = i >> 3;
    w.tile = s / (rows * rep);
    r = s - w.tile * (rows * rep);
    const int row = r / rep;
    u = row * 8 + ((x - row) & 7);
    r -= row * rep;
  } else {
    w.tile = i / (units * rep);
    r = i - w.tile * (units * rep);
    u = r / rep;
    r -= u * rep;
  }
  w.none = u >= units;
  w.b = u / p.G;
  w.h = (u - w.b * p.G) * rep + r;
  if (late_first) w.tile = tiles - 1 - w.tile;
  return w;
}
inline unsigned work_blocks(const WinParams& p, int tiles, int rep) {
  return (unsigned)(main_blocks(p.B * p.G, tiles, rep) + (p.q_off ? TAIL * p.G * rep : 0));
}

// Rows of a packed tensor that belong to no sequence become zero: columns col0 .. col0 + d - 1 of rows < off[0] and
// >= off[B] (called by the blocks of the extra grid layer; `part` of `parts` blocks).
template <typename T>
__device__ __forceinline__ void zero_rest(T* out, int64_t ld, int64_t col0, int d, const int32_t* off, int B, int64_t rows,
                                          int part, int parts) {
  const int64_t a = max((int64_t)0, min((int64_t)off[0], rows)), z = max(a, min((int64_t)off[B], rows));
  const int64_t n = a + (rows - z);
  for (int64_t e = (int64_t)part * 256 + threadIdx.x; e < n * d; e += (int64_t)parts * 256) {
    const int64_t r = e / d;
    out[(r < a ? r : z + (r - a)) * ld + col0 + (e - r * d)] = T(0);
  }
}

}  // namespace skwin

// bf16 matrix-core path (window_attn_mfma.hip)
bool sk_window_mfma_supported(const skwin::WinParams& p, int dtype);
int sk_window_fwd_mfma(const skwin::WinParams& p, hipStream_t stream);
int sk_window_bwd_mfma(const skwin::WinParams& p, hipStream_t stream);
