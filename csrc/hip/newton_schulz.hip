// Orthogonalisation of matrices by Newton-Schulz products, and the Muon optimizer step around it (gfx950).
//
//   X_0 = G / (|G|_F + eps)                       A_k = X_k X_k^T   (X_k^T X_k where G has more rows than columns)
//   B_k = b A_k + c A_k A_k                       X_{k+1} = a X_k + B_k X_k   (a X_k + X_k B_k)
//   (a, b, c) = (3.4445, -4.7750, 2.0315)
//
// which takes every singular value s of G / |G| to f(f(...f(s))), f(s) = a s + b s^3 + c s^5: values above ~1e-2 end in
// 0.68 .. 1.21.  Small singular values grow by a = 3.44 per iteration, and so does a rounding error made next to them:
// with operands rounded to 16 bits the result is 1e-3 (well conditioned) to 1e-1 (low rank) off, with fp32 operands
// 1e-6 to 2e-5.  There is no fp32 matrix instruction at more than a sixteenth of the fp16 rate, so the fp32 operands
// are kept as two fp16 planes, v = hi + 2^-11 lo (22 bits), and a product is three v_mfma_f32_32x32x16_f16: hi*hi into one
// fp32 accumulator, hi*lo + lo*hi into another, 2^-11 of which is added at the end; the missing lo*lo is below 2^-22 of the
// sum of magnitudes.  fp16 and not bf16 planes: the iterates are bounded (|f| <= 1.2024 on [0, 1.2024], so |X| <= 1.21, |A| <=
// 1.45, |B| <= 2.81 in every entry), so a power of two puts them into fp16's range with 11 bits each instead of 8.
//
// Scales: X is held times S = 2^15, A and B times 2^14: nothing overflows 65504.  An entry that is small next to the others
// grows by up to 3.44 per iteration relative to them, as much as its rounding error, so small entries need their bits as
// well: a matrix with rows of 1e-6 is right only if these are.  That is why lo is held times 2^11, which keeps it in fp16's
// normal range for as long as hi is: values of X keep 22 bits down to 2^-29 (of A and B to 2^-28) and are rounded to
// multiples of 2^-50 below, where |X_0| is 1.  (With lo as it is, 2^-18 and 2^-40, and the scale going by the matrix's typical
// entry: 128 x 256 with half of its rows times 1e-6 was 5e-4 of the norm off after 10 iterations, fp32 products 2e-6; in
// rows of 1e-8 no bit was left.)  What is rounded away there grows to 3.44^12 2^-51 = 1e-9 of an entry in 12 iterations,
// which is below what fp32 products lose; later ones would let it through.
//
// Where the norm is not far above eps, |X_0| = |G| / (|G| + eps) is small, and grows by at most a < 4 per iteration: X_k is
// held times another 2^e_k, e_k = max(0, e_0 - 2 k), and A_k and B_k times 2^(2 e_k), so that vanishing gradients keep their
// bits.  e_0 is found on the device (with the norm) so that 2^e_0 |X_0| is in [0.45, 0.9) or e_0 is 0: where c A A is scaled
// away B_k is b A_k alone, up to 4.775 * 0.81 * 2^14 = 63370 (with 2^e_0 |X_0| up to 1 it overflowed 65504 on matrices in
// which one row has nearly all of such a norm, and the result was NaN).
//
// A and B are symmetric: only tiles on and below the diagonal are computed, their mirror images are copies.  All
// matrices of an optimizer step (or of a batch) go through each stage in one launch, from work lists that name (matrix,
// tile row, tile column), longest first.  The operands live in a workspace whose planes are padded with zeros to whole
// tiles, so the products need no bounds checks; a row holds its two planes in turns of 32 values, hi then lo, so that the
// 32 k of a step are one 128-byte line per row (apart, each plane's 64 bytes fetched a line of which half was used).
//
// Measured: 4096 x 4096, an iteration A 191 us, B 194 us, X 346 us: 1.1 .. 1.2 PFLOP/s in the matrix cores, next to 1.45
// of the fastest large fp16 product on this card.  ResNet-50's 54 matrices, an iteration A 61 + 12, B 32, X 108 us: X's
// tiles have as few as two k-steps, so that what they take is their first loads and the 128 KB of X that each reads and
// writes at its end; norm and first iterate 56 and 65 us at 5 TB/s, the last X with the parameters 140.  Up to a few hundred
// rows an iteration is four launches of 4 .. 15 us, 5 of them a tile's first loads and its end.
//
// Errors of fp32 results after five iterations are 0.2 .. 0.6 times those of fp32 with sums by blocks on sides of up to 64 and
// 0.6 .. 1.25 times on longer ones (0.3 .. 0.6 times those of the fp32 library products from 2500 on), single matrices of
// a few entries up to 2.5 times; after twelve up to twice.
#include "row_io.h"

typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));

#define NS_A 3.4445f
#define NS_B (-4.7750f)
#define NS_C 2.0315f
#define NS_GRAM_SCALE 16384.f  // of A and B
#define NS_LO 2048.f           // of a lo plane against its hi plane

// One matrix.  Offsets in elements of the buffer they point into.
struct NsMat {
  long long at;    // of the matrix in the input / output / parameter buffers (rows * cols contiguous values)
  long long x;     // X and the next X in the workspace: two plane pairs [rp][cp]
  long long a;     // A and B: two plane pairs [mp][mp]
  long long part;  // first of its `parts` partial sums of squares
  int rows, cols;
  int rp, cp, mp;  // padded rows, columns and min(rows, cols)
  int parts;
  int chunk;       // elements per partial sum
  int tall;        // rows > cols
  float scale;     // S (the same for every matrix)
  float lr_scale;  // sqrt(max(1, rows / cols))
};

// One workgroup of a product stage: the tile (ti, tj) of `edge` x `edge` values, summed over k0 <= k < k1.  Where the
// reduction is cut in several jobs, each leaves its fp32 sums in slab `slab` (in units of 64 x 64 values), else -1; the
// job that joins them (NsArgs::gram_joins, poly_joins) has the first one's number and k0 = how many there are.
struct NsJob {
  int mat;  // -1: nothing (the lists are interleaved from eight queues of equal length)
  int ti, tj, edge;
  int k0, k1;
  int slab, pad;
};

struct NsArgs {
  const NsMat* mats;
  const int4* chunks;       // {matrix, chunk, -, -}
  const int4* packs;        // {matrix, tile row, tile column, -}: 64 x 64 tiles of the padded matrix
  const NsJob* gram;        // tiles of A, tj <= ti
  const NsJob* gram_joins;
  const NsJob* poly;        // tiles of B, tj <= ti
  const NsJob* poly_joins;
  const NsJob* full;        // tiles of X
  const NsJob* small;       // slices of matrices whose shorter side is at most 64 (then there are no other jobs)
  int nsmall, small_slices;
  int nchunks, npacks, ngram, ngram_joins, npoly, npoly_joins, nfull;
  int steps;
  int dtype;           // of `in` (and `out`): IO_*
  int large;           // which lists hold tiles of 128: 1 gram, 2 poly, 4 full
  const void* in;      // the matrices, or their gradients
  void* out;           // orthogonalised matrices (null: parameter update)
  float* buf;          // momentum (null: none)
  float* w;            // parameters
  bf16* w16;           // their bf16 copy, or null
  const float* hyper;  // {step size, gradient scale}
  double* part;        // the partial sums, then e_0 of every matrix
  float* slabs;
  f16* ws;
  long long nparts;
  float eps, mu, wd;
  int nesterov;
};

// ---------------------------------------------------------------- norm and first iterate
// the value to orthogonalise: the gradient, or the momentum update of it.  Evaluated twice (for the norm, then for X_0)
// from the same stored values and without contraction, so both see the same bits.
__device__ __forceinline__ float ns_direction(float g, float buf, float mu, int nesterov) {
#pragma clang fp contract(off)
  return nesterov ? g + mu * buf : buf;
}
__device__ __forceinline__ float ns_momentum(float g, float buf, float mu) {
#pragma clang fp contract(off)
  return mu * buf + g;
}

// Sums of squares in 64 bits (fp32 squares would overflow at 2e19 and vanish at 1e-23), one per chunk of a matrix, and
// the momentum update on the way.
template <typename T, bool MOMENTUM>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsArgs p) {
  __shared__ double red[4];
  const int4 job = p.chunks[blockIdx.x];
  const NsMat m = p.mats[job.x];
  const long long n = (long long)m.rows * m.cols;
  const long long lo = (long long)job.y * m.chunk, hi = lo + m.chunk < n ? lo + m.chunk : n;
  const T* in = (const T*)p.in + m.at;
  float* buf = MOMENTUM ? p.buf + m.at : nullptr;
  const float gs = MOMENTUM ? p.hyper[1] : 1.f;
  double s = 0.0;
  for (long long i = lo + threadIdx.x * 8; i < hi; i += 256 * 8) {
    float g[8], b[8];
    const int left = hi - i < 8 ? (int)(hi - i) : 8;
    row_load<T, 8>(in + i, 0, left, g);
    if (MOMENTUM) {
      row_load<float, 8>(buf + i, 0, left, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[j] *= gs;
        b[j] = ns_momentum(g[j], b[j], p.mu);
        g[j] = ns_direction(g[j], b[j], p.mu, p.nesterov);
      }
      row_store<float, 8>(buf + i, 0, left, b);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s += j < left ? (double)g[j] * (double)g[j] : 0.0;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) p.part[m.part + job.y] = (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ void ns_split(float v, f16& hi, f16& lo) {
  hi = (f16)v;
  lo = (f16)((v - (float)hi) * NS_LO);
}
__device__ __forceinline__ float ns_value(f16 hi, f16 lo) { return fmaf((float)lo, 1.f / NS_LO, (float)hi); }

// A plane pair [rows][ld]: the hi value (row, col); its lo value is 32 further on.
__device__ __forceinline__ size_t ns_at(int ld, int row, int col) {
  return (size_t)row * 2 * ld + ((col >> 5) << 6) + (col & 31);
}
// eight consecutive values of a row, col a multiple of 8
__device__ __forceinline__ void ns_get(const f16* at, float (&v)[8]) {
  const f16x8 h = *(const f16x8*)at, l = *(const f16x8*)(at + 32);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = ns_value(h[j], l[j]);
}
__device__ __forceinline__ void ns_put(f16* at, const float (&v)[8]) {
  f16x8 h, l;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f16 a, b;
    ns_split(v[j], a, b);
    h[j] = a;
    l[j] = b;
  }
  *(f16x8*)at = h;
  *(f16x8*)(at + 32) = l;
}

// What G is multiplied with for X_0 as it is held, and e_0, from the partial sums; `red` is LDS for four values.
__device__ __forceinline__ double ns_first_scale(const NsArgs& p, const NsMat& m, double* red, int& lift) {
  double s = 0.0;
  for (int i = threadIdx.x; i < m.parts; i += 256) s += p.part[m.part + i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  const double size = norm / (norm + (double)p.eps);
  lift = 0;
  if (size > 0.0 && size < 1.0) (void)frexp(size / 0.9, &lift);   // size * 2^-lift in [0.45, 0.9)
  lift = lift < 0 ? -lift : 0;
  return ldexp((double)m.scale / (norm + (double)p.eps), lift);
}

// X_0 times S as two fp16 planes, zeros in the padding.  A workgroup writes 64 x 64 values; its reads are on their way
// while the norm is put together.
template <typename T, bool MOMENTUM>
__global__ __launch_bounds__(256) void ns_pack_kernel(NsArgs p) {
  __shared__ double red[4];
  const int4 job = p.packs[blockIdx.x];
  const NsMat m = p.mats[job.x];
  const T* in = (const T*)p.in + m.at;
  const float* buf = MOMENTUM ? p.buf + m.at : nullptr;
  const float gs = MOMENTUM ? p.hyper[1] : 1.f;
  f16* x = p.ws + m.x;
  const int col = job.z * 64 + (threadIdx.x & 7) * 8, row0 = job.y * 64 + (threadIdx.x >> 3);
  float g[2][8], b[2][8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = row0 + h * 32;
#pragma unroll
    for (int j = 0; j < 8; ++j) g[h][j] = b[h][j] = 0.f;
    if (row < m.rows && col < m.cols) {
      row_load<T, 8>(in + (size_t)row * m.cols, col, m.cols, g[h]);
      if (MOMENTUM) row_load<float, 8>(buf + (size_t)row * m.cols, col, m.cols, b[h]);
    }
  }
  int lift;
  const double scale = ns_first_scale(p, m, red, lift);
  if (job.y == 0 && job.z == 0 && threadIdx.x == 0) p.part[p.nparts + job.x] = (double)lift;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (MOMENTUM) g[h][j] = ns_direction(g[h][j] * gs, b[h][j], p.mu, p.nesterov);
      g[h][j] = (float)((double)g[h][j] * scale);
    }
    ns_put(x + ns_at(m.cp, row0 + h * 32, col), g[h]);
  }
}

// ---------------------------------------------------------------- products
#define NS_BK 32

// Tiles in LDS.  k contiguous: T rows of 128 bytes, 16-byte chunk plane * 4 + k / 8 at slot chunk ^ ns_swz(row): 16 rows
// reading the same chunk touch every bank once.
__device__ __forceinline__ int ns_swz(int row) { return (row >> 1) & 7; }
// k is the row: 32 rows of 4 T bytes, blocks of 32 columns hi and lo in turn; a transposing read touches 64 bytes in each of
// four consecutive rows, which all start at bank 0.
__device__ __forceinline__ int ns_swz_tr(int row) { return (row & 3) << 2; }

// An operand of a product: a plane pair; element (i, k) of the operand at row i, column k, or (k-major) at row k,
// column i; `i0` is the tile's first i.
struct NsOperand {
  const f16* base;
  int ld;
  int i0;
};

// 16 bytes a lane from `base` (the same for the wave) + `off` into LDS at `lds` + AT, lane after lane.  No other code of a
// kernel keeps a value in m0.
template <int AT>
__device__ __forceinline__ void ns_to_stage(const f16* base, unsigned off, unsigned lds) {
  asm volatile(
      "s_add_u32 m0, %2, %3\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %1"
      :
      : "v"(off), "s"(base), "s"(lds), "n"(AT)
      : "memory", "scc", "m0");
}

// T x T tile of sum_k P(i, k) Q(j, k), k0 <= k < k1, on 2 x 2 waves.  The accumulator of a wave holds the TRANSPOSED tile
// (Q is the matrix instruction's first operand): lane l, element e of acc[u][v] is column
// j = v * 32 + (e & 3) + 8 (e >> 2) + 4 (l >> 5) of row i = u * 32 + (l & 31), so four consecutive elements are four
// consecutive columns.
//
// k advances by 32; each of the four waves brings half of an operand of the next k-tiles (P, P, Q, Q) into LDS by
// LDS-DMA, NST - 1 k-tiles ahead, with counted waits and raw barriers; the fragments of the next 16 k are read while the
// matrix instructions of the present ones run.
//
// What bounds it is LDS: a k-tile of 128 x 128 is 32 KB written and 64 KB read, 768 cycles at 128 bytes a cycle, next to
// 768 cycles of matrix instructions on each of the four SIMDs; one of 64 x 64 is 48 KB, 384 cycles, next to 192.  NST is 2
// for 128 x 128.  64 x 64 tiles of A and B have four slots where they are at most two to a CU, which is what their registers
// (213) leave room for (36 tiles over 8192 values: 59 -> 46 us, with six no less), else three: ResNet-50's update, whose B
// has 872 tiles over up to 1024 values, 1148 us with three there and 1159 with four.
//
// The sums of hi hi and of the mixed products have accumulators of their own, so that lo may have a scale of its own.  It
// also makes for two thirds fewer roundings in the large sums: 4096 x 4096 fp32 1.7e-6 of the norm off, in one accumulator
// 3.2e-6.  For 128 x 128 that is 128 registers of accumulators next to 64 of fragments: the loop over k-tiles must be a
// single body with one way out, or the compiler holds accumulators twice and spills.
template <int T, int NST, bool PK, bool QK>
__device__ __forceinline__ void ns_product(const NsOperand& P, const NsOperand& Q, int k0, int k1, char* smem,
                                           f32x16 (&acc)[T / 64][T / 64]) {
  constexpr int OPER = T * NS_BK * 4;         // bytes of an operand's k-tile, both planes
  constexpr int STAGE = 2 * OPER;
  constexpr int LPS = OPER / 2048;            // LDS-DMA instructions per wave and k-tile
  constexpr int MT = T / 64;
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wid >> 1, wc = wid & 1;

  // staging: this wave's half of an operand.  What stands beside the matrix instructions is kept short: the offsets of the
  // lanes in registers, the k-tiles' start in scalar ones, places in LDS moved by one addition each to the next slot.
  const bool kmajor = wid < 2 ? PK : QK;
  const int ld = wid < 2 ? P.ld : Q.ld, i0 = wid < 2 ? P.i0 : Q.i0;
  const f16* src = wid < 2 ? P.base : Q.base;
  unsigned off[LPS];                          // bytes: at most 128 rows of 2^20 columns
  size_t step;                                // elements between two k-tiles
  if (kmajor) {
    constexpr int RPI = 256 / T;              // k rows per instruction: 2 or 4; this wave brings 16
#pragma unroll
    for (int i = 0; i < LPS; ++i) {
      const int r = (wid & 1) * 16 + i * RPI + lane / (64 / RPI), slot = lane % (64 / RPI);
      off[i] = (unsigned)r * 4 * ld + ((slot ^ ns_swz_tr(r)) << 4);
    }
    src += (size_t)k0 * 2 * ld + 2 * i0;
    step = (size_t)NS_BK * 2 * ld;
  } else {
#pragma unroll
    for (int i = 0; i < LPS; ++i) {           // 8 rows per instruction
      const int r = (wid & 1) * (T / 2) + i * 8 + (lane >> 3), slot = lane & 7;
      off[i] = (unsigned)r * 4 * ld + ((slot ^ ns_swz(r)) << 4);
    }
    src += (size_t)i0 * 2 * ld + 2 * k0;
    step = 2 * NS_BK;
  }
  // (a scalar register that the vector unit wrote can be read as an address five instructions later; where that is left to
  // the compiler it counts them, behind inline assembly it does not look)
  asm volatile("s_nop 4");
  const unsigned lds = (unsigned)(uintptr_t)(LDS_AS char*)smem;
  const unsigned lds_wave = lds + wid * (OPER / 2);
  // (`i` is a constant once the loops around are unrolled; a slot is given by its first byte)
  auto stage_one = [&](int slot, int i) {
    const unsigned at = lds_wave + slot;
    if (i == 0) ns_to_stage<0>(src, off[0], at);
    if (i == 1) ns_to_stage<1 * 1024>(src, off[1], at);
    if (i == 2) ns_to_stage<2 * 1024>(src, off[2], at);
    if (i == 3) ns_to_stage<3 * 1024>(src, off[3], at);
    if constexpr (LPS == 8) {
      if (i == 4) ns_to_stage<4 * 1024>(src, off[4], at);
      if (i == 5) ns_to_stage<5 * 1024>(src, off[5], at);
      if (i == 6) ns_to_stage<6 * 1024>(src, off[6], at);
      if (i == 7) ns_to_stage<7 * 1024>(src, off[7], at);
    }
    if (i == LPS - 1) src += step;
  };

  // fragments: a lane's places in the first slot, for the two planes and, where the swizzle mixes them with the place,
  // the halves of k (k contiguous) or the blocks of 32 rows (k-major); everything else is a constant to add
  auto places = [&](bool km, int row0, unsigned oper, unsigned (&at)[2][2]) {
#pragma unroll
    for (int lo = 0; lo < 2; ++lo)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (km) {
          const int col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3), krow = 8 * (lane >> 5) + ((lane & 15) >> 2);
          const int chunk = ((row0 >> 5) + x) * 8 + lo * 4 + (col >> 3);
          at[lo][x] = lds + oper + krow * (T * 4) + ((chunk ^ ns_swz_tr(krow)) << 4) + (col & 7) * 2;
        } else {
          const int row = row0 + (lane & 31);
          at[lo][x] = lds + oper + row * 128 + (((lo * 4 + x * 2 + (lane >> 5)) ^ ns_swz(row)) << 4);
        }
      }
  };
  unsigned p_at[2][2], q_at[2][2];
  places(PK, wr * (T / 2), 0, p_at);
  places(QK, wc * (T / 2), OPER, q_at);
  auto frag = [&](bool km, const unsigned (&at)[2][2], int u, int ks, int lo) -> f16x8 {
    if (km) {
      union { s16x4 h[2]; f16x8 v; } r;
#pragma unroll
      for (int q = 0; q < 2; ++q)
        r.h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (LDS_AS s16x4*)(uintptr_t)(at[lo][u] + (ks * 16 + 4 * q) * (T * 4)));
      return r.v;
    }
    return *(const LDS_AS f16x8*)(uintptr_t)(at[lo][ks] + u * 4096);
  };
  f32x16 cross[MT][MT];                       // sums of hi lo and lo hi, times NS_LO
  f16x8 ph[2][MT], pl[2][MT], qh[2][MT], ql[2][MT];
  constexpr int FRAGS = 4 * MT;               // of a step of 16 k: Q hi, P hi, Q lo, P lo
  auto load_frag = [&](int ks, int to, int i) {
    const int u = i % MT;
    if (i / MT == 0) qh[to][u] = frag(QK, q_at, u, ks, 0);
    if (i / MT == 1) ph[to][u] = frag(PK, p_at, u, ks, 0);
    if (i / MT == 2) ql[to][u] = frag(QK, q_at, u, ks, 1);
    if (i / MT == 3) pl[to][u] = frag(PK, p_at, u, ks, 1);
  };
  // the matrix instructions of a step of 16 k; `between` issues other work behind each, which runs in its shadow
  auto multiply = [&](int from, auto between) {
#pragma unroll
    for (int n = 0; n < 3 * MT * MT; ++n) {
      const int u = n / MT % MT, v = n % MT;
      const f16x8 q = n / (MT * MT) == 1 ? ql[from][v] : qh[from][v];
      const f16x8 w = n / (MT * MT) == 2 ? pl[from][u] : ph[from][u];
      f32x16& to = n < MT * MT ? acc[u][v] : cross[u][v];
      to = __builtin_amdgcn_mfma_f32_32x32x16_f16(q, w, to, 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      between(n);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int u = 0; u < MT; ++u)
#pragma unroll
    for (int v = 0; v < MT; ++v)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[u][v][e] = cross[u][v][e] = 0.f;

  const int nk = (k1 - k0) / NS_BK;
  auto stage = [&](int slot) {
#pragma unroll
    for (int i = 0; i < LPS; ++i) stage_one(slot, i);
  };
#pragma unroll
  for (int s = 0; s < NST - 1; ++s)
    if (s < nk) stage(s * STAGE);
  // waits until k-tile kt has arrived (the NST - 2 behind it may be on their way) and this wave's reads are done; after
  // the barrier that holds for every wave
  auto arrive = [&](int kt) {
    if (kt + NST - 2 < nk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * LPS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  arrive(0);
  if (NST - 1 < nk) stage((NST - 1) * STAGE);
#pragma unroll
  for (int i = 0; i < FRAGS; ++i) load_frag(0, 0, i);
  // Issued in a block, the eight LDS-DMA and eight LDS reads of a step would hold the wave for as long as its matrix
  // instructions take; one behind each of these they cost next to nothing.
  constexpr int N = 3 * MT * MT;
  constexpr int RPM = (FRAGS + N - 1) / N;    // reads, and LDS-DMA, behind one matrix instruction
  constexpr int SPM = (LPS + N - 1) / N;
  auto second_half = [&]() {
    multiply(0, [&](int n) {
#pragma unroll
      for (int i = n * RPM; i < n * RPM + RPM; ++i)
        if (i < FRAGS) load_frag(1, 1, i);
    });
  };
  // (The last k-tile stands by itself: with one loop for all, the wait counts in front of the second group would have to
  // hold for the pass without new reads as well, and wait for the new reads in all others.  The loop is not unrolled over
  // the slots: the compiler would keep a second set of accumulators for its ways out.)
  int slot = 0;
  for (int kt = 0; kt + 1 < nk; ++kt) {
    second_half();
    arrive(kt + 1);  // ... and this k-tile has been read by every wave: its slot takes the one NST further on
    const int here = slot;
    slot = here == (NST - 1) * STAGE ? 0 : here + STAGE;
#pragma unroll
    for (int lo = 0; lo < 2; ++lo)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        p_at[lo][x] += slot - here;
        q_at[lo][x] += slot - here;
      }
    const bool more = kt + NST < nk;
    multiply(1, [&](int n) {
#pragma unroll
      for (int i = n * RPM; i < n * RPM + RPM; ++i)
        if (i < FRAGS) load_frag(0, 0, i);
      if (more)
#pragma unroll
        for (int i = n * SPM; i < n * SPM + SPM; ++i)
          if (i < LPS) stage_one(here, i);
    });
  }
  second_half();
  multiply(1, [](int) {});
#pragma unroll
  for (int u = 0; u < MT; ++u)
#pragma unroll
    for (int v = 0; v < MT; ++v)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[u][v][e] = fmaf(cross[u][v][e], 1.f / NS_LO, acc[u][v][e]);
}

// fp32 tile in LDS: 16-byte writes of 8 rows at a time hit every bank once at this pitch
#define NS_PITCH(T) ((T) + 4)
// LDS of a launch with large tiles or four slots (two workgroups to a CU), and of others
#define NS_LDS_LARGE (128 * NS_PITCH(128) * 4)
#define NS_LDS_SMALL (3 * 4 * 64 * NS_BK * 2)
static_assert(NS_LDS_LARGE >= 2 * 4 * 128 * NS_BK * 2 && NS_LDS_LARGE >= 4 * 4 * 64 * NS_BK * 2, "stages fit");
static_assert(NS_LDS_SMALL >= 64 * NS_PITCH(64) * 4, "the fp32 tile fits");

// accumulators -> the tile [i][j] in LDS
template <int T>
__device__ __forceinline__ void ns_to_lds(const f32x16 (&acc)[T / 64][T / 64], float* tile) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int i0 = (wid >> 1) * (T / 2) + (lane & 31), j0 = (wid & 1) * (T / 2) + 4 * (lane >> 5);
  __syncthreads();  // every wave is done with the stages
#pragma unroll
  for (int u = 0; u < T / 64; ++u)
#pragma unroll
    for (int v = 0; v < T / 64; ++v)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *(f32x4*)(tile + (i0 + u * 32) * NS_PITCH(T) + j0 + v * 32 + 2 * e) =
            f32x4{acc[u][v][e], acc[u][v][e + 1], acc[u][v][e + 2], acc[u][v][e + 3]};
  __syncthreads();
}

// e_k of a matrix
__device__ __forceinline__ int ns_lift(const NsArgs& p, int mat, int k) {
  const int e = (int)p.part[p.nparts + mat] - 2 * k;
  return e > 0 ? e : 0;
}

// The fp32 tile in LDS, sums over all k, becomes the tile of A, or with POLY of B = b A + c A A, and its mirror image.
// ROWS of its rows, from row `r0` of the tile on, are in LDS.
template <int T, int ROWS, bool POLY>
__device__ __forceinline__ void ns_symmetric_out(const NsArgs& p, const NsMat& m, int ti, int tj, int r0, int lift, float* tile) {
  f16* a = p.ws + m.a;
  f16* out = POLY ? a + (size_t)2 * m.mp * m.mp : a;
  const int i0 = ti * T + r0, j0 = tj * T;
  const float f = POLY ? ldexpf(NS_C / NS_GRAM_SCALE, -2 * lift) : NS_GRAM_SCALE / (m.scale * m.scale);
  // rows of the tile: eight consecutive columns a thread
  for (int e = threadIdx.x; e < ROWS * T / 8; e += 256) {
    const int r = e / (T / 8), c = e % (T / 8) * 8;
    const size_t at = ns_at(m.mp, i0 + r, j0 + c);
    float* t = tile + r * NS_PITCH(T) + c;
    float v[8];
    if (POLY) ns_get(a + at, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = POLY ? NS_B * v[j] + f * t[j] : f * t[j];
    ns_put(out + at, v);
    if (ti != tj)
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = v[j];
  }
  if (ti == tj) return;
  __syncthreads();
  // mirror image: consecutive lanes take consecutive columns of the tile in LDS, eight rows each
  for (int e = threadIdx.x; e < ROWS * T / 8; e += 256) {
    const int c = e % T, r = e / T * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = tile[(r + j) * NS_PITCH(T) + c];
    ns_put(out + ns_at(m.mp, j0 + c, i0 + r), v);
  }
}

// Tile of A = X X^T (or X^T X) or, with POLY, of A A; with a slab, only the sums over the job's share of k.
template <int T, int NST, bool POLY>
__device__ __forceinline__ void ns_symmetric(const NsArgs& p, const NsMat& m, const NsJob& job, int k, int lift, char* smem) {
  f32x16 acc[T / 64][T / 64];
  const f16* x = p.ws + m.x + (k & 1 ? (size_t)2 * m.rp * m.cp : 0);
  const f16* a = p.ws + m.a;
  const int i0 = job.ti * T, j0 = job.tj * T;
  if (POLY)
    ns_product<T, NST, false, false>({a, m.mp, i0}, {a, m.mp, j0}, job.k0, job.k1, smem, acc);
  else if (m.tall)
    ns_product<T, NST, true, true>({x, m.cp, i0}, {x, m.cp, j0}, job.k0, job.k1, smem, acc);
  else
    ns_product<T, NST, false, false>({x, m.cp, i0}, {x, m.cp, j0}, job.k0, job.k1, smem, acc);
  float* tile = (float*)smem;
  ns_to_lds<T>(acc, tile);
  if (job.slab >= 0) {
    float* slab = p.slabs + (size_t)job.slab * 4096;
    for (int e = threadIdx.x; e < T * T / 4; e += 256)
      *(f32x4*)(slab + e * 4) = *(const f32x4*)(tile + e / (T / 4) * NS_PITCH(T) + e % (T / 4) * 4);
    return;
  }
  ns_symmetric_out<T, T, POLY>(p, m, job.ti, job.tj, 0, lift, tile);
}

// Sums of the slabs of a tile, in order; a workgroup takes 32 of its rows (the mean tile has few slabs of 64 KB, and one
// workgroup would read them at the pace of its own loads).
#define NS_JOIN_ROWS 32
template <int T, bool POLY>
__device__ __forceinline__ void ns_join_slabs(const NsArgs& p, const NsMat& m, const NsJob& job, int r0, int lift, float* tile) {
  constexpr int N = NS_JOIN_ROWS * T / 4 / 256;
  const float* slab = p.slabs + (size_t)job.slab * 4096 + r0 * T + threadIdx.x * 4;
  f32x4 v[N];
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = *(const f32x4*)(slab + n * 1024);
  for (int i = 1; i < job.k0; ++i)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const f32x4 w = *(const f32x4*)(slab + (size_t)i * T * T + n * 1024);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[n][j] += w[j];
    }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int e = n * 256 + threadIdx.x;
    *(f32x4*)(tile + e / (T / 4) * NS_PITCH(T) + e % (T / 4) * 4) = v[n];
  }
  __syncthreads();
  ns_symmetric_out<T, NS_JOIN_ROWS, POLY>(p, m, job.ti, job.tj, r0, lift, tile);
}

enum { NS_NEXT = 0, NS_OUT = 1, NS_APPLY = 2 };

// Eight consecutive values of the result, into the output or the parameters.
template <int WHAT, typename O>
__device__ __forceinline__ void ns_result(const NsArgs& p, const NsMat& m, int row, int col, const float* o, float keep,
                                          float rate) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = o[j];
  const size_t flat = m.at + (size_t)row * m.cols;
  if (WHAT == NS_OUT) {
    row_store<O, 8>((O*)p.out + flat, col, m.cols, v);
  } else {
    float w[8];
    row_load<float, 8>(p.w + flat, col, m.cols, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = w[j] * keep - rate * v[j];
    row_store<float, 8>(p.w + flat, col, m.cols, w);
    if (p.w16 != nullptr) row_store<bf16, 8>(p.w16 + flat, col, m.cols, w);
  }
}

// Tile of a X + B X (or a X + X B): the next iterate, the result, or the parameter update with it.
template <int T, int WHAT, typename O>
__device__ __forceinline__ void ns_advance(const NsArgs& p, const NsMat& m, const NsJob& job, int k, int lift, int lift_next,
                                           char* smem) {
  constexpr int NST = T == 128 ? 2 : 3;
  f32x16 acc[T / 64][T / 64];
  const size_t xs = (size_t)2 * m.rp * m.cp;
  const f16* x = p.ws + m.x + (k & 1 ? xs : 0);
  f16* next = p.ws + m.x + (k & 1 ? 0 : xs);
  const f16* b = p.ws + m.a + (size_t)2 * m.mp * m.mp;
  const int i0 = job.ti * T, j0 = job.tj * T;
  if (m.tall)
    ns_product<T, NST, false, false>({x, m.cp, i0}, {b, m.mp, j0}, job.k0, job.k1, smem, acc);
  else
    ns_product<T, NST, false, true>({b, m.mp, i0}, {x, m.cp, j0}, job.k0, job.k1, smem, acc);
  float* tile = (float*)smem;
  ns_to_lds<T>(acc, tile);
  const float lr = WHAT == NS_APPLY ? p.hyper[0] : 0.f;
  const float keep = 1.f - lr * p.wd, rate = lr * m.lr_scale;
  // the result leaves without its scale, the next iterate with its own
  const float fx = ldexpf(NS_A, lift_next - lift), ft = ldexpf(1.f / NS_GRAM_SCALE, lift_next - 3 * lift);
  const float unscale = ldexpf(1.f / m.scale, -lift_next);
  for (int e = threadIdx.x; e < T * T / 8; e += 256) {
    const int r = e / (T / 8), c = e % (T / 8) * 8;
    const int row = i0 + r, col = j0 + c;
    if (WHAT != NS_NEXT && (row >= m.rows || col >= m.cols)) continue;
    const size_t at = ns_at(m.cp, row, col);
    const float* t = tile + r * NS_PITCH(T) + c;
    float v[8];
    ns_get(x + at, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fx * v[j] + ft * t[j];
    if (WHAT == NS_NEXT) {
      ns_put(next + at, v);
      continue;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= unscale;
    ns_result<WHAT, O>(p, m, row, col, v, keep, rate);
  }
}

template <bool POLY, int SLOTS>
__global__ __launch_bounds__(256, 2) void ns_symmetric_kernel(NsArgs p, int k) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const NsJob job = (POLY ? p.poly : p.gram)[blockIdx.x];
  if (job.mat < 0) return;
  const NsMat m = p.mats[job.mat];
  const int lift = POLY ? ns_lift(p, job.mat, k) : 0;
  if (job.edge == 128)
    ns_symmetric<128, 2, POLY>(p, m, job, k, lift, smem);
  else
    ns_symmetric<64, SLOTS, POLY>(p, m, job, k, lift, smem);
}

template <bool POLY>
__global__ __launch_bounds__(256) void ns_join_kernel(NsArgs p, int k) {
  __shared__ __attribute__((aligned(16))) float tile[NS_JOIN_ROWS * NS_PITCH(128)];
  const NsJob job = (POLY ? p.poly_joins : p.gram_joins)[blockIdx.x];
  const int r0 = blockIdx.y * NS_JOIN_ROWS;
  if (r0 >= job.edge) return;
  const NsMat m = p.mats[job.mat];
  const int lift = POLY ? ns_lift(p, job.mat, k) : 0;
  if (job.edge == 128)
    ns_join_slabs<128, POLY>(p, m, job, r0, lift, tile);
  else
    ns_join_slabs<64, POLY>(p, m, job, r0, lift, tile);
}

template <int WHAT, typename O>
__global__ __launch_bounds__(256, 2) void ns_advance_kernel(NsArgs p, int k) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const NsJob job = p.full[blockIdx.x];
  if (job.mat < 0) return;
  const NsMat m = p.mats[job.mat];
  const int lift = ns_lift(p, job.mat, k), lift_next = ns_lift(p, job.mat, k + 1);
  if (job.edge == 128)
    ns_advance<128, WHAT, O>(p, m, job, k, lift, lift_next, smem);
  else
    ns_advance<64, WHAT, O>(p, m, job, k, lift, lift_next, smem);
}

// ---------------------------------------------------------------- short sides of at most 64
// One launch an iteration.  A workgroup owns a slice of X, `edge` blocks of 64 x 64 along its long side, from block
// `tj` on; A, 64 x 64, is the sum of all slices' partial products, which every workgroup of the matrix adds up for
// itself (in slice order, so that all hold the same A) and turns into B; then it advances its blocks and leaves the partial
// product of the new ones.  64 x 576 is a chain of small launches whatever is done, bound by their latency: in
// separate stages a call of five iterations took 80 us, this way 46.
//
// The matrix instruction adds up eight products at a time after cutting them off at 2^-23 of the largest, and near the end,
// where A is close to the identity, that is the product of two diagonal values each time: the others lose up to a unit in
// the last place, always towards zero.  So A = d I + E with d about the mean of the diagonal (every fourth of its values; the
// algebra holds for any d, but all workgroups of a matrix must take the same), and
//   B = (b d + c d^2) I + F,   F = (b + 2 c d) E + c E E,   X_{k+1} = (a + b d + c d^2) X_k + F X_k:
// E and F are small where A is close to the identity, and so is all that their products and their 22 bits lose (12 x 500:
// 7.4e-7 of the norm off with d = 0, 2.4e-7 with this, 7.9e-7 in fp32 products).  It takes 0.5 us an iteration, so results
// that are rounded to 16 bits, and updates of parameters, which they reach times a small rate, are made with d = 0: 0.3 .. 1.3
// times the error of fp32 products.
//
// Tiles in LDS: 64 rows of 256 bytes, two blocks of 32 columns, hi and lo.  One swizzle serves both ways of reading:
// 16 rows at one chunk (all four bits of the row differ) and 64 bytes in four consecutive rows (its low bits on top).
#define NS_TILE 16384
__device__ __forceinline__ int ns_mix(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }
// byte offset of the 16-byte chunk that holds (row, col)
__device__ __forceinline__ int ns_chunk(int row, int col, int lo) {
  return row * 256 + ((((col >> 5) * 8 + lo * 4 + ((col & 31) >> 3)) ^ ns_mix(row)) << 4);
}

__device__ __forceinline__ f32x16 ns_zero() {
  f32x16 z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}

// 64 x 64 product of two tiles over 64 k, added to `acc`; the wave's quarter, transposed as in ns_product
template <bool PK, bool QK>
__device__ __forceinline__ void ns_small_product(const char* P, const char* Q, f32x16& acc) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int tr_k = 8 * (lane >> 5) + ((lane & 15) >> 2), tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  auto frag = [&](const char* tile, bool km, int row0, int kk, int lo) -> f16x8 {
    if (km) {
      union { s16x4 h[2]; f16x8 v; } r;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int krow = kk * 16 + tr_k + 4 * q;
        const char* at = tile + ns_chunk(krow, row0 + tr_col, lo) + (tr_col & 7) * 2;
        r.h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)at);
      }
      return r.v;
    }
    return *(const f16x8*)(tile + ns_chunk(row0 + (lane & 31), kk * 16 + (lane >> 5) * 8, lo));
  };
  const int i0 = (wid >> 1) * 32, j0 = (wid & 1) * 32;
  f32x16 cross = ns_zero();
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    const f16x8 ph = frag(P, PK, i0, kk, 0), qh = frag(Q, QK, j0, kk, 0);
    const f16x8 pl = frag(P, PK, i0, kk, 1), ql = frag(Q, QK, j0, kk, 1);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh, ph, acc, 0, 0, 0);
    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql, ph, cross, 0, 0, 0);
    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh, pl, cross, 0, 0, 0);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = fmaf(cross[e], 1.f / NS_LO, acc[e]);
}

// four consecutive values of a tile, col a multiple of 4
__device__ __forceinline__ void ns_small_get(const char* tile, int row, int col, float (&v)[4]) {
  const int in = (col & 7) * 2;
  const f16x4 h = *(const f16x4*)(tile + ns_chunk(row, col, 0) + in), l = *(const f16x4*)(tile + ns_chunk(row, col, 1) + in);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = ns_value(h[j], l[j]);
}
__device__ __forceinline__ void ns_small_put(char* tile, int row, int col, const float (&v)[4]) {
  f16x4 h, l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f16 a, b;
    ns_split(v[j], a, b);
    h[j] = a;
    l[j] = b;
  }
  const int in = (col & 7) * 2;
  *(f16x4*)(tile + ns_chunk(row, col, 0) + in) = h;
  *(f16x4*)(tile + ns_chunk(row, col, 1) + in) = l;
}

// a block of X: 64 rows of 256 bytes, `ld` elements apart per plane
__device__ __forceinline__ void ns_small_fetch(const f16* x, int ld, row_u32x4 (&v)[4]) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int row = n * 16 + (threadIdx.x >> 4), chunk = threadIdx.x & 15;
    v[n] = *(const row_u32x4*)(x + (size_t)row * 2 * ld + chunk * 8);
  }
}
__device__ __forceinline__ void ns_small_to_tile(const row_u32x4 (&v)[4], char* tile) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int row = n * 16 + (threadIdx.x >> 4), chunk = threadIdx.x & 15;
    *(row_u32x4*)(tile + row * 256 + ((chunk ^ ns_mix(row)) << 4)) = v[n];
  }
}
__device__ __forceinline__ void ns_small_from_tile(const char* tile, f16* x, int ld) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int row = n * 16 + (threadIdx.x >> 4), chunk = threadIdx.x & 15;
    *(row_u32x4*)(x + (size_t)row * 2 * ld + chunk * 8) = *(const row_u32x4*)(tile + row * 256 + ((chunk ^ ns_mix(row)) << 4));
  }
}
// partial product of this slice: [i][j], four consecutive j a store
__device__ __forceinline__ void ns_small_slab(const f32x16& acc, float* slab) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int i = (wid >> 1) * 32 + (lane & 31), j = (wid & 1) * 32 + 4 * (lane >> 5);
#pragma unroll
  for (int e = 0; e < 16; e += 4)
    *(f32x4*)(slab + i * 64 + j + 2 * e) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
}
__device__ __forceinline__ f16* ns_small_block(const NsArgs& p, const NsMat& m, int k, int block) {
  f16* x = p.ws + m.x + (k & 1 ? (size_t)2 * m.rp * m.cp : 0);
  return x + (m.tall ? (size_t)block * 64 * 2 * m.cp : (size_t)block * 128);
}

// X_0 of a slice and its partial product
template <typename T, bool MOMENTUM>
__global__ __launch_bounds__(256) void ns_small_first_kernel(NsArgs p) {
  __shared__ __attribute__((aligned(16))) char tile[NS_TILE];
  __shared__ double red[4];
  const NsJob job = p.small[blockIdx.x];
  const NsMat m = p.mats[job.mat];
  const T* in = (const T*)p.in + m.at;
  const float* buf = MOMENTUM ? p.buf + m.at : nullptr;
  const float gs = MOMENTUM ? p.hyper[1] : 1.f;
  int lift;
  const double scale = ns_first_scale(p, m, red, lift);
  if (job.ti == 0 && threadIdx.x == 0) p.part[p.nparts + job.mat] = (double)lift;
  f32x16 acc = ns_zero();
  for (int block = job.tj; block < job.tj + job.edge; ++block) {
    const int row0 = m.tall ? block * 64 : 0, col0 = m.tall ? 0 : block * 64;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = h * 32 + (threadIdx.x >> 3), c = (threadIdx.x & 7) * 8, row = row0 + r, col = col0 + c;
      float g[8], b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = b[j] = 0.f;
      if (row < m.rows && col < m.cols) {
        row_load<T, 8>(in + (size_t)row * m.cols, col, m.cols, g);
        if (MOMENTUM) row_load<float, 8>(buf + (size_t)row * m.cols, col, m.cols, b);
      }
      f16x8 vh, vl;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (MOMENTUM) g[j] = ns_direction(g[j] * gs, b[j], p.mu, p.nesterov);
        f16 hi, lo;
        ns_split((float)((double)g[j] * scale), hi, lo);
        vh[j] = hi;
        vl[j] = lo;
      }
      *(f16x8*)(tile + ns_chunk(r, c, 0)) = vh;
      *(f16x8*)(tile + ns_chunk(r, c, 1)) = vl;
    }
    __syncthreads();
    if (m.tall)
      ns_small_product<true, true>(tile, tile, acc);
    else
      ns_small_product<false, false>(tile, tile, acc);
    ns_small_from_tile(tile, ns_small_block(p, m, 0, block), m.cp);
    __syncthreads();
  }
  ns_small_slab(acc, p.slabs + (size_t)(job.slab + job.ti) * 4096);
}

// Iteration k of a slice; the partial products of iteration k are in half k % 2 of the slabs.
template <int WHAT, typename O, bool SHIFT>
__global__ __launch_bounds__(256, 3) void ns_small_kernel(NsArgs p, int k) {
  __shared__ __attribute__((aligned(16))) char lds[2 * NS_TILE + 64 * NS_PITCH(64) * 4];
  __shared__ f32x4 diagonal[4];  // every fourth value of A's
  char* tb = lds;                 // F
  char* tx = lds + NS_TILE;       // E, then X
  char* tn = lds + 2 * NS_TILE;   // the next X; its fp32 tile where it is the result
  const NsJob job = p.small[blockIdx.x];
  const NsMat m = p.mats[job.mat];
  const int lift = ns_lift(p, job.mat, k), lift_next = ns_lift(p, job.mat, k + 1);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int i = (wid >> 1) * 32 + (lane & 31), j = (wid & 1) * 32 + 4 * (lane >> 5);
  row_u32x4 x[4];
  ns_small_fetch(ns_small_block(p, m, k, job.tj), m.cp, x);
  float shift = 0.f;  // d, in the scale of A
  {  // A, and E
    const float* slab = p.slabs + (size_t)((k & 1) * p.small_slices + job.slab) * 4096 + threadIdx.x * 4;
    f32x4 v[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) v[n] = *(const f32x4*)(slab + n * 1024);
#pragma unroll 4
    for (int q = 1; q < job.k0; ++q)
#pragma unroll
      for (int n = 0; n < 4; ++n) v[n] += *(const f32x4*)(slab + (size_t)q * 4096 + n * 1024);
    const float f = NS_GRAM_SCALE / (m.scale * m.scale);
    const int row = threadIdx.x >> 4, col = (threadIdx.x & 15) * 4;   // (of n = 0)
    const int side = m.tall ? m.cols : m.rows;
    if (SHIFT) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (n * 16 + row == col) ((float*)diagonal)[n * 4 + (row >> 2)] = v[n][0] * f;
      __syncthreads();
      const f32x4 four = (diagonal[0] + diagonal[1]) + (diagonal[2] + diagonal[3]);
      shift = ((four[0] + four[1]) + (four[2] + four[3])) / (float)((side + 3) >> 2);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float a[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) a[q] = v[n][q] * f - (SHIFT && n * 16 + row == col + q && n * 16 + row < side ? shift : 0.f);
      ns_small_put(tx, n * 16 + row, col, a);
    }
  }
  const float d = SHIFT ? ldexpf(shift / NS_GRAM_SCALE, -2 * lift) : 0.f;
  __syncthreads();
  {  // F
    f32x16 acc = ns_zero();
    ns_small_product<false, false>(tx, tx, acc);
    const float f = ldexpf(NS_C / NS_GRAM_SCALE, -2 * lift);
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      float v[4];
      ns_small_get(tx, i, j + 2 * e, v);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = (NS_B + 2.f * NS_C * d) * v[q] + f * acc[e + q];
      ns_small_put(tb, i, j + 2 * e, v);
    }
  }
  __syncthreads();
  const float fx = ldexpf(NS_A + (NS_B + NS_C * d) * d, lift_next - lift), ft = ldexpf(1.f / NS_GRAM_SCALE, lift_next - 3 * lift);
  const float unscale = ldexpf(1.f / m.scale, -lift_next);
  const float lr = WHAT == NS_APPLY ? p.hyper[0] : 0.f;
  const float keep = 1.f - lr * p.wd, rate = lr * m.lr_scale;
  f32x16 gram = ns_zero();
  for (int block = job.tj; block < job.tj + job.edge; ++block) {
    ns_small_to_tile(x, tx);
    if (block + 1 < job.tj + job.edge) ns_small_fetch(ns_small_block(p, m, k, block + 1), m.cp, x);
    __syncthreads();
    f32x16 acc = ns_zero();
    if (m.tall)
      ns_small_product<false, false>(tx, tb, acc);
    else
      ns_small_product<false, true>(tb, tx, acc);
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      float v[4];
      ns_small_get(tx, i, j + 2 * e, v);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = fx * v[q] + ft * acc[e + q];
      if (WHAT == NS_NEXT)
        ns_small_put(tn, i, j + 2 * e, v);
      else
        *(f32x4*)((float*)tn + i * NS_PITCH(64) + j + 2 * e) =
            f32x4{v[0] * unscale, v[1] * unscale, v[2] * unscale, v[3] * unscale};
    }
    __syncthreads();
    if (WHAT == NS_NEXT) {
      if (m.tall)
        ns_small_product<true, true>(tn, tn, gram);
      else
        ns_small_product<false, false>(tn, tn, gram);
      ns_small_from_tile(tn, ns_small_block(p, m, k + 1, block), m.cp);
    } else {
      const int row0 = m.tall ? block * 64 : 0, col0 = m.tall ? 0 : block * 64;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = h * 32 + (threadIdx.x >> 3), c = (threadIdx.x & 7) * 8;
        if (row0 + r < m.rows && col0 + c < m.cols)
          ns_result<WHAT, O>(p, m, row0 + r, col0 + c, (float*)tn + r * NS_PITCH(64) + c, keep, rate);
      }
    }
    __syncthreads();
  }
  if (WHAT == NS_NEXT) ns_small_slab(gram, p.slabs + (size_t)((k + 1 & 1) * p.small_slices + job.slab + job.ti) * 4096);
}

// ---------------------------------------------------------------- host
template <void (*KERNEL)(NsArgs, int)>
static int ns_tiles(int blocks, bool large, const NsArgs& a, int k, hipStream_t st) {
  // the dynamic-LDS limit is a per-device function attribute: remembered per device
  static bool attr_set[64] = {};
  int dev = 0;
  (void)hipGetDevice(&dev);
  dev = (dev >= 0 && dev < 64) ? dev : 0;
  if (!attr_set[dev]) {
    const int rc = (int)hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, NS_LDS_LARGE);
    if (rc != 0) return rc;
    attr_set[dev] = true;
  }
  hipLaunchKernelGGL(KERNEL, dim3(blocks), dim3(256), large ? NS_LDS_LARGE : NS_LDS_SMALL, st, a, k);
  return (int)hipGetLastError();
}

template <bool POLY>
static int ns_symmetric_tiles(int blocks, bool large, const NsArgs& a, int k, hipStream_t st) {
  if (blocks <= 512) return ns_tiles<ns_symmetric_kernel<POLY, 4>>(blocks, true, a, k, st);
  return ns_tiles<ns_symmetric_kernel<POLY, 3>>(blocks, large, a, k, st);
}

template <bool POLY>
static int ns_join(int tiles, const NsArgs& a, int k, hipStream_t st) {
  hipLaunchKernelGGL((ns_join_kernel<POLY>), dim3(tiles, 128 / NS_JOIN_ROWS), dim3(256), 0, st, a, k);
  return (int)hipGetLastError();
}

template <typename T, bool MOMENTUM>
static int ns_first(const NsArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((ns_norm_kernel<T, MOMENTUM>), dim3(a.nchunks), dim3(256), 0, st, a);
  if (a.nsmall > 0)
    hipLaunchKernelGGL((ns_small_first_kernel<T, MOMENTUM>), dim3(a.nsmall), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((ns_pack_kernel<T, MOMENTUM>), dim3(a.npacks), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

// the advancing stage of iteration k
template <int WHAT, typename O>
static int ns_step(const NsArgs& a, int k, hipStream_t st) {
  if (a.nsmall == 0) return ns_tiles<ns_advance_kernel<WHAT, O>>(a.nfull, (a.large & 4) != 0, a, k, st);
  constexpr bool FP32 = WHAT == NS_OUT && sizeof(O) == 4;
  if constexpr (WHAT == NS_NEXT)
    if (a.out != nullptr && a.dtype == IO_F32) {
      hipLaunchKernelGGL((ns_small_kernel<WHAT, O, true>), dim3(a.nsmall), dim3(256), 0, st, a, k);
      return (int)hipGetLastError();
    }
  hipLaunchKernelGGL((ns_small_kernel<WHAT, O, FP32>), dim3(a.nsmall), dim3(256), 0, st, a, k);
  return (int)hipGetLastError();
}

// All matrices of the lists: norm (and momentum), first iterate, `steps` iterations, the last of which writes the result
// or the parameters.
extern "C" int dtfa_newton_schulz(const NsArgs* args, hipStream_t st) {
  const NsArgs a = *args;
  if (a.nchunks <= 0 || a.steps < 1) return -1;
  if (a.nsmall <= 0 && (a.npacks <= 0 || a.ngram <= 0 || a.npoly <= 0 || a.nfull <= 0)) return -1;
  if ((a.out == nullptr) == (a.w == nullptr) || (a.w != nullptr) != (a.buf != nullptr) || (a.w != nullptr && a.hyper == nullptr))
    return -2;
  if (a.dtype != IO_BF16 && a.dtype != IO_F32 && (a.dtype != IO_F16 || a.buf != nullptr)) return -3;
  int rc;
  if (a.buf != nullptr)
    rc = a.dtype == IO_BF16 ? ns_first<bf16, true>(a, st) : ns_first<float, true>(a, st);
  else
    rc = a.dtype == IO_BF16 ? ns_first<bf16, false>(a, st) : a.dtype == IO_F16 ? ns_first<f16, false>(a, st)
         : ns_first<float, false>(a, st);
  for (int k = 0; k < a.steps && rc == 0; ++k) {
    if (a.nsmall == 0) {
      rc = ns_symmetric_tiles<false>(a.ngram, (a.large & 1) != 0, a, k, st);
      if (rc == 0 && a.ngram_joins > 0) rc = ns_join<false>(a.ngram_joins, a, k, st);
      if (rc == 0) rc = ns_symmetric_tiles<true>(a.npoly, (a.large & 2) != 0, a, k, st);
      if (rc == 0 && a.npoly_joins > 0) rc = ns_join<true>(a.npoly_joins, a, k, st);
      if (rc != 0) break;
    }
    if (k + 1 < a.steps)
      rc = ns_step<NS_NEXT, float>(a, k, st);
    else if (a.out == nullptr)
      rc = ns_step<NS_APPLY, float>(a, k, st);
    else if (a.dtype == IO_BF16)
      rc = ns_step<NS_OUT, bf16>(a, k, st);
    else if (a.dtype == IO_F16)
      rc = ns_step<NS_OUT, f16>(a, k, st);
    else
      rc = ns_step<NS_OUT, float>(a, k, st);
  }
  return rc;
}
