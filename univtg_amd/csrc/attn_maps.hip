// Attention over score maps: (1) one softmax map with a learned relative position bias by buckets ("relpos"), (2) differential attention, the
// difference of two softmax maps with a learned weight per head ("diff").  Forward and backward, queries of one length over keys of another,
// shared key / value heads, strided operands, key mask, causal mask, bf16 and fp16 operands with fp32 scores, statistics and sums.
//
//   relpos  x_ij = scale q_i.k_j + T[bucket(j - i - q_offset), h]     o = softmax(x) v
//   diff    x^m_ij = scale q^m_i.k^m_j  (m = 1, 2)                    o = (softmax(x^1) - lam_h softmax(x^2)) v,  v twice as wide as a q / k map
//
// Every score tile is computed transposed to the operand that follows it (queries along lanes for o and dq, keys along lanes for dk and dv),
// so that the probabilities go from the accumulators of one MFMA into the operand of the next without leaving their lane; the operand that has
// to be transposed is read with ds_read_b64_tr_b16.  Tiles reach LDS by LDS-DMA (16 bytes per lane, no register round trip).
//
// Probabilities and score gradients are rounded to the operands' 16 bits, once, where they become operands of the matrix pipe: their products are off by
// about as much as storing them in 16 bits costs anyway.  Against 64 bits o is 1.3 times (one map) to 1.5 times (two, whose difference cancels) as far off
// as its own rounding makes it.  A second product with what the rounding left takes that to 1.0, and the forward from 220 to 262 us (32 x 1232, 8 heads of
// 128), from 388 to 507 (causal 2 x 8191, 16 heads of 64), from 568 to 756 (2 x 6007, 8 heads of two maps of 64): not taken.
#include "uvtg_kernels.h"
#include "../../include/uvtg.h"
#include <string.h>
#include <math.h>

namespace {

typedef __attribute__((ext_vector_type(2))) _Float16 half2_t;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float ROW_OFF = 1e30f;       // "log2 of the sum" of a query row that has no probabilities: exp2(x - ROW_OFF) is an exact 0
constexpr int PAD = 96;                // entries on either side of the bias window: the positions of a wave's 32 queries x 64 keys span 95
constexpr int SLAB = 32 * 72;          // elements of a wave's store slab
constexpr int WIN = 256;               // key tiles whose masks a workgroup holds in LDS at a time

struct MapArgs {
  const bf16_t *q, *k, *v, *o, *o2, *dO;       // raw 16-bit values of either type
  const float *table, *lam;
  const int* buckets;
  const unsigned char* kvalid;
  bf16_t *out, *out2, *dq, *dk, *dv;
  float *lse, *rvec, *part, *acc, *amax;
  const float* lse_in;
  long long q_sb, q_ss, q_sh, q_sm, k_sb, k_ss, k_sh, k_sm, v_sb, v_ss, v_sh, mask_sb;     // element strides
  int B, H, Hkv, G, Sq, Sk, NB, R, off, causal;
  int seen;                                     // keys from here on are seen by no query (causal), so that their rows may hold anything: masked, as by kvalid
  float scale, c;                               // c = scale log2(e)
  int hb, nsplit;                               // split kernel: heads packed into a row block, key ranges
  int glo, gw;                                  // bias gradient: first reachable relative position, number of them
};

template <bool HALF> __device__ __forceinline__ f32x16 mma(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (HALF) return mfma32h(a, b, c); else return mfma32(a, b, c);
}
template <bool HALF> __device__ __forceinline__ unsigned pack2(float lo, float hi) {
  if constexpr (HALF) { const f32x2 v = {lo, hi}; return __builtin_bit_cast(unsigned, __builtin_convertvector(v, half2_t)); }
  else return pack_bf2(lo, hi);
}
template <bool HALF> __device__ __forceinline__ float to_f(short x) {
  if constexpr (HALF) return (float)__builtin_bit_cast(_Float16, x); else return bf2f((bf16_t)x);
}
template <bool HALF> __device__ __forceinline__ bf16_t from_f(float x) {
  if constexpr (HALF) return __builtin_bit_cast(bf16_t, (_Float16)x); else return f2bf(x);
}
// eight packed values (a half of a 32 x 32 block's registers) as an MFMA operand
__device__ __forceinline__ s16x8 frag(const unsigned* p) { return __builtin_bit_cast(s16x8, (u32x4){p[0], p[1], p[2], p[3]}); }
__device__ __forceinline__ s16x8 cat4(s16x4 a, s16x4 b) { return (s16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
// a probability from its log2: the statistics of a row with scores of 1e9 are tens of units coarse, and no probability may exceed 1 for that (the
// clamp is a modifier of the exponential itself).  A NaN has to stay one: the modifier turns it into 0 unless the wave's DX10_CLAMP (bit 8 of the mode
// register) is off, which costs nothing where an instruction per score would.
__device__ __forceinline__ float prob(float x) { return __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(x), 0.f, 1.f); }
__device__ __forceinline__ void clamp_keeps_nan() { __builtin_amdgcn_s_setreg(1 | 8 << 6, 0); }
// the other half-wave's value, without LDS
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return __int_as_float(r[0]) + __int_as_float(r[1]);
}
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}
// log2 of a number that is 1 but for roundings (or, for coarse statistics, is not)
__device__ __forceinline__ float log2_near_1(float s) {
  const float d = s - 1.f;
  return fabsf(d) < 1e-3f ? d * LOG2E * fmaf(-0.5f, d, 1.f) : __builtin_amdgcn_logf(s);
}
// The matrix pipe's sums are off by a little to one side (measured: dP about 1e-8 of its terms low).  lam's gradient adds one such sum per row of all
// queries, which cancel, and so would keep it: half of dP's products are formed with the other sign, where the error has it too (two maps of 32,
// 4 x 3869 queries over 2657 keys, fp16: 1.1e-5 of dlam before, under 1e-6 with it).  ds does not feel a constant in dP.
__device__ __forceinline__ s16x8 negated(s16x8 x) { return x ^ (short)0x8000; }
// fp16 score gradients: of a small dO (a mean over a batch, no loss scale) most would fall below the type's normal range (dO of 2^-10 over 4000 keys: dq and
// dk off by 5e-3, where storing them in 16 bits makes 6e-4).  They are formed from dO times the power of two that brings its largest entry to 1 .. 2, and dq and dk are divided by it
// in the factor that they are stored with; an entry of 1 or more leaves everything as it is.  (Not further up: |dS| may reach |dO| |v| channels / 2.)
__device__ __forceinline__ float lift_of(float amax) {                     // (NaN, infinity: 1)
  const int e = (int)((__float_as_uint(amax) >> 23) & 255) - 127;
  return __uint_as_float((unsigned)(127 + min(max(-e, 0), 15)) << 23);
}
__device__ __forceinline__ float inverse_of(float lift) { return __uint_as_float((254u << 23) - __float_as_uint(lift)); }
template <int N> __device__ __forceinline__ float amax_half(const s16x8 (&x)[N]) {     // (as whole numbers, whose order is the values'; a NaN is the largest)
  typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
  u16x2 m = 0;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const u32x4 w = __builtin_bit_cast(u32x4, x[i]);
#pragma unroll
    for (int e = 0; e < 4; e++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
  }
  return (float)__builtin_bit_cast(_Float16, (unsigned short)(m[0] > m[1] ? m[0] : m[1]));
}
__device__ __forceinline__ float top_of_wave(float x) {                    // (steps as in wave_sum_dpp)
  x = fmaxf(x, dpp_mov<0xB1>(x));
  x = fmaxf(x, dpp_mov<0x4E>(x));
  x = fmaxf(x, dpp_mov<0x141>(x));
  x = fmaxf(x, dpp_mov<0x140>(x));
  const int b = __float_as_int(x);
  return fmaxf(fmaxf(__int_as_float(__builtin_amdgcn_readlane(b, 0)), __int_as_float(__builtin_amdgcn_readlane(b, 16))),
               fmaxf(__int_as_float(__builtin_amdgcn_readlane(b, 32)), __int_as_float(__builtin_amdgcn_readlane(b, 48))));
}
__device__ __forceinline__ void zero(f32x16& x) {
#pragma unroll
  for (int r = 0; r < 16; r++) x[r] = 0.f;
}
__device__ __forceinline__ unsigned long long uniform64(unsigned long long m) {
  return (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(m & 0xffffffffull)) |
         ((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(m >> 32)) << 32);
}

// An LDS tile of W-element rows that is read by rows (ds_read_b128) and transposed (ds_read_b64_tr_b16): 16-byte chunk c of row r is stored at
// chunk c ^ f(r).  16 consecutive rows put one chunk index on 16 different 16-byte slots of the 256-byte bank row, and 4 consecutive rows put
// the 64 bytes of a transposing read on 4 different quarters of it: neither kind of read has a bank conflict.
template <int W> struct Tile {
  __device__ static __forceinline__ int f(int r) {
    if constexpr (W == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (W == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
  }
  __device__ static __forceinline__ int off(int r, int col) { return r * W + ((((col >> 3) ^ f(r))) << 3) + (col & 7); }
  // the permutation is an XOR: 16-element column steps are XORs of the offset, 16 rows further it is the same, 8 rows further one bit differs
  __device__ static __forceinline__ int cols(int base, int dcol) { return base ^ dcol; }
  __device__ static __forceinline__ int rows8(int base) { return (base ^ 16) + 8 * W; }
};

// A chain of N fragment reads and the MFMAs that use them, R reads ahead of their use: left alone the scheduler sinks each read to its MFMA, and
// every MFMA then waits out an LDS round trip.  fill() may run well before run(), under other arithmetic.
__device__ __forceinline__ void fence();
template <int N, int R, typename Load> __device__ __forceinline__ void fill(s16x8 (&f)[R], Load&& load) {
#pragma unroll
  for (int i = 0; i < (N < R ? N : R); i++) f[i] = load(i);
}
template <int N, int R, typename Load, typename Use> __device__ __forceinline__ void run(s16x8 (&f)[R], Load&& load, Use&& use) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    use(i, f[i % R]);
    if (i + R < N) f[i % R] = load(i + R);
    fence();
  }
}
// Fragments by LDS byte address: `at` is the lane's place in a tile whose start is a multiple of its row size, so that a column step is an XOR of the
// address (one VALU operation) and a step of 16 rows, another tile of the stage, an immediate.  opaque() keeps the compiler from hoisting the XORs
// out of the loop: it would spend a register on each of them, and spill.
__device__ __forceinline__ unsigned lds_at(const bf16_t* p) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const bf16_t*)p; }
__device__ __forceinline__ unsigned opaque(unsigned x) { asm volatile("" : "+v"(x)); return x; }
__device__ __forceinline__ s16x8 row_frag(unsigned at, int i, int bytes) {
  return *(const __attribute__((address_space(3))) s16x8*)(uintptr_t)((at ^ (32 * i)) + bytes);
}
__device__ __forceinline__ s16x8 col_frag(unsigned at0, unsigned at1, int i, int bytes) {
  typedef __attribute__((address_space(3))) s16x4* lptr;
  return cat4(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(uintptr_t)((at0 ^ (64 * i)) + bytes)),
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(uintptr_t)((at1 ^ (64 * i)) + bytes)));
}
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// ROWS rows of a strided matrix -> LDS tile, `nw` waves sharing the work; rows behind `last` repeat it.  A whole tile of ordinary rows is addressed by
// a scalar base and a 32-bit lane offset that does not depend on the tile (an instruction covers 512 / W rows, and NW waves step by a multiple of the
// permutation's period); the last tile, and rows more than 64 MB apart, by 64-bit lane addresses.
// The request itself is inline assembly: behind the builtin the compiler makes every LDS read that might touch the destination wait for ALL requests
// in flight, so that a tile requested ahead stalls the reads of the tile at hand (measured: two thirds of these kernels' time).  What orders requests
// and reads here is dma_wait() and the barrier behind it.  (The s_nop: a vector memory instruction reads its scalar address 5 wait states after a vector
// instruction may have written it.)
__device__ __forceinline__ void dma16(const void* base, unsigned offset, unsigned lds) {
  unsigned m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(m0) : "v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane((int)lds)) : "memory");
}
__device__ __forceinline__ void dma16(const void* lane_ptr, unsigned lds) {
  unsigned m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(m0) : "v"(lane_ptr), "s"(__builtin_amdgcn_readfirstlane((int)lds)) : "memory");
}
template <int W, int ROWS, int NW> __device__ __forceinline__ void load_tile(const bf16_t* base, long long stride, int row0, int last, bf16_t* tile, int wave, int lane) {
  constexpr int RPI = 512 / W, NI = ROWS / RPI, PERIOD = W == 128 ? 4 : W == 64 ? 2 : 1;
  const int lr = lane / (W / 8), lc = lane % (W / 8);
  const unsigned lds = lds_at(tile);
  if (row0 + ROWS - 1 <= last && stride < (1 << 25)) {
#pragma unroll
    for (int i = 0; i < (NI + NW - 1) / NW; i++) {
      const int n = i * NW + wave;
      if (NI % NW == 0 || n < NI)
        dma16(base + ((long long)row0 + n * RPI) * stride, 2u * (unsigned)(lr * (int)stride + ((lc ^ Tile<W>::f((NW % PERIOD ? n : wave) * RPI + lr)) * 8)), lds + n * 1024);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < (NI + NW - 1) / NW; i++) {
    const int n = i * NW + wave;
    if (NI % NW == 0 || n < NI) {
      const int r = n * RPI + lr;
      dma16(base + (long long)min(row0 + r, last) * stride + (lc ^ Tile<W>::f(r)) * 8, lds + n * 1024);
    }
  }
}
// The same for the loops over tiles, which keep a lane's row and chunk of a request ready.  Rows behind the last are clamped to it.  (One request per
// few MFMAs instead of all of a tile's together measured 5 - 12 % slower: a request holds its wave about as long wherever it stands.)
template <int W, int ROWS, int NW> struct Loader {
  static constexpr int RPI = 512 / W, NI = ROWS / RPI, PIECES = (NI + NW - 1) / NW, PERIOD = W == 128 ? 4 : W == 64 ? 2 : 1;
  static_assert(NW == 1 || NW % PERIOD == 0, "a wave's requests of a tile share one lane offset, or differ from it by an XOR");
  const char* base;
  unsigned stride;                              // bytes (the host refuses rows further than 128 MB apart)
  int last, wave, row, chunk;
  __device__ __forceinline__ Loader(const bf16_t* b, long long stride_, int last_, int wave_, int lane)
      : base((const char*)b), stride(2u * (unsigned)stride_), last(last_), wave(wave_), row(lane / (W / 8)) {
    chunk = ((lane % (W / 8)) ^ Tile<W>::f(wave * RPI + row)) * 16;
  }
  __device__ __forceinline__ void tile(int row0, unsigned lds, long long disp) const {
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
      const int n = i * NW + wave, r0 = min(row0 + n * RPI, last);
      if (NI % NW == 0 || n < NI)
        dma16(base + disp + (unsigned long long)(unsigned)r0 * stride,                                 // (opaque: not kept ready)
              (unsigned)min((int)opaque(row), last - r0) * stride + (chunk ^ (16 * Tile<W>::f(NW == 1 ? i % PERIOD * RPI : 0))), lds + n * 1024);
    }
  }
};
// zero the rows of a landed tile whose mask bit is clear: a masked key's k / v row may hold anything, infinities and NaN included
template <int W> __device__ __forceinline__ void clear_rows(bf16_t* tile, unsigned long long mask, int rows, int tid, int nt) {
  for (int i = tid; i < rows * (W / 8); i += nt)
    if (!((mask >> (i / (W / 8))) & 1)) *(u32x4*)(tile + i * 8) = (u32x4){0, 0, 0, 0};
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Key masks of the tiles of 64 keys, one 64-bit word each: of up to WIN tiles from w0 on in LDS, or plain arithmetic where there is no mask
struct Masks {
  const unsigned char* kv;
  unsigned long long* words;
  int w0, Sk, ntiles, wave, lane;
  __device__ __forceinline__ Masks(const MapArgs& a, int b, int ntiles_, unsigned long long* words_, int wave_, int lane_)
      : kv(a.kvalid ? a.kvalid + (size_t)b * a.mask_sb : nullptr), words(words_), w0(0), Sk(a.seen), ntiles(ntiles_), wave(wave_), lane(lane_) {}
  __device__ __forceinline__ void load() {       // (a barrier before and behind)
    if (!kv) return;
    const int n = min(WIN, ntiles - w0);
#pragma unroll 4
    for (int t = wave; t < n; t += 4) {
      const int key = (w0 + t) * 64 + lane;
      const unsigned long long m = __builtin_amdgcn_ballot_w64(key < Sk && kv[min(key, Sk - 1)] != 0);
      if (lane == 0) words[t] = m;
    }
  }
  __device__ __forceinline__ unsigned long long at(int t) const {
    if (kv) return uniform64(words[t - w0]);
    return t * 64 + 64 <= Sk ? ~0ull : (1ull << (Sk - t * 64)) - 1;
  }
  // first tile from t on with a key that is not masked (ntiles: none), and its mask; every wave of the workgroup calls it with the same t
  __device__ __forceinline__ int find(int t, unsigned long long& m) {
    for (; t < ntiles; t++) {
      if (kv && t >= w0 + WIN) {
        __syncthreads();
        w0 += WIN;
        load();
        __syncthreads();
      }
      m = at(t);
      if (m) return t;
    }
    return ntiles;
  }
};

// Bias of relative positions rlo .. rhi for one head, times log2(e): entry (rel - rlo).  Positions behind +-R take the bias of +-R.
__device__ __forceinline__ void load_bias(const MapArgs& a, int h, int rlo, int rhi, float* sB, int tid, int nt) {
  for (int i = tid; i <= rhi - rlo; i += nt) {
    const int rel = min(max(rlo + i, -a.R), a.R);
    const int bk = min(max(a.buckets[rel + a.R], 0), a.NB - 1);      // (an entry outside the table would be a read out of range)
    sB[i] = a.table[(size_t)bk * a.H + h] * LOG2E;
  }
}

// Window of positions whose bias a workgroup with positions lowest .. highest holds in LDS: at most PAD behind +-R, never without the position
// at or behind an end that it reaches
__device__ __forceinline__ void bias_window(const MapArgs& a, int lowest, int highest, int& rlo, int& rhi) {
  rlo = min(max(lowest, -a.R - PAD), a.R);
  rhi = min(max(highest, -a.R), a.R + PAD);
}

// 1-D grid -> (row block, batch, head).  Workgroups go round-robin over the 8 XCDs, each with an L2 of its own: XCD x takes a contiguous range
// of the list, so that the blocks of a head, then the heads that share its keys, run on one XCD; batch before key head, because the samples of
// a ragged batch differ in cost and a launch ends with its slowest XCD.
__device__ __forceinline__ void block_id(int nblk, const MapArgs& a, int heads, int& blk, int& b, int& h) {
  const int total = gridDim.x, qn = total / 8, r = total % 8, xcd = blockIdx.x % 8, idx = blockIdx.x / 8;
  const int v = (xcd < r ? xcd * (qn + 1) : r * (qn + 1) + (xcd - r) * qn) + idx;
  blk = v % nblk;
  const int g = heads / a.Hkv, p = v / nblk, hi = p / g;
  b = hi % a.B;
  h = (hi / a.B) * g + p % g;
}

// [W / 32] accumulators (rows = channels, lane = row of the output) times a factor per lane -> 16-bit rows of W contiguous channels, through a
// wave-private LDS slab: 16 bytes per lane, W / 8 lanes per row.  keep: all ones, or 0 for a lane whose row is stored as zeros (NaN included)
template <bool HALF, int W, typename F>
__device__ __forceinline__ void store_rows(const f32x16* acc, float factor, bf16_t* slab, int lane, F&& row_ptr, unsigned keep = ~0u) {
  constexpr int PW = W < 64 ? W : 64, STR = PW + 8, CPR = PW / 8;
  const int l31 = lane & 31, g = lane >> 5;
#pragma unroll
  for (int pass = 0; pass < W / PW; pass++) {
#pragma unroll
    for (int i = 0; i < PW / 32; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const f32x16& x = acc[pass * (PW / 32) + i];
        u32x2 t;
        t[0] = pack2<HALF>(x[4 * j] * factor, x[4 * j + 1] * factor) & keep;
        t[1] = pack2<HALF>(x[4 * j + 2] * factor, x[4 * j + 3] * factor) & keep;
        *(u32x2*)(slab + l31 * STR + i * 32 + 8 * j + 4 * g) = t;
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 32 * CPR / 64; i++) {
      const int idx = lane + 64 * i, row = idx / CPR, ch = idx % CPR;
      bf16_t* p = row_ptr(row);
      const u32x4 v = *(const u32x4*)(slab + row * STR + ch * 8);
      if (p) *(u32x4*)(p + pass * PW + ch * 8) = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// Scores of a 32-key x 32-query block held as f32x16 (register r <-> key (r & 3) + 8 (r >> 2) + 4 g, lane <-> query): -inf where the key's mask
// bit is clear or the key is behind `lim` (the last key the lane's query sees, relative to the block)
__device__ __forceinline__ void mask_scores(f32x16& s, unsigned mask32, int lim, int g, float off) {
  const unsigned m = mask32 >> (4 * g);
  const int l = lim - 4 * g;
#pragma unroll
  for (int r = 0; r < 16; r++) {
    const int key = (r & 3) + 8 * (r >> 2);
    if (!((m >> key) & 1) || key > l) s[r] = off;
  }
}

// ------------------------------------------------------------------------------------------------
// forward: one workgroup = 128 queries of one head, a wave of 32 each, 64-key tiles in two LDS stages.  The first two tiles are requested before
// anything else is known; from then on the requests of the next tile go out between the MFMAs of the current one.
//   one pass over the keys: m the running maximum of a row's scores, l = sum exp(x - m), o = sum exp(x - m) v, both times exp(m - m') when m rises
// Bound by the matrix and the vector pipe by turns: a 64-key tile costs a wave 32 MFMAs of 32 cycles (128 channels) and about as many cycles of vector
// work, half of it exponentials, and two waves per SIMD (registers) overlap the two in part.  MFMA 35 % and vector 43 % of the busy cycles at 128 channels,
// 40 % and 71 % with three waves at 64.  Measured: 32 x 1232 (half of the keys valid), 8 heads of 128: 227 us, 660 TF/s; causal 2 x 8191, 16 heads of 64:
// 431 us (399 at best), 640 TF/s; two maps of 64, 2 x 6007, 8 heads: 534 us, 526 TF/s.  Row blocks of 256 (8 waves) were 5 - 20 % slower.
// ------------------------------------------------------------------------------------------------
template <bool HALF, int D, int MAPS>
__global__ __launch_bounds__(256, 2) void maps_fwd_kernel(const MapArgs a) {
  constexpr int DV = MAPS * D, KT = 64 * D, STAGE = MAPS * KT + 64 * DV, NK = D / 16, ND = DV / 32, NB = MAPS == 2 ? 1 : 2, RA = 4;
  constexpr bool BIAS = MAPS == 1;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  bf16_t* stage = (bf16_t*)smem;
  unsigned long long* sMask = (unsigned long long*)(smem + 2 * STAGE * 2);
  float* sB = (float*)(sMask + WIN);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, l31 = lane & 31, i16 = lane & 15, qd = (lane >> 4) & 1;
  const int nqb = (a.Sq + 127) / 128;
  int blk, b, h;
  block_id(nqb, a, a.H, blk, b, h);
  if (a.causal) blk = nqb - 1 - blk;                     // the longest rows first
  const int kh = h / a.G, qb = blk * 128, q0 = qb + wave * 32, q_raw = q0 + l31, qrow = min(q_raw, a.Sq - 1);
  const bool live = q0 < a.Sq;
  const int last_q = min(qb + 127, a.Sq - 1);
  int ntiles = (a.Sk + 63) / 64;
  if (a.causal) ntiles = last_q + a.off < 0 ? 0 : min(ntiles, (last_q + a.off) / 64 + 1);
  typedef Loader<D, 64, 4> KL;
  typedef Loader<DV, 64, 4> VL;
  const KL kl(a.k + (long long)b * a.k_sb + (long long)kh * a.k_sh, a.k_ss, a.Sk - 1, wave, lane);
  const VL vl(a.v + (long long)b * a.v_sb + (long long)kh * a.v_sh, a.v_ss, a.Sk - 1, wave, lane);
  auto request = [&](int kt, int buf) {
    const unsigned s = lds_at(stage) + buf * STAGE * 2;
#pragma unroll
    for (int m = 0; m < MAPS; m++) kl.tile(kt * 64, s + m * KT * 2, 2 * m * a.k_sm);
    vl.tile(kt * 64, s + MAPS * KT * 2, 0);
  };
  if (ntiles > 0) request(0, 0);
  if (ntiles > 1) request(1, 1);

  s16x8 qf[MAPS][NK];
#pragma unroll
  for (int m = 0; m < MAPS; m++)
#pragma unroll
    for (int ks = 0; ks < NK; ks++)
      qf[m][ks] = *(const s16x8*)(a.q + (long long)b * a.q_sb + (long long)qrow * a.q_ss + (long long)h * a.q_sh + m * a.q_sm + 16 * ks + 8 * g);
  Masks masks(a, b, ntiles, sMask, wave, lane);
  masks.load();
  int rlo, rhi;
  bias_window(a, -(last_q + a.off), ntiles * 64 - 1 - qb - a.off, rlo, rhi);
  if constexpr (BIAS) load_bias(a, h, rlo, rhi, sB, tid, 256);
  f32x16 oacc[MAPS][ND];
  float m_run[MAPS], l_run[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; m++) {
    m_run[m] = -INFINITY; l_run[m] = 0.f;
#pragma unroll
    for (int i = 0; i < ND; i++) zero(oacc[m][i]);
  }
  const int koff = 2 * Tile<D>::off(l31, 8 * g);                                                      // bytes
  const int toff0 = 2 * Tile<DV>::off(4 * g + (i16 >> 2), 16 * qd + 4 * (i16 & 3)), toff1 = 2 * Tile<DV>::rows8(toff0 / 2);
  __syncthreads();
  float bl = 0.f, br = 0.f;
  if constexpr (BIAS) { bl = rlo <= -a.R ? sB[0] : 0.f; br = rhi >= a.R ? sB[rhi - rlo] : 0.f; }
  unsigned long long mask = ntiles > 0 ? masks.at(0) : 0, mask_n = ntiles > 1 ? masks.at(1) : 0;
#pragma nounroll
  for (int t = 0, tn = min(1, ntiles), buf = 0; t < ntiles;) {
    dma_wait();
    __syncthreads();
    const bool req = tn > 1 && tn < ntiles;                // (the second tile has been requested before the loop)
    bf16_t* sK = stage + buf * STAGE;
    bf16_t* sV = sK + MAPS * KT;
    if (mask != ~0ull) {
      clear_rows<DV>(sV, mask, 64, tid, 256);
      __syncthreads();
    }
    const int key0 = t * 64;
    const int seen = a.causal ? q0 + min(31, a.Sq - 1 - q0) + a.off - key0 : 64;      // last key (relative) that any query of the wave sees
    const bool work = live && seen >= 0;
    if (req && !work) request(tn, buf ^ 1);
    if (work) {
      const bool part = mask != ~0ull || (a.causal && q0 + a.off < key0 + 63);
      // NB blocks of 32 keys per softmax step: two for one map; one for two, whose accumulators leave no registers for more
      constexpr int NS = MAPS * NK * NB, NP = 2 * NB * ND;
#pragma unroll 1
      for (int kp = 0; kp < 2; kp += NB) {
        unsigned pk[MAPS][NB][8];
        f32x16 sc[MAPS][NB];
        s16x8 fa[RA];
        const unsigned ka = opaque(lds_at(sK) + koff + kp * 64 * D), va0 = opaque(lds_at(sV) + toff0 + kp * 64 * DV), va1 = opaque(lds_at(sV) + toff1 + kp * 64 * DV);
        auto krow = [&](int i) { return row_frag(ka, i / NB % NK, (i / NB / NK * KT + i % NB * 32 * D) * 2); };
        auto vcol = [&](int i) { return col_frag(va0, va1, i % ND, (i / ND) * 16 * DV * 2); };
#pragma unroll
        for (int m = 0; m < MAPS; m++)
#pragma unroll
          for (int kb = 0; kb < NB; kb++) zero(sc[m][kb]);
        fill<NS>(fa, krow);
        fence();
        run<NS>(fa, krow, [&](int i, s16x8 x) {
          sc[i / NB / NK][i % NB] = mma<HALF>(x, qf[i / NB / NK][i / NB % NK], sc[i / NB / NK][i % NB]);
        });
        if (req && kp == 0) request(tn, buf ^ 1);          // (while the score MFMAs run)
        fill<NP>(fa, vcol);                                // (arrive under the softmax arithmetic)
        fence();
#pragma unroll
        for (int m = 0; m < MAPS; m++) {
          f32x16 (&s)[NB] = sc[m];
          // log2-domain scores are cc s + cb: the scale and a bias that is the same over the tile cost nothing, they ride in the exponent's FMA
          float cc = a.c, cb = 0.f;
          if constexpr (BIAS) {
            const int rmin = key0 - q0 - 31 - a.off, rmax = key0 + 63 - q0 - a.off;
            if (rmin >= a.R) cb = br;
            else if (rmax <= -a.R) cb = bl;
            else {
              const float* bp = sB + (key0 - min(q_raw, last_q) - a.off + 4 * g - rlo);
#pragma unroll
              for (int kb = 0; kb < NB; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[kb][r] = fmaf(s[kb][r], a.c, bp[(kp + kb) * 32 + (r & 3) + 8 * (r >> 2)]);
              cc = 1.f;
            }
          }
          if (part) {
            const int lim = a.causal ? q_raw + a.off - key0 : 64;
#pragma unroll
            for (int kb = 0; kb < NB; kb++) mask_scores(s[kb], (unsigned)(mask >> (32 * (kp + kb))), lim - 32 * (kp + kb), g, -INFINITY);
          }
          float mx = s[0][0];
#pragma unroll
          for (int kb = 0; kb < NB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[kb][r]);
          mx = fmaf(half_max(mx), cc, cb);
          // the reference point of the exponentials follows the running maximum only when it has fallen 8 (a factor of 256) behind: the sums are
          // fp32 and the probabilities at most 2^8, and the accumulators are rescaled a few times per row instead of at every new maximum
          if (__builtin_amdgcn_ballot_w64(mx > m_run[m] + 8.f)) {
            const float mn = fmaxf(m_run[m], mx);
            const float al = ex2(m_run[m] - (mn == -INFINITY ? 0.f : mn));
            m_run[m] = mn; l_run[m] *= al;
#pragma unroll
            for (int i = 0; i < ND; i++)
#pragma unroll
              for (int r = 0; r < 16; r++) oacc[m][i][r] *= al;
          }
          const float e0 = cb - (m_run[m] == -INFINITY ? 0.f : m_run[m]);
          float rs = 0.f;
#pragma unroll
          for (int kb = 0; kb < NB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
              const float p0 = ex2(fmaf(s[kb][r], cc, e0)), p1 = ex2(fmaf(s[kb][r + 1], cc, e0));
              rs += p0 + p1;
              pk[m][kb][r / 2] = pack2<HALF>(p0, p1);
            }
          l_run[m] += rs;                                  // (this half-wave's keys; the halves meet at the end)
        }
        fence();
        run<NP>(fa, vcol, [&](int i, s16x8 x) {
          const int grp = i / ND;                          // 16 keys
#pragma unroll
          for (int m = 0; m < MAPS; m++) oacc[m][i % ND] = mma<HALF>(x, frag(pk[m][grp / 2] + 4 * (grp % 2)), oacc[m][i % ND]);
        });
      }
    }
    t = tn; mask = mask_n; buf ^= 1;
    tn = masks.find(tn + 1, mask_n);
  }
  dma_wait();                                              // no LDS-DMA may outlive the workgroup
  __syncthreads();
  if (!live) return;
  float inv[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; m++) {
    const float l = half_sum(l_run[m]);
    inv[m] = l == 0.f ? 0.f : 1.f / l;
    if (a.lse && g == 0 && q_raw < a.Sq) a.lse[(((size_t)b * a.H + h) * MAPS + m) * a.Sq + q_raw] = l == 0.f ? -INFINITY : m_run[m] * LN2 + __logf(l);
  }
  bf16_t* slab = stage + wave * SLAB;
  auto rows = [&](bf16_t* base) {
    return [=](int row) -> bf16_t* { return q0 + row < a.Sq ? base + (((size_t)b * a.Sq + q0 + row) * a.H + h) * DV : nullptr; };
  };
  if constexpr (MAPS == 2) {
    if (a.out2) store_rows<HALF, DV>(oacc[MAPS - 1], inv[MAPS - 1], slab, lane, rows(a.out2));
    const float w = -a.lam[h] * inv[MAPS - 1];
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) oacc[0][i][r] = fmaf(oacc[0][i][r], inv[0], w * oacc[MAPS - 1][i][r]);
    inv[0] = 1.f;
  }
  store_rows<HALF, DV>(oacc[0], inv[0], slab, lane, rows(a.out));
}

// ------------------------------------------------------------------------------------------------
// forward of few rows: one workgroup = up to 32 rows (queries of the heads that share a key head) x one range of keys; its 4 waves take 32-key
// tiles in turn and never wait for each other before the end.  Bound by the bytes of k and v: every key row is read once per row block.  A single query
// over 16 x 32765 keys (16 heads, 4 of keys, 128 channels): 188 us, 4.9 TB/s; 5 over 16 x 20011, two maps of 64: 126 us, 4.4 TB/s.  One query over 257
// keys: 11 us, the chain of dependent memory accesses (bias, tile, tile, join).
// ------------------------------------------------------------------------------------------------
template <bool HALF, int D, int MAPS>
__global__ __launch_bounds__(256, 2) void maps_fwd_split_kernel(const MapArgs a) {
  constexpr int DV = MAPS * D, KT = 32 * D, STAGE = MAPS * KT + 32 * DV, NK = D / 16, ND = DV / 32, RA = DV == 2 * D && D == 64 ? 3 : 4;
  constexpr int NLK = MAPS * 32 * D / 512, NLV = 32 * DV / 512;                 // LDS-DMA instructions of a tile's k and v
  constexpr bool BIAS = MAPS == 1;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  bf16_t* stage = (bf16_t*)smem;                                               // [4 waves][STAGE], then fp32 [4][DV][32] in the same place
  constexpr int SB = 4 * STAGE * 2 > 4 * DV * 32 * 4 ? 4 * STAGE * 2 : 4 * DV * 32 * 4;
  unsigned* sMask = (unsigned*)(smem + SB);                                    // [2 WIN] 32-key masks
  float* sML = (float*)(sMask + 2 * WIN);                                      // [MAPS][2][4][32] maxima and sums of the waves
  float* sB = sML + MAPS * 2 * 4 * 32;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, l31 = lane & 31, i16 = lane & 15, qd = (lane >> 4) & 1;
  // grid: x = row block (head group hg of hb heads, 32-row block qb of its hb * Sq rows), y = key range, z = batch x key head
  const int rows_h = a.hb * a.Sq, nrb = (rows_h + 31) / 32, hg = blockIdx.x / nrb, rb = blockIdx.x % nrb;
  const int b = blockIdx.z / a.Hkv, kh = blockIdx.z % a.Hkv;
  const int nh = min(a.hb, a.G - hg * a.hb), nrows = min(32, nh * a.Sq - rb * 32);
  if (nrows <= 0) return;
  const int row = rb * 32 + min(l31, nrows - 1), hl = row / a.Sq, qi = row % a.Sq, h = kh * a.G + hg * a.hb + hl;
  const bf16_t* kb_ = a.k + (long long)b * a.k_sb + (long long)kh * a.k_sh;
  const bf16_t* vb_ = a.v + (long long)b * a.v_sb + (long long)kh * a.v_sh;

  s16x8 qf[MAPS][NK];
#pragma unroll
  for (int m = 0; m < MAPS; m++)
#pragma unroll
    for (int ks = 0; ks < NK; ks++)
      qf[m][ks] = *(const s16x8*)(a.q + (long long)b * a.q_sb + (long long)qi * a.q_ss + (long long)h * a.q_sh + m * a.q_sm + 16 * ks + 8 * g);
  f32x16 oacc[MAPS][ND];
  float m_run[MAPS], l_run[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; m++) {
    m_run[m] = -INFINITY; l_run[m] = 0.f;
#pragma unroll
    for (int i = 0; i < ND; i++) zero(oacc[m][i]);
  }
  // positions of the block's queries: all of 0 .. Sq - 1 when several heads are packed, else 32 of them
  const int qlo = a.hb > 1 ? 0 : rb * 32, qhi = a.hb > 1 ? a.Sq - 1 : min(rb * 32 + 31, a.Sq - 1);
  int tiles = (a.Sk + 31) / 32;
  if (a.causal) tiles = qhi + a.off < 0 ? 0 : min(tiles, (qhi + a.off) / 32 + 1);
  const int per = (tiles + a.nsplit - 1) / a.nsplit, t0 = min(blockIdx.y * per, tiles), t1 = min(t0 + per, tiles);
  const int rlo = min(max(t0 * 32 - qhi - a.off, -a.R), a.R), rhi = min(max(t1 * 32 - 1 - qlo - a.off, -a.R), a.R), bw = rhi - rlo + 1;
  if constexpr (BIAS) for (int i = 0; i < nh; i++) load_bias(a, kh * a.G + hg * a.hb + i, rlo, rhi, sB + i * bw, tid, 256);

  bf16_t* sK = stage + wave * STAGE;
  bf16_t* sV = sK + MAPS * KT;
  const int koff = 2 * Tile<D>::off(l31, 8 * g);                                                      // bytes
  const int toff0 = 2 * Tile<DV>::off(4 * g + (i16 >> 2), 16 * qd + 4 * (i16 & 3)), toff1 = 2 * Tile<DV>::rows8(toff0 / 2);
  typedef Loader<D, 32, 1> KL;
  typedef Loader<DV, 32, 1> VL;
  const KL kl(kb_, a.k_ss, a.Sk - 1, 0, lane);
  const VL vl(vb_, a.v_ss, a.Sk - 1, 0, lane);
  auto request_k = [&](int kt) {
#pragma unroll
    for (int m = 0; m < MAPS; m++) kl.tile(kt * 32, lds_at(sK) + m * KT * 2, 2 * m * a.k_sm);
  };
  auto request_v = [&](int kt) { vl.tile(kt * 32, lds_at(sV), 0); };
  const unsigned char* kv = a.kvalid ? a.kvalid + (size_t)b * a.mask_sb : nullptr;
  for (int w0 = t0; w0 < t1; w0 += 2 * WIN) {
    const int wn = min(2 * WIN, t1 - w0);
    __syncthreads();
#pragma unroll 4
    for (int t = 2 * wave; t < wn; t += 8) {               // two 32-key masks per ballot
      const int key = (w0 + t) * 32 + lane;
      const unsigned long long m = __builtin_amdgcn_ballot_w64(key < a.seen && (!kv || kv[key] != 0));
      if (lane == 0) { sMask[t] = (unsigned)m; sMask[t + 1] = (unsigned)(m >> 32); }
    }
    __syncthreads();
    auto next = [&](int t) { while (t < wn && __builtin_amdgcn_readfirstlane((int)sMask[t]) == 0) t += 4; return t; };
    int t = next(wave);
    if (t < wn) { request_k(w0 + t); request_v(w0 + t); }
    while (t < wn) {
      const int tn = next(t + 4);
      const bool more = tn < wn;
      const unsigned mask = (unsigned)__builtin_amdgcn_readfirstlane((int)sMask[t]);
      const int key0 = (w0 + t) * 32;
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NLV) : "memory");          // k of this tile has landed (its v was requested behind it)
      unsigned pk[MAPS][8];
      s16x8 fa[RA];
#pragma unroll
      for (int m = 0; m < MAPS; m++) {                     // one map's scores at a time: the accumulators of two leave no registers for both
        f32x16 s;
        zero(s);
        const unsigned ka = opaque(lds_at(sK) + koff);
        auto krow = [&](int i) { return row_frag(ka, i, m * KT * 2); };
        fill<NK>(fa, krow);
        fence();
        run<NK>(fa, krow, [&](int i, s16x8 x) { s = mma<HALF>(x, qf[m][i], s); });
        if (m == MAPS - 1) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");              // the reads of k are done: its place may be written
          if (more) request_k(w0 + tn);
        }
        if constexpr (BIAS) {
          const float* bp = sB + hl * bw;
          const int rel = key0 + 4 * g - qi - a.off;
#pragma unroll
          for (int r = 0; r < 16; r++) s[r] = fmaf(s[r], a.c, bp[min(max(rel + (r & 3) + 8 * (r >> 2), rlo), rhi) - rlo]);
        } else {
#pragma unroll
          for (int r = 0; r < 16; r++) s[r] *= a.c;
        }
        mask_scores(s, mask, a.causal ? qi + a.off - key0 : 32, g, -INFINITY);
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[r]);
        mx = half_max(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m_run[m] + 8.f)) {
          const float mn = fmaxf(m_run[m], mx);
          const float al = ex2(m_run[m] - (mn == -INFINITY ? 0.f : mn));
          m_run[m] = mn; l_run[m] *= al;
#pragma unroll
          for (int i = 0; i < ND; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) oacc[m][i][r] *= al;
        }
        const float e0 = m_run[m] == -INFINITY ? 0.f : -m_run[m];
        float rs = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float p0 = ex2(s[r] + e0), p1 = ex2(s[r + 1] + e0);
          rs += p0 + p1;
          pk[m][r / 2] = pack2<HALF>(p0, p1);
        }
        l_run[m] += rs;
        fence();
      }
      if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NLK) : "memory");                        // v of this tile
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (mask != ~0u) { clear_rows<DV>(sV, mask, 32, lane, 64); asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
      const unsigned va0 = opaque(lds_at(sV) + toff0), va1 = opaque(lds_at(sV) + toff1);
      auto vcol = [&](int i) { return col_frag(va0, va1, i % ND, (i / ND) * 16 * DV * 2); };
      fill<2 * ND>(fa, vcol);
      fence();
      run<2 * ND>(fa, vcol, [&](int i, s16x8 x) {
#pragma unroll
        for (int m = 0; m < MAPS; m++) oacc[m][i % ND] = mma<HALF>(x, frag(pk[m] + 4 * (i / ND)), oacc[m][i % ND]);
      });
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) request_v(w0 + tn);
      t = tn;
    }
  }
  // join the four waves: factors from the common maximum, then a sum in wave order
#pragma unroll
  for (int m = 0; m < MAPS; m++) {
    const float l = half_sum(l_run[m]);
    if (g == 0) { sML[(m * 2 + 0) * 128 + wave * 32 + l31] = m_run[m]; sML[(m * 2 + 1) * 128 + wave * 32 + l31] = l; }
  }
  float* sO = (float*)smem;
  const int orow = tid & 31, oc = tid >> 5;                                   // 8 threads per row, DV / 8 channels each
  const int r2 = rb * 32 + orow, oh = kh * a.G + hg * a.hb + r2 / a.Sq, oq = r2 % a.Sq;
  constexpr int CPT = DV / 8;
  float res[MAPS][CPT], mt[MAPS], lt[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; m++) {
    __syncthreads();                                                           // tiles read, maxima written; the other map's sums read
    const float* M = sML + (m * 2) * 128;
    const float mm = fmaxf(fmaxf(M[l31], M[32 + l31]), fmaxf(M[64 + l31], M[96 + l31]));
    const float fac = ex2(m_run[m] - (mm == -INFINITY ? 0.f : mm));
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) sO[(wave * DV + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * g) * 32 + l31] = oacc[m][i][r] * fac;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < CPT; e++) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < 4; w++) x += sO[(w * DV + oc * CPT + e) * 32 + orow];
      res[m][e] = x;
    }
    const float mo = fmaxf(fmaxf(M[orow], M[32 + orow]), fmaxf(M[64 + orow], M[96 + orow]));
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) l += M[128 + w * 32 + orow] * ex2(M[w * 32 + orow] - (mo == -INFINITY ? 0.f : mo));
    mt[m] = mo; lt[m] = l;
  }
  if (orow >= nrows) return;
  const size_t orow_g = ((size_t)b * a.H + oh) * a.Sq + oq;
  if (a.nsplit > 1) {                                                          // partial: [B, H, Sq][split][MAPS][DV + 2]
    float* w = a.acc + (orow_g * a.nsplit + blockIdx.y) * (MAPS * (DV + 2));
#pragma unroll
    for (int m = 0; m < MAPS; m++) {
#pragma unroll
      for (int e = 0; e < CPT; e++) w[m * (DV + 2) + oc * CPT + e] = res[m][e];
      if (oc == 0) { w[m * (DV + 2) + DV] = mt[m]; w[m * (DV + 2) + DV + 1] = lt[m]; }
    }
    return;
  }
  float inv[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; m++) {
    inv[m] = lt[m] == 0.f ? 0.f : 1.f / lt[m];
    if (a.lse && oc == 0) a.lse[(((size_t)b * a.H + oh) * MAPS + m) * a.Sq + oq] = lt[m] == 0.f ? -INFINITY : mt[m] * LN2 + __logf(lt[m]);
  }
  const size_t ob = (((size_t)b * a.Sq + oq) * a.H + oh) * DV + oc * CPT;
  const float w = MAPS == 2 ? a.lam[oh] : 0.f;
#pragma unroll
  for (int e = 0; e < CPT; e++) {
    float x = res[0][e] * inv[0];
    if constexpr (MAPS == 2) {
      const float y = res[MAPS - 1][e] * inv[MAPS - 1];
      if (a.out2) a.out2[ob + e] = from_f<HALF>(y);
      x -= w * y;
    }
    a.out[ob + e] = from_f<HALF>(x);
  }
}

// joins the key ranges of maps_fwd_split_kernel: one wave per row, ranges in order (5 - 7 us for 256 - 1280 rows of 8 ranges: latency)
template <bool HALF, int D, int MAPS>
__global__ __launch_bounds__(256) void maps_join_kernel(const MapArgs a) {
  constexpr int DV = MAPS * D, CPL = (DV + 63) / 64, W = MAPS * (DV + 2);
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);        // (b, h, query)
  if (row >= (long long)a.B * a.H * a.Sq) return;
  const int i = (int)(row % a.Sq);
  const long long bh = row / a.Sq;
  const int h = (int)(bh % a.H), b = (int)(bh / a.H);
  const float* p = a.acc + (size_t)row * a.nsplit * W;
  float o[MAPS][CPL];
#pragma unroll
  for (int m = 0; m < MAPS; m++) {
    float mx = -INFINITY;
    for (int s = lane; s < a.nsplit; s += 64) mx = fmaxf(mx, p[(size_t)s * W + m * (DV + 2) + DV]);
    mx = wave_max(mx);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float l = 0.f;
#pragma unroll
    for (int c = 0; c < CPL; c++) o[m][c] = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.nsplit; s++) {
      const float* w = p + (size_t)s * W + m * (DV + 2);
      const float f = ex2(w[DV] - mu);
      l += w[DV + 1] * f;
#pragma unroll
      for (int c = 0; c < CPL; c++) if (DV >= 64 || lane < DV) o[m][c] += w[lane + 64 * c] * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < CPL; c++) o[m][c] *= inv;
    if (a.lse && lane == 0) a.lse[(bh * MAPS + m) * a.Sq + i] = l == 0.f ? -INFINITY : mx * LN2 + __logf(l);
  }
  const size_t ob = (((size_t)b * a.Sq + i) * a.H + h) * DV;
#pragma unroll
  for (int c = 0; c < CPL; c++) {
    if (DV < 64 && lane >= DV) continue;
    float x = o[0][c];
    if constexpr (MAPS == 2) {
      if (a.out2) a.out2[ob + lane + 64 * c] = from_f<HALF>(o[MAPS - 1][c]);
      x -= a.lam[h] * o[MAPS - 1][c];
    }
    a.out[ob + lane + 64 * c] = from_f<HALF>(x);
  }
}

// ------------------------------------------------------------------------------------------------
// backward, queries: dq and the row sums r_i = sum_j p_ij dp_ij.  One workgroup = 128 queries of one head, tiles as in the forward.
// ds = p (dp - r) needs r before the first key: rowsum(dO o) gives it up to the rounding of o, which is enough for dq (16 bits), and the exact
// fp32 sum falls out of the same registers (one FMA per element): the key kernel forms ds, the bias table's and lam's gradients from that.  Both are
// divided by the row's sum of p, which is 1 up to the rounding of lse (1e-6): the ds of a row then add up to 0, where a bucket that holds nearly all of
// a row would keep the difference and nothing else.
// Row statistics leave as [B][H][64-query tile][MAPS][2][64] floats: log2 of the row sum (ROW_OFF for a row without one), r.
// Bound as the forward: three products per pair of positions instead of two.  32 x 1232, 8 heads of 128: 330 us, 680 TF/s; causal 4 x 4096, 16 heads of
// two maps of 64: 762 us (713 at best), 540 TF/s (of which the sums of p and dP's signs, for the precision of r: 3 - 5 %).  (Exponentials placed under the MFMAs of dP by hand were 13 % slower.)
// ------------------------------------------------------------------------------------------------
template <bool HALF, int D, int MAPS>
__global__ __launch_bounds__(256, 2) void maps_bwd_q_kernel(const MapArgs a) {
  clamp_keeps_nan();
  constexpr int DV = MAPS * D, KT = 64 * D, STAGE = MAPS * KT + 64 * DV, NK = D / 16, NV = DV / 16, ND = D / 32, RA = 4;
  constexpr bool BIAS = MAPS == 1;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  bf16_t* stage = (bf16_t*)smem;
  unsigned long long* sMask = (unsigned long long*)(smem + 2 * STAGE * 2);
  float* sB = (float*)(sMask + WIN);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, l31 = lane & 31, i16 = lane & 15, qd = (lane >> 4) & 1;
  const int nqb = (a.Sq + 127) / 128;
  int blk, b, h;
  block_id(nqb, a, a.H, blk, b, h);
  if (a.causal) blk = nqb - 1 - blk;
  const int kh = h / a.G, qb = blk * 128, q0 = qb + wave * 32, q_raw = q0 + l31, qrow = min(q_raw, a.Sq - 1);
  const bool live = q0 < a.Sq;
  const int last_q = min(qb + 127, a.Sq - 1);
  int ntiles = (a.Sk + 63) / 64;
  if (a.causal) ntiles = last_q + a.off < 0 ? 0 : min(ntiles, (last_q + a.off) / 64 + 1);
  typedef Loader<D, 64, 4> KL;
  typedef Loader<DV, 64, 4> VL;
  const KL kl(a.k + (long long)b * a.k_sb + (long long)kh * a.k_sh, a.k_ss, a.Sk - 1, wave, lane);
  const VL vl(a.v + (long long)b * a.v_sb + (long long)kh * a.v_sh, a.v_ss, a.Sk - 1, wave, lane);
  auto request = [&](int kt, int buf) {
    const unsigned s = lds_at(stage) + buf * STAGE * 2;
#pragma unroll
    for (int m = 0; m < MAPS; m++) kl.tile(kt * 64, s + m * KT * 2, 2 * m * a.k_sm);
    vl.tile(kt * 64, s + MAPS * KT * 2, 0);
  };
  if (ntiles > 0) request(0, 0);
  if (ntiles > 1) request(1, 1);
  s16x8 qf[MAPS][NK], of[NV];
  float L[MAPS], del[MAPS], racc[MAPS], psum[MAPS], drop = 1.f;
  const float lam = MAPS == 2 ? a.lam[h] : 0.f;
  {
    const size_t ro = (((size_t)b * a.Sq + qrow) * a.H + h) * DV + 8 * g;
#pragma unroll
    for (int m = 0; m < MAPS; m++) {
#pragma unroll
      for (int ks = 0; ks < NK; ks++)
        qf[m][ks] = *(const s16x8*)(a.q + (long long)b * a.q_sb + (long long)qrow * a.q_ss + (long long)h * a.q_sh + m * a.q_sm + 16 * ks + 8 * g);
      const float l = a.lse_in[(((size_t)b * a.H + h) * MAPS + m) * a.Sq + qrow];
      L[m] = l == -INFINITY ? ROW_OFF : l * LOG2E;
      del[m] = 0.f; racc[m] = 0.f; psum[m] = 0.f;
    }
#pragma unroll
    for (int ks = 0; ks < NV; ks++) of[ks] = *(const s16x8*)(a.dO + ro + 16 * ks);
#pragma unroll
    for (int ks = 0; ks < NV; ks++) {
      const s16x8 x = *(const s16x8*)(a.o + ro + 16 * ks);
      s16x8 y;
      if constexpr (MAPS == 2) y = *(const s16x8*)(a.o2 + ro + 16 * ks);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float d = to_f<HALF>(of[ks][e]);
        if constexpr (MAPS == 2) {
          const float o2 = to_f<HALF>(y[e]);
          del[0] += d * fmaf(lam, o2, to_f<HALF>(x[e]));
          del[MAPS - 1] += d * o2;
        } else del[0] += d * to_f<HALF>(x[e]);
      }
    }
#pragma unroll
    for (int m = 0; m < MAPS; m++) del[m] = half_sum(del[m]);
    if constexpr (HALF) {                                  // every row by its own power of two; the key kernel takes one for all rows that it adds up
      const float am = half_max(amax_half(of)), lift = lift_of(am), top = top_of_wave(am);
      drop = inverse_of(lift);
      if (live && lane == 0) a.amax[((size_t)b * a.H + h) * ((a.Sq + 31) / 32) + q0 / 32] = top;
#pragma unroll
      for (int m = 0; m < MAPS; m++) del[m] *= lift;
#pragma unroll
      for (int ks = 0; ks < NV; ks++)
        of[ks] = __builtin_bit_cast(s16x8, __builtin_bit_cast(half8_t, of[ks]) * (_Float16)(MAPS == 2 && ks >= NV / 4 && ks < 3 * NV / 4 ? -lift : lift));
    } else if constexpr (MAPS == 2) {
#pragma unroll
      for (int ks = NV / 4; ks < 3 * NV / 4; ks++) of[ks] = negated(of[ks]);
    }
  }
  Masks masks(a, b, ntiles, sMask, wave, lane);
  masks.load();
  int rlo, rhi;
  bias_window(a, -(last_q + a.off), ntiles * 64 - 1 - qb - a.off, rlo, rhi);
  if constexpr (BIAS) load_bias(a, h, rlo, rhi, sB, tid, 256);
  f32x16 acc[MAPS][ND];
#pragma unroll
  for (int m = 0; m < MAPS; m++)
#pragma unroll
    for (int i = 0; i < ND; i++) zero(acc[m][i]);
  const int koff = 2 * Tile<D>::off(l31, 8 * g), voff = 2 * Tile<DV>::off(l31, 8 * g);                // bytes
  const int toff0 = 2 * Tile<D>::off(4 * g + (i16 >> 2), 16 * qd + 4 * (i16 & 3)), toff1 = 2 * Tile<D>::rows8(toff0 / 2);
  __syncthreads();
  float bl = 0.f, br = 0.f;
  if constexpr (BIAS) { bl = rlo <= -a.R ? sB[0] : 0.f; br = rhi >= a.R ? sB[rhi - rlo] : 0.f; }
  unsigned long long mask = ntiles > 0 ? masks.at(0) : 0, mask_n = ntiles > 1 ? masks.at(1) : 0;
#pragma nounroll
  for (int t = 0, tn = min(1, ntiles), buf = 0; t < ntiles;) {
    dma_wait();
    __syncthreads();
    const bool req = tn > 1 && tn < ntiles;
    bf16_t* sK = stage + buf * STAGE;
    bf16_t* sV = sK + MAPS * KT;
    if (mask != ~0ull) {
#pragma unroll
      for (int m = 0; m < MAPS; m++) clear_rows<D>(sK + m * KT, mask, 64, tid, 256);
      clear_rows<DV>(sV, mask, 64, tid, 256);
      __syncthreads();
    }
    const int key0 = t * 64;
    const int seen = a.causal ? q0 + min(31, a.Sq - 1 - q0) + a.off - key0 : 64;
    const bool work = live && seen >= 0;
    if (req && !work) request(tn, buf ^ 1);
    if (work) {
      const bool part = mask != ~0ull || (a.causal && q0 + a.off < key0 + 63);
      constexpr int NS = NV + MAPS * NK, NP = 2 * MAPS * ND;
#pragma unroll 1
      for (int kb = 0; kb < 2; kb++) {
        f32x16 dp, s[MAPS];
        s16x8 fa[RA];
        const unsigned ka = opaque(lds_at(sK) + koff + kb * 64 * D), va = DV == D ? ka : opaque(lds_at(sV) + voff + kb * 64 * DV);
        const unsigned ta0 = opaque(lds_at(sK) + toff0 + kb * 64 * D), ta1 = opaque(lds_at(sK) + toff1 + kb * 64 * D);
        auto kvrow = [&](int i) { return i < NV ? row_frag(va, i, DV == D ? MAPS * KT * 2 : 0) : row_frag(ka, (i - NV) % NK, (i - NV) / NK * KT * 2); };
        auto kcol = [&](int i) { return col_frag(ta0, ta1, i % ND, (i / (2 * ND) * KT + i / ND % 2 * 16 * D) * 2); };
        zero(dp);
#pragma unroll
        for (int m = 0; m < MAPS; m++) zero(s[m]);
        fill<NS>(fa, kvrow);
        fence();
        run<NS>(fa, kvrow, [&](int i, s16x8 x) {
          const int j = i < NV ? 0 : i - NV;
          if (MAPS == 2 && (i == NV / 4 || i == 3 * NV / 4)) dp = -dp;
          if (i < NV) dp = mma<HALF>(x, of[i < NV ? i : 0], dp); else s[j / NK] = mma<HALF>(x, qf[j / NK][j % NK], s[j / NK]);
        });
        if (req && kb == 0) request(tn, buf ^ 1);
        fill<NP>(fa, kcol);
        fence();
        unsigned pk[MAPS][8];
#pragma unroll
        for (int m = 0; m < MAPS; m++) {
          float cc = a.c, cb = 0.f;
          if constexpr (BIAS) {
            const int rmin = key0 - q0 - 31 - a.off, rmax = key0 + 63 - q0 - a.off;
            if (rmin >= a.R) cb = br;
            else if (rmax <= -a.R) cb = bl;
            else {
              const float* bp = sB + (key0 - min(q_raw, last_q) - a.off + 4 * g - rlo);
#pragma unroll
              for (int r = 0; r < 16; r++) s[m][r] = fmaf(s[m][r], a.c, bp[kb * 32 + (r & 3) + 8 * (r >> 2)]);
              cc = 1.f;
            }
          }
          if (part) mask_scores(s[m], (unsigned)(mask >> (32 * kb)), (a.causal ? q_raw + a.off - key0 : 64) - 32 * kb, g, -INFINITY);
          const float e0 = cb - L[m];
          const float f = m == 0 ? 1.f : -lam;
          float rb = 0.f, pb = 0.f;                        // (sums of a block, then of blocks: a long row's last terms meet no long sum)
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            const float p0 = prob(fmaf(s[m][r], cc, e0)), p1 = prob(fmaf(s[m][r + 1], cc, e0));
            rb = fmaf(p0, dp[r], rb); rb = fmaf(p1, dp[r + 1], rb);
            pb += p0 + p1;
            pk[m][r / 2] = pack2<HALF>((m ? f * p0 : p0) * (dp[r] - del[m]), (m ? f * p1 : p1) * (dp[r + 1] - del[m]));
          }
          racc[m] += rb; psum[m] += pb;
        }
        fence();
        run<NP>(fa, kcol, [&](int i, s16x8 x) {
          acc[i / (2 * ND)][i % ND] = mma<HALF>(x, frag(pk[i / (2 * ND)] + 4 * (i / ND % 2)), acc[i / (2 * ND)][i % ND]);
        });
      }
    }
    t = tn; mask = mask_n; buf ^= 1;
    tn = masks.find(tn + 1, mask_n);
  }
  dma_wait();
  __syncthreads();
  if (!live) return;
#pragma unroll
  for (int m = 0; m < MAPS; m++) {
    const float s = half_sum(psum[m]), r = s == 0.f ? 0.f : half_sum(racc[m]) / s * drop;          // (NaN stays NaN)
    float* st = a.rvec + ((((size_t)b * a.H + h) * ((a.Sq + 63) / 64) + q0 / 64) * MAPS + m) * 128 + (q0 & 32) + l31;
    st[g * 64] = g ? r : q_raw < a.Sq && s != 0.f ? L[m] + log2_near_1(s) : ROW_OFF;
    if (MAPS == 2 && m == MAPS - 1) {                      // lam's gradient: the wave's 32 rows, [H][B][32-row block]
      const float w = wave_sum_dpp(g == 0 && q_raw < a.Sq ? r : 0.f);
      const int n32 = (a.Sq + 31) / 32;
      if (lane == 0) a.part[((size_t)h * a.B + b) * n32 + q0 / 32] = w;
    }
  }
  bf16_t* slab = stage + wave * SLAB;
#pragma unroll
  for (int m = 0; m < MAPS; m++)
    store_rows<HALF, D>(acc[m], a.scale * drop, slab, lane, [=](int row) -> bf16_t* {
      return q0 + row < a.Sq ? a.dq + ((((size_t)b * a.Sq + q0 + row) * a.H + h) * MAPS + m) * D : nullptr; });
}

// ------------------------------------------------------------------------------------------------
// backward, keys: dk, dv and (relpos) the bias gradient by relative position.  One workgroup = 128 keys of one key head; it walks the queries of
// every head of the group in tiles of 64, so that the shared heads' gradients are summed in registers, in a fixed order.  8 waves: wave w has keys
// 32 (w & 3) .. and of each tile the queries 32 (w >> 2) .., and the two waves of a key block add up at the end: two waves per SIMD, whose LDS round
// trips, exponentials and MFMAs overlap (one wave of 4 per SIMD, with everything in 420 registers, spent two thirds of its time waiting).
// Bound by the pipes and by LDS, of which a block near the diagonal uses twice as much (its score gradients are summed along the diagonals): 32 x 1232,
// 8 heads of 128: 500 us, 597 TF/s over four products; causal 4 x 4096, 16 heads of two maps of 64: 694 us, 792 TF/s.
// ------------------------------------------------------------------------------------------------
template <bool HALF, int D, int MAPS>
__global__ __launch_bounds__(512, 2) void maps_bwd_k_kernel(const MapArgs a) {
  clamp_keeps_nan();
  constexpr int DV = MAPS * D, QT = 64 * D, STAGE = MAPS * QT + 64 * DV, NK = D / 16, NV = DV / 16, ND = D / 32, NDV = DV / 32;
  constexpr bool BIAS = MAPS == 1, VLDS = DV == 128;       // 128 channels: v's fragments stay in LDS, beside the accumulators they would not fit
  constexpr int RA = VLDS ? 3 : 4, RV = 2;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  bf16_t* stage = (bf16_t*)smem;
  bf16_t* sV = stage + 2 * STAGE;
  float* sStat = (float*)(sV + (VLDS ? 128 * DV : 0));     // [2][2][2][64]: log2 of the row sums, r of a tile's maps
  float* sDiag = sStat + 2 * 256;                          // [8 waves][16 queries][48]: score gradients, row q shifted by q
  float* sAny = sDiag + (BIAS ? 8 * 768 : 0);              // [8]
  float* sB = sAny + 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, l31 = lane & 31, i16 = lane & 15, qd = (lane >> 4) & 1;
  const int kw = wave & 3, qh = wave >> 2;
  const int nkb = (a.Sk + 127) / 128;
  int blk, b, kh;
  block_id(nkb, a, a.Hkv, blk, b, kh);
  const int k0 = blk * 128 + kw * 32, key = k0 + l31, krow = min(key, a.Sk - 1);
  const int first = a.causal ? max(0, (blk * 128 - a.off)) / 64 : 0, nq64 = (a.Sq + 63) / 64;          // tiles of queries that see a key
  typedef Loader<D, 64, 8> QL;
  typedef Loader<DV, 64, 8> OL;
  QL ql(a.q + (long long)b * a.q_sb + (long long)kh * a.G * a.q_sh, a.q_ss, a.Sq - 1, wave, lane);
  OL ol(a.dO + ((size_t)b * a.Sq * a.H + kh * a.G) * DV, (long long)a.H * DV, a.Sq - 1, wave, lane);
  const float* stat = a.rvec + ((size_t)b * a.H + kh * a.G) * nq64 * MAPS * 128;
  auto request = [&](int qt, int buf) {
    const unsigned s = lds_at(stage) + buf * STAGE * 2;
#pragma unroll
    for (int m = 0; m < MAPS; m++) ql.tile(qt * 64, s + m * QT * 2, 2 * m * a.q_sm);
    ol.tile(qt * 64, s + MAPS * QT * 2, 0);
    if (wave == 7) dma16(stat + (size_t)qt * MAPS * 128, opaque(lane * 16), lds_at((bf16_t*)sStat) + buf * 1024);     // the tile's row statistics
  };
  auto request_two = [&]() {
    if (first < nq64) request(first, 0);
    if (first + 1 < nq64) request(first + 1, 1);
  };
  request_two();
  // lane = key in every product: whatever a masked key's row holds reaches only its own gradient rows, which are zeroed before the store
  const bool kok = key < a.seen && (!a.kvalid || a.kvalid[(size_t)b * a.mask_sb + krow] != 0);
  const bf16_t* vb_ = a.v + (long long)b * a.v_sb + (long long)kh * a.v_sh;
  s16x8 kf[MAPS][NK], vf[VLDS ? 1 : NV];
#pragma unroll
  for (int m = 0; m < MAPS; m++)
#pragma unroll
    for (int ks = 0; ks < NK; ks++)
      kf[m][ks] = *(const s16x8*)(a.k + (long long)b * a.k_sb + (long long)krow * a.k_ss + (long long)kh * a.k_sh + m * a.k_sm + 16 * ks + 8 * g);
  if constexpr (VLDS) load_tile<DV, 128, 8>(vb_, a.v_ss, blk * 128, a.Sk - 1, sV, wave, lane);
  else
#pragma unroll
    for (int ks = 0; ks < NV; ks++) vf[ks] = *(const s16x8*)(vb_ + (long long)krow * a.v_ss + 16 * ks + 8 * g);
  f32x16 dk[MAPS][ND], dv[NDV];
#pragma unroll
  for (int m = 0; m < MAPS; m++)
#pragma unroll
    for (int i = 0; i < ND; i++) zero(dk[m][i]);
#pragma unroll
  for (int i = 0; i < NDV; i++) zero(dv[i]);
  const int qoff = 2 * Tile<D>::off(l31, 8 * g), ooff = 2 * Tile<DV>::off(l31, 8 * g);               // bytes
  const int tq0 = 2 * Tile<D>::off(4 * g + (i16 >> 2), 16 * qd + 4 * (i16 & 3)), tq1 = 2 * Tile<D>::rows8(tq0 / 2);
  const int to0 = 2 * Tile<DV>::off(4 * g + (i16 >> 2), 16 * qd + 4 * (i16 & 3)), to1 = 2 * Tile<DV>::rows8(to0 / 2);
  int rlo, rhi;
  bias_window(a, blk * 128 - (a.Sq + 63) - a.off, blk * 128 + 127 - first * 64 - a.off, rlo, rhi);
  const int nk32 = (a.Sk + 31) / 32;
  // sums along the 63 diagonals of a 32 x 32 block in two passes of 16 queries: row q of a pass is written q entries to the left into 47 columns of
  // 48 (the last, and what no key falls on, stays zero for good); lane l collects relative position l - 31 of the block, column l - 16 of the first
  // pass and column l of the second
  float* diag = sDiag + wave * 768;
  if constexpr (BIAS) {
#pragma unroll
    for (int i = 0; i < 12; i++) diag[i * 64 + lane] = 0.f;
  }
  float drop = 1.f;
  const bool live = __builtin_amdgcn_ballot_w64(kok) != 0;
  if (lane == 0) sAny[wave] = live ? 1.f : 0.f;
  int nqt = max(0, nq64 - first);
  for (int hg = 0; hg < a.G; hg++) {
    const int h = kh * a.G + hg;
    const float lam = MAPS == 2 ? a.lam[h] : 0.f;
    float fl = 0.f, fr = 0.f, bl = 0.f, br = 0.f;          // sums and bias of the positions at and behind -R / +R
    float* part = nullptr;
    float top = 0.f;
    const int ntop = a.G * ((a.Sq + 31) / 32);
    const float* tops = a.amax + ((size_t)b * a.H + kh * a.G) * ((a.Sq + 31) / 32);
    const int at = HALF ? (int)opaque(lane) : 0;           // (opaque: no address kept over the loop)
    if (HALF && at < ntop) top = tops[at];                 // (used behind the wait that the bias needs anyway)
    if (hg > 0) {
      __syncthreads();                                     // the previous head's tiles, bias and statistics are read
      ql.base += 2 * a.q_sh; ol.base += 2 * DV; stat += (size_t)nq64 * MAPS * 128;
      if (nqt > 0) request_two();
    }
    if constexpr (BIAS) {
      load_bias(a, h, rlo, rhi, sB, tid, 512);
      if (k0 < a.Sk) {
        part = a.part + ((((size_t)h * a.B + b) * nk32 + k0 / 32) * 2 + qh) * a.gw;
        for (int i = lane; i < a.gw; i += 64) part[i] = 0.f;                    // (done before the first tile's wait)
      }
    }
    __syncthreads();
    if (hg == 0 && __builtin_amdgcn_readfirstlane(__float_as_int(sAny[0] + sAny[1] + sAny[2] + sAny[3])) == 0) nqt = 0;     // no key of the workgroup is valid
    if constexpr (BIAS) { bl = rlo <= -a.R ? sB[0] : 0.f; br = rhi >= a.R ? sB[rhi - rlo] : 0.f; }
    float lift = 1.f;                                      // from the largest entry of the group's dO
    if constexpr (HALF) {
      for (int i = at + 64; i < ntop; i += 64) top = fmaxf(top, tops[i]);
      lift = lift_of(top_of_wave(top));
      drop = inverse_of(lift);
    }
#pragma nounroll
    for (int n = 0; n < nqt; n++) {
      const int qt = first + n, buf = n & 1, q0 = qt * 64 + qh * 32;
      dma_wait();
      if (HALF && wave == 7 && lift != 1.f) {              // (the wave that requested the tile's statistics: r by the lift, too)
#pragma unroll
        for (int m = 0; m < MAPS; m++) sStat[buf * 256 + m * 128 + 64 + lane] *= lift;
      }
      __syncthreads();
      const bool req = n > 0 && n + 1 < nqt;
      const bool work = live && q0 < a.Sq && !(a.causal && q0 + 31 + a.off < k0);
      if (req && !work) request(qt + 1, buf ^ 1);
      if (work) {
        const bf16_t* sQ = stage + buf * STAGE + qh * 32 * D;
        const bf16_t* sO = stage + buf * STAGE + MAPS * QT + qh * 32 * DV;
        const float* st = sStat + buf * 256 + qh * 32;
        constexpr int NS = MAPS * NK, NP = NDV + MAPS * ND;
        f32x16 s[MAPS], dp;
        zero(dp);
#pragma unroll
        for (int m = 0; m < MAPS; m++) zero(s[m]);
        s16x8 fa[RA], fv[VLDS ? RV : 1];
        const unsigned qa = opaque(lds_at(sQ) + qoff), oa = DV == D ? qa : opaque(lds_at(sO) + ooff);
        constexpr int OB = DV == D ? MAPS * QT * 2 : 0;    // (one map: dO's tile is q's, one tile further)
        auto qorow = [&](int i) { return i < NS ? row_frag(qa, i % NK, i / NK * QT * 2) : row_frag(oa, i - NS, OB); };
        const unsigned va = VLDS ? opaque(lds_at(sV) + kw * 64 * DV + ooff) : 0;
        fill<NS + NV>(fa, qorow);
        fence();
#pragma unroll
        for (int i = 0; i < NS + NV; i++) {
          if (i < NS) s[i < NS ? i / NK : 0] = mma<HALF>(fa[i % RA], kf[i < NS ? i / NK : 0][i % NK], s[i < NS ? i / NK : 0]);
          else dp = mma<HALF>(fa[i % RA], VLDS ? fv[(i + RV - NS) % RV] : vf[VLDS || i < NS ? 0 : i - NS], dp);
          if (i + RA < NS + NV) fa[i % RA] = qorow(i + RA);
          if (VLDS && i + RV >= NS && i + RV < NS + NV) fv[(i + RV - NS) % RV] = row_frag(va, i + RV - NS, 0);
          fence();
        }
        if (req) request(qt + 1, buf ^ 1);                 // (while the score MFMAs run)
        const unsigned qt0 = opaque(lds_at(sQ) + tq0), qt1 = opaque(lds_at(sQ) + tq1);
        const unsigned ot0 = DV == D ? qt0 : opaque(lds_at(sO) + to0), ot1 = DV == D ? qt1 : opaque(lds_at(sO) + to1);
        // transposed fragments, 16 queries (hf) x 32 channels: dO's NDV blocks, then q's ND blocks of each map
        auto tcol = [&](int i) {
          const int hf = i / NP, c = i % NP;
          if (c < NDV) return col_frag(ot0, ot1, c, OB + 32 * hf * DV);
          return col_frag(qt0, qt1, (c - NDV) % ND, (c - NDV) / ND * QT * 2 + 32 * hf * D);
        };
        if constexpr (!VLDS) { fill<2 * NP>(fa, tcol); fence(); }                // (arrive under the softmax arithmetic)
        // register r <-> query q0 + (r & 3) + 8 (r >> 2) + 4 g, lane <-> key
        const int rb = k0 - q0 - a.off;                    // relative position of the block's first key and first query
        const bool right = BIAS && rb - 31 >= a.R, left = BIAS && rb + 31 <= -a.R, close = BIAS && !right && !left;
        float cc = a.c, cb = 0.f;
        if constexpr (BIAS) {
          if (right) cb = br;
          else if (left) cb = bl;
          else {
            const float* bp = sB + (rb + l31 - 4 * g - 27 - rlo);
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
              for (int e = 0; e < 4; e++) s[0][4 * j + e] = fmaf(s[0][4 * j + e], a.c, bp[27 - e - 8 * j]);
            }
            cc = 1.f;
          }
        }
        if (a.causal && q0 + a.off < k0 + 31) {            // key seen by queries at key - off and behind
          const int lim = key - q0 - a.off - 4 * g;
#pragma unroll
          for (int m = 0; m < MAPS; m++)
#pragma unroll
            for (int r = 0; r < 16; r++) if ((r & 3) + 8 * (r >> 2) < lim) s[m][r] = -INFINITY;
        }
        unsigned pp[8], pd[MAPS][8];
        float far = 0.f, dsum = 0.f;
#pragma unroll
        for (int ps = 0; ps < 2; ps++) {                   // 16 queries
          float ds0[8];
#pragma unroll
          for (int j = 2 * ps; j < 2 * ps + 2; j++) {
            f32x4 L[MAPS], r_[MAPS];
#pragma unroll
            for (int m = 0; m < MAPS; m++) {
              L[m] = *(const f32x4*)(st + m * 128 + 8 * j + 4 * g);
              r_[m] = *(const f32x4*)(st + m * 128 + 64 + 8 * j + 4 * g);
            }
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              float p[2], d0[2], d1[2];
#pragma unroll
              for (int u = 0; u < 2; u++) {
                const int r = 4 * j + e + u;
                p[u] = prob(fmaf(s[0][r], cc, cb - L[0][e + u]));
                d0[u] = p[u] * (HALF ? fmaf(dp[r], lift, -r_[0][e + u]) : dp[r] - r_[0][e + u]);
                if constexpr (BIAS) { far += d0[u]; ds0[r - 8 * ps] = d0[u]; }
                if constexpr (MAPS == 2) {
                  const float p2 = -lam * prob(fmaf(s[MAPS - 1][r], cc, -L[MAPS - 1][e + u]));
                  d1[u] = p2 * (HALF ? fmaf(dp[r], lift, -r_[MAPS - 1][e + u]) : dp[r] - r_[MAPS - 1][e + u]);
                  p[u] += p2;
                }
              }
              pp[2 * j + e / 2] = pack2<HALF>(p[0], p[1]);
              pd[0][2 * j + e / 2] = pack2<HALF>(d0[0], d0[1]);
              if constexpr (MAPS == 2) pd[MAPS - 1][2 * j + e / 2] = pack2<HALF>(d1[0], d1[1]);
            }
            if constexpr (MAPS == 2) fence();              // (the next statistics would not fit beside both maps)
          }
          if constexpr (BIAS) {
            if (close) {
              if (kok) {                                   // (a masked key's entries stay zero, too)
#pragma unroll
                for (int r = 0; r < 8; r++) diag[(4 * g + (r & 3) + 8 * (r >> 2)) * 47 + 15 + l31] = ds0[r];
              }
              __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
              __builtin_amdgcn_wave_barrier();
              float t[4] = {0.f, 0.f, 0.f, 0.f};
              const float* col = diag + (ps ? (lane < 47 ? lane : 47) : (lane >= 16 && lane < 63 ? lane - 16 : 47));
#pragma unroll
              for (int i = 0; i < 16; i++) t[i & 3] += col[i * 48];
              __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
              __builtin_amdgcn_wave_barrier();
              dsum += (t[0] + t[1]) + (t[2] + t[3]);
            }
          }
        }
        if constexpr (BIAS) {
          if constexpr (HALF) { far *= drop; dsum *= drop; }
          if (close) {
            const int rel = rb + lane - 31;                // (the wave's blocks are 64 queries apart: no other one has these positions)
            if (lane < 63) {
              if (rel >= a.R) fr += dsum;
              else if (rel <= -a.R) fl += dsum;
              else if (rel >= a.glo && rel < a.glo + a.gw) part[rel - a.glo] = dsum;
            }
          } else {
            far = kok ? far : 0.f;
            if (right) fr += far; else fl += far;
          }
        }
        fence();
        if constexpr (VLDS) { fill<2 * NP>(fa, tcol); fence(); }
        run<2 * NP>(fa, tcol, [&](int i, s16x8 f) {
          const int hf = i / NP, c = i % NP;
          if (c < NDV) dv[c] = mma<HALF>(f, frag(pp + 4 * hf), dv[c]);
          else dk[(c - NDV) / ND][(c - NDV) % ND] = mma<HALF>(f, frag(pd[(c - NDV) / ND] + 4 * hf), dk[(c - NDV) / ND][(c - NDV) % ND]);
        });
      }
    }
    if constexpr (BIAS) {
      if (part) {
        fl = wave_sum_dpp(fl); fr = wave_sum_dpp(fr);
        if (lane == 0) {                                   // (position -R / +R outside the reachable window: its sum is 0)
          if (-a.R >= a.glo && -a.R < a.glo + a.gw) part[-a.R - a.glo] = fl;
          if (a.R >= a.glo && a.R < a.glo + a.gw) part[a.R - a.glo] = fr;
        }
      }
    }
  }
  dma_wait();
  // the two waves of a key block meet: the upper one hands over its dk and takes the lower one's dv, one accumulator tile of all four pairs at a time
  constexpr int NT = MAPS * ND > NDV ? MAPS * ND : NDV;
  float* swap = (float*)smem;                              // [8 waves][16 registers][64 lanes] = 32 KB
#pragma unroll
  for (int i = 0; i < NT; i++) {
    __syncthreads();
    float* w = swap + wave * 1024 + lane;
    const float* o = swap + (wave ^ 4) * 1024 + lane;
    if (qh ? i < MAPS * ND : i < NDV) {
#pragma unroll
      for (int r = 0; r < 16; r++) w[r * 64] = qh ? dk[(i < MAPS * ND ? i : 0) / ND][(i < MAPS * ND ? i : 0) % ND][r] : dv[i < NDV ? i : 0][r];
    }
    __syncthreads();
    if (qh ? i < NDV : i < MAPS * ND) {
#pragma unroll
      for (int r = 0; r < 16; r++) {
        if (qh) dv[i < NDV ? i : 0][r] += o[r * 64]; else dk[(i < MAPS * ND ? i : 0) / ND][(i < MAPS * ND ? i : 0) % ND][r] += o[r * 64];
      }
    }
  }
  __syncthreads();
  if (k0 >= a.Sk) return;
  bf16_t* slab = stage + wave * SLAB;
  if (!qh) {
#pragma unroll
    for (int m = 0; m < MAPS; m++) {
#pragma unroll
      for (int i = 0; i < ND; i++) if (!kok) zero(dk[m][i]);
      store_rows<HALF, D>(dk[m], a.scale * drop, slab, lane, [=](int row) -> bf16_t* {
        return k0 + row < a.Sk ? a.dk + ((((size_t)b * a.Sk + k0 + row) * a.Hkv + kh) * MAPS + m) * D : nullptr; });
    }
  } else {
#pragma unroll
    for (int i = 0; i < NDV; i++) if (!kok) zero(dv[i]);
    store_rows<HALF, DV>(dv, 1.f, slab, lane, [=](int row) -> bf16_t* {
      return k0 + row < a.Sk ? a.dv + (((size_t)b * a.Sk + k0 + row) * a.Hkv + kh) * DV : nullptr; });
  }
}

// ------------------------------------------------------------------------------------------------
// backward of short rows (Sq, Sk <= 128, every head its own keys): one workgroup = one head of one sample at a time, everything in LDS, every operand
// read once.  8 waves: wave w has queries 32 (w & 3) .. and keys 64 (w >> 2) .. of the scores (lane <-> query); the two halves of a row meet in r, so
// that ds is formed from the exact row sums without a second pass.  dS and then P go through LDS in 16 bits to the products, whose 32 x 32 tiles of
// dq, dk and dv the waves share evenly.  Workgroups stay and fetch their next head under the stores.
// Bound by memory and by the phases' latency: q, k, v, dO in, dq, dk, dv out, 392 MB for 256 x 107 positions and 8 heads of 128: 77 us at the rate of a
// copy, 120 us measured (221 us by the two passes of longer rows).
// ------------------------------------------------------------------------------------------------
template <bool HALF, int D, int MAPS>
__global__ __launch_bounds__(512, MAPS * D == 32 ? 4 : 2) void maps_bwd_short_kernel(const MapArgs a) {
  clamp_keeps_nan();
  constexpr int DV = MAPS * D, KT = 128 * D, VT = 128 * DV, NK = D / 16, NV = DV / 16, NC = DV / 32, ND = D / 32, RA = DV == 32 ? 2 : 4;
  constexpr int NT = NC == 4 ? 2 : 1;                      // 32 x 32 tiles of dq, of dk and of dv per wave (DV = 32: of the first four waves)
  constexpr bool BIAS = MAPS == 1;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  // queries of a round of dS and of P, and dS's place: 128 channels: that of v; 64: its own; 32: that of the diagonals, so that two workgroups fit a CU
  constexpr int RS = DV == 32 || D < DV && DV == 128 ? 64 : 128, RP = DV == 32 ? 64 : 128;
  bf16_t* sK = (bf16_t*)smem;                              // [MAPS][128][D], then (with v's place) P
  bf16_t* sV = sK + VT;                                    // [128][DV]
  bf16_t* sQ = sV + VT;                                    // [MAPS][128][D]
  bf16_t* sO = sQ + VT;                                    // [128][DV]
  float* sR = (float*)(sO + VT);                           // [2 halves][MAPS][2][128] row sums of p dp and of p
  float* sX = sR + 4 * MAPS * 128;                         // [8 waves][768]: skewed score gradients as in the key kernel, then store slabs
  float* sRow = sX + 8 * 768;                              // [8 waves][96] bias gradient of the wave's 95 positions
  float* sEnd = sRow + (BIAS ? 8 * 96 : 0);                // [8 waves][2] its sums at and behind -R, +R
  float* sB = sEnd + (BIAS ? 64 : 0);                      // [256] bias by position
  float* sTop = sB + (BIAS ? 256 : 0);                     // [8 waves] largest entries of dO (fp16), to the next multiple of 256 bytes
  bf16_t* sS = DV == 128 ? sV : DV == 32 ? (bf16_t*)sX : (bf16_t*)(sTop + 64);                       // [MAPS][RS][128]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w4 = wave & 3, half = wave >> 2;
  auto request = [&](int b, int h, int lane) {
#pragma unroll
    for (int m = 0; m < MAPS; m++) {
      load_tile<D, 128, 8>(a.k + (long long)b * a.k_sb + (long long)h * a.k_sh + m * a.k_sm, a.k_ss, 0, a.Sk - 1, sK + m * KT, wave, lane);
      load_tile<D, 128, 8>(a.q + (long long)b * a.q_sb + (long long)h * a.q_sh + m * a.q_sm, a.q_ss, 0, a.Sq - 1, sQ + m * KT, wave, lane);
    }
    load_tile<DV, 128, 8>(a.v + (long long)b * a.v_sb + (long long)h * a.v_sh, a.v_ss, 0, a.Sk - 1, sV, wave, lane);
    load_tile<DV, 128, 8>(a.dO + ((size_t)b * a.Sq * a.H + h) * DV, (long long)a.H * DV, 0, a.Sq - 1, sO, wave, lane);
  };
  const int heads = a.B * a.H;
  auto sample = [&](int id, int& b, int& h) {              // XCD x takes a contiguous range of the (head, sample) pairs
    const int r = heads % 8, xcd = id % 8, v = heads / 8 * xcd + min(xcd, r) + id / 8;
    h = v / a.B;
    b = v - h * a.B;
  };
  int b, h, b_next, h_next, h_last = -1;
  sample(blockIdx.x, b, h);
  request(b, h, threadIdx.x & 63);
#pragma unroll 1
  for (int id = blockIdx.x; id < heads; id += gridDim.x, b = b_next, h = h_next) {
    // (opaque: nothing is kept ready over the loop)
    const int tid = opaque(threadIdx.x), lane = tid & 63, g = lane >> 5, l31 = lane & 31, i16 = lane & 15, qd = (lane >> 4) & 1;
    const int q0 = w4 * 32, q_raw = q0 + l31, qrow = min(q_raw, a.Sq - 1), key0 = half * 64;
    const bool live = q0 < a.Sq;
    float L[MAPS];
#pragma unroll
    for (int m = 0; m < MAPS; m++) {
      const float l = a.lse_in[(((size_t)b * a.H + h) * MAPS + m) * a.Sq + qrow];
      L[m] = q_raw >= a.Sq || l == -INFINITY ? ROW_OFF : l * LOG2E;
    }
    const float lam = MAPS == 2 ? a.lam[h] : 0.f;
    // masks of both halves of the keys
    const unsigned char* kv = a.kvalid ? a.kvalid + (size_t)b * a.mask_sb : nullptr;
    unsigned long long mask[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int key = 64 * i + lane;
      mask[i] = __builtin_amdgcn_ballot_w64(key < a.seen && (!kv || kv[min(key, a.Sk - 1)] != 0));
    }
    const int rlo = -(a.Sq - 1) - a.off, rhi = 127 - a.off;  // positions of the workgroup
    float* row = sRow + wave * 96;
    if constexpr (BIAS) {
      if (h != h_last) load_bias(a, h, rlo, rhi, sB, tid, 512);
      h_last = h;
    }
    dma_wait();
    __syncthreads();
    if ((mask[0] & mask[1]) != ~0ull) {                      // masked rows, and the repeated ones behind the last
#pragma unroll
      for (int i = 0; i < 2; i++)
        if (mask[i] != ~0ull) {
#pragma unroll
          for (int m = 0; m < MAPS; m++) clear_rows<D>(sK + m * KT + i * 64 * D, mask[i], 64, tid, 512);
          clear_rows<DV>(sV + i * 64 * DV, mask[i], 64, tid, 512);
        }
      __syncthreads();
    }
    // One workgroup per CU, all at the same place: the memory would idle under the products.  The next head's operands come to L2 meanwhile, a lane
    // touching a line of 128 bytes (144 -> 126 us for 256 x 107, 8 heads of 128; two workgroups per CU overlap by themselves, 106 us against 108).
    const bool more = id + (int)gridDim.x < heads;
    sample(more ? id + gridDim.x : id, b_next, h_next);
    int touched[2] = {0, 0};
    if constexpr (DV > 32) {
      constexpr int LK = MAPS * (D > 64 ? D / 64 : 1), LV = DV / 64;
      const int t = tid & 255, S = (half ? a.Sq : a.Sk) - 1, lk = t % LK, lv = t % LV;
      const bf16_t* x = half ? a.q + (long long)b_next * a.q_sb + (long long)h_next * a.q_sh : a.k + (long long)b_next * a.k_sb + (long long)h_next * a.k_sh;
      const bf16_t* y = half ? a.dO + ((size_t)b_next * a.Sq * a.H + h_next) * DV : a.v + (long long)b_next * a.v_sb + (long long)h_next * a.v_sh;
      touched[0] = *(const int*)(x + (long long)min(t / LK, S) * (half ? a.q_ss : a.k_ss) + (MAPS == 2 ? lk * (half ? a.q_sm : a.k_sm) : lk * 64));
      touched[1] = *(const int*)(y + (long long)min(t / LV, S) * (half ? (long long)a.H * DV : a.v_ss) + lv * 64);
    }
    const int koff = 2 * Tile<D>::off(l31, 8 * g), voff = 2 * Tile<DV>::off(l31, 8 * g);                // bytes
    const int toff0 = 2 * Tile<D>::off(4 * g + (i16 >> 2), 16 * qd + 4 * (i16 & 3)), toff1 = 2 * Tile<D>::rows8(toff0 / 2);
    const int ooff0 = 2 * Tile<DV>::off(4 * g + (i16 >> 2), 16 * qd + 4 * (i16 & 3)), ooff1 = 2 * Tile<DV>::rows8(ooff0 / 2);
    const int xoff0 = 2 * Tile<128>::off(4 * g + (i16 >> 2), 16 * qd + 4 * (i16 & 3)), xoff1 = 2 * Tile<128>::rows8(xoff0 / 2);
    // ---- scores of 32 queries x 2 blocks of 32 keys: p of every map, dP, and this half's row sums
    f32x16 p[MAPS][2], dp[2];
    float rs[MAPS], ps[MAPS];
#pragma unroll
    for (int m = 0; m < MAPS; m++) { rs[m] = ps[m] = 0.f; zero(p[m][0]); zero(p[m][1]); }
    zero(dp[0]); zero(dp[1]);
    bool on[2];                                              // the block has a (query, key) pair
#pragma unroll
    for (int kb = 0; kb < 2; kb++) on[kb] = live && (unsigned)(mask[half] >> (32 * kb)) != 0 && (!a.causal || min(q0 + 31, a.Sq - 1) + a.off >= key0 + 32 * kb);
    float top = 0.f, lift = 1.f;
    if (on[0] || on[1]) {
      s16x8 qf[MAPS][NK], of[NV];
#pragma unroll
      for (int m = 0; m < MAPS; m++)
#pragma unroll
        for (int ks = 0; ks < NK; ks++) qf[m][ks] = row_frag(lds_at(sQ + m * KT + q0 * D) + koff, ks, 0);
#pragma unroll
      for (int ks = 0; ks < NV; ks++) of[ks] = row_frag(lds_at(sO + q0 * DV) + voff, ks, 0);
      if constexpr (HALF) top = top_of_wave(amax_half(of));
      if constexpr (MAPS == 2) {
#pragma unroll
        for (int ks = NV / 4; ks < 3 * NV / 4; ks++) of[ks] = negated(of[ks]);
      }
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        if (!on[kb]) continue;
        const unsigned ka = opaque(lds_at(sK + (key0 + 32 * kb) * D) + koff), va = opaque(lds_at(sV + (key0 + 32 * kb) * DV) + voff);
        auto kvrow = [&](int i) { return i < NV ? row_frag(va, i, 0) : row_frag(ka, (i - NV) % NK, (i - NV) / NK * KT * 2); };
        s16x8 fa[RA];
        fill<NV + MAPS * NK>(fa, kvrow);
        fence();
        run<NV + MAPS * NK>(fa, kvrow, [&](int i, s16x8 x) {
          const int j = i < NV ? 0 : i - NV;
          if (MAPS == 2 && (i == NV / 4 || i == 3 * NV / 4)) dp[kb] = -dp[kb];
          if (i < NV) dp[kb] = mma<HALF>(x, of[i < NV ? i : 0], dp[kb]); else p[j / NK][kb] = mma<HALF>(x, qf[j / NK][j % NK], p[j / NK][kb]);
        });
        const unsigned mk = (unsigned)(mask[half] >> (32 * kb));
        const bool part = mk != ~0u || (a.causal && q0 + a.off < key0 + 32 * kb + 31);
#pragma unroll
        for (int m = 0; m < MAPS; m++) {
          float cc = a.c;
          if constexpr (BIAS) {
            const float* bp = sB + (key0 + 32 * kb - qrow - a.off + 4 * g - rlo);
#pragma unroll
            for (int r = 0; r < 16; r++) p[m][kb][r] = fmaf(p[m][kb][r], a.c, bp[(r & 3) + 8 * (r >> 2)]);
            cc = 1.f;
          }
          if (part) mask_scores(p[m][kb], mk, a.causal ? q_raw + a.off - key0 - 32 * kb : 32, g, -INFINITY);
#pragma unroll
          for (int r = 0; r < 16; r++) {
            p[m][kb][r] = prob(fmaf(p[m][kb][r], cc, -L[m]));
            rs[m] = fmaf(p[m][kb][r], dp[kb][r], rs[m]);
            ps[m] += p[m][kb][r];
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MAPS; m++) {
      rs[m] = half_sum(rs[m]); ps[m] = half_sum(ps[m]);
      sR[((half * MAPS + m) * 2 + g) * 128 + q_raw] = g ? ps[m] : rs[m];
    }
    if (HALF && lane == 0) sTop[wave] = top;
    __syncthreads();
    if constexpr (HALF) {
      const f32x4 x = *(const f32x4*)sTop, y = *(const f32x4*)(sTop + 4);
      lift = lift_of(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]))));
    }
#pragma unroll
    for (int m = 0; m < MAPS; m++) {                         // (divided by the row's sum of p, as in the query kernel)
      const float x = sR[(2 * m + 1) * 128 + q_raw] + sR[(2 * (MAPS + m) + 1) * 128 + q_raw];
      ps[m] = x == 0.f ? 0.f : 1.f / x;
      rs[m] = (sR[2 * m * 128 + q_raw] + sR[2 * (MAPS + m) * 128 + q_raw]) * ps[m];
      if (m) ps[m] *= -lam;
    }
    if (MAPS == 2 && half == 0 && live) {                    // lam's gradient: the wave's 32 rows, [H][B][32-row block]
      const float w = wave_sum_dpp(g == 0 && q_raw < a.Sq ? rs[MAPS - 1] : 0.f);
      if (lane == 0) a.part[((size_t)h * a.B + b) * ((a.Sq + 31) / 32) + w4] = w;
    }
    const float drop = inverse_of(lift);
    if constexpr (HALF) {
#pragma unroll
      for (int m = 0; m < MAPS; m++) rs[m] *= lift;
    }
    // ---- P and dS, packed as operands
    unsigned pp[2][8], pd[MAPS][2][8];
    float* diag = sX + wave * 768;
    if constexpr (BIAS) {
#pragma unroll
      for (int i = 0; i < 12; i++) diag[i * 64 + lane] = 0.f;
      row[lane] = 0.f;
      if (lane < 32) row[64 + lane] = 0.f;
    }
    float fl = 0.f, fr = 0.f;
#pragma unroll
    for (int kb = 0; kb < 2; kb++) {
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        float x[2], d[MAPS][2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          x[u] = p[0][kb][r + u] * ps[0];
          d[0][u] = x[u] * (HALF ? fmaf(dp[kb][r + u], lift, -rs[0]) : dp[kb][r + u] - rs[0]);
          if constexpr (MAPS == 2) {
            const float y = ps[MAPS - 1] * p[MAPS - 1][kb][r + u];
            d[MAPS - 1][u] = y * (HALF ? fmaf(dp[kb][r + u], lift, -rs[MAPS - 1]) : dp[kb][r + u] - rs[MAPS - 1]);
            x[u] += y;
          }
          if constexpr (BIAS) dp[kb][r + u] = d[0][u];
        }
        pp[kb][r / 2] = opaque(pack2<HALF>(x[0], x[1]));     // (opaque: formed here, by all waves at once, not in the rounds below)
#pragma unroll
        for (int m = 0; m < MAPS; m++) pd[m][kb][r / 2] = opaque(pack2<HALF>(d[m][0], d[m][1]));
      }
      if constexpr (BIAS) {
        if (on[kb]) {
          // sums along the block's diagonals as in the key kernel, keys and queries exchanged: lane l collects position l - 31 of the block
          float v = 0.f;
#pragma unroll
          for (int ps = 0; ps < 2; ps++) {                   // 16 keys
#pragma unroll
            for (int r = 0; r < 8; r++) diag[(4 * g + (r & 3) + 8 * (r >> 2)) * 49 + 31 - l31] = dp[kb][8 * ps + r];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const float* col = diag + (ps ? (lane >= 16 && lane < 63 ? lane - 16 : 47) : (lane < 47 ? lane : 47));
            float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 16; i++) t[i & 3] += col[i * 48];
            v += (t[0] + t[1]) + (t[2] + t[3]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
          }
          if constexpr (HALF) v *= drop;
          const int rel = key0 + 32 * kb - q0 - a.off + lane - 31;
          if (lane < 63) {
            if (rel >= a.R) fr += v;
            else if (rel <= -a.R) fl += v;
            else row[32 * kb + lane] += v;
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
    if constexpr (BIAS) {
      fl = wave_sum_dpp(fl); fr = wave_sum_dpp(fr);
      if (lane == 0) { sEnd[wave * 2] = fl; sEnd[wave * 2 + 1] = fr; }
    }
    // tiles of the wave: queries 32 qb, channels 32 qc of dq; keys 32 kb .. 32 + channels 32 kc .. of dk and dv
    auto qb = [&](int j) { return MAPS == 2 && NT == 2 ? 2 * j + half : NC == 1 ? wave : wave >> 1; };
    auto qc = [&](int j) { return MAPS == 2 && NT == 2 ? w4 : NC == 1 ? 0 : NT * (wave & 1) + j; };
    const int kblk = NC == 1 ? wave : wave >> 1, kc = NC == 1 ? 0 : NT * (wave & 1);
    const bool keys = 32 * kblk < a.Sk && kblk < 4;
    f32x16 dq[NT], dk[NT], dv[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) { zero(dq[j]); zero(dk[j]); zero(dv[j]); }
    // products over `n` queries: the left operand's channels `c`, the right one's keys, both transposed; chunks of 16, the next one's fragments on their
    // way under the MFMAs of the current one
    auto products = [&](f32x16 (&acc)[NT], unsigned l0, unsigned l1, int lrow, int c, unsigned r0, unsigned r1, int n) {
      const int n16 = (n + 15) / 16;
      auto load = [&](int i, s16x8& fb, s16x8 (&fa)[NT]) {
        fb = col_frag(r0 + i * 4096, r1 + i * 4096, kblk, 0);
#pragma unroll
        for (int j = 0; j < NT; j++) fa[j] = col_frag(l0 + i * lrow, l1 + i * lrow, c + j, 0);
      };
      auto mul = [&](const s16x8& fb, const s16x8 (&fa)[NT]) {
#pragma unroll
        for (int j = 0; j < NT; j++) acc[j] = mma<HALF>(fa[j], fb, acc[j]);
      };
      s16x8 fb0, fb1, fa0[NT], fa1[NT];
      load(0, fb0, fa0);
#pragma unroll 1
      for (int i = 0; i < n16; i += 2) {
        load(min(i + 1, n16 - 1), fb1, fa1);
        fence();
        mul(fb0, fa0);
        fence();
        load(min(i + 2, n16 - 1), fb0, fa0);
        fence();
        if (i + 1 < n16) mul(fb1, fa1);
      }
    };
    auto put = [&](bf16_t* tile, const unsigned (&x)[2][8], int row) {
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int j = 0; j < 4; j++) *(u32x2*)(tile + Tile<128>::off(row, key0 + 32 * kb + 8 * j + 4 * g)) = (u32x2){x[kb][2 * j], x[kb][2 * j + 1]};
    };
    // ---- dq and dk: dS of RS queries at a time
#pragma unroll 1
    for (int qr = 0; qr < a.Sq; qr += RS) {
      if (qr || DV == 32) __syncthreads();                   // the last round's dS, or the diagonals, are read (v: all waves have met in the row sums since)
      if (live && q0 >= qr && q0 < qr + RS) {
#pragma unroll
        for (int m = 0; m < MAPS; m++) put(sS + m * RS * 128, pd[m], q0 - qr + l31);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NT; j++) {
        if (32 * qb(j) < qr || 32 * qb(j) >= min(qr + RS, a.Sq)) continue;
        const int m = qc(j) / ND;
        const unsigned ra = opaque(lds_at(sS) + m * RS * 256 + (32 * qb(j) - qr) * 256 + 2 * Tile<128>::off(l31, 4 * g));
        const unsigned ta0 = opaque(lds_at(sK) + m * KT * 2 + toff0), ta1 = opaque(lds_at(sK) + m * KT * 2 + toff1);
        const int c = qc(j) % ND;
        // 16 keys a step, in the order in which a transposing read of k delivers them
        auto kcol = [&](int i) { return col_frag(ta0, ta1, c, i * 32 * D); };
        typedef const __attribute__((address_space(3))) s16x4* rptr;
        auto dsrow = [&](int i) { return cat4(*(rptr)(uintptr_t)(ra ^ (32 * i)), *(rptr)(uintptr_t)(ra ^ (32 * i) ^ 16)); };
        s16x8 fa[RA], fb[RA];
        fill<8>(fa, kcol);
        fill<8>(fb, dsrow);
        fence();
#pragma unroll
        for (int i = 0; i < 8; i++) {
          dq[j] = mma<HALF>(fa[i % RA], fb[i % RA], dq[j]);
          if (i + RA < 8) { fa[i % RA] = kcol(i + RA); fb[i % RA] = dsrow(i + RA); }
          fence();
        }
      }
      if (keys) {
        const int m = kc / ND;
        const unsigned qa = lds_at(sQ) + m * KT * 2 + qr * D * 2, sa = lds_at(sS) + m * RS * 256;
        products(dk, opaque(qa + toff0), opaque(qa + toff1), 32 * D, kc % ND, opaque(sa + xoff0), opaque(sa + xoff1), min(RS, a.Sq - qr));
      }
    }
    // ---- dv: P of RP queries at a time
#pragma unroll 1
    for (int qr = 0; qr < a.Sq; qr += RP) {
      __syncthreads();                                       // k, or the last round's P, is read
      if (live && q0 >= qr && q0 < qr + RP) put(sK, pp, q0 - qr + l31);
      __syncthreads();
      if (keys) {
        const unsigned oa = lds_at(sO) + qr * DV * 2;
        products(dv, opaque(oa + ooff0), opaque(oa + ooff1), 32 * DV, kc, opaque(lds_at(sK) + xoff0), opaque(lds_at(sK) + xoff1), min(RP, a.Sq - qr));
      }
    }
    __syncthreads();                                         // every tile is read: the next head's arrive under the stores
    asm volatile("" ::"v"(touched[0]), "v"(touched[1]));
    if (more) request(b_next, h_next, opaque(lane));
    if constexpr (BIAS) {
      if (tid < a.gw) {                                      // bias gradient: the waves' sums by position, in wave order
        const int rel = a.glo + tid;
        const int far = rel == a.R ? 1 : rel == -a.R ? 0 : -1;
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < 8; w++) {                        // (column 95 of a wave's positions stays 0)
          const int at = rel - (64 * (w >> 2) - 32 * (w & 3) - a.off - 31);
          x += far >= 0 ? sEnd[w * 2 + far] : sRow[w * 96 + ((unsigned)at < 95u ? at : 95)];
        }
        a.part[((size_t)h * a.B + b) * a.gw + tid] = x;
      }
    }
    // a row with a NaN has one at every key: not in a masked key's gradients
    const unsigned keep = -(unsigned)((mask[kblk >> 1 & 1] >> (32 * (kblk & 1) + l31)) & 1);
    bf16_t* slab = (bf16_t*)(sX + wave * 768);
    const float factor = HALF ? a.scale * drop : a.scale;
#pragma unroll
    for (int j = 0; j < NT; j++) {
      if (32 * qb(j) < a.Sq)
        store_rows<HALF, 32>(&dq[j], factor, slab, lane, [=](int r) -> bf16_t* {
          return 32 * qb(j) + r < a.Sq ? a.dq + (((size_t)b * a.Sq + 32 * qb(j) + r) * a.H + h) * DV + 32 * qc(j) : nullptr; });
      if (keys) {
        auto rows = [=](bf16_t* base) {
          return [=](int r) -> bf16_t* { return 32 * kblk + r < a.Sk ? base + (((size_t)b * a.Sk + 32 * kblk + r) * a.H + h) * DV + 32 * (kc + j) : nullptr; };
        };
        store_rows<HALF, 32>(&dk[j], factor, slab, lane, rows(a.dk), keep);
        store_rows<HALF, 32>(&dv[j], 1.f, slab, lane, rows(a.dv), keep);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// bias table's gradient: part [H][B x 32-key blocks x 2][gw] -> sums over a chunk of rows -> sums over the positions of a bucket.  Fixed order.
// 7 - 9 us and 6 us (9 us alone for 256 parts of 213 positions): 35 MB of parts for 24 x 601 keys, 12 heads, 801 positions.
// ------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void diag_sum_kernel(const float* part, long long rows, int gw, int chunk, float* out) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = blockIdx.x * 64 + lane, h = blockIdx.z;
  const long long r0 = (long long)blockIdx.y * chunk, r1 = r0 + chunk < rows ? r0 + chunk : rows;
  float x = 0.f;
  if (col < gw) {
#pragma unroll 4
    for (long long r = r0 + w; r < r1; r += 4) x += part[(h * rows + r) * gw + col];
  }
  red[w][lane] = x;
  __syncthreads();
  if (w == 0 && col < gw) out[((size_t)h * gridDim.y + blockIdx.y) * gw + col] = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}
// one workgroup per head: position sums in 64 bits (a position's rows shared by as many threads as the workgroup has to spare) and the positions' buckets
// to LDS, then a wave per bucket
__global__ __launch_bounds__(1024) void bucket_sum_kernel(const float* sums, int rows, int gw, int glo, const int* buckets, int R, int NB, int H, float* dtable) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem2[];
  double* sS = (double*)smem2;
  double* sG = sS + gw;
  int* sM = (int*)(sG + 1024);
  const int h = blockIdx.x, lane = threadIdx.x & 63, wide = (gw + 63) & ~63, groups = wide < 1024 ? 1024 / wide : 1, grp = threadIdx.x / wide;
  for (int i = threadIdx.x; i < gw; i += 1024) sM[i] = min(max(buckets[min(max(glo + i, -R), R) + R], 0), NB - 1);
  if (groups > 1) {
    const int i = threadIdx.x - grp * wide;
    double x = 0.;
    if (grp < groups && i < gw) {
#pragma unroll 16
      for (int c = grp; c < rows; c += groups) x += (double)sums[((size_t)h * rows + c) * gw + i];
    }
    sG[threadIdx.x] = x;
    __syncthreads();
    if (threadIdx.x < gw) {
      x = 0.;
      for (int n = 0; n < groups; n++) x += sG[n * wide + threadIdx.x];
      sS[threadIdx.x] = x;
    }
  } else {
    for (int i = threadIdx.x; i < gw; i += 1024) {
      double x = 0.;
#pragma unroll 8
      for (int c = 0; c < rows; c++) x += (double)sums[((size_t)h * rows + c) * gw + i];
      sS[i] = x;
    }
  }
  __syncthreads();
  for (int bk = threadIdx.x >> 6; bk < NB; bk += 16) {
    double x = 0.;
    for (int i = lane; i < gw; i += 64) x += sM[i] == bk ? sS[i] : 0.;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    if (lane == 0) dtable[(size_t)bk * H + h] = (float)x;
  }
}
// lam's gradient: minus the sum of a head's n partial row sums
__global__ __launch_bounds__(256) void lam_sum_kernel(const float* part, long long n, float* dlam) {
  __shared__ double red[4];
  const float* p = part + (size_t)blockIdx.x * n;
  double x = 0.;
#pragma unroll 8
  for (long long i = threadIdx.x; i < n; i += 256) x += (double)p[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  if (threadIdx.x == 0) dlam[blockIdx.x] = -(float)((red[0] + red[1]) + (red[2] + red[3]));
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
constexpr int MAX_REACH = 4095, MAX_BUCKETS = 8192;
constexpr size_t SWAP_BYTES = 8 * 32 * 72 * 2 > 8 * 16 * 64 * 4 ? 8 * 32 * 72 * 2 : 8 * 16 * 64 * 4;   // end of the key kernel: exchange, then store slabs
constexpr int DIAG_BYTES = 8 * 768 * 4;                   // skewed score gradients of the key kernel's waves

int check_attn(const uvtg_attn_dims* d, int maps) {
  if (!d) return -10;
  if (d->struct_size != (int)sizeof(uvtg_attn_dims)) return -18;
  if (d->B <= 0 || d->H <= 0 || d->Hkv <= 0 || d->Sq <= 0 || d->Sk <= 0) return -11;
  if (d->dtype != 0 && d->dtype != 1) return -30;
  if (d->H % d->Hkv) return -31;
  if (d->D != 32 && d->D != 64 && !(d->D == 128 && maps == 1)) return maps == 1 ? -5 : -32;
  if (!(d->scale > 0.f) || !isfinite(d->scale)) return -33;
  if (d->Sq > (1 << 24) || d->Sk > (1 << 24) || d->q_offset > (1 << 28) || d->q_offset < -(1 << 28)) return -34;
  if ((long long)d->B * d->H > 65535 * 64ll || (long long)d->B * d->Hkv > 65535) return -34;
  // a grid holds less than 2^32 threads: 512 for 128 rows of the key kernel
  if ((long long)((d->Sq + 127) / 128) * d->B * d->H >= 1 << 23 || (long long)((d->Sk + 127) / 128) * d->B * d->Hkv >= 1 << 23 || d->H > 65535) return -34;
  const long long st[] = {d->q_sb, d->q_ss, d->q_sh, d->k_sb, d->k_ss, d->k_sh, d->v_sb, d->v_ss, d->v_sh, maps == 2 ? d->q_sm : 0, maps == 2 ? d->k_sm : 0};
  for (long long s : st) if (s % 8 || s < 0) return -35;
  if (d->kvalid_sb < 0) return -35;
  if (d->q_ss > (1 << 26) || d->k_ss > (1 << 26) || d->v_ss > (1 << 26)) return -38;
  if (maps == 1) {
    if (d->reach < 1 || d->reach > MAX_REACH) return -36;
    if (d->n_buckets < 1 || d->n_buckets > MAX_BUCKETS) return -37;
  }
  return 0;
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Few rows: the split kernel, row blocks of 32 instead of 128 and the keys cut into ranges.  A row block of 128 takes about 5 + c Sk us on its own,
// c = 0.022 (one map of 128 channels) or 0.044 (two of 64), as long as there are workgroups for every CU; the split kernel with the join takes about
// 11 us + 0.08 us per 1000 keys of each of its row blocks.  Measured, row blocks against split, us (8 heads of 128; of two maps of 64):
//   1 x 128 queries: 512 keys 18, 13; 28, 16   2048 keys 52, 17; 95, 21   4 x 256: 512 keys 19, 24; 29, 30   4096 keys 98, 93; 185, 99
//   7 x 256, 1024 keys: 31, 54; 52, 63   32 x 128, 2048 keys: 63, 158; 101, 163   64 x 32, 1024 keys: 47, 48; 59, 52   64 x 32, 107 keys: 11, 11; 14, 16
// Under 512 keys the gain is 3 - 6 us at most, and is given up: there, above 32 queries, a sample's bits do not depend on how many others there are.  From
// 512 keys on, and for up to 32 queries, the number of ranges does depend on the batch, and with it the order of a row's sums.
// Up to 32 queries the two differ little and the heads of a group share a row block, so that their keys are read once.
struct SplitPlan { int use, hb, blocks, nsplit; };         // heads packed per row block, row blocks per key head, key ranges
SplitPlan plan_split(const uvtg_attn_dims* d, int maps) {
  SplitPlan p = {0, 1, 0, 1};
  const int G = d->H / d->Hkv;
  if (d->Sq < 32) {
    p.hb = 32 / d->Sq < G ? 32 / d->Sq : G;
    const int win = maps == 1 ? (2 * d->reach + 1 < d->Sk + d->Sq ? 2 * d->reach + 1 : d->Sk + d->Sq) : 0;
    while (p.hb > 1 && (long long)p.hb * win * 4 > 32768) p.hb--;
  }
  p.blocks = ((G + p.hb - 1) / p.hb) * ((p.hb * d->Sq + 31) / 32);
  const long long base = (long long)p.blocks * d->B * d->Hkv;
  p.use = d->Sq <= 32 || (base <= 128 * maps && d->Sk >= 512);
  if (!p.use) return p;
  // about two workgroups per CU, of at least 256 keys (8 heads of 128, ranges of at least 512, 256, 128 keys: 128 queries over 2048 18, 17, 20 us; one
  // query over 2048 15, 12, 11 us, over 8192 17, 15, 17 us)
  const long long want = (512 + base - 1) / base, most = d->Sk / 256;
  p.nsplit = (int)(want < most ? want : most);
  if (p.nsplit > 128) p.nsplit = 128;
  if (p.nsplit < 1) p.nsplit = 1;
  return p;
}
// relative positions that any (query, key) pair has, clamped to +-R
void reachable(const uvtg_attn_dims* d, int& glo, int& gw) {
  const int R = d->reach;
  auto cl = [R](long long x) { return (int)(x < -R ? -R : x > R ? R : x); };
  glo = cl(-(long long)(d->Sq - 1) - d->q_offset);
  gw = cl((long long)d->Sk - 1 - d->q_offset) - glo + 1;
}
size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
// whole rows in one workgroup: one pass over the operands (256 x 107, 8 heads of 128: 120 us against 221 us of the two passes)
bool short_rows(const uvtg_attn_dims* d) { return d->Sq <= 128 && d->Sk <= 128 && d->H == d->Hkv; }
struct BwdWs { size_t rvec, part, sums, amax, total; long long rows; int chunk, chunks, direct; };
BwdWs bwd_ws(const uvtg_attn_dims* d, int maps) {
  BwdWs w;
  w.rvec = 0;
  size_t at = align256((size_t)d->B * d->H * ((d->Sq + 63) / 64) * maps * 512 + 512);     // (a tile's statistics are fetched 1024 bytes at a time)
  w.amax = at;
  if (d->dtype && !short_rows(d)) at += align256((size_t)d->B * d->H * ((d->Sq + 31) / 32) * 4);
  w.part = at;
  if (maps == 1) {
    int glo, gw;
    reachable(d, glo, gw);
    w.rows = short_rows(d) ? d->B : (long long)d->B * ((d->Sk + 31) / 32) * 2;
    w.chunk = w.rows > 64 * 128 ? (int)((w.rows + 63) / 64) : 128;
    w.chunks = (int)((w.rows + w.chunk - 1) / w.chunk);
    // few parts (at most 64 per thread of the second kernel): without the first one
    w.direct = w.rows * ((gw + 63) & ~63) <= 64 * 1024;
    at += align256((size_t)d->H * w.rows * gw * 4);
    w.sums = at;
    if (!w.direct) at += align256((size_t)d->H * w.chunks * gw * 4);
  } else {
    w.rows = (long long)d->B * ((d->Sq + 31) / 32);
    w.chunk = w.chunks = w.direct = 0;
    at += align256((size_t)d->H * w.rows * 4);
    w.sums = at;
  }
  w.total = at;
  return w;
}

MapArgs map_args(const uvtg_attn_dims* d) {
  MapArgs a;
  memset(&a, 0, sizeof(a));
  a.q_sb = d->q_sb; a.q_ss = d->q_ss; a.q_sh = d->q_sh; a.q_sm = d->q_sm;
  a.k_sb = d->k_sb; a.k_ss = d->k_ss; a.k_sh = d->k_sh; a.k_sm = d->k_sm;
  a.v_sb = d->v_sb; a.v_ss = d->v_ss; a.v_sh = d->v_sh; a.mask_sb = d->kvalid_sb;
  a.B = d->B; a.H = d->H; a.Hkv = d->Hkv; a.G = d->H / d->Hkv; a.Sq = d->Sq; a.Sk = d->Sk; a.NB = d->n_buckets; a.R = d->reach;
  a.off = d->q_offset; a.causal = d->causal != 0; a.seen = a.causal ? max(0, min(d->Sk, d->Sq + d->q_offset)) : d->Sk; a.scale = d->scale; a.c = d->scale * LOG2E;
  return a;
}

// entries of the bias window of a workgroup of `rows` rows
size_t window_bytes(const uvtg_attn_dims* d, int maps, int rows, long long other) {
  if (maps == 2) return 0;
  const long long w = 2ll * (d->reach + PAD) + 1, most = other + rows + 192;
  return (size_t)(w < most ? w : most) * 4;
}

// LDS of the kernels that walk key tiles: two stages (or, at the end, the waves' store slabs), masks, bias window
template <int D, int MAPS> size_t lds_rows(const uvtg_attn_dims* d) {
  const size_t tiles = 2 * 64 * 2 * MAPS * D * 2, slabs = 4 * SLAB * 2;
  return (tiles > slabs ? tiles : slabs) + WIN * 8 + window_bytes(d, MAPS, 128, d->Sk);
}
template <bool HALF, int D, int MAPS> int run_fwd(const uvtg_attn_dims* d, MapArgs a, hipStream_t s) {
  constexpr int DV = MAPS * D;
  const SplitPlan p = plan_split(d, MAPS);
  if (!p.use) {
    hipLaunchKernelGGL((maps_fwd_kernel<HALF, D, MAPS>), dim3((unsigned)((d->Sq + 127) / 128) * d->H * d->B), dim3(256), (lds_rows<D, MAPS>(d)), s, a);
    UVTG_CHECK_LAUNCH();
    return 0;
  }
  a.hb = p.hb; a.nsplit = p.nsplit;
  constexpr size_t tiles = 4 * 32 * (MAPS * D + DV) * 2, sums = 4 * DV * 32 * 4;
  const long long win = MAPS == 1 ? (2ll * d->reach + 1 < d->Sk + d->Sq + 64ll ? 2ll * d->reach + 1 : d->Sk + d->Sq + 64ll) : 0;
  const size_t lds = (tiles > sums ? tiles : sums) + 2 * WIN * 4 + MAPS * 2 * 128 * 4 + (size_t)p.hb * win * 4;
  hipLaunchKernelGGL((maps_fwd_split_kernel<HALF, D, MAPS>), dim3(p.blocks, p.nsplit, d->B * d->Hkv), dim3(256), lds, s, a);
  UVTG_CHECK_LAUNCH();
  if (p.nsplit > 1) {
    hipLaunchKernelGGL((maps_join_kernel<HALF, D, MAPS>), dim3((unsigned)(((long long)d->B * d->H * d->Sq + 3) / 4)), dim3(256), 0, s, a);
    UVTG_CHECK_LAUNCH();
  }
  return 0;
}
template <bool HALF, int D, int MAPS> int run_bwd(const uvtg_attn_dims* d, MapArgs a, float* dsum, char* ws, hipStream_t s) {
  constexpr int DV = MAPS * D;
  const BwdWs w = bwd_ws(d, MAPS);
  a.rvec = (float*)(ws + w.rvec);
  a.part = (float*)(ws + w.part);
  a.amax = (float*)(ws + w.amax);
  if (MAPS == 1) reachable(d, a.glo, a.gw);
  if (short_rows(d)) {
    constexpr size_t lds = 4 * 128 * DV * 2 + 4 * MAPS * 512 + DIAG_BYTES + (MAPS == 1 ? 8 * 96 * 4 + 256 + 1024 : 0) + 256 + (DV == 64 ? MAPS * 128 * 256 : 0);
    // workgroups that stay: one per CU, two where registers allow
    const int wgs = (DV == 32 ? 2 : 1) * persistent_cus();
    hipLaunchKernelGGL((maps_bwd_short_kernel<HALF, D, MAPS>), dim3(d->H * d->B < wgs ? d->H * d->B : wgs), dim3(512), lds, s, a);
    UVTG_CHECK_LAUNCH();
  } else {
    hipLaunchKernelGGL((maps_bwd_q_kernel<HALF, D, MAPS>), dim3((unsigned)((d->Sq + 127) / 128) * d->H * d->B), dim3(256), (lds_rows<D, MAPS>(d)), s, a);
    UVTG_CHECK_LAUNCH();
    const size_t need_k = 2 * 64 * (MAPS * D + DV) * 2 + (DV == 128 ? 128 * DV * 2 : 0) + 2 * 1024 + (MAPS == 1 ? DIAG_BYTES : 0) + 32 + window_bytes(d, MAPS, 128, d->Sq);
    const size_t lds_k = need_k > SWAP_BYTES ? need_k : SWAP_BYTES;
    hipLaunchKernelGGL((maps_bwd_k_kernel<HALF, D, MAPS>), dim3((unsigned)((d->Sk + 127) / 128) * d->Hkv * d->B), dim3(512), lds_k, s, a);
    UVTG_CHECK_LAUNCH();
  }
  if (!dsum) return 0;
  if (MAPS == 1) {
    float* sums = (float*)(ws + w.sums);
    if (!w.direct) {
      hipLaunchKernelGGL(diag_sum_kernel, dim3((a.gw + 63) / 64, w.chunks, d->H), dim3(256), 0, s, a.part, w.rows, a.gw, w.chunk, sums);
      UVTG_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(bucket_sum_kernel, dim3(d->H), dim3(1024), (size_t)a.gw * 12 + 1024 * 8, s, w.direct ? a.part : sums, w.direct ? (int)w.rows : w.chunks, a.gw, a.glo,
                       a.buckets, a.R, a.NB, a.H, dsum);
  } else hipLaunchKernelGGL(lam_sum_kernel, dim3(d->H), dim3(256), 0, s, a.part, w.rows, dsum);
  UVTG_CHECK_LAUNCH();
  return 0;
}

template <int MAPS> int dispatch_fwd(const uvtg_attn_dims* d, const MapArgs& a, hipStream_t s) {
#define GO(D_) if (d->D == D_) return d->dtype ? run_fwd<true, D_, MAPS>(d, a, s) : run_fwd<false, D_, MAPS>(d, a, s);
  GO(32) GO(64)
  if constexpr (MAPS == 1) { GO(128) }
#undef GO
  return -5;
}
template <int MAPS> int dispatch_bwd(const uvtg_attn_dims* d, const MapArgs& a, float* dsum, char* ws, hipStream_t s) {
#define GO(D_) if (d->D == D_) return d->dtype ? run_bwd<true, D_, MAPS>(d, a, dsum, ws, s) : run_bwd<false, D_, MAPS>(d, a, dsum, ws, s);
  GO(32) GO(64)
  if constexpr (MAPS == 1) { GO(128) }
#undef GO
  return -5;
}

}  // namespace

extern "C" size_t uvtg_attn_ws_bytes(const uvtg_attn_dims* d, int maps, int backward) {
  if ((maps != 1 && maps != 2) || check_attn(d, maps)) return 0;
  if (backward) return bwd_ws(d, maps).total;
  const SplitPlan p = plan_split(d, maps);
  return p.use && p.nsplit > 1 ? (size_t)d->B * d->H * d->Sq * p.nsplit * maps * (maps * d->D + 2) * 4 : 0;
}
extern "C" int uvtg_relpos_attention_fwd(const uvtg_attn_dims* d, const void* q, const void* k, const void* v, const float* table, const int* buckets,
                                         const unsigned char* kvalid, void* o, float* lse, void* ws, uvtg_stream_t st) {
  if (int e = check_attn(d, 1)) return e;
  if (!q || !k || !v || !table || !buckets || !o || (!ws && uvtg_attn_ws_bytes(d, 1, 0))) return -20;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o)) return -35;
  MapArgs a = map_args(d);
  a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.table = table; a.buckets = buckets; a.kvalid = kvalid;
  a.out = (bf16_t*)o; a.lse = lse; a.acc = (float*)ws;
  return dispatch_fwd<1>(d, a, (hipStream_t)st);
}
extern "C" int uvtg_relpos_attention_bwd(const uvtg_attn_dims* d, const void* q, const void* k, const void* v, const float* table, const int* buckets,
                                         const unsigned char* kvalid, const void* o, const float* lse, const void* dO, void* dq, void* dk, void* dv,
                                         float* dtable, void* ws, uvtg_stream_t st) {
  if (int e = check_attn(d, 1)) return e;
  if (!q || !k || !v || !table || !buckets || !o || !lse || !dO || !dq || !dk || !dv || !ws) return -20;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(dO) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv)) return -35;
  MapArgs a = map_args(d);
  a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.table = table; a.buckets = buckets; a.kvalid = kvalid;
  a.o = (const bf16_t*)o; a.lse_in = lse; a.dO = (const bf16_t*)dO; a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv;
  return dispatch_bwd<1>(d, a, dtable, (char*)ws, (hipStream_t)st);
}
extern "C" int uvtg_diff_attention_fwd(const uvtg_attn_dims* d, const void* q, const void* k, const void* v, const float* lam, const unsigned char* kvalid,
                                       void* o, void* o2, float* lse, void* ws, uvtg_stream_t st) {
  if (int e = check_attn(d, 2)) return e;
  if (!q || !k || !v || !lam || !o || (!ws && uvtg_attn_ws_bytes(d, 2, 0))) return -20;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(o2)) return -35;
  MapArgs a = map_args(d);
  a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.lam = lam; a.kvalid = kvalid;
  a.out = (bf16_t*)o; a.out2 = (bf16_t*)o2; a.lse = lse; a.acc = (float*)ws;
  return dispatch_fwd<2>(d, a, (hipStream_t)st);
}
extern "C" int uvtg_diff_attention_bwd(const uvtg_attn_dims* d, const void* q, const void* k, const void* v, const float* lam, const unsigned char* kvalid,
                                       const void* o, const void* o2, const float* lse, const void* dO, void* dq, void* dk, void* dv, float* dlam, void* ws,
                                       uvtg_stream_t st) {
  if (int e = check_attn(d, 2)) return e;
  if (!q || !k || !v || !lam || !o || !o2 || !lse || !dO || !dq || !dk || !dv || !ws) return -20;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(o2) || !aligned16(dO) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
    return -35;
  MapArgs a = map_args(d);
  a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.lam = lam; a.kvalid = kvalid;
  a.o = (const bf16_t*)o; a.o2 = (const bf16_t*)o2; a.lse_in = lse; a.dO = (const bf16_t*)dO; a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv;
  return dispatch_bwd<2>(d, a, dlam, (char*)ws, (hipStream_t)st);
}
