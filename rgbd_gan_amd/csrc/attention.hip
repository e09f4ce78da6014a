// Attention over the tokens of a pixel grid with a learned relative position bias, forward and backward.
//
//   s_ij = scale q_i . k_j;  cap > 0: s_ij = cap tanh(s_ij / cap);  s_ij += table[h][bucket(offset of i from j)];
//   keys j >= lengths[b] do not exist;  p = softmax over the keys;  o_i = sum_j p_ij v_j, and 0 for a row without keys.
//   ds = p (dp - delta), dp_ij = do_i . v_j, delta_i = do_i . o_i;  dtable[h][u] = sum of ds over the pairs of bucket u;
//   through the cap ds (1 - tanh^2);  dq = scale ds k, dk = scale ds^T q, dv = p^T do.
//
// Token t sits at row t / cols, column t % cols of the grid.  With P(t) = t + (cols - 1) (t / cols) the offset (dy, dx) of a
// pair is the single number P(i) - P(j), so the bias of a tile of scores is a short run of the (2 rows - 1)(2 cols - 1) offsets.
//
// Matrix products run on v_mfma_f32_32x32x16_bf16.  Scores are computed TRANSPOSED (keys x queries: the keys are the A
// operand), so a lane holds one query and 16 of its keys: row maximum and sum need one exchange between lane l and l + 32,
// the rescaling of the output is one factor a lane, and the 16 probabilities are, packed to bf16, the B operand of the second
// product as they stand (its K order follows the accumulator's: 4 keys of one half, 4 of the other), while the A operand comes
// out of LDS through the transposing read.  Probabilities and score gradients are rounded to bf16 as operands of these products, which
// makes o, dq, dk and dv two bf16 roundings off where arithmetic in fp32 would be one (2.4e-3 against 1.7e-3 in relative 2-norm); o's
// probabilities go in as three terms, with fp32's digits, where the table learns (FINE) and for few query rows.  Maxima, sums,
// statistics and the table's gradient stay in fp32.
//
// Times below: us on one MI355X, where a 2 GB copy reaches 5.05 TB/s and an 8192^3 bf16 product of the library 1130 TFLOP/s.  "32 px":
// 32 samples of a 32x32 map, 4 heads of 64; "64 px": 8 of 64x64, 2 heads of 64, capped scores; "128 px": 4 of 128x128, one head of 64;
// "line": 2 of 4096 tokens, 4 query heads on 2 of 128.
#include <type_traits>

#include "common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
// rows of a streamed tile (keys forward and in dq, queries in dk / dv): two buffers of two operands are 32 KB of LDS at head sizes 64 and
// 128, 16 KB at 32
constexpr int kt_of(int D) { return D == 128 ? 32 : 64; }
constexpr int BLK = 128;                  // rows a workgroup owns: 4 waves x 32
constexpr int WIN_PAD = 4;
// LDS bytes for the window: with the tiles (32 KB) three workgroups a compute unit forward, two of dq with its blocks (69 KB)
constexpr int WIN_FWD = 20480, WIN_DQ = 10240;
constexpr float NO_ROW = 0x1p100f;          // log2-sum-exp of a row that is not there: p = exp2(x - 2^100) = 0 for every finite x
constexpr float NEG_INF = -__builtin_inff();
// Where a row's sum of probabilities may lie before the forward pass moves its reference.  The output is summed as p v before the division by that
// sum, so a sum of S takes S from the range of |v| that fp32 can add up.  Up to 2^24, what the largest number of keys reaches next to a
// reference at their maximum, finite outputs stay finite for |v| below 1e29 (runs of keys joined included), and scores of order 1 over 2^14
// keys (a sum near 2^15) never leave it.  Down to 2^-40 the products keep bf16's digits (the matrix unit keeps numbers below 2^-126) for
// |v| above 1e-27.  A row that has moved pays a subtraction a score, 128 px 385 us against 357: a bias that falls by 50 with the distance puts the
// first keys of most rows below 2^-40, one that falls by 20 does not (but below 2^-10: 384).
constexpr float SUM_LOW = 0x1p-40f, SUM_HIGH = 0x1p24f;

struct AttnArgs {
    const unsigned short *q, *k, *v, *d_o, *o, *o_lo;
    unsigned short *out, *out_lo, *dq, *dk, *dv;
    float *lse, *delta, *part, *dtable;
    const float* table; const int* map; const int* lengths;
    int64_t q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh;
    int64_t dq_sb, dq_sl, dq_sh, dk_sb, dk_sl, dk_sh, dv_sb, dv_sl, dv_sh;
    int B, H, Hkv, rep, Lq, Lk;
    int rows, cols, pos_cols, q_start, n_buckets;
    int kt, n_qb, n_kb, n_kt, seg_tiles, win_bytes, splits;
    float* runs; int64_t run_floats;      // output or dq in runs of keys: their fp32 sums (splits, B, Lq, H, D)
    int span;                             // width of a row of bias-gradient partials (distances a workgroup meets)
    float scale, cap;
};

// ---- positions.  `cols` here is pos_cols: the grid's columns, or a number no token reaches where the grid is a single row.
__device__ __forceinline__ int pos_of(int t, int cols) { return t + (cols - 1) * (t / cols); }

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// ---- LDS tiles: `rows` x D bf16, 16-byte chunks permuted so that both ways of reading a tile spread over the 64 banks: the
//      row-major 16-byte reads of 32 consecutive rows and the transposing 8-byte reads of 4 consecutive rows x 64 bytes.
template <int D> __device__ __forceinline__ int swz(int row) {
    if (D == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    if (D == 64) return (((row >> 1) & 1) << 2) | (((row >> 2) & 1) << 1) | ((row >> 3) & 1);
    return (row >> 2) & 3;
}

template <int D> struct Frags {
    int rb;                               // row-major fragment: byte address of (row lane & 31, chunk lane / 32)
    int tb;                               // transposed fragment: (row 4 (lane / 32) + q, columns 16 mblk + 4 p)
    __device__ __forceinline__ Frags(int lane) {
        const int r = lane & 31, half = lane >> 5;
        rb = r * (2 * D) + ((half ^ swz<D>(r)) << 4);
        const int q = (lane & 15) >> 2, p = lane & 3, mblk = (lane >> 4) & 1;
        const int row = 4 * half + q;
        tb = row * (2 * D) + (((mblk * 2 + (p >> 1)) ^ swz<D>(row)) << 4) + (p & 1) * 8;
    }
    // rows row0 .. row0 + 31 (row0 a multiple of 32), columns 16 ks + 8 half + 0..7
    __device__ __forceinline__ bf16x8 row(const char* tile, int row0, int ks) const {
        return *reinterpret_cast<const bf16x8*>(tile + row0 * (2 * D) + (rb ^ (ks << 5)));
    }
    // column 32 dblk + (lane & 31) of rows row0 + {4 half + 0..3, 8 + 4 half + 0..3} (row0 a multiple of 16)
    __device__ __forceinline__ bf16x8 col(const char* tile, int row0, int dblk) const {
        constexpr int EX = D == 64 ? 16 : 32;        // what row + 8 changes in swz
        const char* t = tile + row0 * (2 * D);
        const s16x4 a = tr(t + (tb ^ (dblk << 6)));
        const s16x4 b = tr(t + 16 * D + (tb ^ EX ^ (dblk << 6)));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    static __device__ __forceinline__ s16x4 tr(const char* p) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(const_cast<char*>(p)));
    }
};

// One tile of KT rows x D from global memory straight into LDS (global_load_lds: no registers, 16 bytes a lane, a wave's 1 KB in a
// row; the permutation of the chunks is in the source addresses).  Rows at or beyond `valid` repeat the last valid one: whatever
// memory holds there, a NaN included, is never read.  M0 carries the LDS address; nothing the compiler emits for gfx950 reads it.
// The caller waits with dma_wait() before the barrier that publishes the tile.
template <int D, int KT> struct Dma {
    static constexpr int CH = D / 8, NP = KT * CH / 256;
    unsigned off[NP];                     // bytes from the tile's first row
    int64_t step;                         // bytes of KT rows
    const char* base;
    int valid;                            // rows from the next tile's first on
    unsigned lds;
    __device__ __forceinline__ void offsets(int64_t sl, int rows) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int pc = threadIdx.x + 256 * i, row = pc / CH, ch = (pc % CH) ^ swz<D>(row);
            off[i] = (unsigned)min(row, rows - 1) * (unsigned)(2 * sl) + 16 * ch;
        }
    }
    __device__ __forceinline__ void init(const unsigned short* p, int64_t sl, int rows, const char* tile) {
        base = reinterpret_cast<const char*>(p);
        step = 2 * KT * sl;
        valid = rows;
        lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)tile + 1024 * wave_id();
        offsets(sl, rows);
    }
    // the next tile, `buf_bytes` behind the first buffer
    __device__ __forceinline__ void next(int64_t sl, int buf_bytes) {
        if (valid < KT) offsets(sl, valid);
        const uint64_t b = (uint64_t)(uintptr_t)base;                 // (uniform by construction; said so where the compiler lost it)
        const uint64_t from = (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)b);
        const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane((int)lds) + buf_bytes;
#pragma unroll
        for (int i = 0; i < NP; ++i)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                         :: "s"(to + 4096 * i), "v"(off[i]), "s"(from) : "memory", "m0");
        base += step;
        valid -= KT;
    }
};
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ f32x16 mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8 pack8(const f32x16& v, int i0) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(v[i0 + 2 * i], v[i0 + 2 * i + 1]);
    return __builtin_bit_cast(bf16x8, o);
}
__device__ __forceinline__ float other_half_max(float x) { return fmaxf(x, __shfl_xor(x, 32, 64)); }
__device__ __forceinline__ float other_half_sum(float x) { return x + __shfl_xor(x, 32, 64); }

// LDS operations of one wave complete in order; this keeps the compiler to that order where lanes read what others wrote
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The loads of `f` are waited for here: left to the first use, inside the loop, that wait would also wait for the loop's own loads
// of the next tile (one counter, in order) -- which doubled the time of a tile.
template <int N> __device__ __forceinline__ void arrived(bf16x8 (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        u32x4 v = __builtin_bit_cast(u32x4, f[i]);
        asm volatile("" : "+v"(v));
        f[i] = __builtin_bit_cast(bf16x8, v);
    }
}

// What rounding a value to bf16 drops, in 16 bits and all of it: fp32's low half.  hi is the nearest, so the value's bits are hi * 2^16 +
// the low half read as a signed number; a tie goes to the even hi, and one that went down is stored a unit lower (2^-24 of the value).
__device__ __forceinline__ unsigned low_half(float v) {
    const unsigned b = __float_as_uint(v);
    return (b & 0x1ffffu) == 0x8000u ? 0x7fffu : b & 0xffffu;
}
__device__ __forceinline__ float whole(unsigned hi, unsigned lo) { return __uint_as_float((hi << 16) + (unsigned)(int)(short)lo); }

// tanh of 16 values.  Below 0.5 an odd polynomial (least squares on Chebyshev nodes, relative error 1.1e-7: there the quotient
// form would lose digits by cancellation, and capped scores mostly lie there); beyond it 1 - 2 / (e^2x + 1).
__device__ __forceinline__ float tanh_small(float x) {
    const float u = x * x;
    float r = 0.017141319811344147f;
    r = r * u + -0.05298924073576927f;
    r = r * u + 0.13324828445911407f;
    r = r * u + -0.3333307206630707f;
    r = r * u + 1.f;
    return r * x;
}
__device__ __forceinline__ void tanh16(f32x16& v, float f) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) { v[i] *= f; top = fmaxf(top, fabsf(v[i])); }
    if (!__any(top >= 0.5f)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = tanh_small(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(2.f * LOG2E * v[i]);
            const float t = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
            v[i] = fabsf(v[i]) < 0.5f ? tanh_small(v[i]) : t;
        }
    }
}

// The workgroup's place: consecutive ids go round the 8 XCDs, so give each XCD a run of neighbours (they share keys and values).
__device__ __forceinline__ int xcd_run(int id, int total) {
    const int q = total >> 3, r = total & 7, x = id & 7;
    return x * q + min(x, r) + (id >> 3);
}

// A bias in the exponent of 2.  One at or below -1e30 (a mask written as the type's lowest number) is -inf: a row that has nothing else
// would otherwise carry a log-sum-exp in which the sum is below the last digit, and its gradients would be wrong.
__device__ __forceinline__ float in_log2(float bias) { return bias <= -1e30f ? NEG_INF : bias * LOG2E; }

// ---- the bias of a run of tiles (a segment), in LDS.  The workgroup's own rows are tokens at places own_first .. own_last, the
//      streamed ones begin at other_first and span `span` places.  Entry j is the offset whose place grows with the streamed row, so a
//      lane reads upwards; SIGN +1: the streamed rows are queries.  Values are kept times log2(e): the softmax runs on exp2.
template <int SIGN>
__device__ __forceinline__ void stage_window(float* win, const AttnArgs& a, int h, int own_first, int own_last, int other_first, int span) {
    const int n = (own_last - own_first) + span + 1 + WIN_PAD;
    const int c0 = (2 * a.cols - 1) * (a.rows - 1) + a.cols - 1, size = (2 * a.cols - 1) * (2 * a.rows - 1);
    const float* row = a.table + (int64_t)h * a.n_buckets;
    const int base = SIGN > 0 ? other_first - own_last + c0 : own_last - other_first + c0;
    for (int j = threadIdx.x; j < n; j += 256) {
        const int e = base + SIGN * j;                                // beyond the map: a streamed row that is no token
        const int u = min(max(a.map[min(max(e, 0), size - 1)], 0), a.n_buckets - 1);
        win[j] = e >= 0 && e < size ? in_log2(row[u]) : 0.f;
    }
}

// Where in the window the streamed rows of a block of 32 lie, in bytes, from the segment's first on.
// BIAS 2 (regular grids): a block's four groups of 8 rows lie at distances that are the same for every block, the rows of a half of
// a group are neighbours, and from block to block the place grows by a fixed step (rows of the grid divide 32) or by 32 and, at the
// end of a row of the grid, by columns - 1 more: a handful of scalars.  BIAS 1 (any grid): a table of the segment's rows.
template <int BIAS> struct Places {
    int blk, x, step, wrap, cols, g[4];
    __device__ __forceinline__ void init(const AttnArgs& a, int first) {
        if (BIAS != 2) return;
        const bool narrow = a.rows > 1 && a.cols < 32;
        blk = 0;
        cols = a.pos_cols;
        x = narrow ? 0 : first % cols;
        step = 4 * (narrow ? 32 + 32 / a.cols * (a.cols - 1) : 32);
        wrap = narrow ? 0 : 4 * (cols - 1);
        if (narrow) cols = 1 << 30;
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = 4 * (8 * i + (narrow ? (a.cols - 1) * (8 * i / a.cols) : 0));
    }
    // bytes from a lane's own place: rows 4 half .. 4 half + 3 of a group
    static __device__ __forceinline__ int half_off(const AttnArgs& a, int half) {
        return BIAS == 2 ? 4 * (4 * half + (a.rows > 1 && a.cols == 4 ? 3 * half : 0)) : 0;
    }
    __device__ __forceinline__ void next() {
        if (BIAS != 2) return;
        blk += step;
        x += 32;
        if (x >= cols) { x -= cols; blk += wrap; }
    }
    // the table of BIAS 1: places of the segment's rows (tokens first .. first + n - 1, repeated from the last that exists on)
    static __device__ __forceinline__ void table(int* at, const AttnArgs& a, int first, int n, int last) {
        if (BIAS != 1) return;
        const int p0 = pos_of(first, a.pos_cols);
        for (int i = threadIdx.x; i < n; i += 256) at[i] = 4 * (pos_of(min(first + i, last), a.pos_cols) - p0);
    }
};

// 16 biases of a lane: rows 8 (i / 4) + 4 half + i % 4 of a block of 32; `at`: the block's rows in the table of BIAS 1.
template <int BIAS>
__device__ __forceinline__ f32x16 read_bias(const char* win, const Places<BIAS>& pl, const int* at, int half, int lane_off) {
    f32x16 o = {};
    if (BIAS == 2) {
        const char* w0 = win + (lane_off + pl.blk);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float* w = reinterpret_cast<const float*>(w0 + pl.g[g]);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[4 * g + i] = w[i];
        }
    } else if (BIAS == 1) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[4 * g + i] = *reinterpret_cast<const float*>(win + at[8 * g + 4 * half + i] + lane_off);
    }
    return o;
}

// Scores of 16 (lane, streamed row) pairs in units of log2, from raw products (which may carry a constant in units of 1 / f).
// With a cap the tanh stays in `th`.
template <int BIAS, bool CAP>
__device__ __forceinline__ void to_logits(f32x16& x, f32x16& th, const AttnArgs& a, const f32x16& bias) {
    if (CAP) {
        th = x;
        tanh16(th, a.scale / a.cap);
    }
    const float f = CAP ? a.cap * LOG2E : a.scale * LOG2E;
    const f32x16& r = CAP ? th : x;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = BIAS ? r[i] * f + bias[i] : r[i] * f;
}

// Operands of a block of 32 streamed rows, read as a group ahead of their use: the compiler, left alone, reads each next to its
// matrix instruction and waits out the LDS latency every time.
template <int D> struct RowOps {
    bf16x8 f[D / 16];
    __device__ __forceinline__ void load(const Frags<D>& fr, const char* tile, int row0) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) f[ks] = fr.row(tile, row0, ks);
    }
    // products with the workgroup's own 32 rows (a lane each), from c on
    __device__ __forceinline__ f32x16 times(const bf16x8* own, f32x16 c) const {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) c = mfma(f[ks], own[ks], c);
        return c;
    }
};
template <int D> struct ColOps {
    bf16x8 f[2][D / 32];
    __device__ __forceinline__ void load(const Frags<D>& fr, const char* tile, int row0) {
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) f[g][d] = fr.col(tile, row0 + 16 * g, d);
    }
};
#define PHASE() __builtin_amdgcn_sched_barrier(0)

__device__ __forceinline__ f32x16 splat(float v) {
    f32x16 r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = v;
    return r;
}

__device__ __forceinline__ int keys_of(const AttnArgs& a, int b) {
    return a.lengths ? min(max(a.lengths[b], 0), a.Lk) : a.Lk;
}

// First of n tiles of a run.
__device__ __forceinline__ int run_first(int n, int runs, int run) { return min(n, (n + runs - 1) / runs * run); }

// ======================================================================================================= forward
// A workgroup owns 128 queries of a head, a wave 32 of them, and streams tiles of keys and values (64 rows, 32 at head size 128) through
// two LDS buffers: the next tile's loads run under the whole of this one's work.  What bounds it is issue, not a pipe: of the cycles of a
// SIMD at 128 px the matrix instructions take 34 %, the vector ones (16 exponentials of 4 slots each, 60 others a 32 x 32 block) 54 %, and
// with two waves they overlap little (with the cap 32 and 77 %, 64 px).  Leaving out, one at a time, the exponentials, half of the second
// product, the bias reads or the tiles' loads shortens it by 9 .. 12 % each; both blocks' first products ahead of the softmax change nothing.
// Three workgroups a compute unit at head size 64 (registers and LDS; four spill), two at 128.  32 px 48 without bias, 59 .. 63 with; 128 px
// 360 .. 430 (640 .. 760 TFLOP/s; its 512 workgroups are two a compute unit), with a cap of 50 600; three times its samples 780 TFLOP/s, capped
// 540.  Few workgroups: the keys are cut into
// `splits` runs, whose fp32 outputs, references and sums a second launch joins.
// LDS: K[2] V[2] tiles | window | table of the segment's places (BIAS 1).
// FINE: the probabilities go into the second product as three bf16 terms (24 bits): delta = do . o must be that exact where the fp32
// gradient of the table is wanted, whose sums cancel.  Its error against 64 bits over seven forms of 18 to 4096 tokens: one term 0.5 .. 1.5e-3,
// two 0.5 .. 2.8e-6, three 0.2 .. 0.6e-6, fp32 torch operations 0.1 .. 1.9e-6.  V's operands serve all three.  32 px: one term 63, two 76, three
// 84 .. 88 (the terms' subtractions, not the products).
template <int D, int BIAS, bool CAP, bool FINE>
__global__ __launch_bounds__(256, D == 128 ? 2 : D == 64 ? 3 : 4) void attn_fwd_kernel(AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int KT = kt_of(D), TB = KT * 2 * D, KS = D / 16, DB = D / 32;
    char* win = smem + 4 * TB;
    int* at = reinterpret_cast<int*>(win + a.win_bytes);

    const int id = xcd_run(blockIdx.x, gridDim.x);
    const int split = id % a.splits, own = id / a.splits, qb = own % a.n_qb, bh = own / a.n_qb, h = bh % a.H, b = bh / a.H, hk = h / a.rep;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int row = qb * BLK + wave * 32 + (lane & 31);
    const Frags<D> fr(lane);

    bf16x8 qf[KS];
    {
        const unsigned short* qp = a.q + b * a.q_sb + (int64_t)min(row, a.Lq - 1) * a.q_sl + h * a.q_sh + 8 * half;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
    }
    const int len = keys_of(a, b);
    const int nt = (len + KT - 1) / KT, t0 = run_first(nt, a.splits, split), t1 = run_first(nt, a.splits, split + 1);
    const unsigned short* kp = a.k + b * a.k_sb + (int64_t)t0 * KT * a.k_sl + hk * a.k_sh;
    const unsigned short* vp = a.v + b * a.v_sb + (int64_t)t0 * KT * a.v_sl + hk * a.v_sh;

    const int tq0 = a.q_start + qb * BLK, tq1 = a.q_start + min(qb * BLK + BLK, a.Lq) - 1;
    const int pq0 = BIAS ? pos_of(tq0, a.pos_cols) : 0, pq1 = BIAS ? pos_of(tq1, a.pos_cols) : 0;
    const int lane_off = BIAS ? 4 * (pq1 - pos_of(min(a.q_start + row, tq1), a.pos_cols)) + Places<BIAS>::half_off(a, half) : 0;

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = splat(0.f);
    // The softmax's reference m: probabilities are exp2(x - m).  m stays 0, and no maximum is looked for, while a row's sum stays between
    // SUM_LOW and SUM_HIGH; a row that leaves this range takes as m what makes its sum about 1 (its log-sum-exp so far, or the block's
    // maximum where that is larger) and scales what it has.
    float m = 0.f, l = 0.f;
    bool moved = false;                                              // (of the wave) some m is not 0

    Dma<D, KT> sk, sv;
    Places<BIAS> pl;
    int seg_t = t0;                                                  // the first tile of the segment in the window
    if (BIAS) pl.init(a, t0 * KT);
    if (t0 < t1) {
        sk.init(kp, a.k_sl, len - t0 * KT, smem);
        sv.init(vp, a.v_sl, len - t0 * KT, smem + 2 * TB);
        sk.next(a.k_sl, 0);
        sv.next(a.v_sl, 0);
        dma_wait();
    }
    arrived(qf);
    auto tile = [&](int t, auto parity) {
        constexpr int P = decltype(parity)::value;
        const char* kc = smem + P * TB;
        const char* vc = smem + (2 + P) * TB;
        if (BIAS && (t == t0 || t == seg_t + a.seg_tiles)) {
            __syncthreads();                                         // every wave is done with the last window
            seg_t = t;
            pl.blk = 0;
            const int n = a.seg_tiles * KT, p0 = pos_of(t * KT, a.pos_cols);
            stage_window<-1>(reinterpret_cast<float*>(win), a, h, pq0, pq1, p0, pos_of(t * KT + n - 1, a.pos_cols) - p0);
            Places<BIAS>::table(at, a, t * KT, n, a.Lk - 1);
        }
        __syncthreads();
        if (t + 1 < t1) {
            sk.next(a.k_sl, (P ^ 1) * TB);
            sv.next(a.v_sl, (P ^ 1) * TB);
        }
        PHASE();
        f32x16 x, th;
        const int* at_t = at + (t - seg_t) * KT;
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) {
            RowOps<D> kf;
            kf.load(fr, kc, 32 * u);
            const f32x16 bias = read_bias<BIAS>(win, pl, at_t + 32 * u, half, lane_off);
            if (BIAS) pl.next();
            PHASE();
            x = kf.times(qf, splat(0.f));
            ColOps<D> vf;
            vf.load(fr, vc, 32 * u);
            PHASE();
            auto logits = [&] {
                to_logits<BIAS, CAP>(x, th, a, bias);
                if (t * KT + KT > len) {
                    int k0 = t * KT + 32 * u + 4 * half;
                    asm volatile("" : "+v"(k0));                     // (else the comparisons' operands are computed for every tile)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (k0 + 8 * (i >> 2) + (i & 3) >= len) x[i] = NEG_INF;
                }
            };
            logits();
            if (moved)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] -= m;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x[i] = __builtin_amdgcn_exp2f(x[i]);
                sum += x[i];
            }
            float ln = l + sum;
            if (__any(!(ln > SUM_LOW && ln < SUM_HIGH))) {           // (a NaN comes here too, and stays one)
                const float both = other_half_sum(ln);
                const bool bad = !(both > SUM_LOW && both < SUM_HIGH);
                if (__any(bad)) {
                    kf.load(fr, kc, 32 * u);
                    x = kf.times(qf, splat(0.f));
                    logits();
                    float top = NEG_INF;
#pragma unroll
                    for (int i = 0; i < 16; ++i) top = fmaxf(top, x[i]);
                    top = other_half_max(top);
                    const float have = other_half_sum(l);
                    float mn = have > 0.f ? fmaxf(m + __builtin_amdgcn_logf(have), top) : top;
                    if (!bad || mn == NEG_INF) mn = m;
                    const float al = have > 0.f ? __builtin_amdgcn_exp2f(m - mn) : (have == 0.f ? 0.f : have);
                    m = mn;
                    moved = true;
                    sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        x[i] = __builtin_amdgcn_exp2f(x[i] - m);
                        sum += x[i];
                    }
                    ln = l * al + sum;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[d][i] *= al;
                }
            }
            l = ln;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const bf16x8 pf = pack8(x, 8 * g);
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = mfma(vf.f[g][d], pf, o[d]);
                if (FINE) {
                    bf16x8 rest = pf;
#pragma unroll
                    for (int term = 1; term < 3; ++term) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[8 * g + i] -= (float)rest[i];
                        rest = pack8(x, 8 * g);
#pragma unroll
                        for (int d = 0; d < DB; ++d) o[d] = mfma(vf.f[g][d], rest, o[d]);
                    }
                }
            }
        }
        dma_wait();
    };
    for (int t = t0; t < t1; t += 2) {
        tile(t, std::integral_constant<int, 0>{});
        if (t + 1 < t1) tile(t + 1, std::integral_constant<int, 1>{});
    }
    l = other_half_sum(l);
    if (row >= a.Lq) return;
    if (a.splits > 1) {
        const int64_t at_row = ((int64_t)b * a.Lq + row) * a.H + h;
        float* p = a.runs + split * a.run_floats + at_row * D + 4 * half;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(p + 32 * d + 8 * g) = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
        if (half == 0) *reinterpret_cast<f32x2_t*>(a.part + 2 * (split * (a.run_floats / D) + at_row)) = f32x2_t{m, l};
        return;
    }
    const float il = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);       // no key: 0; a NaN stays one
    if (a.lse && half == 0) a.lse[(int64_t)bh * a.Lq + row] = l == 0.f ? 0.f : m + __builtin_amdgcn_logf(l);
    const int64_t ob = (((int64_t)b * a.Lq + row) * a.H + h) * D + 4 * half;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = o[d][4 * g + i] * il;
            const u32x2 w = {pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
            *reinterpret_cast<u32x2*>(a.out + ob + 32 * d + 8 * g) = w;
            if (a.out_lo) {                                          // delta needs o in fp32
                const u32x2 r = {low_half(f[0]) | low_half(f[1]) << 16, low_half(f[2]) | low_half(f[3]) << 16};
                *reinterpret_cast<u32x2*>(a.out_lo + ob + 32 * d + 8 * g) = r;
            }
        }
}

// Output from the runs' sums, references and probabilities (part: (splits, B, Lq, H, 2)): four values a thread, grid
// (sample, query, head, D / 4) / 256.
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int D) {
    const int64_t e = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x), row = e / D;
    if (e >= a.run_floats) return;
    const int64_t rows = a.run_floats / D;
    float m = NEG_INF, l = 0.f;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    auto of_run = [&](int i) { return *reinterpret_cast<const f32x2_t*>(a.part + 2 * (min(i, a.splits - 1) * rows + row)); };
    for (int i0 = 0; i0 < a.splits; i0 += 4) {
        f32x2_t ml[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) ml[j] = of_run(i0 + j);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (ml[j][1] != 0.f) m = fmaxf(m, ml[j][0]);              // (a run without keys has no reference; one of NaN has)
    }
    for (int i0 = 0; i0 < a.splits; i0 += 4) {
        f32x2_t ml[4];
        f32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            ml[j] = of_run(i0 + j);
            v[j] = *reinterpret_cast<const f32x4*>(a.runs + min(i0 + j, a.splits - 1) * a.run_floats + e);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i0 + j >= a.splits || ml[j][1] == 0.f) continue;
            const float al = __builtin_amdgcn_exp2f(ml[j][0] - m);
            l += ml[j][1] * al;
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += v[j][k] * al;
        }
    }
    const float il = l > 0.f ? 1.f / l : l;                          // no key: 0; a NaN stays one
    const int64_t h = row % a.H, bq = row / a.H, b = bq / a.Lq, qi = bq - b * a.Lq;
    if (a.lse && e % D == 0) a.lse[(b * a.H + h) * a.Lq + qi] = l == 0.f ? 0.f : m + __builtin_amdgcn_logf(l);
    *reinterpret_cast<u32x2*>(a.out + e) = u32x2{pack_bf16x2(s[0] * il, s[1] * il), pack_bf16x2(s[2] * il, s[3] * il)};
    if (a.out_lo)
        *reinterpret_cast<u32x2*>(a.out_lo + e) = u32x2{low_half(s[0] * il) | low_half(s[1] * il) << 16, low_half(s[2] * il) | low_half(s[3] * il) << 16};
}

// ======================================================================================================= forward, few rows
// At most 32 (query, head) pairs share a key / value head: all of them are the lanes of ONE product, so keys and values are read once
// however many heads share them, and the keys are cut into `splits` runs for as many workgroups.  Bound by reading keys and values: a
// wave streams blocks of 32 keys of its own (two buffers, no barrier in the loop), and the waves', then the runs', (maximum, sum,
// output) are joined in a fixed order.  part: (B, Hkv, splits, 32, D + 2) fp32: output, maximum, sum; one run writes the rows itself.
// One query, 4 samples of 16384 keys, 8 heads on 2 of 128 (67 MB): 20 + 4 with bias, 3.3 TB/s, 17 + 4 without; 256 samples of 1024 keys, 8 heads
// of 64 (537 MB): 107, 5.0 TB/s.
// LDS: for each wave K[2] V[2] of 32 rows; the joining reuses it.
template <int D> struct WaveDma {
    static constexpr int NP = D / 16;                                // 1 KB pieces of a block
    unsigned lds;
    __device__ __forceinline__ void init(const char* block) { lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)block; }
    // rows k0 .. k0 + 31 (the last valid one repeated) into the block `bytes` behind
    __device__ __forceinline__ void load(const unsigned short* p, int64_t sl, int k0, int valid, int bytes) const {
        constexpr int RP = 512 / D, CH = D / 8;                       // rows of a piece, chunks of a row
        const int lane = threadIdx.x & 63, r0 = lane / CH, ch = lane % CH;
        const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane((int)lds) + bytes;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int row = i * RP + r0;
            const unsigned short* src = p + (int64_t)min(k0 + row, valid - 1) * sl + ((ch ^ swz<D>(row)) << 3);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(to + 1024 * i), "v"(src) : "memory", "m0");
        }
    }
};

// Value d of a row from its sums: s over the keys, reference m, probabilities l.
__device__ __forceinline__ void write_few(const AttnArgs& a, int64_t row, int64_t lse_row, int D, int d, float s, float m, float l) {
    const float y = l > 0.f ? s / l : (l == 0.f ? 0.f : l);           // no key: 0; a NaN stays one
    a.out[row * D + d] = f32_to_bf16_bits(y);
    if (a.out_lo) a.out_lo[row * D + d] = (unsigned short)low_half(y);
    if (a.lse && d == 0) a.lse[lse_row] = l == 0.f ? 0.f : m + __builtin_amdgcn_logf(l);
}

template <int D, bool BIAS, bool CAP>
__global__ __launch_bounds__(256, 1) void attn_few_kernel(AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int BB = 32 * 2 * D, KS = D / 16, DB = D / 32;          // bytes of a block
    const int split = blockIdx.x % a.splits, bk = blockIdx.x / a.splits, hk = bk % a.Hkv, b = bk / a.Hkv;
    const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5, col = lane & 31;
    const int cols = a.rep * a.Lq;
    const int h = hk * a.rep + min(col, cols - 1) / a.Lq, qi = min(col, cols - 1) % a.Lq;
    const Frags<D> fr(lane);
    char* mine = smem + wave * 4 * BB;
    WaveDma<D> dma;
    dma.init(mine);

    const int len = keys_of(a, b), blocks = (len + 31) / 32;
    const int per = (blocks + a.splits - 1) / a.splits, b1 = min(blocks, (split + 1) * per);
    const unsigned short* kp = a.k + b * a.k_sb + hk * a.k_sh;
    const unsigned short* vp = a.v + b * a.v_sb + hk * a.v_sh;

    // the bias of a lane's 16 (pair, key): places first, then their buckets, one block ahead
    const int pq = BIAS ? pos_of(a.q_start + qi, a.pos_cols) + (2 * a.cols - 1) * (a.rows - 1) + a.cols - 1 : 0;
    const int last = (2 * a.cols - 1) * (2 * a.rows - 1) - 1;
    const float* trow = BIAS ? a.table + (int64_t)h * a.n_buckets : nullptr;
    const float inv_cols = BIAS ? 1.f / (float)a.pos_cols : 0.f;
    int u[16];
    float bias[16];
    auto places = [&](int blk) {
        const int x0 = blk * 32 % a.pos_cols, base = pq - pos_of(blk * 32, a.pos_cols);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int off = 8 * (i >> 2) + 4 * half + (i & 3);
            // rows of the grid that off keys further on have ended: (x0 + off) / cols, a quotient below 2^12 at least 1 / 2048 off an integer
            const int wraps = a.rows > 1 ? (int)(((float)(x0 + off) + 0.5f) * inv_cols) : 0;
            u[i] = a.map[min(max(base - off - wraps * (a.cols - 1), 0), last)];
        }
    };
    auto buckets = [&] {
#pragma unroll
        for (int i = 0; i < 16; ++i) bias[i] = in_log2(trow[min(max(u[i], 0), a.n_buckets - 1)]);
    };

    bf16x8 qf[KS];
    {
        const unsigned short* qp = a.q + b * a.q_sb + (int64_t)qi * a.q_sl + h * a.q_sh + 8 * half;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
    }
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = splat(0.f);
    float m = NEG_INF, l = 0.f;
    int blk = split * per + wave, p = 0;
    if (blk < b1) {
        dma.load(kp, a.k_sl, blk * 32, len, 0);
        dma.load(vp, a.v_sl, blk * 32, len, 2 * BB);
        if (BIAS) { places(blk); buckets(); }
    }
    arrived(qf);
    for (; blk < b1; blk += 4, p ^= 1) {
        float now[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) now[i] = BIAS ? bias[i] : 0.f;
        dma_wait();
        const bool more = blk + 4 < b1;
        if (more) {
            dma.load(kp, a.k_sl, (blk + 4) * 32, len, (p ^ 1) * BB);
            dma.load(vp, a.v_sl, (blk + 4) * 32, len, (2 + (p ^ 1)) * BB);
            if (BIAS) places(blk + 4);
        }
        RowOps<D> kf;
        kf.load(fr, mine + p * BB, 0);
        f32x16 x = kf.times(qf, splat(0.f)), th;
        if (CAP) {
            th = x;
            tanh16(th, a.scale / a.cap);
        }
        const float f = CAP ? a.cap * LOG2E : a.scale * LOG2E;
        float top = NEG_INF;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = (CAP ? th[i] : x[i]) * f + now[i];
            if (blk * 32 + 8 * (i >> 2) + 4 * half + (i & 3) >= len) x[i] = NEG_INF;
            top = fmaxf(top, x[i]);
        }
        top = other_half_max(top);
        const float mn = fmaxf(m, top), ms = mn == NEG_INF ? 0.f : mn, al = __builtin_amdgcn_exp2f(m - ms);
        m = mn;
        l *= al;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= al;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = __builtin_amdgcn_exp2f(x[i] - ms);
            l += x[i];
        }
        ColOps<D> vf;
        vf.load(fr, mine + (2 + p) * BB, 0);
#pragma unroll
        for (int g = 0; g < 2; ++g) {                                // three bf16 terms of p: the matrix cores have time to spare here
            bf16x8 pf = pack8(x, 8 * g);
#pragma unroll
            for (int term = 0; term < 3; ++term) {
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = mfma(vf.f[g][d], pf, o[d]);
                if (term < 2) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[8 * g + i] -= (float)pf[i];
                    pf = pack8(x, 8 * g);
                }
            }
        }
        if (BIAS && more) buckets();
    }
    l = other_half_sum(l);
    // join the waves: (32, D) outputs and 32 (maximum, sum) of each
    __syncthreads();
    float* jo = reinterpret_cast<float*>(smem);                      // (4, 32, D + 1): a lane's column apart from its neighbour's
    float* jm = jo + 4 * 32 * (D + 1);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) jo[(wave * 32 + col) * (D + 1) + 32 * d + 8 * (i >> 2) + 4 * half + (i & 3)] = o[d][i];
    if (half == 0) { jm[wave * 64 + col] = m; jm[wave * 64 + 32 + col] = l; }
    __syncthreads();
    float* part = a.splits > 1 ? a.part + (int64_t)blockIdx.x * 32 * (D + 2) : nullptr;
    for (int e = threadIdx.x; e < cols * D; e += 256) {
        const int c = e / D, d = e % D;
        float mm = NEG_INF, s = 0.f, ll = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, jm[w * 64 + c]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float al = __builtin_amdgcn_exp2f(jm[w * 64 + c] - (mm == NEG_INF ? 0.f : mm));
            s += jo[(w * 32 + c) * (D + 1) + d] * al;
            ll += jm[w * 64 + 32 + c] * al;
        }
        if (part) {
            part[c * (D + 2) + d] = s;
            if (d == 0) { part[c * (D + 2) + D] = mm; part[c * (D + 2) + D + 1] = ll; }
        } else {                                                     // one run: the rows are whole
            const int hc = hk * a.rep + c / a.Lq, qc = c % a.Lq;
            write_few(a, ((int64_t)b * a.Lq + qc) * a.H + hc, ((int64_t)b * a.H + hc) * a.Lq + qc, D, d, s, mm, ll);
        }
    }
}

// A workgroup a (sample, query, head): the runs' partials joined, eight at a time by each of its 512 / D rows of D threads.
constexpr int MAX_SPLITS = 512;
template <int D> __global__ __launch_bounds__(512) void attn_few_join_kernel(AttnArgs a) {
    __shared__ float al[MAX_SPLITS], red[512];
    const int d = threadIdx.x % D, r = threadIdx.x / D, h = blockIdx.x % a.H, qi = blockIdx.x / a.H % a.Lq, b = blockIdx.x / a.H / a.Lq;
    const int hk = h / a.rep, c = h % a.rep * a.Lq + qi;
    const float* part = a.part + (((int64_t)b * a.Hkv + hk) * a.splits * 32 + c) * (D + 2);
    constexpr int64_t RUN = 32 * (D + 2);
    constexpr int R = 512 / D;
    // wave 0: every run's maximum and sum -> its factor, the row's maximum and sum
    __shared__ float row_m, row_l;
    if (threadIdx.x < 64) {
        float mm = NEG_INF, ll = 0.f;
        for (int i = threadIdx.x; i < a.splits; i += 64) { al[i] = part[i * RUN + D]; mm = fmaxf(mm, al[i]); }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 64));
        for (int i = threadIdx.x; i < a.splits; i += 64) {
            al[i] = __builtin_amdgcn_exp2f(al[i] - (mm == NEG_INF ? 0.f : mm));
            ll += part[i * RUN + D + 1] * al[i];
        }
        ll = wave_sum(ll);
        if (threadIdx.x == 0) { row_m = mm; row_l = ll; }
    }
    __syncthreads();
    float s = 0.f;
    for (int i0 = r; i0 < a.splits; i0 += R * 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = part[min(i0 + j * R, a.splits - 1) * RUN + d];
#pragma unroll
        for (int j = 0; j < 8; ++j) s += i0 + j * R < a.splits ? v[j] * al[min(i0 + j * R, MAX_SPLITS - 1)] : 0.f;
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (r) return;
    for (int k = 1; k < R; ++k) s += red[k * D + d];
    write_few(a, blockIdx.x, ((int64_t)b * a.H + h) * a.Lq + qi, D, d, s, row_m, row_l);
}

// ======================================================================================================= dq, delta and the table
// Partials of the table's gradient, without global atomics and in one order of summation.  DT names how a 128 x 64 tile of ds (fp32,
// never rounded) is reduced to sums over pairs of equal offset:
//   BLOCKS    where 32 aligned tokens lie in one row of the grid (columns a multiple of 32, or a single row): within a 32 x 32 block
//             the offset is one number plus (query - key), 63 sums.  A wave puts its block into LDS of its own (no barrier), rows
//             of 32 values and 40 zeros: a lane then adds up one diagonal, 32 reads at fixed distances that run off the block into
//             zeros, no comparison.  part (b, h, query group, key group, 64).  Adding with ds_add_f32 instead: 728, 32 px.  The sums
//             of a tile are stored one tile later: the wait for the next tile's loads would wait for a store that has just gone out.
//   DIAGONALS any other grid: a pair is known by its distance i - j and by whether the column of i wraps (class 0: dx >= 0, class 1:
//             dx < 0).  ds goes through LDS and a thread adds up one diagonal of the tile; a diagonal stays with its thread (distance
//             mod 256) over the tiles it crosses and is stored once: part (b, h, query block, class, distance).  Taken where BLOCKS
//             would do it costs more: 32 px 197 + 22 against 102 + 22.
// Three products a block where the forward pass has two.  32 px: 67 without bias, 74 .. 79 with, 102 .. 112 with the table's sums (16 writes and
// 32 reads of 4 bytes more a lane and block; vector instructions 45 %, matrix ones 23 % of a SIMD's cycles), 64 px 229 .. 250, line 138 + 9.  Two
// workgroups a compute unit; three at head size 32 without the table's sums, with them LDS holds two there as well (and the capped form, kept to
// the registers of three, spills 84 bytes a lane; at head size 128 28).
// Few workgroups: the keys are cut into `splits` runs whose fp32 dq a second launch adds up (a run has its own diagonals, and its own blocks).
// LDS: K[2] V[2] | BLOCKS: a block and its zeros for each wave, DIAGONALS: ds (KT x 128 floats) | window.
enum { DT_NONE = 0, DT_BLOCKS = 1, DT_DIAGONALS = 2 };
constexpr int BS = 72;                    // floats from row to row of a block: rows 4 apart (a wave's halves) are 32 banks apart
constexpr int block_rows(int D) { return D == 128 ? 16 : 32; }       // (16: a block goes through in two halves, for two workgroups' LDS)
constexpr int block_floats(int D) { return 32 + block_rows(D) * BS; }
constexpr int dt_lds(int dt, int D) { return dt == DT_BLOCKS ? 4 * block_floats(D) * 4 : dt == DT_DIAGONALS ? kt_of(D) * BLK * 4 : 0; }

template <int D, int BIAS, bool CAP, int DT>
__global__ __launch_bounds__(256, D == 32 ? 3 : 2) void attn_dq_kernel(AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int BR = block_rows(D), KT = kt_of(D), TB = KT * 2 * D, KS = D / 16, DB = D / 32;
    float* dsl = reinterpret_cast<float*>(smem + 4 * TB);
    char* win = smem + 4 * TB + dt_lds(DT, D);
    int* at = reinterpret_cast<int*>(win + a.win_bytes);
    const int n_kg = a.n_kt * (KT / 32);

    const int id = xcd_run(blockIdx.x, gridDim.x);
    const int split = id % a.splits, own = id / a.splits, qb = own % a.n_qb, bh = own / a.n_qb, h = bh % a.H, b = bh / a.H, hk = h / a.rep;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int row = qb * BLK + wave * 32 + (lane & 31);
    const bool live = row < a.Lq;
    const Frags<D> fr(lane);
    float* blk = dsl + wave_id() * block_floats(D) + 32;                // BLOCKS: row 0, zeros in front of it
    if (DT == DT_BLOCKS) {
        for (int i = lane; i < block_floats(D); i += 64) blk[i - 32] = 0.f;
        wave_fence();
    }

    bf16x8 qf[KS], gf[KS];
    float delta = 0.f;
    {
        const int r = min(row, a.Lq - 1);
        const unsigned short* qp = a.q + b * a.q_sb + (int64_t)r * a.q_sl + h * a.q_sh + 8 * half;
        const int64_t ob = (((int64_t)b * a.Lq + r) * a.H + h) * D + 8 * half;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            qf[ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
            gf[ks] = *reinterpret_cast<const bf16x8*>(a.d_o + ob + 16 * ks);
            const u32x4 ov = *reinterpret_cast<const u32x4*>(a.o + ob + 16 * ks), lv = *reinterpret_cast<const u32x4*>(a.o_lo + ob + 16 * ks);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                delta += (float)gf[ks][2 * i] * whole(ov[i] & 0xffffu, lv[i]);
                delta += (float)gf[ks][2 * i + 1] * whole(ov[i] >> 16, lv[i] >> 16);
            }
        }
    }
    delta = other_half_sum(delta);
    if (live && half == 0 && split == 0) a.delta[(int64_t)bh * a.Lq + row] = delta;
    if (!live) delta = 0.f;
    const float lse = live ? a.lse[(int64_t)bh * a.Lq + row] : NO_ROW;

    const int len = keys_of(a, b);
    const int nt = (len + KT - 1) / KT, t0 = run_first(nt, a.splits, split), t1 = run_first(nt, a.splits, split + 1);
    const unsigned short* kp = a.k + b * a.k_sb + (int64_t)t0 * KT * a.k_sl + hk * a.k_sh;
    const unsigned short* vp = a.v + b * a.v_sb + (int64_t)t0 * KT * a.v_sl + hk * a.v_sh;
    const int tq0 = a.q_start + qb * BLK, tq1 = a.q_start + min(qb * BLK + BLK, a.Lq) - 1;
    const int pq0 = BIAS ? pos_of(tq0, a.pos_cols) : 0, pq1 = BIAS ? pos_of(tq1, a.pos_cols) : 0;
    const int lane_off = BIAS ? 4 * (pq1 - pos_of(min(a.q_start + row, tq1), a.pos_cols)) + Places<BIAS>::half_off(a, half) : 0;

    f32x16 acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = splat(0.f);
    float sum0 = 0.f, sum1 = 0.f;                                    // the thread's diagonal, by class
    // DIAGONALS: partials of this workgroup, place 0 = the smallest distance it meets
    float* part = DT == DT_DIAGONALS ? a.part + (int64_t)id * 2 * a.span
                                     : DT == DT_BLOCKS ? a.part + ((int64_t)own * 4 + wave) * n_kg * 64 : nullptr;
    const int d_min = tq0 - (nt * KT - 1);
    float hold[KT / 32];                                             // BLOCKS: a tile's sums until they are stored

    Dma<D, KT> sk, sv;
    Places<BIAS> pl;
    int seg_t = t0;
    if (BIAS) pl.init(a, t0 * KT);
    if (t0 < t1) {
        sk.init(kp, a.k_sl, len - t0 * KT, smem);
        sv.init(vp, a.v_sl, len - t0 * KT, smem + 2 * TB);
        sk.next(a.k_sl, 0);
        sv.next(a.v_sl, 0);
        dma_wait();
    }
    arrived(qf);
    arrived(gf);
    auto tile = [&](int t, auto parity) {
        constexpr int P = decltype(parity)::value;
        const char* kc = smem + P * TB;
        const char* vc = smem + (2 + P) * TB;
        if (BIAS && (t == t0 || t == seg_t + a.seg_tiles)) {
            __syncthreads();
            seg_t = t;
            pl.blk = 0;
            const int n = a.seg_tiles * KT, p0 = pos_of(t * KT, a.pos_cols);
            stage_window<-1>(reinterpret_cast<float*>(win), a, h, pq0, pq1, p0, pos_of(t * KT + n - 1, a.pos_cols) - p0);
            Places<BIAS>::table(at, a, t * KT, n, a.Lk - 1);
        }
        __syncthreads();
        if (DT == DT_BLOCKS && t > t0)
#pragma unroll
            for (int u = 0; u < KT / 32; ++u) part[(KT / 32 * (t - 1) + u) * 64 + lane] = hold[u];
        if (t + 1 < t1) {
            sk.next(a.k_sl, (P ^ 1) * TB);
            sv.next(a.v_sl, (P ^ 1) * TB);
        }
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) {
            RowOps<D> f;
            f.load(fr, kc, 32 * u);
            f32x16 s = f.times(qf, splat(0.f)), th;
            f.load(fr, vc, 32 * u);
            const f32x16 bias = read_bias<BIAS>(win, pl, at + (t - seg_t) * KT + 32 * u, half, lane_off);
            if (BIAS) pl.next();
            f32x16 dp = f.times(gf, splat(0.f));
            to_logits<BIAS, CAP>(s, th, a, bias);
            if (t * KT + KT > len) {
                int k0 = t * KT + 32 * u + 4 * half;
                asm volatile("" : "+v"(k0));
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (k0 + 8 * (i >> 2) + (i & 3) >= len) s[i] = NEG_INF;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float ds = __builtin_amdgcn_exp2f(s[i] - lse) * (dp[i] - delta);
                if (DT == DT_DIAGONALS) dsl[(32 * u + 8 * (i >> 2) + 4 * half + (i & 3)) * BLK + wave * 32 + (lane & 31)] = ds;
                dp[i] = ds;
                s[i] = CAP ? ds * (1.f - th[i] * th[i]) : ds;
            }
            ColOps<D> kt;
            kt.load(fr, kc, 32 * u);
            // the table's sums: the block's values go out and its diagonals come in while the products run
            float diag[32];
            auto put = [&](int e) {
#pragma unroll
                for (int i = 0; i < BR / 2; ++i) blk[(8 * (i >> 2) + 4 * half + (i & 3)) * BS + (lane & 31)] = dp[BR / 2 * e + i];
                wave_fence();
            };
            auto get = [&](int e) {                                  // lane: query - key = lane - 32
#pragma unroll
                for (int i = 0; i < BR; ++i) diag[i] = blk[i * (BS + 1) + BR * e + lane - 32];
                wave_fence();
            };
            auto total = [&] {
                float t4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < BR; ++i) t4[i & 3] += diag[i];
                return (t4[0] + t4[1]) + (t4[2] + t4[3]);
            };
            if (DT == DT_BLOCKS) { put(0); get(0); }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const bf16x8 pf = pack8(s, 8 * g);
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] = mfma(kt.f[g][d], pf, acc[d]);
            }
            if (DT == DT_BLOCKS) {
                float sum = total();
                if (BR == 16) { put(1); get(1); sum += total(); }
                hold[u] = sum;
            }
        }
        dma_wait();
        if (DT == DT_DIAGONALS) {
            __syncthreads();
            const int k0 = t * KT, lo = tq0 - k0 - (KT - 1);         // smallest distance of this tile
            const int w = ((int)threadIdx.x - lo) & 255;
            const int c = w - (KT - 1), dist = lo + w;               // column of the tile = row + c
            if (c < BLK) {
                const int k_lo = max(0, -c), k_hi = min(KT - 1, BLK - 1 - c);
                const float* p = dsl + k_lo * (BLK + 1) + c;
                int r = dist % a.cols;
                r += r < 0 ? a.cols : 0;
                int x = (k0 + k_lo) % a.cols + r - a.cols;           // >= 0: the column of i wraps
                for (int k = k_lo; k <= k_hi; k += 8, p += 8 * (BLK + 1)) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = k + j <= k_hi ? p[j * (BLK + 1)] : 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float w = x >= 0 ? v[j] : 0.f;
                        sum1 += w;
                        sum0 += v[j] - w;
                        ++x;
                        x -= x == r ? a.cols : 0;                    // the key's own row ends
                    }
                }
                if (c + KT >= BLK || t + 1 == t1) {                        // the diagonal leaves the workgroup's rows, or the run ends
                    part[dist - d_min] = sum0;
                    part[a.span + dist - d_min] = sum1;
                    sum0 = sum1 = 0.f;
                }
            }
        }
    };
    for (int t = t0; t < t1; t += 2) {
        tile(t, std::integral_constant<int, 0>{});
        if (t + 1 < t1) tile(t + 1, std::integral_constant<int, 1>{});
    }
    if (DT == DT_BLOCKS && t0 < t1)
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) part[(KT / 32 * (t1 - 1) + u) * 64 + lane] = hold[u];
    if (!live) return;
    if (a.splits > 1) {
        float* p = a.runs + split * a.run_floats + (((int64_t)b * a.Lq + row) * a.H + h) * D + 4 * half;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(p + 32 * d + 8 * g) = f32x4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
        return;
    }
    unsigned short* qo = a.dq + b * a.dq_sb + (int64_t)row * a.dq_sl + h * a.dq_sh + 4 * half;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const u32x2 w = {pack_bf16x2(acc[d][4 * g] * a.scale, acc[d][4 * g + 1] * a.scale),
                             pack_bf16x2(acc[d][4 * g + 2] * a.scale, acc[d][4 * g + 3] * a.scale)};
            *reinterpret_cast<u32x2*>(qo + 32 * d + 8 * g) = w;
        }
}

// dq from the runs' sums: four values a thread, grid (sample, query, head, D / 4) / 256.
__global__ __launch_bounds__(256) void attn_dq_sum_kernel(AttnArgs a, int D) {
    const int64_t e = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
    if (e >= a.run_floats) return;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < a.splits; i0 += 4) {
        f32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const f32x4*>(a.runs + min(i0 + j, a.splits - 1) * a.run_floats + e);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j < a.splits)
#pragma unroll
                for (int k = 0; k < 4; ++k) s[k] += v[j][k];
    }
    const int64_t row = e / D / a.H, b = row / a.Lq;
    unsigned short* o = a.dq + b * a.dq_sb + (row - b * a.Lq) * a.dq_sl + e / D % a.H * a.dq_sh + e % D;
    *reinterpret_cast<u32x2*>(o) = u32x2{pack_bf16x2(s[0] * a.scale, s[1] * a.scale), pack_bf16x2(s[2] * a.scale, s[3] * a.scale)};
}

// ---- the table's gradient from the partials: sums over samples and places first, then by bucket.
// BLOCKS.  by_block (H, classes, 64): a class is (row difference, column-group difference) of a block's query and key groups, G =
// columns / 32 groups a row (a single row: G = all of them).  grid (classes, H), 16 row lanes x 64 places; `more`: samples behind those
// that are summed already.
__global__ __launch_bounds__(1024) void attn_block_sums_kernel(AttnArgs a, float* by_block, bool more, int q_rows, int k_rows, int gq, int gk) {
    __shared__ float red[1024];
    const int cls = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63, r = threadIdx.x >> 6;
    const int dgs = gq + gk - 1;
    const int dy = cls / dgs - (k_rows - 1), dg = cls % dgs - (gk - 1);       // query group row (from q_row0) - key row, group - group
    const int y0 = max(0, dy), y1 = min(q_rows, k_rows + dy), g0 = max(0, dg), g1 = min(gq, gk + dg);
    const int n_qg = a.n_qb * 4, n_kg = a.n_kt * (a.kt / 32);
    // runs of blocks one step apart (down the rows; along the groups where there is one row), eight at a time, dealt out over the waves
    const bool line = q_rows == 1 && k_rows == 1;
    const int lo = line ? g0 : y0, hi_all = line ? g1 : y1, outer = line ? 1 : max(0, g1 - g0);
    const int chunks = max(0, hi_all - lo + 7) / 8, tasks = a.B * outer * chunks;
    const int64_t step = 64 * (line ? (int64_t)n_kg + 1 : (int64_t)gq * n_kg + gk);
    const float* src = a.part + (int64_t)h * n_qg * n_kg * 64 + lane;
    float s = 0.f;
    for (int task = __builtin_amdgcn_readfirstlane(r); task < tasks; task += 16) {
        const int o = task / chunks, first = lo + task % chunks * 8, b = o / outer, g = line ? 0 : g0 + o % outer;
        const int k_valid = a.kt / 32 * ((keys_of(a, b) + a.kt - 1) / a.kt);      // key groups that were stored
        // last block of the run: a query group that exists, a key group that was stored
        const int hi = line ? min(hi_all, min(n_qg, k_valid + dg))
                            : min(hi_all, min((n_qg - g + gq - 1) / gq, dy + (k_valid - (g - dg) + gk - 1) / gk));
        if (first >= hi) continue;
        const float* p = src + ((int64_t)b * a.H * n_qg + (line ? first : first * gq + g)) * n_kg * 64 +
                         64 * (int64_t)(line ? first - dg : (first - dy) * gk + g - dg);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p[min(j, hi - 1 - first) * step];
#pragma unroll
        for (int j = 0; j < 8; ++j) s += first + j < hi ? v[j] : 0.f;
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (r == 0) {
        for (int k = 1; k < 16; ++k) s += red[k * 64 + lane];
        float* o = by_block + ((int64_t)h * gridDim.x + cls) * 64 + lane;
        *o = more ? *o + s : s;
    }
}

// dtable[h][u] = sum over the offsets of bucket u (order[start[u]] .. ): grid (n_buckets, H).  An offset lies in two neighbouring
// classes of blocks.
__global__ __launch_bounds__(256) void attn_block_bucket_kernel(AttnArgs a, const float* by_block, const int* order, const int* start, int q_row0,
                                                                int k_rows, int q_rows, int gq, int gk) {
    __shared__ float red[4];
    const int u = blockIdx.x, h = blockIdx.y, w = 2 * a.cols - 1, dgs = gq + gk - 1;
    const float* src = by_block + (int64_t)h * (q_rows + k_rows - 1) * dgs * 64;
    float s = 0.f;
    for (int e = start[u] + (int)threadIdx.x; e < start[u + 1]; e += 256) {
        const int off = order[e];
        int dy = off / w - (a.rows - 1), dx = off % w - (a.cols - 1);
        if (a.rows == 1) dx -= a.q_start;                              // groups count from the first query
        dy -= q_row0;
        if (dy < -(k_rows - 1) || dy > q_rows - 1) continue;
        const int lo = dx >> 5, c = dx & 31;                           // dx = 32 lo + c = 32 (lo + 1) - (32 - c)
        const float* row = src + (int64_t)(dy + k_rows - 1) * dgs * 64;
        const int g = lo + gk - 1;
        if (g >= 0 && g < dgs) s += row[g * 64 + 32 + c];
        if (c && g + 1 >= 0 && g + 1 < dgs) s += row[(g + 1) * 64 + c];
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.dtable[(int64_t)h * a.n_buckets + u] = red[0] + red[1] + red[2] + red[3];
}

// DIAGONALS.  by_dist (H, 2, n_dist): grid (distances / 64, 2 classes x H), 16 row lanes x 64 distances.
__global__ __launch_bounds__(1024) void attn_dist_kernel(AttnArgs a, float* by_dist, bool more, int n_dist, int d0) {
    __shared__ float red[1024];
    const int i = blockIdx.x * 64 + (threadIdx.x & 63), r = threadIdx.x >> 6;
    const int cls = blockIdx.y & 1, h = blockIdx.y >> 1, dist = i + d0;
    float s = 0.f;
    for (int e = r; e < a.B * a.n_qb * a.splits; e += 16) {
        const int split = e % a.splits, qb = e / a.splits % a.n_qb, b = e / a.splits / a.n_qb;
        const int nt = (keys_of(a, b) + a.kt - 1) / a.kt, t0 = run_first(nt, a.splits, split), t1 = run_first(nt, a.splits, split + 1);
        const int tq0 = a.q_start + qb * BLK, place = dist - (tq0 - (nt * a.kt - 1));
        if (t0 == t1 || dist < tq0 - (t1 * a.kt - 1) || dist > tq0 + BLK - 1 - t0 * a.kt) continue;     // no pair of the run's
        s += a.part[((((int64_t)b * a.H + h) * a.n_qb + qb) * a.splits + split) * 2 * a.span + (int64_t)cls * a.span + place];
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (r == 0 && i < n_dist) {
        for (int k = 1; k < 16; ++k) s += red[k * 64 + (threadIdx.x & 63)];
        float* o = by_dist + ((int64_t)h * 2 + cls) * n_dist + i;
        *o = more ? *o + s : s;
    }
}

__global__ __launch_bounds__(256) void attn_dist_bucket_kernel(AttnArgs a, const float* by_dist, const int* order, const int* start, int n_dist,
                                                               int d0) {
    __shared__ float red[4];
    const int u = blockIdx.x, h = blockIdx.y, w = 2 * a.cols - 1;
    const float* src = by_dist + (int64_t)h * 2 * n_dist;
    float s = 0.f;
    for (int e = start[u] + (int)threadIdx.x; e < start[u + 1]; e += 256) {
        const int off = order[e], dy = off / w - (a.rows - 1), dx = off % w - (a.cols - 1);
        const int place = dy * a.cols + dx - d0;
        if (place >= 0 && place < n_dist) s += src[(int64_t)(dx < 0) * n_dist + place];
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.dtable[(int64_t)h * a.n_buckets + u] = red[0] + red[1] + red[2] + red[3];
}

// ======================================================================================================= dk, dv
// A workgroup owns 128 keys of one key / value head and streams the queries of every head that shares it: scores here are
// queries x keys, a lane holds one key.  No sum leaves the workgroup; where keys and heads alone are too few workgroups for the chip,
// the tiles of queries are cut into `splits` runs whose fp32 sums a second launch adds up: part (splits, B, Hkv, Lk, 2 D).
// Four products a block; the row sums' logarithm and delta come in as the products' initial values, which saves their subtraction.
// 32 px 78 without bias, 89 .. 97 with, 64 px 216 .. 247, line 226 .. 239 + 9.  Three waves a SIMD at head size 32 (the capped forms spill 24 .. 32
// bytes a lane), two at 64 (three spill), one at 128: dk, dv
// and the wave's own keys and values are 192 registers there, a block's scores and operands the rest of 450; within 256 they spill.
// LDS: Q[2] dO[2] | lse[2][64] | delta[2][64] | window | table of the segment's places (BIAS 1).
template <int D, int BIAS, bool CAP>
__global__ __launch_bounds__(256, D == 128 ? 1 : D == 64 ? 2 : 3) void attn_dkv_kernel(AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int KT = kt_of(D), TB = KT * 2 * D, KS = D / 16, DB = D / 32;
    float* ls = reinterpret_cast<float*>(smem + 4 * TB);
    float* dl = ls + 2 * KT;
    char* win = reinterpret_cast<char*>(dl + 2 * KT);
    int* at = reinterpret_cast<int*>(win + a.win_bytes);

    const int id = xcd_run(blockIdx.x, gridDim.x);
    const int split = id % a.splits, kb = id / a.splits % a.n_kb, bk = id / a.splits / a.n_kb, hk = bk % a.Hkv, b = bk / a.Hkv;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int key = kb * BLK + wave * 32 + (lane & 31);
    const Frags<D> fr(lane);
    const int len = keys_of(a, b);

    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[d] = dv[d] = splat(0.f);

    if (kb * BLK < len && a.Lq > 0) {
        bf16x8 kf[KS], vf[KS];
        {
            const int r = min(key, len - 1);                         // keys beyond the length repeat the last one; their sums are dropped
            const unsigned short* kp = a.k + b * a.k_sb + (int64_t)r * a.k_sl + hk * a.k_sh + 8 * half;
            const unsigned short* vp = a.v + b * a.v_sb + (int64_t)r * a.v_sl + hk * a.v_sh + 8 * half;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                kf[ks] = *reinterpret_cast<const bf16x8*>(kp + 16 * ks);
                vf[ks] = *reinterpret_cast<const bf16x8*>(vp + 16 * ks);
            }
        }
        const int tk0 = kb * BLK, tk1 = min(kb * BLK + BLK, a.Lk) - 1;
        const int pk0 = BIAS ? pos_of(tk0, a.pos_cols) : 0, pk1 = BIAS ? pos_of(tk1, a.pos_cols) : 0;
        const int lane_off = BIAS ? 4 * (pk1 - pos_of(min(key, tk1), a.pos_cols)) + Places<BIAS>::half_off(a, half) : 0;
        const int nqt = (a.Lq + KT - 1) / KT;
        const float neg_inv_f = -1.f / (a.scale * LOG2E);

        Dma<D, KT> sq, sg;
        float next_l = 0.f, next_d = 0.f;
        auto load = [&](int h, int t, int buf, bool first) {          // tile t of head h into buffer buf
            if (t == 0 || first) {
                sq.init(a.q + b * a.q_sb + h * a.q_sh + (int64_t)t * KT * a.q_sl, a.q_sl, a.Lq - t * KT, smem);
                sg.init(a.d_o + (((int64_t)b * a.Lq + t * KT) * a.H + h) * D, (int64_t)a.H * D, a.Lq - t * KT, smem + 2 * TB);
            }
            sq.next(a.q_sl, buf * TB);
            sg.next((int64_t)a.H * D, buf * TB);
            if (threadIdx.x < KT) {
                const int r = t * KT + threadIdx.x;
                const int64_t at_row = (int64_t)(b * a.H + h) * a.Lq + r;
                next_l = r < a.Lq ? a.lse[at_row] : NO_ROW;
                next_d = r < a.Lq ? a.delta[at_row] : 0.f;
            }
        };
        auto store = [&](int p) {
            if (threadIdx.x < KT) {
                ls[p * KT + threadIdx.x] = CAP ? next_l : next_l * neg_inv_f;     // the scores' products start from -lse / f
                dl[p * KT + threadIdx.x] = -next_d;                               // ... and dp's from -delta
            }
            dma_wait();
        };
        Places<BIAS> pl;
        const int n_all = nqt * a.rep, per = (n_all + a.splits - 1) / a.splits, n0 = split * per, n1 = min(n_all, n0 + per);
        int h = hk * a.rep + n0 / nqt, t = n0 % nqt, seg_t = 0;      // the tile at hand: head, tile of its queries
        if (n0 < n1) {
            load(h, t, 0, true);
            store(0);
        }
        arrived(kf);
        arrived(vf);
        auto tile = [&](int n, auto parity) {
            constexpr int P = decltype(parity)::value;
            const char* qc = smem + P * TB;
            const char* gc = smem + (2 + P) * TB;
            const float* lc = ls + P * KT;
            const float* dc = dl + P * KT;
            if (BIAS && (n == n0 || t == 0 || t == seg_t + a.seg_tiles)) {
                __syncthreads();
                if (n == n0 || t == 0) pl.init(a, a.q_start + t * KT);
                seg_t = t;
                pl.blk = 0;
                const int rows = a.seg_tiles * KT, first = a.q_start + t * KT, p0 = pos_of(first, a.pos_cols);
                stage_window<1>(reinterpret_cast<float*>(win), a, h, pk0, pk1, p0, pos_of(first + rows - 1, a.pos_cols) - p0);
                Places<BIAS>::table(at, a, first, rows, a.q_start + a.Lq - 1);
            }
            __syncthreads();
            const int* at_t = at + (t - seg_t) * KT;
            if (++t == nqt) { t = 0; ++h; }
            if (n + 1 < n1) load(h, t, P ^ 1, false);
            PHASE();
            auto rows16 = [&](const float* v, int u) {                // a value per streamed row of the block, as the products lie
                f32x16 r;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(v + 32 * u + 8 * g + 4 * half);
#pragma unroll
                    for (int i = 0; i < 4; ++i) r[4 * g + i] = x[i];
                }
                return r;
            };
#pragma unroll
            for (int u = 0; u < KT / 32; ++u) {
                f32x16 s = CAP ? splat(0.f) : rows16(lc, u), th, le;
                RowOps<D> f;
                f.load(fr, qc, 32 * u);
                PHASE();
                s = f.times(kf, s);
                f.load(fr, gc, 32 * u);
                f32x16 dp = rows16(dc, u);
                const f32x16 bias = read_bias<BIAS>(win, pl, at_t + 32 * u, half, lane_off);
                if (BIAS) pl.next();
                if (CAP) le = rows16(lc, u);
                PHASE();
                dp = f.times(vf, dp);
                ColOps<D> gt, qt;
                gt.load(fr, gc, 32 * u);
                if (D <= 64) qt.load(fr, qc, 32 * u);
                PHASE();
                to_logits<BIAS, CAP>(s, th, a, bias);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[i] = __builtin_amdgcn_exp2f(CAP ? s[i] - le[i] : s[i]);
                    dp[i] *= s[i];
                    if (CAP) dp[i] *= 1.f - th[i] * th[i];
                }
                if (D > 64) qt.load(fr, qc, 32 * u);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const bf16x8 pf = pack8(s, 8 * g), df = pack8(dp, 8 * g);
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        dv[d] = mfma(gt.f[g][d], pf, dv[d]);
                        dk[d] = mfma(qt.f[g][d], df, dk[d]);
                    }
                }
            }
            if (n + 1 < n1) store(P ^ 1);
        };
        for (int n = n0; n < n1; n += 2) {
            tile(n, std::integral_constant<int, 0>{});
            if (n + 1 < n1) tile(n + 1, std::integral_constant<int, 1>{});
        }
    }
    if (key >= a.Lk) return;
    const bool in = key < len;
    if (a.splits > 1) {                                              // (keys beyond the length: attn_kv_sum_kernel does not read them)
        if (!in) return;
        float* p = a.part + (((int64_t)split * a.B * a.Hkv + bk) * a.Lk + key) * 2 * D + 4 * half;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                *reinterpret_cast<f32x4*>(p + 32 * d + 8 * g) = f32x4{dk[d][4 * g], dk[d][4 * g + 1], dk[d][4 * g + 2], dk[d][4 * g + 3]};
                *reinterpret_cast<f32x4*>(p + D + 32 * d + 8 * g) = f32x4{dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]};
            }
        return;
    }
    unsigned short* ko = a.dk + b * a.dk_sb + (int64_t)key * a.dk_sl + hk * a.dk_sh + 4 * half;
    unsigned short* vo = a.dv + b * a.dv_sb + (int64_t)key * a.dv_sl + hk * a.dv_sh + 4 * half;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            u32x2 w = {pack_bf16x2(dk[d][4 * g] * a.scale, dk[d][4 * g + 1] * a.scale),
                       pack_bf16x2(dk[d][4 * g + 2] * a.scale, dk[d][4 * g + 3] * a.scale)};
            u32x2 x = {pack_bf16x2(dv[d][4 * g], dv[d][4 * g + 1]), pack_bf16x2(dv[d][4 * g + 2], dv[d][4 * g + 3])};
            if (!in) w = x = u32x2{0, 0};
            *reinterpret_cast<u32x2*>(ko + 32 * d + 8 * g) = w;
            *reinterpret_cast<u32x2*>(vo + 32 * d + 8 * g) = x;
        }
}

// dk, dv from the runs' sums: four values a thread, grid (tokens x heads x 2 D / 4 / 256).
__global__ __launch_bounds__(256) void attn_kv_sum_kernel(AttnArgs a, int D) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, per = D / 2;           // groups of four a (sample, head, key)
    const int64_t row = e / per, total = (int64_t)a.B * a.Hkv * a.Lk;
    if (row >= total) return;
    const int c = (int)(e % per) * 4, key = (int)(row % a.Lk), hk = (int)(row / a.Lk % a.Hkv), b = (int)(row / a.Lk / a.Hkv);
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (key < keys_of(a, b)) {
        const float* p = a.part + row * 2 * D + c;
        const int64_t run = total * 2 * D;
        for (int i0 = 0; i0 < a.splits; i0 += 4) {
            f32x4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const f32x4*>(p + min(i0 + j, a.splits - 1) * run);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i0 + j < a.splits)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[k] += v[j][k];
        }
    }
    const bool is_k = c < D;
    const float f = is_k ? a.scale : 1.f;
    unsigned short* o = is_k ? a.dk + b * a.dk_sb + (int64_t)key * a.dk_sl + hk * a.dk_sh + c
                             : a.dv + b * a.dv_sb + (int64_t)key * a.dv_sl + hk * a.dv_sh + c - D;
    *reinterpret_cast<u32x2*>(o) = u32x2{pack_bf16x2(s[0] * f, s[1] * f), pack_bf16x2(s[2] * f, s[3] * f)};
}

// ======================================================================================================= host side
// The bias window of a segment of `tiles` streamed tiles next to 128 owned rows, and (irregular grids) the table of its places.
int64_t span_of(int64_t n, int rows, int cols) {                      // the most P(last) - P(first) can be over n consecutive tokens
    return n <= 1 ? 0 : (n - 1) + (rows > 1 ? (n - 2 + cols) / cols * (cols - 1) : 0);
}
struct Window { int tiles, win_bytes; size_t lds; };
// As many tiles as `budget` bytes hold; tiles 0: not even one.
Window window_of(int bias, int owned, int streamed, int rows, int cols, int KT, int budget) {
    Window w{};
    if (bias == 0 || streamed == 0) return w;
    for (int t = ceil_div(streamed, KT); t > 0; t = t > 64 ? t / 2 : t - 1) {
        const int64_t win = 4 * (span_of(owned < BLK ? owned : BLK, rows, cols) + span_of((int64_t)t * KT, rows, cols) + 1 + WIN_PAD);
        const int64_t all = (win + 15) / 16 * 16 + (bias == 1 ? 4 * (int64_t)t * KT : 0);
        if (all <= budget) { w.tiles = t; w.win_bytes = (int)((win + 15) / 16 * 16); w.lds = (size_t)all; break; }
    }
    return w;
}

int check_desc(const rgbd_attn_desc* d, const char* who) {
    RGBD_REQUIRE(d != nullptr, "%s: null descriptor", who);
    RGBD_REQUIRE(d->B >= 0 && d->H > 0 && d->Hkv > 0 && d->Lq >= 0 && d->Lk >= 0 && d->H % d->Hkv == 0,
                 "%s: bad sizes B=%d H=%d Hkv=%d Lq=%d Lk=%d (Hkv must divide H)", who, d->B, d->H, d->Hkv, d->Lq, d->Lk);
    RGBD_REQUIRE(d->D == 32 || d->D == 64 || d->D == 128, "%s: head size %d is not one of 32, 64, 128", who, d->D);
    // (a launch has fewer than 2^32 threads)
    RGBD_REQUIRE(d->Lq < (1 << 24) && d->Lk < (1 << 24) && (int64_t)d->H * d->D < (1 << 24) &&
                 (int64_t)d->B * d->H * (ceil_div(d->Lq, BLK) + ceil_div(d->Lk, BLK)) < (1 << 23), "%s: too many heads or tokens", who);
    // (the kernels divide by both, and by their quotient)
    RGBD_REQUIRE(d->cap == 0.f || (d->cap >= 1e-12f && d->cap <= 1e12f), "%s: cap must be 0 or in [1e-12, 1e12], got %g", who, d->cap);
    RGBD_REQUIRE(fabsf(d->scale) >= 1e-12f && fabsf(d->scale) <= 1e12f, "%s: |scale| must lie in [1e-12, 1e12], got %g", who, d->scale);
    const int64_t st[9] = {d->q_sb, d->q_sl, d->q_sh, d->k_sb, d->k_sl, d->k_sh, d->v_sb, d->v_sl, d->v_sh};
    for (int i = 0; i < 9; ++i) RGBD_REQUIRE(st[i] % 8 == 0, "%s: strides must be multiples of 8 elements", who);
    for (int i = 1; i < 9; i += 3) RGBD_REQUIRE(st[i] >= 0 && st[i] < (1 << 24), "%s: token strides must lie in [0, 2^24) elements", who);
    RGBD_REQUIRE((((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v) & 15) == 0, "%s: q, k, v must be 16-byte aligned", who);
    if (d->table) {
        RGBD_REQUIRE(d->map != nullptr && d->n_buckets > 0, "%s: a bias table needs its bucket map", who);
        RGBD_REQUIRE(d->rows > 0 && d->cols > 0 && (int64_t)d->rows * d->cols < (1 << 24), "%s: bad grid %d x %d", who, d->rows, d->cols);
        RGBD_REQUIRE(d->rows == 1 || d->cols <= 1024, "%s: a grid of more than one row has at most 1024 columns, got %d", who, d->cols);
        RGBD_REQUIRE(d->q_start >= 0 && (int64_t)d->q_start + d->Lq <= (int64_t)d->rows * d->cols && d->Lk <= (int64_t)d->rows * d->cols,
                     "%s: tokens outside the %d x %d grid (q_start=%d Lq=%d Lk=%d)", who, d->rows, d->cols, d->q_start, d->Lq, d->Lk);
    }
    return 0;
}

AttnArgs args_of(const rgbd_attn_desc* d) {
    AttnArgs a{};
    a.q = (const unsigned short*)d->q; a.k = (const unsigned short*)d->k; a.v = (const unsigned short*)d->v;
    a.q_sb = d->q_sb; a.q_sl = d->q_sl; a.q_sh = d->q_sh;
    a.k_sb = d->k_sb; a.k_sl = d->k_sl; a.k_sh = d->k_sh;
    a.v_sb = d->v_sb; a.v_sl = d->v_sl; a.v_sh = d->v_sh;
    a.table = d->table; a.map = d->map; a.lengths = d->lengths;
    a.B = d->B; a.H = d->H; a.Hkv = d->Hkv; a.rep = d->H / d->Hkv; a.Lq = d->Lq; a.Lk = d->Lk;
    a.rows = d->table ? d->rows : 1; a.cols = d->table ? d->cols : 1 << 24; a.q_start = d->table ? d->q_start : 0;
    a.pos_cols = a.rows > 1 ? a.cols : 1 << 30; a.n_buckets = d->n_buckets;
    a.scale = d->scale; a.cap = d->cap;
    a.n_qb = ceil_div(d->Lq, BLK); a.n_kb = ceil_div(d->Lk, BLK); a.kt = kt_of(d->D); a.n_kt = ceil_div(d->Lk, a.kt);
    a.lse = d->lse;
    return a;
}

// 0 no bias; 2 regular, 1 irregular grid (struct Places) for streamed tokens that begin at `first`.
int bias_mode(const rgbd_attn_desc* d, int first) {
    if (!d->table) return 0;
    const bool wide = d->rows == 1 || (d->cols % 32 == 0 && first % 32 == 0);
    const bool narrow = (d->cols == 4 || d->cols == 8 || d->cols == 16) && first % d->cols == 0;
    return wide || narrow ? 2 : 1;
}

#define BY_BIAS_CAP(KERNEL, D, ...)                                                                                     \
    do {                                                                                                                \
        if (cap) {                                                                                                      \
            if (bias == 0) LAUNCH((KERNEL<D, 0, true __VA_ARGS__>));                                                    \
            else if (bias == 1) LAUNCH((KERNEL<D, 1, true __VA_ARGS__>));                                               \
            else LAUNCH((KERNEL<D, 2, true __VA_ARGS__>));                                                              \
        } else {                                                                                                        \
            if (bias == 0) LAUNCH((KERNEL<D, 0, false __VA_ARGS__>));                                                   \
            else if (bias == 1) LAUNCH((KERNEL<D, 1, false __VA_ARGS__>));                                              \
            else LAUNCH((KERNEL<D, 2, false __VA_ARGS__>));                                                             \
        }                                                                                                               \
    } while (0)
#define LAUNCH(K)                                                                                                       \
    do {                                                                                                                \
        if (!rgbd_reserve_lds((const void*)&K, (int)lds)) { rgbd_set_error("attention: cannot reserve %d bytes of LDS", (int)lds); return -2; } \
        hipLaunchKernelGGL(K, dim3(grid), dim3(256), lds, s, a);                                                        \
    } while (0)

template <int D> int launch_fwd(const AttnArgs& a, int bias, bool cap, bool fine, unsigned grid, size_t lds, hipStream_t s) {
    if (!fine) { BY_BIAS_CAP(attn_fwd_kernel, D, , false); return 0; }
    if (cap) { if (bias == 1) LAUNCH((attn_fwd_kernel<D, 1, true, true>)); else LAUNCH((attn_fwd_kernel<D, 2, true, true>)); }
    else { if (bias == 1) LAUNCH((attn_fwd_kernel<D, 1, false, true>)); else LAUNCH((attn_fwd_kernel<D, 2, false, true>)); }
    return 0;
}
template <int D> int launch_dq(const AttnArgs& a, int bias, bool cap, int dt, unsigned grid, size_t lds, hipStream_t s) {
    if (dt == DT_NONE) { BY_BIAS_CAP(attn_dq_kernel, D, , DT_NONE); return 0; }
    if (dt == DT_BLOCKS) {                                            // 32 aligned tokens in a row: four are too
        if (cap) LAUNCH((attn_dq_kernel<D, 2, true, DT_BLOCKS>));
        else LAUNCH((attn_dq_kernel<D, 2, false, DT_BLOCKS>));
        return 0;
    }
    if (cap) { if (bias == 1) LAUNCH((attn_dq_kernel<D, 1, true, DT_DIAGONALS>)); else LAUNCH((attn_dq_kernel<D, 2, true, DT_DIAGONALS>)); }
    else { if (bias == 1) LAUNCH((attn_dq_kernel<D, 1, false, DT_DIAGONALS>)); else LAUNCH((attn_dq_kernel<D, 2, false, DT_DIAGONALS>)); }
    return 0;
}
template <int D> int launch_dkv(const AttnArgs& a, int bias, bool cap, unsigned grid, size_t lds, hipStream_t s) {
    BY_BIAS_CAP(attn_dkv_kernel, D);
    return 0;
}

// Few (query, head) pairs over many keys: the number of runs the keys are cut into, 0 for the other form.  Both read a key block once a
// workgroup, but the other form does it once for every query head.  us for one query, 4 samples, 8 query heads on 2 of 64, this form / the other
// (joins included): 256 keys 6.0 / 7.1, 512 keys 9.6 / 10.1, 1024 keys 9.7 / 13.4; 64 samples of 512 keys 10.4 / 14.5; 4 queries, 256 samples of 1024
// keys (one run) 27 / 69; 4 samples of 16384 keys, 8 on 2 of 128: 21 / 42.  Where no head shares keys the two are alike (256 samples of 1024 keys, 8 heads
// of 64: 107 / 104), and up to 256 keys one launch of the other form is within 1 us.
int few_splits(const rgbd_attn_desc* d) {
    if ((int64_t)d->H / d->Hkv * d->Lq > 32 || d->Lk <= 256 || (int64_t)d->B * d->H * d->Lq >= 1 << 20) return 0;
    const int64_t groups = (int64_t)d->B * d->Hkv, want = d->D == 128 ? 256 : 512;   // workgroups that fit the chip at once (LDS)
    int64_t s = (want + groups - 1) / groups;
    const int64_t most = ceil_div(d->Lk, 32 * 8);                     // two blocks for every wave
    if (s > most) s = most;
    if (s > MAX_SPLITS) s = MAX_SPLITS;
    return (int)(s < 1 ? 1 : s);
}
template <int D> int launch_few(const AttnArgs& a, bool bias, bool cap, hipStream_t s) {
    const unsigned grid = (unsigned)a.B * a.Hkv * a.splits;
    const size_t lds = 4 * 4 * 32 * 2 * D > 4 * (4 * 32 * (D + 1) + 256) ? 4 * 4 * 32 * 2 * D : 4 * (4 * 32 * (D + 1) + 256);
    if (bias) { if (cap) LAUNCH((attn_few_kernel<D, true, true>)); else LAUNCH((attn_few_kernel<D, true, false>)); }
    else { if (cap) LAUNCH((attn_few_kernel<D, false, true>)); else LAUNCH((attn_few_kernel<D, false, false>)); }
    if (a.splits > 1) hipLaunchKernelGGL((attn_few_join_kernel<D>), dim3(a.B * a.H * a.Lq), dim3(512), 0, s, a);
    return 0;
}

// Runs of query tiles for dk, dv: as many as fill the chip once (one workgroup a compute unit at head size 128, two at 64, three at 32:
// registers), of at least eight tiles each.  The runs' sums are written and read once more in fp32, which two runs of small heads do
// not earn back.  us cut / whole, the second launch included: 8 x 1024, 8 query heads on 2 of 64 (4 runs) 51 / 90; 1 x 2048, 4 on 2 of 64
// (8 runs) 25 / 87; 5 x 713, 6 on 2 of 32 (4 runs) 20 / 36; 2 x 4096, 4 on 2 of 128 (4 runs) 222 / 386; 2 x 2048 x 4 of 128 (2 runs) 76 / 102;
// but 4 x 2048 x 4 of 64 (2 runs) 52 / 49, 12 x 1024 x 4 of 32 (2 runs) 33 / 25, 4 x 1024 x 4 of 64 in 4 runs of 4 tiles 26 / 24.
int kv_splits(const rgbd_attn_desc* d) {
    const int64_t groups = (int64_t)d->B * d->Hkv * ceil_div(d->Lk, BLK), want = d->D == 128 ? 256 : d->D == 64 ? 512 : 768;
    if (groups == 0) return 1;
    int64_t s = want / groups;
    const int64_t most = (int64_t)d->H / d->Hkv * ceil_div(d->Lq, kt_of(d->D)) / 8;
    if (s > most) s = most;
    if (s > 64) s = 64;
    return s < (d->D == 128 ? 2 : 3) ? 1 : (int)s;
}

// Runs of keys for the forward pass and dq where their workgroups leave compute units idle: as many as fill the chip twice over, of at least
// `least` tiles each (6 forward, 2 for dq); with a workgroup on every compute unit already, only from 32 tiles on.  us cut (with the launch
// that joins the runs) / whole, forward, dq: 64x64 x 2 heads of 64, one sample (8 runs) 39 / 102, 41 / 118, two samples (4 runs) 55 / 104,
// 60 / 121; 4 x 32x32 x 4 of 64, capped (2 and 4 runs) 29 / 38, 33 / 45; 5 x 713 x 6 of 32 (2 runs) 29 / 31, 49 / 69; line (2 runs) 145 / 164,
// 148 / 172; 8 x 16x16 x 4 of 64 (2 runs for dq) 21 / 29; but 8 x 32x32 x 4 of 64, 256 workgroups of 16 tiles, 36 / 33, 42 / 41.
int key_runs(const rgbd_attn_desc* d, int least) {
    const int64_t groups = (int64_t)d->B * d->H * ceil_div(d->Lq, BLK), tiles = ceil_div(d->Lk, kt_of(d->D));
    if (groups == 0 || (groups >= 256 && tiles < 32)) return 1;
    int64_t s = 512 / groups;
    if (s > tiles / least) s = tiles / least;
    if (s > 64) s = 64;
    return (int)(s < 1 ? 1 : s);
}
int fwd_splits(const rgbd_attn_desc* d) { return key_runs(d, 6); }
int dq_splits(const rgbd_attn_desc* d) { return key_runs(d, 2); }

// Floats of the backward workspace: delta, the table's partials of `chunk` samples (PART_FLOATS at most, or one sample), what the first
// reduction leaves of them, the runs' dk and dv.
constexpr int64_t PART_FLOATS = 128 << 20;
struct BwdSizes { int64_t delta, part, sums, kv, dq; int mode, dq_runs, chunk, span, n_dist, d0, q_row0, q_rows, k_rows, gq, gk; };
BwdSizes bwd_sizes(const rgbd_attn_desc* d, bool dt) {
    BwdSizes z{};
    z.chunk = d->B;
    z.delta = ((int64_t)d->B * d->H * d->Lq + 3) / 4 * 4;
    const int ks = kv_splits(d);
    z.kv = ks > 1 ? (int64_t)ks * d->B * d->Hkv * d->Lk * 2 * d->D : 0;
    z.dq_runs = dq_splits(d);
    z.dq = z.dq_runs > 1 ? (int64_t)z.dq_runs * d->B * d->Lq * d->H * d->D : 0;
    if (!dt || d->Lq == 0 || d->Lk == 0) return z;
    const int KT = kt_of(d->D), n_qb = ceil_div(d->Lq, BLK), n_kt = ceil_div(d->Lk, KT);
    if (d->rows == 1 || (d->cols % 32 == 0 && d->q_start % d->cols == 0)) {
        z.mode = DT_BLOCKS;
        z.part = (int64_t)d->H * n_qb * 4 * n_kt * (KT / 32) * 64;
        z.gq = d->rows == 1 ? n_qb * 4 : d->cols / 32;
        z.gk = d->rows == 1 ? n_kt * (KT / 32) : d->cols / 32;
        z.q_row0 = d->rows == 1 ? 0 : d->q_start / d->cols;
        z.q_rows = d->rows == 1 ? 1 : ceil_div(d->Lq, d->cols);
        z.k_rows = d->rows == 1 ? 1 : ceil_div(d->Lk, d->cols);
        z.sums = (int64_t)d->H * (z.q_rows + z.k_rows - 1) * (z.gq + z.gk - 1) * 64;
    } else {
        z.mode = DT_DIAGONALS;
        z.span = n_kt * KT + BLK;
        z.part = (int64_t)d->H * n_qb * z.dq_runs * 2 * z.span;
        z.d0 = d->q_start - (n_kt * KT - 1);                          // distances from there to q_start + n_qb * BLK - 1
        z.n_dist = d->q_start + n_qb * BLK - z.d0;
        z.sums = (int64_t)d->H * 2 * z.n_dist;
    }
    // (a 64 x 64 map's partials are 4 MB a sample and head; above 512 MB dq runs over as many samples at a time as fit in that, one at least)
    const int64_t fit = z.part < PART_FLOATS ? PART_FLOATS / z.part : 1;
    z.chunk = fit < d->B ? (int)fit : d->B;
    z.part *= z.chunk;
    z.sums = (z.sums + 3) / 4 * 4;
    return z;
}

}  // namespace

extern "C" int64_t rgbd_attention_fwd_workspace(const rgbd_attn_desc* d) {
    if (check_desc(d, "rgbd_attention_fwd_workspace")) return -1;
    if (d->B == 0 || d->Lq == 0) return 0;
    const int few = few_splits(d), runs = few ? 1 : fwd_splits(d);
    if (few > 1) return (int64_t)d->B * d->Hkv * few * 32 * (d->D + 2);
    return runs > 1 ? (int64_t)runs * d->B * d->Lq * d->H * (d->D + 2) : 0;
}

extern "C" int rgbd_attention_fwd(const rgbd_attn_desc* d, void* o, void* o_lo, float* workspace, void* stream) {
    if (check_desc(d, "rgbd_attention_fwd")) return -1;
    if (d->B == 0 || d->Lq == 0) return 0;
    RGBD_REQUIRE(d->q && o && (d->Lk == 0 || (d->k && d->v)), "rgbd_attention_fwd: null pointer");
    RGBD_REQUIRE((((uintptr_t)o | (uintptr_t)o_lo) & 15) == 0, "rgbd_attention_fwd: outputs must be 16-byte aligned");
    AttnArgs a = args_of(d);
    a.out = (unsigned short*)o;
    a.out_lo = (unsigned short*)o_lo;
    const bool cap = d->cap > 0.f;
    hipStream_t s = (hipStream_t)stream;
    a.splits = few_splits(d);
    if (a.splits) {
        RGBD_REQUIRE(workspace || a.splits == 1, "rgbd_attention_fwd: null workspace");
        a.part = workspace;
        const int rc = d->D == 32 ? launch_few<32>(a, d->table, cap, s) : d->D == 64 ? launch_few<64>(a, d->table, cap, s) : launch_few<128>(a, d->table, cap, s);
        if (rc) return rc;
        RGBD_CHECK_LAUNCH("rgbd_attention_fwd (few rows)");
        return 0;
    }
    const int bias = bias_mode(d, 0);
    const Window w = window_of(bias, d->Lq, d->Lk, a.rows, a.cols, a.kt, WIN_FWD);
    RGBD_REQUIRE(bias == 0 || d->Lk == 0 || w.tiles > 0, "rgbd_attention_fwd: the bias of one tile does not fit (%d x %d grid)", a.rows, a.cols);
    a.seg_tiles = w.tiles;
    a.win_bytes = w.win_bytes;
    a.splits = fwd_splits(d);
    a.run_floats = (int64_t)d->B * d->Lq * d->H * d->D;
    a.runs = workspace;
    a.part = workspace + a.splits * a.run_floats;
    RGBD_REQUIRE(a.splits == 1 || (workspace && ((uintptr_t)workspace & 15) == 0), "rgbd_attention_fwd: null or unaligned workspace");
    const size_t lds = 4 * a.kt * 2 * d->D + w.lds;
    const unsigned grid = (unsigned)a.B * a.H * a.n_qb * a.splits;
    const bool fine = d->fine && bias;
    const int rc = d->D == 32   ? launch_fwd<32>(a, bias, cap, fine, grid, lds, s)
                   : d->D == 64 ? launch_fwd<64>(a, bias, cap, fine, grid, lds, s)
                                : launch_fwd<128>(a, bias, cap, fine, grid, lds, s);
    if (rc) return rc;
    if (a.splits > 1) hipLaunchKernelGGL(attn_join_kernel, dim3((unsigned)((a.run_floats / 4 + 255) / 256)), dim3(256), 0, s, a, d->D);
    RGBD_CHECK_LAUNCH("rgbd_attention_fwd");
    return 0;
}

extern "C" int64_t rgbd_attention_bwd_workspace(const rgbd_attn_desc* d, int want_table) {
    if (check_desc(d, "rgbd_attention_bwd_workspace")) return -1;
    const BwdSizes z = bwd_sizes(d, want_table && d->table);
    return z.delta + z.part + z.sums + z.kv + z.dq + 4;
}

extern "C" int rgbd_attention_bwd(const rgbd_attn_desc* d, const rgbd_attn_grad* g, float* workspace, void* stream) {
    const char* who = "rgbd_attention_bwd";
    if (check_desc(d, who)) return -1;
    RGBD_REQUIRE(g != nullptr, "%s: null gradient descriptor", who);
    const bool dt = g->dtable != nullptr;
    RGBD_REQUIRE(!dt || (d->table && g->order && g->start), "%s: the table's gradient needs the table and its buckets' offsets", who);
    hipStream_t s = (hipStream_t)stream;
    const bool empty = d->B == 0 || d->Lq == 0 || d->Lk == 0;
    if (dt && empty) {
        const hipError_t e = rgbd_zero_async(g->dtable, (size_t)d->H * d->n_buckets * 4, s);
        RGBD_REQUIRE(e == hipSuccess, "%s: %s", who, hipGetErrorString(e));
    }
    if (d->B == 0) return 0;
    RGBD_REQUIRE(workspace && (d->Lq == 0 || (d->q && d->lse && g->d_o && g->o && g->o_lo && g->dq)) &&
                 (d->Lk == 0 || (d->k && d->v && g->dk && g->dv)), "%s: null pointer", who);
    const int64_t st[9] = {g->dq_sb, g->dq_sl, g->dq_sh, g->dk_sb, g->dk_sl, g->dk_sh, g->dv_sb, g->dv_sl, g->dv_sh};
    for (int i = 0; i < 9; ++i) RGBD_REQUIRE(st[i] % 8 == 0, "%s: strides must be multiples of 8 elements", who);
    RGBD_REQUIRE((((uintptr_t)g->d_o | (uintptr_t)g->o | (uintptr_t)g->o_lo | (uintptr_t)g->dq | (uintptr_t)g->dk | (uintptr_t)g->dv |
                   (uintptr_t)workspace) & 15) == 0, "%s: buffers must be 16-byte aligned", who);
    AttnArgs a = args_of(d);
    a.d_o = (const unsigned short*)g->d_o; a.o = (const unsigned short*)g->o; a.o_lo = (const unsigned short*)g->o_lo;
    a.dq = (unsigned short*)g->dq; a.dk = (unsigned short*)g->dk; a.dv = (unsigned short*)g->dv;
    a.dq_sb = g->dq_sb; a.dq_sl = g->dq_sl; a.dq_sh = g->dq_sh;
    a.dk_sb = g->dk_sb; a.dk_sl = g->dk_sl; a.dk_sh = g->dk_sh;
    a.dv_sb = g->dv_sb; a.dv_sl = g->dv_sl; a.dv_sh = g->dv_sh;
    a.dtable = g->dtable;
    const BwdSizes z = bwd_sizes(d, dt);
    a.delta = workspace;
    a.part = workspace + z.delta;
    a.span = z.span;
    float* sums = a.part + z.part;
    const bool cap = d->cap > 0.f;

    if (d->Lq > 0) {
        const int bias = bias_mode(d, 0);
        const Window w = window_of(bias, d->Lq, d->Lk, a.rows, a.cols, a.kt, z.mode ? WIN_DQ : WIN_FWD);
        RGBD_REQUIRE(bias == 0 || d->Lk == 0 || w.tiles > 0, "%s: the bias of one tile does not fit (%d x %d grid)", who, a.rows, a.cols);
        a.seg_tiles = w.tiles;
        a.win_bytes = w.win_bytes;
        const size_t lds = 4 * a.kt * 2 * d->D + dt_lds(z.mode, d->D) + w.lds;
        a.splits = z.dq_runs;
        a.run_floats = (int64_t)d->B * d->Lq * d->H * d->D;
        a.runs = workspace + z.delta + z.part + z.sums + z.kv;
        for (int b0 = 0; b0 < d->B; b0 += z.chunk) {
            AttnArgs c = a;
            c.B = d->B - b0 < z.chunk ? d->B - b0 : z.chunk;
            const int64_t rows = (int64_t)b0 * a.H * a.Lq;
            c.q += b0 * a.q_sb; c.k += b0 * a.k_sb; c.v += b0 * a.v_sb; c.dq += b0 * a.dq_sb;
            c.d_o += rows * d->D; c.o += rows * d->D; c.o_lo += rows * d->D;
            c.lse += rows; c.delta += rows; c.runs += rows * d->D;
            if (c.lengths) c.lengths += b0;
            const unsigned grid = (unsigned)c.B * a.H * a.n_qb * a.splits;
            const int rc = d->D == 32   ? launch_dq<32>(c, bias, cap, z.mode, grid, lds, s)
                           : d->D == 64 ? launch_dq<64>(c, bias, cap, z.mode, grid, lds, s)
                                        : launch_dq<128>(c, bias, cap, z.mode, grid, lds, s);
            if (rc) return rc;
            RGBD_CHECK_LAUNCH("rgbd_attention_bwd (dq)");
            if (z.mode == DT_BLOCKS)
                hipLaunchKernelGGL(attn_block_sums_kernel, dim3((z.q_rows + z.k_rows - 1) * (z.gq + z.gk - 1), a.H), dim3(1024), 0, s, c, sums,
                                   b0 > 0, z.q_rows, z.k_rows, z.gq, z.gk);
            else if (z.mode == DT_DIAGONALS)
                hipLaunchKernelGGL(attn_dist_kernel, dim3(ceil_div(z.n_dist, 64), 2 * a.H), dim3(1024), 0, s, c, sums, b0 > 0, z.n_dist, z.d0);
        }
        if (a.splits > 1)
            hipLaunchKernelGGL(attn_dq_sum_kernel, dim3((unsigned)((a.run_floats / 4 + 255) / 256)), dim3(256), 0, s, a, d->D);
        if (z.mode == DT_BLOCKS)
            hipLaunchKernelGGL(attn_block_bucket_kernel, dim3(a.n_buckets, a.H), dim3(256), 0, s, a, sums, g->order, g->start, z.q_row0, z.k_rows,
                               z.q_rows, z.gq, z.gk);
        else if (z.mode == DT_DIAGONALS)
            hipLaunchKernelGGL(attn_dist_bucket_kernel, dim3(a.n_buckets, a.H), dim3(256), 0, s, a, sums, g->order, g->start, z.n_dist, z.d0);
        RGBD_CHECK_LAUNCH("rgbd_attention_bwd (table)");
    }
    if (d->Lk > 0) {
        const int bias = d->Lq > 0 ? bias_mode(d, d->q_start) : 0;
        const Window w = window_of(bias, d->Lk, d->Lq, a.rows, a.cols, a.kt, WIN_FWD);
        RGBD_REQUIRE(bias == 0 || w.tiles > 0, "%s: the bias of one tile does not fit (%d x %d grid)", who, a.rows, a.cols);
        a.seg_tiles = w.tiles;
        a.win_bytes = w.win_bytes;
        const size_t lds = 4 * a.kt * 2 * d->D + 4 * a.kt * 4 + w.lds;
        a.splits = kv_splits(d);
        a.part = workspace + z.delta + z.part + z.sums;
        const unsigned grid = (unsigned)a.B * a.Hkv * a.n_kb * a.splits;
        const int rc = d->D == 32 ? launch_dkv<32>(a, bias, cap, grid, lds, s) : d->D == 64 ? launch_dkv<64>(a, bias, cap, grid, lds, s)
                                                                                            : launch_dkv<128>(a, bias, cap, grid, lds, s);
        if (rc) return rc;
        if (a.splits > 1)
            hipLaunchKernelGGL(attn_kv_sum_kernel, dim3((unsigned)(((int64_t)a.B * a.Hkv * a.Lk * (d->D / 2) + 255) / 256)), dim3(256), 0, s, a, d->D);
        RGBD_CHECK_LAUNCH("rgbd_attention_bwd (dk, dv)");
    }
    return 0;
}
