// Losses over a large number of classes, forward and backward, without the logits in memory: softmax cross entropy of a linear
// head, the additive angular margin of models/SoftMaxLoss.py:99-138 on cosines with several weight rows to a class, and the
// divergence from a teacher of which the largest logits are kept.
//
// With z_nc = scale * x_n . w_c, o_n = log of the sum of exp(z_nc) over the classes that are not the row's target t:
//   loss_n = log(1 + exp(o_n - z_nt)),   dz_nc = P_nc - [c = t],   P = softmax(z),   dx = dz W,   dW = dz^T x.
// The target is kept out of the sum so that neither the loss of a row that is nearly certain nor its P_nt - 1 is the difference
// of two numbers that are nearly the same.  The forward is one product x W^T whose tiles leave as a maximum and a sum of
// exponentials to a row (logits_kernel), and a kernel that puts a row's tiles together (finish_kernel).  The backward works the
// logits out again, a range of classes at a time, rounds dz to the operands' type - what a head that keeps its logits would have
// handed its products - and multiplies it twice (products_kernel): by W for dx, transposed by x for dW.
#include <atomic>
#include <cmath>
#include <type_traits>

#include "na1d_encoder.h"

namespace na1d {
namespace loss {

using namespace enc;

// =============================================================================
// Tiles
// =============================================================================
// Every operand comes through LDS in pieces of 64 rows of 128 bytes, written there by the loads themselves; what a step of 64 of
// the contraction needs of a tile is extent / 64 such pieces.  An operand whose contraction runs along its rows in memory has
// the tile's rows (64 to a piece) and 64 values of each; one whose contraction runs from row to row ("turned") has 64 rows of
// the contraction and 64 of the tile's columns, which come out of LDS transposed (ds_read_b64_tr_b16).  The 16-byte units of a
// row are XOR-swizzled by three bits of its number, by which the sixteen rows of a row operand's read, and the rows {0-3, 8-11} or
// {4-7, 12-15} of half a wave's transposed read, spread over all banks; no one choice of bits does for both (an operand's
// read takes 4 cycles and a transposed one 2, with the other's choice 8 and 4; the kernels' counters show no conflicts).
constexpr int kStep = 64;                     // of the contraction
constexpr int kPieceRow = 2 * kStep;          // bytes
constexpr int kPiece = 64 * kPieceRow;
template <bool TURNED> __device__ inline int swizzle(int row) {
    return TURNED ? ((row >> 3) & 1) << 2 | ((row >> 1) & 1) << 1 | ((row >> 2) & 1) : (row >> 1) & 7;
}

// Where an operand's tile comes from.  All members but the lane's are wave-uniform.
template <int EXTENT, int NW, bool TURNED> struct Source {
    static constexpr int kLoads = EXTENT * kPieceRow / kChunk / NW;          // of a wave in a step
    static constexpr int kBytes = EXTENT * kPieceRow;
    static_assert(EXTENT * kPieceRow % (kChunk * NW) == 0 && (!TURNED || EXTENT % 64 == 0) && NW % 4 == 0, "whole chunks");
    const char *at;          // first byte of the tile
    int64_t bytes, step;     // from there to the end of what may be read; from one step to the next
    int pitch, width;        // bytes: from row to row; of a row, from the tile's first one on
    int lane_at, unit;       // this lane's place in chunk `wave`
    // `rows`: rows that exist from the tile's first one on (of the tile, or, turned, of the contraction)
    __device__ inline void init(const char *first, int64_t rows, int64_t row_pitch, int64_t row_width, int wave, int lane) {
        at = first;
        pitch = (int)row_pitch;
        width = (int)row_width;
        bytes = rows > 0 ? (rows - 1) * row_pitch + row_width : 0;
        step = TURNED ? kStep * row_pitch : kPieceRow;
        unit = ((lane & 7) ^ swizzle<TURNED>(8 * wave + (lane >> 3))) * 16;          // chunks of a wave are 32 rows apart, or 64
        lane_at = (8 * wave + (lane >> 3)) * pitch + unit;
    }
    __device__ inline void load(LDS_PTR(char) to, int s, int wave) const {
        const int64_t left = bytes - s * step;
        const Rsrc src = make_rsrc(at + s * step, (int)(left < 0 ? 0 : left < (1 << 30) ? left : (1 << 30)));
        const int from = TURNED || s * kPieceRow + unit < width ? lane_at : kNowhere;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int c = j * NW;                                            // + wave
            int off = from;
            if constexpr (TURNED) {
                off += c % 8 * 8 * pitch + c / 8 * kPieceRow;
                if (c / 8 * kPieceRow + unit >= width) off = kNowhere;
            } else {
                off += c * 8 * pitch;
            }
            load_to_lds<16, kReadShared>(src, to + (c + wave) * kChunk, off);
        }
    }
};
// A tile of weight rows of which K belong to a class: the 16-row tiles of a wave (MT of them, a multiple of K) are K of the same 16
// classes, one behind the other, so that a lane has all of a class's products.  (Row operands only.)
template <int EXTENT, int NW, int MT, int K> struct ClassSource {
    static constexpr int kLoads = EXTENT * kPieceRow / kChunk / NW, kBytes = EXTENT * kPieceRow;
    static_assert(EXTENT * kPieceRow % (kChunk * NW) == 0 && NW % 4 == 0 && MT % K == 0, "whole chunks, whole classes");
    const char *at;
    int64_t bytes;
    int width, lane_at, unit;
    int chunk_at[kLoads];
    // `classes`: those that exist from the tile's first one on, row_pitch bytes from row to row
    __device__ inline void init(const char *first, int64_t classes, int64_t row_pitch, int64_t row_width, int wave, int lane) {
        const int pitch = (int)row_pitch * K;
        at = first;
        width = (int)row_width;
        bytes = classes > 0 ? (classes - 1) * (int64_t)pitch + (K - 1) * row_pitch + row_width : 0;
        unit = ((lane & 7) ^ swizzle<false>(8 * wave + (lane >> 3))) * 16;
        lane_at = (lane >> 3) * pitch + unit;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int chunk = j * NW + wave, tile = chunk >> 1, of_wave = tile % MT;
            chunk_at[j] = (tile / MT * (16 * MT / K) + of_wave / K * 16 + (chunk & 1) * 8) * pitch + of_wave % K * (int)row_pitch;
        }
    }
    __device__ inline void load(LDS_PTR(char) to, int s, int wave) const {
        const int64_t left = bytes - s * kPieceRow;
        const Rsrc src = make_rsrc(at + s * kPieceRow, (int)(left < 0 ? 0 : left < (1 << 30) ? left : (1 << 30)));
        const int from = s * kPieceRow + unit < width ? lane_at : kNowhere;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) load_to_lds<16, kReadShared>(src, to + (j * NW + wave) * kChunk, from + chunk_at[j]);
    }
};
// Operands of the 16 x 16 x 32 product out of such a tile: 16 of its extent (number t) and half h of the step's 64.
template <bool TURNED> struct Reader;
template <> struct Reader<false> {
    int lane_at;
    __device__ inline void init(int n, int g) { lane_at = n * kPieceRow + ((g ^ swizzle<false>(n)) << 4); }
    __device__ inline u32x4 read(LDS_PTR(char) tile, int t, int h) const {
        return *reinterpret_cast<LDS_PTR(u32x4)>(tile + t * 16 * kPieceRow + (lane_at ^ h * 64));
    }
};
template <> struct Reader<true> {
    int lane_at;
    __device__ inline void init(int n, int g) {
        const int row = 8 * g + (n >> 2);
        lane_at = row * kPieceRow + ((((n & 3) >> 1) ^ swizzle<true>(row)) << 4) + 8 * (n & 1);
    }
    __device__ inline u32x4 read(LDS_PTR(char) tile, int t, int h) const {
        LDS_PTR(char) p = tile + (t >> 2) * kPiece + h * 32 * kPieceRow;
        const int at = lane_at ^ (t & 3) * 32;
        const u32x2 a = read_tr(p + at), b = read_tr(p + 4 * kPieceRow + (at ^ 16));
        return u32x4{a.x, a.y, b.x, b.y};
    }
};

// A workgroup's tile: WM x WN waves of MT x NT products of 16 x 16; STAGES steps of operands in LDS.
template <int MT_, int NT_, int WM_, int WN_, int STAGES_> struct Shape {
    static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, STAGES = STAGES_;
    static constexpr int kWavesOf = WM * WN, kThreadsOf = 64 * kWavesOf, BM = 16 * MT * WM, BN = 16 * NT * WN;
    static constexpr int kSlot = (BM + BN) * kPieceRow, kLds = STAGES * kSlot;
};
template <bool MAX> __device__ inline float joined(float x, float y) { return MAX ? __builtin_fmaxf(x, y) : x + y; }
template <bool MAX = false> __device__ inline float sum_of_16(float x) {        // (or the largest) over the lanes of one g
    x = joined<MAX>(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0xb1, 0xf, 0xf, true)));
    x = joined<MAX>(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x4e, 0xf, 0xf, true)));
    x = joined<MAX>(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x141, 0xf, 0xf, true)));
    return joined<MAX>(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x140, 0xf, 0xf, true)));
}
template <bool MAX> __device__ inline float over_wave(float x) {
    float a, b;
    swap_rows16(sum_of_16<MAX>(x), a, b);
    swap_rows32(joined<MAX>(a, b), a, b);
    return joined<MAX>(a, b);
}
__device__ inline void turn_over() { asm volatile("s_barrier" ::: "memory"); }
template <int COUNT> __device__ inline void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COUNT) : "memory"); }

// acc[i][j] += A[16 of M, number wm * MT + i] . B[16 of N, number wn * NT + j]^T; lane (n, g) holds M 4g .. 4g + 3 and N n.
//
// Four waves: a step's operands are asked for STAGES - 1 steps ahead; one barrier to a step.  Two workgroups to a CU overlap.
template <class DT, class S, class A, class B, class RA, class RB>
__device__ inline void accumulate_ahead(f32x4 (&acc)[S::MT][S::NT], const A &a, const B &b, const RA &ra, const RB &rb, int steps, LDS_PTR(char) lds, int wave, int wm,
                                        int wn) {
    constexpr int kAhead = S::STAGES - 1, kLoads = A::kLoads + B::kLoads;
    auto stage = [&](int s, int slot) {
        a.load(lds + slot * S::kSlot, s, wave);
        b.load(lds + slot * S::kSlot + A::kBytes, s, wave);
    };
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
        if (s < steps) stage(s, s);
    int slot = 0, next = kAhead;
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        if (s + kAhead <= steps)
            wait_loads<(kAhead - 1) * kLoads>();
        else
            wait_loads<0>();
        barrier_lds();                       // everyone's loads of this step are there, everyone is done with the step before
        if (s + kAhead < steps) stage(s + kAhead, next);
        LDS_PTR(char) from = lds + slot * S::kSlot;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 x[S::MT], y[S::NT];
#pragma unroll
            for (int i = 0; i < S::MT; ++i) x[i] = ra.read(from, wm * S::MT + i, h);
#pragma unroll
            for (int j = 0; j < S::NT; ++j) y[j] = rb.read(from + A::kBytes, wn * S::NT + j, h);
#pragma unroll
            for (int i = 0; i < S::MT; ++i)
#pragma unroll
                for (int j = 0; j < S::NT; ++j) acc[i][j] = Mma<DT>::k32(x[i], y[j], acc[i][j]);
        }
        slot = slot + 1 == S::STAGES ? 0 : slot + 1;
        next = next + 1 == S::STAGES ? 0 : next + 1;
    }
}

// Eight waves, one workgroup to a CU: two groups of four, a wave of each on every SIMD, which take turns.  A step is four quarters
// of MT / 2 x NT products; while one group multiplies, the other reads the next quarter's operands out of LDS and asks for the next
// step's from memory.  A group's reads have returned before the barrier that ends its turn, so its turn at the next step may write
// where the other group's last turn has read; a step's loads are waited for at the end of its last reading turn, a barrier before
// anyone reads them.  16384 x 1024 by 8192 x 1024 rows, with the softmax: 1130 TFLOP/s (four waves in tiles of 128 x 128: 960; eight
// waves that read and multiply as the compiler orders it: 1085).
template <class DT, class S, class A, class B, class RA, class RB>
__device__ inline void accumulate_in_turns(f32x4 (&acc)[S::MT][S::NT], const A &a, const B &b, const RA &ra, const RB &rb, int steps, LDS_PTR(char) lds, int wave, int wm,
                                           int wn) {
    static_assert(S::kWavesOf == 8 && S::STAGES == 2 && S::MT % 2 == 0, "two groups of four waves, two steps in LDS");
    constexpr int kHalf = S::MT / 2;
    if (steps <= 0) return;
    a.load(lds, 0, wave);
    b.load(lds + A::kBytes, 0, wave);
    wait_loads<0>();
    barrier_lds();
    if (wave >= 4) turn_over();
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        LDS_PTR(char) from = lds + (s & 1) * S::kSlot;
        LDS_PTR(char) to = lds + (~s & 1) * S::kSlot;
        u32x4 y[S::NT];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int h = c >> 1, i0 = (c & 1) * kHalf;
            u32x4 x[kHalf];
            if ((c & 1) == 0) {
#pragma unroll
                for (int j = 0; j < S::NT; ++j) y[j] = rb.read(from + A::kBytes, wn * S::NT + j, h);
            }
#pragma unroll
            for (int i = 0; i < kHalf; ++i) x[i] = ra.read(from, wm * S::MT + i0 + i, h);
            __builtin_amdgcn_sched_barrier(0);
            if (c == 0 && s + 1 < steps) b.load(to + A::kBytes, s + 1, wave);
            if (c == 1 && s + 1 < steps) a.load(to, s + 1, wave);
            if (c == 3) wait_loads<0>();
            barrier_lds();
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < kHalf; ++i)
#pragma unroll
                for (int j = 0; j < S::NT; ++j) acc[i0 + i][j] = Mma<DT>::k32(x[i], y[j], acc[i0 + i][j]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            turn_over();
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (wave < 4) turn_over();
}
template <class DT, class S, class A, class B, class RA, class RB>
__device__ inline void accumulate(f32x4 (&acc)[S::MT][S::NT], const A &a, const B &b, const RA &ra, const RB &rb, int steps, LDS_PTR(char) lds, int wave, int wm, int wn) {
    if constexpr (S::kWavesOf == 8)
        accumulate_in_turns<DT, S>(acc, a, b, ra, rb, steps, lds, wave, wm, wn);
    else
        accumulate_ahead<DT, S>(acc, a, b, ra, rb, steps, lds, wave, wm, wn);
}

// =============================================================================
// The heads
// =============================================================================
constexpr int kFar = 0x7f000000;             // no class
// What a row has to do with its target, left by the forward for the backward.
struct alignas(16) RowStat {
    float lse2;        // log2 of the sum of exp(z) over all classes, the target's with its margin; +inf: the row does not count
    float at_target;   // P_t - 1, times the margin's slope; of a teacher's row the largest |P - q| of its entries
    int target;        // class, or kFar
    int sub;           // of its weight rows the nearest
};
// What a row multiplies its probabilities by: dz = f exp2(z2 - lse2).  Gradients of single logits are rounded to 16 bits, where fp16
// ends at 6e-8 and either type is at its most exact just below a power of two; so all are multiplied by one number, which the
// products' ends take away again.  It brings the largest that there may be to between kTopDz / 2 and kTopDz, and of the steps of a
// factor of two it takes the eighth by which the rows' largest ones (the target's, -(1 - P_t) of a whole) lose least in
// rounding: most of a gradient's length is theirs.  (Over 40 heads of random sizes a gradient was up to 1.52 times as far from 64 bits as
// one that is rounded but once; 1.79 times with the largest brought to kTopDz itself.)
constexpr float kTopDz = 32640.f;            // 255 * 2^7
struct Upstream {
    const float *dloss, *count;     // count NULL: dloss has a value for every row
    const float *most;              // what to bring to kTopDz, for an upstream gradient of 1 (with `count`) or as it is
    float factor;
    int mean;
    struct Read { float dloss, count, most; };                      // asked for, to be waited for later
    __device__ inline Read read() const { return {count ? dloss[0] : 1.f, count ? count[0] : 1.f, *most}; }
    __device__ inline float base(const Read &v) const { return count ? factor * (mean ? v.dloss / v.count : v.dloss) : factor; }
    __device__ inline float base() const { return base(read()); }
    __device__ inline float up(float base) const { return up(base, read()); }
    __device__ inline float up(float base, const Read &v) const {
        const float top = __builtin_fabsf(base) * v.most;
        return top > 0.f && top < 3.0e38f ? __builtin_fminf(kTopDz / top, 0x1p100f) : 1.f;
    }
    __device__ inline float down() const { return 1.f / up(base()); }
};
struct Head {
    const char *x, *w;
    int64_t x_pitch, w_pitch;       // bytes
    int N, V, D, subs;
    float scale2;                   // scale * log2(e)
    const float *inv_x, *inv_w;     // 1 / |row| (cosines only)
};
// A class's index in ids of either width; what does not fit 32 bits is no class.
__device__ inline int load_id(const void *ids, int64_t i, int wide) {
    if (!wide) return reinterpret_cast<const int32_t *>(ids)[i];
    const int64_t v = reinterpret_cast<const int64_t *>(ids)[i];
    return v < INT32_MIN || v > INT32_MAX ? (v < 0 ? INT32_MIN : INT32_MAX) : (int)v;
}
// A row of zeros (no longer than kLeastNorm) has cosine 0 with everything and no gradient.  The factor of its products is a small
// number and not 0, so that a masked logit of -inf stays one.  A row whose squares have no sum in fp32 has no cosine: a weight's factor is no
// number, a row's of x is 0, by which finish_kernel knows it - it need not count.
constexpr float kLeastNorm = 1e-12f, kNoNorm = 1e-30f;

constexpr int kNormBlocks = 1024;
// 1 / |row| of 16-bit rows, sixteen lanes to a row; the first `rows_a` are a's.  And the largest of each workgroup's rows of b.
// Bound by memory: 101024 rows of 512 channels 18 us, 5.8 TB/s.
template <class DT>
__global__ void __launch_bounds__(256)
norms_kernel(float *__restrict__ inv_a, float *__restrict__ inv_b, float *__restrict__ most_b, const char *__restrict__ a, const char *__restrict__ b, int64_t a_pitch,
             int64_t b_pitch, int64_t rows_a, int64_t rows_b, int D) {
    constexpr int kAtOnce = 2;                                                  // rows of a lane in flight
    __shared__ float most[4];
    const int lane = threadIdx.x & 15, wave = threadIdx.x >> 6;
    const int64_t step = (int64_t)gridDim.x * 16, rows = rows_a + rows_b;
    float top = 0.f;
    for (int64_t r0 = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); r0 < rows; r0 += kAtOnce * step) {
        float s[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int64_t r = min(r0 + i * step, rows - 1);
            const char *row = r < rows_a ? a + r * a_pitch : b + (r - rows_a) * b_pitch;
            s[i] = 0.f;
#pragma unroll 2
            for (int c = lane * 8; c < D; c += 128) {
                const u32x4 v = *reinterpret_cast<const u32x4 *>(row + 2 * c);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x2 p = widen<DT>(v[k]);
                    s[i] = __builtin_fmaf(p.x, p.x, s[i]);
                    s[i] = __builtin_fmaf(p.y, p.y, s[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int64_t r = r0 + i * step;
            const float sum = sum_of_16(s[i]), inv = sum > 3.4e38f ? (r < rows_a ? 0.f : __builtin_nanf("")) : sum > kLeastNorm * kLeastNorm ? 1.f / __builtin_sqrtf(sum) : sum != sum ? sum : kNoNorm;
            if (r >= rows) continue;
            if (lane == 0) (r < rows_a ? inv_a[r] : inv_b[r - rows_a]) = inv;
            if (r >= rows_a) top = __builtin_fmaxf(top, inv);
        }
    }
    top = over_wave<true>(top);
    if ((threadIdx.x & 63) == 0) most[wave] = top;
    __syncthreads();
    if (threadIdx.x == 0) most_b[blockIdx.x] = __builtin_fmaxf(__builtin_fmaxf(most[0], most[1]), __builtin_fmaxf(most[2], most[3]));
}

// Tile number -> (class tile, row tile): groups of kGroup class tiles by all row tiles, so that what runs side by side on an XCD
// shares both operands in its L2.
constexpr int kGroup = 8;
__device__ inline void tile_of(uint32_t item, int m_tiles, int n_tiles, int &m, int &n) {
    const uint32_t per = (uint32_t)kGroup * n_tiles, group = item / per, in = item - group * per;
    const uint32_t wide = min((uint32_t)kGroup, (uint32_t)m_tiles - group * kGroup);
    n = (int)(in / wide);
    m = (int)(group * kGroup + in - (uint32_t)n * wide);
}

struct Logits {
    Head h;
    int class0, classes;            // of this range; the tiles cut it up
    int m_tiles, n_tiles;
    // forward: a maximum and a sum (log2 domain) to a class tile and row
    f32x2 *part;
    const void *ids;                // targets, or NULL: no class is kept out
    int ids_wide;
    f32x2 *at;                      // [N]: the target's product (cosines: over the weight's length) and which of its weight rows
    // backward
    Upstream up;
    const RowStat *stats;
    char *dz;                       // 16-bit [N, subs, plane]
    int64_t plane;                  // columns to a sub-centre, a multiple of 64
    float *col_part;                // cosines: sums of dz * cosine over a wave's rows: [n_tiles * WN, subs, plane]
};

// 1 / length of a tile's weight rows c .. c + 3 (classes from c0 on, `there` of them; 0 for those that there are not).  The places
// behind the last class belong to `saved` too.
template <int SUBS> __device__ inline f32x4 inverse_lengths(const Head &h, int c0, int c, int there, int sub) {
    f32x4 v;
    if constexpr (SUBS != 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = h.inv_w[(int64_t)(c0 + min(c + k, there - 1)) * h.subs + sub];
    } else {
        v = *reinterpret_cast<const f32x4 *>(h.inv_w + c0 + c);
    }
    if (c + 4 > there)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = c + k < there ? v[k] : 0.f;
    return v;
}

// Logits of a tile of classes (M) by rows (N).  SUBS: 0, one weight row to a class; 2 and more, that many, side by side in a lane's
// sums (ClassSource); 1, any number, one product after the other with the largest kept (and which, a byte to a value).
// 4000 x 20000 classes of 2 rows, 512 channels, bf16: forward 322 us one after the other in tiles of 64 x 128, 222 us side by side in
// tiles of 128 x 128 (backward 706 and 654 us); 12562 x 2166 of 2, 224 channels: 98 and 73 us (175 and 153 us).
template <class DT, class S, bool COS, int SUBS, bool BACK>
__global__ void __launch_bounds__(S::kThreadsOf, 2)
logits_kernel(Logits a) {
    constexpr bool LOOP = SUBS == 1;
    constexpr int K = SUBS > 1 ? SUBS : 1, CT = S::MT / K, BC = S::BM / K;     // rows in a lane's sums, 16-class tiles of a wave, classes of the tile
    extern __shared__ __attribute__((aligned(16))) char smem[];
    LDS_PTR(char) lds = (LDS_PTR(char))smem;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int wm = wave % S::WM, wn = wave / S::WM;
    int mt, nt;
    tile_of(xcd_item(blockIdx.x, gridDim.x), a.m_tiles, a.n_tiles, mt, nt);
    const int c0 = a.class0 + mt * BC, r0 = nt * S::BN;                        // first class and row
    const int there = min(a.class0 + a.classes, a.h.V) - c0;                   // classes of the tile that exist
    const int subs = SUBS ? a.h.subs : 1;
    std::conditional_t<(K > 1), ClassSource<S::BM, S::kWavesOf, S::MT, K>, Source<S::BM, S::kWavesOf, false>> ws;
    Source<S::BN, S::kWavesOf, false> xs;
    xs.init(a.h.x + r0 * a.h.x_pitch, min(S::BN, a.h.N - r0), a.h.x_pitch, 2 * (int64_t)a.h.D, wave, lane);
    Reader<false> reader;
    reader.init(n, g);
    const int steps = (a.h.D + kStep - 1) / kStep;
    f32x4 acc[S::MT][S::NT];
    f32x4 best[LOOP ? S::MT : 1][LOOP ? S::NT : 1];
    uint32_t which[LOOP ? S::MT : 1][LOOP ? S::NT : 1];
    const int first = 16 * wm * CT + 4 * g;                                    // this lane's class of the tile in its first 16-class tile
    // What the ends read of the rows is asked for in front of the products.  Of a 64-bit target the lower half will do: a row whose
    // upper half is not its sign has no target, and what it leaves is not read.
    int target[S::NT];
    float row_inv[S::NT], row_up[S::NT];
    RowStat row_stats[S::NT];
    Upstream::Read up_read{};
    if constexpr (BACK) up_read = a.up.read();
#pragma unroll
    for (int j = 0; j < S::NT; ++j) {
        const int64_t r = min(r0 + 16 * (wn * S::NT + j) + n, a.h.N - 1);
        if constexpr (!BACK) target[j] = a.ids ? reinterpret_cast<const int32_t *>(a.ids)[a.ids_wide ? 2 * r : r] : -1;
        if constexpr (BACK) row_stats[j] = a.stats[r], row_up[j] = a.up.count ? 1.f : a.up.dloss[r];
        row_inv[j] = COS ? a.h.inv_x[r] : 1.f;
    }
#pragma unroll 1
    for (int sub = 0; sub < (LOOP ? subs : 1); ++sub) {
        const char *rows = a.h.w + (int64_t)c0 * subs * a.h.w_pitch + sub * a.h.w_pitch;
        ws.init(rows, min(BC, there), K > 1 ? a.h.w_pitch : a.h.w_pitch * subs, 2 * (int64_t)a.h.D, wave, lane);
#pragma unroll
        for (int i = 0; i < S::MT; ++i)
#pragma unroll
            for (int j = 0; j < S::NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        f32x4 ahead[LOOP ? S::MT : 1];                                          // asked for in front of the product
        if constexpr (LOOP)
#pragma unroll
            for (int i = 0; i < S::MT; ++i) ahead[i] = inverse_lengths<SUBS>(a.h, c0, first + 16 * i, there, sub);
        if (LOOP && sub) barrier_lds();
        accumulate<DT, S>(acc, ws, xs, reader, reader, steps, lds, wave, wm, wn);
        if constexpr (COS) {
#pragma unroll
            for (int i = 0; i < S::MT; ++i) {
                f32x4 inv;
                if constexpr (LOOP)
                    inv = ahead[i];
                else
                    inv = inverse_lengths<SUBS>(a.h, c0, first + 16 * (i / K), there, i % K);
#pragma unroll
                for (int j = 0; j < S::NT; ++j) {
                    acc[i][j] *= inv;
                    if constexpr (LOOP) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const bool better = sub == 0 || acc[i][j][r] > best[i][j][r] || acc[i][j][r] != acc[i][j][r];
                            best[i][j][r] = better ? acc[i][j][r] : best[i][j][r];
                            which[i][j] = sub == 0 ? 0u : better ? (which[i][j] & ~(0xffu << 8 * r)) | (uint32_t)sub << 8 * r : which[i][j];
                        }
                    }
                }
            }
        }
    }
    // Logits of 16-class tile p by the rows of column j, and (SUBS) of which weight row of the class each is.
    auto logits_of = [&](int p, int j, uint32_t &of) {
        f32x4 v = LOOP ? best[LOOP ? p : 0][LOOP ? j : 0] : acc[p * K][j];
        of = LOOP ? which[LOOP ? p : 0][LOOP ? j : 0] : 0u;
#pragma unroll
        for (int i = 1; i < K; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float o = acc[p * K + i][j][r];
                const bool better = o > v[r] || o != o;
                v[r] = better ? o : v[r];
                of = better ? (of & ~(0xffu << 8 * r)) | (uint32_t)i << 8 * r : of;
            }
        return v;
    };

    if constexpr (!BACK) {
        barrier_lds();                                                          // the operands' place is taken over
        LDS_PTR(f32x2) met = (LDS_PTR(f32x2))lds;                               // [WM][BN]
#pragma unroll
        for (int j = 0; j < S::NT; ++j) {
            const int row = 16 * (wn * S::NT + j) + n;
            const int64_t r = min(r0 + row, a.h.N - 1);
            const float c2 = a.h.scale2 * row_inv[j];
            f32x4 v[CT];
            uint32_t of[CT];
#pragma unroll
            for (int p = 0; p < CT; ++p) v[p] = logits_of(p, j, of[p]);
            if (there < BC) {
#pragma unroll
                for (int p = 0; p < CT; ++p)
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[p][k] = first + 16 * p + k < there ? v[p][k] : kNegInf;
            }
            const uint32_t t = (uint32_t)(target[j] - c0 - 16 * wm * CT);       // as a class of this wave's
            if (a.ids && __builtin_amdgcn_ballot_w64(t < 16 * CT)) {
                float mine = 0.f;
                uint32_t of_mine = 0;
                bool found = false;
#pragma unroll
                for (int p = 0; p < CT; ++p)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool here = (uint32_t)(4 * g + 16 * p + k) == t;
                        mine = here ? v[p][k] : mine;
                        if constexpr (SUBS != 0) of_mine = here ? of[p] >> 8 * k & 0xffu : of_mine;
                        found |= here;
                        v[p][k] = here ? kNegInf : v[p][k];
                    }
                if (found && r0 + row < a.h.N) a.at[r] = f32x2{mine, (float)of_mine};
            }
            float top = kNegInf;
#pragma unroll
            for (int p = 0; p < CT; ++p)
#pragma unroll
                for (int k = 0; k < 4; ++k) top = __builtin_fmaxf(top, v[p][k]);
            top = xor_max(top) * c2;
            const float off = top == kNegInf ? 0.f : top;
            float sum = 0.f;
#pragma unroll
            for (int p = 0; p < CT; ++p)
#pragma unroll
                for (int k = 0; k < 4; ++k) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(v[p][k], c2, -off));
            sum = xor_sum(sum);
            if (g == 0) met[wm * S::BN + row] = f32x2{top, sum};
        }
        barrier_lds();
        for (int row = threadIdx.x; row < S::BN; row += S::kThreadsOf) {
            if (r0 + row >= a.h.N) break;
            f32x2 v = met[row];
#pragma unroll
            for (int i = 1; i < S::WM; ++i) {
                const f32x2 o = met[i * S::BN + row];
                const float top = __builtin_fmaxf(v.x, o.x), off = top == kNegInf ? 0.f : top;
                v = f32x2{top, v.y * __builtin_amdgcn_exp2f(v.x - off) + o.y * __builtin_amdgcn_exp2f(o.x - off)};
            }
            a.part[(int64_t)mt * a.h.N + r0 + row] = v;
        }
    } else {
        const int64_t pitch = 2 * a.plane * subs;                               // bytes of a row of dz
        const int col = mt * BC + 16 * wm * CT;                                 // this wave's first column of the range
        const Rsrc out = make_rsrc(a.dz + r0 * pitch, (int)((int64_t)min(S::BN, a.h.N - r0) * pitch));
        // dz for weights of length 1 takes the products' place (LOOP: the largest ones stay in `best`); sums of dz times the cosine
        f32x4 sums[COS ? S::MT : 1];
        if constexpr (COS)
#pragma unroll
            for (int i = 0; i < S::MT; ++i) sums[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float base = a.up.base(up_read), common = base * a.up.up(base, up_read);
#pragma unroll
        for (int j = 0; j < S::NT; ++j) {
            const int row = 16 * (wn * S::NT + j) + n;
            RowStat rg = row_stats[j];
            const float ix = row_inv[j], c2 = a.h.scale2 * ix;
            float f = common * row_up[j] * ix;
            if (rg.sub < 0 || (COS && ix == kNoNorm)) f = 0.f;
            // Rows behind the last have no share in the sums.  Their products are 0, which may be far above the logarithm of the last row's sum.
            if (r0 + row >= a.h.N) f = 0.f, rg.lse2 = __builtin_inff();
            const float e = f * rg.at_target;
            const int64_t t = (int64_t)rg.target - c0;
            const bool hit = t >= 16 * wm * CT && t < 16 * (wm + 1) * CT;
            const bool any = __builtin_amdgcn_ballot_w64(hit) != 0;
#pragma unroll
            for (int p = 0; p < CT; ++p) {
                uint32_t of;
                const f32x4 v = logits_of(p, j, of);
                f32x4 d;
#pragma unroll
                for (int k = 0; k < 4; ++k) d[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(v[k], c2, -rg.lse2)) * f;
                if (any) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool at = first + 16 * p + k == t;
                        d[k] = at ? e : d[k];
                        of = at ? (of & ~(0xffu << 8 * k)) | (uint32_t)rg.sub << 8 * k : of;
                    }
                }
                if (there < BC) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) d[k] = first + 16 * p + k < there ? d[k] : 0.f;
                }
                if constexpr (LOOP) {
                    acc[p][j] = d;
                    which[p][j] = of;
                } else {
#pragma unroll
                    for (int i = 0; i < K; ++i) {
                        f32x4 own = d;
                        if constexpr (K > 1)
#pragma unroll
                            for (int k = 0; k < 4; ++k) own[k] = (of >> 8 * k & 0xffu) == (uint32_t)i ? d[k] : 0.f;
                        if constexpr (COS) sums[p * K + i] += own * v;
                        acc[p * K + i][j] = own;
                    }
                }
            }
            if constexpr (COS) __builtin_amdgcn_sched_barrier(0);               // a column of tiles at a time: registers
        }
        auto scale_of = [&](int p, int sub) {                                   // a weight row of zeros has no gradient
            f32x4 inv = inverse_lengths<SUBS>(a.h, c0, first + 16 * p, there, sub);
#pragma unroll
            for (int k = 0; k < 4; ++k) inv[k] = inv[k] == kNoNorm ? 0.f : inv[k];
            return inv;
        };
        const int width = (int)max((int64_t)0, min((int64_t)32 * CT, 2 * (a.plane - col)));
        auto store = [&](int j, int sub, const u32x2 (&o)[CT]) {
            const int at = (int)((16 * (wn * S::NT + j) + n) * pitch + 2 * (sub * a.plane + col));
            if constexpr (CT == 1)
                __builtin_amdgcn_raw_buffer_store_b64(o[0], out, g * 8 < width ? at + g * 8 : kNowhere, 0, 0);
            else
                store_tile<16 * CT, 0>(out, at, o, g, width);
        };
        auto store_sums = [&](int p, int sub, f32x4 v) {
            if (!a.col_part) return;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = sum_of_16(v[k]);
            if (n == 0 && 32 * p + 8 * g < width)
                *reinterpret_cast<f32x4 *>(a.col_part + ((int64_t)(nt * S::WN + wn) * subs + sub) * a.plane + col + 16 * p + 4 * g) = v;
        };
        if constexpr (!LOOP) {
#pragma unroll
            for (int i = 0; i < K; ++i) {
                if constexpr (COS)
#pragma unroll
                    for (int p = 0; p < CT; ++p) {
                        const f32x4 inv = scale_of(p, i);
#pragma unroll
                        for (int j = 0; j < S::NT; ++j) acc[p * K + i][j] *= inv;
                    }
#pragma unroll
                for (int j = 0; j < S::NT; ++j) {
                    u32x2 o[CT];
#pragma unroll
                    for (int p = 0; p < CT; ++p) o[p] = narrow4<DT>(acc[p * K + i][j]);
                    store(j, i, o);
                }
                if constexpr (COS)
#pragma unroll
                    for (int p = 0; p < CT; ++p) store_sums(p, i, sums[p * K + i]);
            }
        } else {
#pragma unroll 1
            for (int sub = 0; sub < subs; ++sub) {
                f32x4 inv[CT];
#pragma unroll
                for (int p = 0; p < CT; ++p) inv[p] = scale_of(p, sub), sums[p] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < S::NT; ++j) {
                    u32x2 o[CT];
#pragma unroll
                    for (int p = 0; p < CT; ++p) {
                        f32x4 d = acc[p][j];
#pragma unroll
                        for (int k = 0; k < 4; ++k) d[k] = (which[p][j] >> 8 * k & 0xffu) == (uint32_t)sub ? d[k] : 0.f;
                        sums[p] += d * best[p][j];
                        o[p] = narrow4<DT>(d * inv[p]);
                    }
                    store(j, sub, o);
                }
#pragma unroll
                for (int p = 0; p < CT; ++p) store_sums(p, sub, sums[p]);
            }
        }
    }
}

// =============================================================================
// A row's tiles put together, the target's logit, the loss
// =============================================================================
// Waits more than it works: 8192 rows of 256 tiles 6 us.  A teacher's entries are products of their own, read row by row: 4096 x 64 of 768
// channels 74 us, 419 MB behind the L2s at 5.7 TB/s, out of the last level of cache (the weight is 74 MB).
struct Finish {
    Head h;
    const f32x2 *part, *at;
    int m_tiles, rows;              // rows to a workgroup, a power of two up to 16
    const void *ids;
    int ids_wide, top;              // teacher's entries of a row, 0: targets
    const void *teacher;
    int teacher_type;               // NA1D_BF16, NA1D_FP16, NA1D_FP32
    int64_t ignore;
    int cosines;
    float cos_m, sin_m, threshold, drop, temperature;
    RowStat *stats;
    float *coeff;                   // teacher: p - q of every entry, [N, top]
    float *loss;                    // [N]
    uint8_t *hits;                  // [N], or NULL
};
__device__ inline float teacher_value(const void *p, int64_t i, int type) {
    if (type == NA1D_FP32) return reinterpret_cast<const float *>(p)[i];
    const uint16_t v = reinterpret_cast<const uint16_t *>(p)[i];
    return type == NA1D_BF16 ? BF16::to_f32(v) : FP16::to_f32(v);
}
constexpr int kFinishThreads = 256;
// The derivative of the margin's cosine has the sine in its denominator; it is bounded there.
constexpr float kLeastSine2 = 1e-6f;

template <class DT>
__global__ void __launch_bounds__(kFinishThreads)
finish_kernel(Finish a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    f32x2 *met = reinterpret_cast<f32x2 *>(smem);                               // [lanes][rows]: 256 of them
    float *lse = reinterpret_cast<float *>(met + kFinishThreads);               // [16]
    const int entries = (a.top + 3) & ~3;                                       // of a row here; the last ones may be of no class
    float *z = lse + 16;                                                        // teacher, [rows][entries]: products,
    int *ids = reinterpret_cast<int *>(z + a.rows * entries);                   // classes,
    float *share = reinterpret_cast<float *>(ids + a.rows * entries);           // and their q
    const int R = a.rows, lanes = kFinishThreads / R, r = threadIdx.x & (R - 1), l = threadIdx.x / R;
    const int64_t r0 = (int64_t)blockIdx.x * R;
    {
        f32x2 v = {kNegInf, 0.f};
        const int64_t row = min(r0 + r, (int64_t)a.h.N - 1);
#pragma unroll 4
        for (int t = l; t < a.m_tiles; t += lanes) {
            const f32x2 o = a.part[(int64_t)t * a.h.N + row];
            const float top = __builtin_fmaxf(v.x, o.x), off = top == kNegInf ? 0.f : top;
            v = f32x2{top, v.y * __builtin_amdgcn_exp2f(v.x - off) + o.y * __builtin_amdgcn_exp2f(o.x - off)};
        }
        met[threadIdx.x] = v;
    }
    // a teacher's entries: 16 lanes to an entry
    const int lane16 = threadIdx.x & 15;
    for (int e = threadIdx.x >> 4; e < R * entries; e += kFinishThreads / 16) {
        const int64_t row = r0 + e / entries;
        const int k = e % entries;
        float s = 0.f;
        int id = -1;
        if (row < a.h.N && k < a.top) {
            id = load_id(a.ids, row * a.top + k, a.ids_wide);
            if (id >= 0 && id < a.h.V) {
                const char *xr = a.h.x + row * a.h.x_pitch, *w = a.h.w + id * a.h.w_pitch;
#pragma unroll 4
                for (int c = lane16 * 8; c < a.h.D; c += 128) {
                    const u32x4 p = *reinterpret_cast<const u32x4 *>(xr + 2 * c), q = *reinterpret_cast<const u32x4 *>(w + 2 * c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x2 u = widen<DT>(p[i]), v = widen<DT>(q[i]);
                        s = __builtin_fmaf(u.x, v.x, s);
                        s = __builtin_fmaf(u.y, v.y, s);
                    }
                }
            }
        }
        s = sum_of_16(s);
        if (lane16 == 0) z[e] = s, ids[e] = id;
    }
    __syncthreads();
    // The tiles' sums meet, R rows at a time.
    for (int half = lanes / 2; half; half >>= 1) {
        if (l < half) {
            const f32x2 v = met[threadIdx.x], o = met[threadIdx.x + half * R];
            const float top = __builtin_fmaxf(v.x, o.x), off = top == kNegInf ? 0.f : top;
            met[threadIdx.x] = f32x2{top, v.y * __builtin_amdgcn_exp2f(v.x - off) + o.y * __builtin_amdgcn_exp2f(o.x - off)};
        }
        __syncthreads();
    }
    const float largest = met[threadIdx.x & (R - 1)].x;                         // of the other classes' logits, for threads below R
    if ((int)threadIdx.x < R) lse[threadIdx.x] = met[threadIdx.x].x + __builtin_log2f(met[threadIdx.x].y);
    __syncthreads();
    if (!a.top) {
        const int64_t row = r0 + threadIdx.x;
        if ((int)threadIdx.x < R && row < a.h.N) {
            const int64_t raw = a.ids_wide ? reinterpret_cast<const int64_t *>(a.ids)[row] : (int64_t)reinterpret_cast<const int32_t *>(a.ids)[row];
            RowStat st = {__builtin_inff(), 0.f, kFar, -1};
            float loss = raw == a.ignore ? 0.f : __builtin_nanf("");
            bool hit = false;
            if (raw != a.ignore && raw >= 0 && raw < a.h.V) {
                float best = a.at[row].x, slope = 1.f;
                if (a.cosines && a.h.inv_x[row] == 0.f) best = __builtin_nanf("");
                st.sub = (int)a.at[row].y;
                hit = best * (a.h.scale2 * (a.cosines ? a.h.inv_x[row] : 1.f)) >= largest;         // as the tiles' maxima were worked out
                if (a.cosines) {
                    const float c = best * a.h.inv_x[row], sine2 = 1.f - c * c;
                    best = c;
                    if (c > a.threshold) {
                        best = c * a.cos_m - __builtin_sqrtf(__builtin_fmaxf(sine2, 0.f)) * a.sin_m;
                        slope = a.cos_m + a.sin_m * c / __builtin_sqrtf(__builtin_fmaxf(sine2, kLeastSine2));
                    } else if (c <= a.threshold) {
                        best = c - a.drop;
                    }
                }
                const float zt = best * a.h.scale2, others = lse[threadIdx.x], d = others - zt;         // log2 domain
                const float e = __builtin_amdgcn_exp2f(-__builtin_fabsf(d)), more = log1pf(e);
                loss = __builtin_fmaxf(d, 0.f) * kLn2 + more;
                if (d != d) loss = d;
                st.lse2 = (d > 0.f ? others : zt) + more * kLog2e;
                st.at_target = -(d > 0.f ? 1.f : e) / (1.f + e) * slope;
                st.target = (int)raw;
            }
            a.stats[row] = st;
            a.loss[row] = loss;
            if (a.hits) a.hits[row] = hit;
        }
    } else {
        // A teacher's row: a wave to each.
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        for (int q0 = wave; q0 < R; q0 += kFinishThreads / 64) {
            const int64_t row = r0 + q0;
            if (row >= a.h.N) break;
            const int *id = ids + q0 * entries;
            float *q = share + q0 * entries;
            const float *zr = z + q0 * entries;
            float top = kNegInf, total = 0.f;
            bool bad = false, nan = false;
            for (int k = lane; k < a.top; k += 64) {
                const float t = id[k] >= 0 && id[k] < a.h.V ? teacher_value(a.teacher, row * a.top + k, a.teacher_type) * (1.f / a.temperature) : kNegInf;
                bad |= id[k] >= a.h.V;
                nan |= t != t;
                top = __builtin_fmaxf(top, t);
                q[k] = t;
            }
            top = over_wave<true>(top);
            const float off = top == kNegInf ? 0.f : top;
            for (int k = lane; k < a.top; k += 64) total += __builtin_amdgcn_exp2f((q[k] - off) * kLog2e);
            total = over_wave<false>(total);
            bad = __builtin_amdgcn_ballot_w64(bad) != 0;
            nan = __builtin_amdgcn_ballot_w64(nan) != 0;
            const bool counts = !bad && (top > kNegInf || nan);
            const float log_total = __builtin_log2f(total), inv = 1.f / total, lse2 = lse[q0];
            float sum = 0.f;
            for (int k = lane; k < a.top; k += 64) {
                const float logq = (q[k] - off) * kLog2e - log_total, share = __builtin_amdgcn_exp2f((q[k] - off) * kLog2e) * inv, z2 = zr[k] * a.h.scale2;
                if (share != 0.f) sum += share * (logq - (z2 - lse2));
                q[k] = share;
            }
            if (lane < entries - a.top) q[a.top + lane] = 0.f;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");              // every lane reads the others' shares
            float typical = 0.f;
            for (int k = lane; k < a.top; k += 64) {
                float same = 0.f;                                               // an entry that is there twice has both shares
                const int own = id[k];
#pragma unroll 4
                for (int m = 0; m < entries; m += 4) {
                    const u32x4 them = *reinterpret_cast<const u32x4 *>(id + m);
                    const f32x4 theirs = *reinterpret_cast<const f32x4 *>(q + m);
#pragma unroll
                    for (int i = 0; i < 4; ++i) same += (int)them[i] == own ? theirs[i] : 0.f;
                }
                const float d = counts && own >= 0 ? __builtin_amdgcn_exp2f(zr[k] * a.h.scale2 - lse2) - same : 0.f;
                a.coeff[row * a.top + k] = d;
                typical = __builtin_fmaxf(typical, __builtin_fabsf(d));
            }
            sum = over_wave<false>(sum);
            typical = over_wave<true>(typical);
            RowStat st = {__builtin_inff(), 0.f, kFar, -1};
            float loss = bad ? __builtin_nanf("") : 0.f;
            if (counts) {
                loss = sum * kLn2 * a.temperature * a.temperature;
                st.lse2 = lse2;
                st.at_target = typical;
                st.sub = 0;
            }
            if (lane == 0) a.stats[row] = st, a.loss[row] = loss;
            if (lane == 0 && a.hits) a.hits[row] = 0;
        }
    }
}

// The sum or mean of the rows' losses in a fixed order, how many rows count, and what dz are to be scaled by (Upstream).  A number f
// rounded to b bits is off by 2^-b of the power of two below it: for each of kSteps scales within a factor of two, the sum of those
// powers squared over the typical f of up to 1024 rows (of all rows: 3 us more at 16000).
// (As the work of the finish kernel's last workgroup it is no launch of its own, but the fences of all the others cost more than
// that: 128 rows 15.8 us against 5.2 + 1.9, 999 rows 50 against 9.)
constexpr int kSteps = 8;
struct Reduce {
    float *total, *count, *most;
    const float *loss, *dloss, *inv_x, *inv_w, *most_w;       // dloss: of every row, in a backward (NULL otherwise); most_w [kNormBlocks]; all may be NULL
    const RowStat *stats;
    int N, subs, mean;
};
__global__ void __launch_bounds__(1024)
reduce_kernel(Reduce a) {
    __shared__ double sums[16];
    __shared__ int counts[16];
    __shared__ float tops[16], mosts[16], losts[16][kSteps];
    double s = 0.0;
    int c = 0;
    float top = 0.f, most = a.most_w ? 0.f : 1.f, some = 0.f;
    if (a.N > 1024 || (int)threadIdx.x < a.N) {
        const int64_t r = a.N > 1024 ? (int64_t)threadIdx.x * a.N >> 10 : threadIdx.x;
        const RowStat st = a.stats[r];
        some = __builtin_fabsf(st.at_target) * (a.dloss ? __builtin_fabsf(a.dloss[r]) : 1.f);
        if (a.inv_x && st.sub >= 0) some *= a.inv_x[r] * a.inv_w[(int64_t)st.target * a.subs + st.sub];
        some = st.sub < 0 ? 0.f : __builtin_fminf(some, 0x1p60f);              // (0 times what is no number is none)
    }
#pragma unroll 8
    for (int r = threadIdx.x; r < a.N; r += 1024) {
        const RowStat st = a.stats[r];
        if (a.loss) s += (double)a.loss[r];
        const float up = a.dloss ? __builtin_fabsf(a.dloss[r]) : 1.f;
        const float f = __builtin_fmaxf(1.f, __builtin_fabsf(st.at_target)) * (a.inv_x ? a.inv_x[r] : 1.f) * up;
        c += st.sub >= 0;
        top = __builtin_fmaxf(top, st.sub >= 0 ? f : 0.f);
    }
    if (a.most_w) most = a.most_w[threadIdx.x];
    static_assert(kNormBlocks == 1024, "one to a thread");
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o), c += __shfl_xor(c, o);
    top = over_wave<true>(top), most = over_wave<true>(most);
    const float below = __uint_as_float(__float_as_uint(some) & 0x7f800000u);
    float lost[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) lost[i] = over_wave<false>((some * __builtin_exp2f((float)i / kSteps) >= 2.f * below ? 4.f : 1.f) * (below * below));
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (lane == 0) {
        sums[wave] = s, counts[wave] = c, tops[wave] = top, mosts[wave] = most;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) losts[wave][i] = lost[i];
    }
    __syncthreads();
    if (wave) return;
    float mine = 0.f;                                                           // lanes 0 to 7: a scale each
#pragma unroll
    for (int i = 0; i < 16; ++i) mine += losts[i][lane % kSteps];
    mine *= __builtin_amdgcn_exp2f(-2.f / kSteps * (float)(lane % kSteps));
    float least = mine;
#pragma unroll
    for (int o = 1; o < kSteps; o <<= 1) least = __builtin_fminf(least, __shfl_xor(least, o));
    const uint64_t at = __builtin_amdgcn_ballot_w64(mine == least);             // none of numbers that are none
    const float best = at ? __builtin_amdgcn_exp2f((float)(__builtin_ctzll(at) % kSteps) / kSteps) : 1.f;
    if (lane) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += sums[i], c += counts[i], top = __builtin_fmaxf(top, tops[i]), most = __builtin_fmaxf(most, mosts[i]);
    const float largest = top * most, all = kTopDz / (best * largest);          // rounded down to a power of two, all * best is the scale
    *a.most = all > 1e-30f && all < 1e30f ? kTopDz / (best * __uint_as_float(__float_as_uint(all) & 0x7f800000u)) : largest;
    if (!a.loss) return;
    *a.count = (float)(c > 1 ? c : 1);
    *a.total = (float)(a.mean ? s / (double)(c > 1 ? c : 1) : s);
}

// =============================================================================
// Backward
// =============================================================================
// The teacher's entries of dz, which the logits' kernel left as those of any class.  Entries of one class write the same value.  A row
// that does not count has its zeros already; its coefficients are zeros too, but what comes from upstream need not be a number.
template <class DT>
__global__ void __launch_bounds__(256)
entries_kernel(uint16_t *__restrict__ dz, const float *__restrict__ coeff, const RowStat *__restrict__ stats, Upstream up, const void *__restrict__ ids, int ids_wide, int N, int top,
               int class0, int classes, int64_t plane) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)N * top) return;
    const int64_t row = i / top, c = (int64_t)load_id(ids, i, ids_wide) - class0;
    if (c < 0 || c >= classes || stats[row].sub < 0) return;
    const float base = up.base();
    dz[row * plane + c] = (uint16_t)Mma<DT>::pack(coeff[i] * (base * up.up(base) * (up.count ? 1.f : up.dloss[row])), 0.f);
}

// dx (fp32, all ranges' and splits' shares): x rows (N side) by channels (M side), contracted over a range's classes; and dW:
// weight rows by channels, contracted over the rows.  Both in one launch, so that the one's last workgroups run beside the other's first.
// Bound by the matrix cores where there are many rows: 8192 rows, 16384 classes, 1024 channels 450 us, 1220 TFLOP/s (the library's two products 895 and
// 1087); by dz (read twice) and dW where there are few: 1024 rows, 100000 classes, 512 channels 288 us, 730 TFLOP/s.
struct Product {
    const char *dz, *other;         // other: W, or x
    int64_t plane, other_pitch;     // of dz; bytes from one row of `other` to the next
    int N, D, subs;
    int classes, columns, class0;   // of this range; its columns of dz, whole steps
    int m_tiles, n_tiles, splits, per;          // per: of the contraction to a split, a multiple of kStep
    float *part;                    // fp32 [splits, rows, D]; dW: rows from the range's first on
    int64_t part_stride;
    int add;                        // to what is there
    Upstream up;
    // dW at once
    char *out;                      // 16-bit [V * subs, D], or NULL: to part
    const char *w;                  // cosines: dW loses its part along w
    int64_t w_pitch;
    const float *inv_w, *col_part;
    int col_parts;
};
template <class DT, class S, bool DW>
__device__ inline void product(const Product &a, uint32_t item, LDS_PTR(char) lds) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int wm = wave % S::WM, wn = wave / S::WM;
    const uint32_t mt = item % (uint32_t)a.m_tiles, rest = item / (uint32_t)a.m_tiles;
    const int nt = (int)(rest % (uint32_t)a.n_tiles), split = (int)(rest / (uint32_t)a.n_tiles);
    const int d0 = (int)mt * S::BM;
    const int64_t pitch = 2 * a.plane * a.subs;
    f32x4 acc[S::MT][S::NT];
#pragma unroll
    for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int j = 0; j < S::NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    Reader<true> turned;
    turned.init(n, g);
    Source<S::BM, S::kWavesOf, true> as;
    float along = 0.f;                                                          // cosines: of class threadIdx.x of the tile
    const int tiles_of_plane = DW ? a.n_tiles / a.subs : 1;
    const int sub = DW ? nt / tiles_of_plane : 0, col0 = DW ? (nt - sub * tiles_of_plane) * S::BN : 0, r0 = DW ? 0 : nt * S::BN;
    if constexpr (DW) {
        if (a.out && a.w && (int)threadIdx.x < S::BN && col0 + (int)threadIdx.x < a.classes) {
            const float *of = a.col_part + sub * a.plane + col0 + threadIdx.x, inv = a.inv_w[(int64_t)(a.class0 + col0 + threadIdx.x) * a.subs + sub];
#pragma unroll 8
            for (int p = 0; p < a.col_parts; ++p) along += of[(int64_t)p * a.subs * a.plane];
            along *= inv == kNoNorm ? 0.f : inv * inv;
        }
        const int64_t first = (int64_t)split * a.per, rows = min((int64_t)a.per, a.N - first);
        Source<S::BN, S::kWavesOf, true> bs;
        as.init(a.other + first * a.other_pitch + 2 * d0, rows, a.other_pitch, 2 * (int64_t)(a.D - d0), wave, lane);
        bs.init(a.dz + first * pitch + 2 * (sub * a.plane + col0), rows, pitch, 2 * (a.plane - col0), wave, lane);
        accumulate<DT, S>(acc, as, bs, turned, turned, (int)((rows + kStep - 1) / kStep), lds, wave, wm, wn);
    } else {
        Reader<false> straight;
        straight.init(n, g);
        Source<S::BN, S::kWavesOf, false> bs;
        const int first = split * a.per, wide = min(a.per, a.columns - first);
#pragma unroll 1
        for (int k = 0; k < a.subs; ++k) {
            if (k) barrier_lds();
            as.init(a.other + ((int64_t)(a.class0 + first) * a.subs + k) * a.other_pitch + 2 * d0, min(wide, a.classes - first), a.other_pitch * a.subs,
                    2 * (int64_t)(a.D - d0), wave, lane);
            bs.init(a.dz + r0 * pitch + 2 * (k * a.plane + first), min(S::BN, a.N - r0), pitch, 2 * (int64_t)wide, wave, lane);
            accumulate<DT, S>(acc, as, bs, turned, straight, (wide + kStep - 1) / kStep, lds, wave, wm, wn);
        }
    }
    const int m0 = d0 + 16 * wm * S::MT;                                        // this wave's channels
    if (DW && a.out) {
        const float unscale = a.up.down();
        const int left = a.classes - col0;                                      // classes of the tile
        const int64_t row0 = (int64_t)(a.class0 + col0) * a.subs + sub;
        const int out_pitch = 2 * a.D * a.subs, width = max(0, min(32 * S::MT, 2 * (a.D - m0)));
        const Rsrc os = make_rsrc(a.out + row0 * 2 * a.D, left > 0 ? (int)min((int64_t)(min(left, S::BN) - 1) * out_pitch + 2 * a.D, (int64_t)1 << 30) : 0);
        LDS_PTR(float) part = (LDS_PTR(float))lds;
        const int w_pitch = (int)(a.w_pitch * a.subs);
        const Rsrc wr = make_rsrc(a.w ? a.w + row0 * a.w_pitch : a.other, a.w && left > 0 ? (min(left, S::BN) - 1) * w_pitch + 2 * a.D : 0);
        if (a.w) {
            barrier_lds();                                                      // the operands' place is taken over
            if ((int)threadIdx.x < S::BN) part[threadIdx.x] = along;
            barrier_lds();
        }
#pragma unroll
        for (int j = 0; j < S::NT; ++j) {
            const int c = 16 * (wn * S::NT + j) + n;
            if (a.w) {                                                          // the rows of w as store_tile's: 16 bytes to a lane
                const float less = part[c];
#pragma unroll
                for (int p = 0; p < S::MT / 2; ++p) {
                    const int at = (2 * p + (g & 1)) * 32 + (g >> 1) * 16;
                    const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wr, at < width ? c * w_pitch + 2 * m0 + at : kNowhere, 0, 0));
                    const u32x2 lo = __builtin_amdgcn_permlane16_swap(v.x, v.z, false, false), hi = __builtin_amdgcn_permlane16_swap(v.y, v.w, false, false);
                    acc[2 * p][j] -= less * widen4<DT>(u32x2{lo.x, hi.x});
                    acc[2 * p + 1][j] -= less * widen4<DT>(u32x2{lo.y, hi.y});
                }
            }
            u32x2 o[S::MT];
#pragma unroll
            for (int i = 0; i < S::MT; ++i) o[i] = narrow4<DT>(acc[i][j] * unscale);
            store_tile<16 * S::MT, 0>(os, c * out_pitch + 2 * m0, o, g, width);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < S::NT; ++j) {
        const int in = 16 * (wn * S::NT + j) + n;
        const int64_t row = DW ? (int64_t)(col0 + in) * a.subs + sub : r0 + in;
        if (DW ? col0 + in >= a.classes : r0 + in >= a.N) continue;
        float *to = a.part + split * a.part_stride + row * a.D;
#pragma unroll
        for (int i = 0; i < S::MT; ++i) {
            const int d = m0 + 16 * i + 4 * g;
            if (d >= a.D) continue;
            f32x4 v = acc[i][j];
            if (a.add) v += *reinterpret_cast<const f32x4 *>(to + d);
            *reinterpret_cast<f32x4 *>(to + d) = v;
        }
    }
}

// Both in one launch, the dx part's workgroups first.  (Either may be empty.)
template <class DT, class SX, class SW>
__global__ void __launch_bounds__(SX::kThreadsOf, 2)
products_kernel(Product dx, Product dw, uint32_t dx_items, uint32_t dw_items) {
    static_assert(SX::kThreadsOf == SW::kThreadsOf, "one launch");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    LDS_PTR(char) lds = (LDS_PTR(char))smem;
    if (blockIdx.x < dx_items)
        product<DT, SX, false>(dx, xcd_item(blockIdx.x, dx_items), lds);
    else
        product<DT, SW, true>(dw, xcd_item(blockIdx.x - dx_items, dw_items), lds);
}

// The shares of all splits of a row put together, less their part along the row's own vector (cosines).  WAVES waves to a row share
// its splits: four where there are 8 or more, sixteen where there are 32 and few rows (whole backwards with sixteen and with four: 20 rows of 512 channels, 61
// splits 42 and 44 us; 700 of 96, 60 splits 83 and 76).  Bound by memory: 8192 rows of 1024 channels, two splits 18 us, 84 MB at 4.7 TB/s.
struct Fold {
    char *out;
    const float *part;
    int64_t stride, rows;
    int splits, D;
    Upstream up;
    const char *own;                // cosines: the rows themselves, and 1 / their length
    int64_t own_pitch;
    const float *inv;
};
template <class DT, int WAVES>
__global__ void __launch_bounds__(WAVES > 1 ? 64 * WAVES : 256)
fold_kernel(Fold a) {
    __shared__ f32x4 met[WAVES > 1 ? WAVES : 1][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = WAVES > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (row >= a.rows) return;
    const float *part = a.part + row * a.D;
    float f = a.up.down();
    auto sum = [&](int d) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (d < a.D)
#pragma unroll 8
            for (int s = WAVES > 1 ? wave : 0; s < a.splits; s += WAVES) v += *reinterpret_cast<const f32x4 *>(part + s * a.stride + d);
        if constexpr (WAVES > 1) {
            __syncthreads();
            met[wave][lane] = v;
            __syncthreads();
            v = met[0][lane];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) v += met[i][lane];
        }
        return v;
    };
    auto own = [&](int d) { return d < a.D ? widen4<DT>(*reinterpret_cast<const u32x2 *>(a.own + row * a.own_pitch + 2 * d)) : f32x4{0.f, 0.f, 0.f, 0.f}; };
    constexpr int kKept = 2;                                                    // of a row's 256 channels, for the second look at them
    f32x4 kept[kKept];
    float along = 0.f;
    auto add = [&](f32x4 v) { along += v[0] + v[1] + (v[2] + v[3]); };
    if (a.own) {
#pragma unroll
        for (int i = 0; i < kKept; ++i)
            if (256 * i < a.D) kept[i] = sum(256 * i + lane * 4), add(kept[i] * own(256 * i + lane * 4));
        for (int d = 256 * kKept; d < a.D; d += 256) add(sum(d + lane * 4) * own(d + lane * 4));
        const float inv = a.inv[row];
        along = over_wave<false>(along) * inv * inv;
        if (inv == kNoNorm) f = 0.f, along = 0.f;
    }
    auto store = [&](int d, f32x4 v) {
        if (a.own) v -= along * own(d);
        if (d < a.D && (WAVES == 1 || wave == 0)) *reinterpret_cast<u32x2 *>(a.out + (row * a.D + d) * 2) = narrow4<DT>(v * f);
    };
#pragma unroll
    for (int i = 0; i < kKept; ++i)
        if (256 * i < a.D) store(256 * i + lane * 4, a.own ? kept[i] : sum(256 * i + lane * 4));
    for (int d = 256 * kKept; d < a.D; d += 256) store(d + lane * 4, sum(d + lane * 4));
}

// =============================================================================
// Plans and launches
// =============================================================================
template <class T> inline T ceil_div(T a, T b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
// Places of the forward's results in `saved`, which the backward reads.
struct Saved {
    int64_t count, stats, coeff, inv_x, inv_w, most, bytes;     // count: and the largest factor behind it
    explicit Saved(const na1d_head &h) {
        int64_t at = 0;
        auto take = [&](int64_t n) { const int64_t p = at; at += round_up(n, 256); return p; };
        const bool cosines = h.kind == NA1D_HEAD_MARGIN, teacher = h.kind == NA1D_HEAD_TEACHER;
        count = take(16);
        stats = take(h.N * (int64_t)sizeof(RowStat));
        coeff = take(teacher ? 4 * h.N * h.top : 0);
        inv_x = take(cosines ? 4 * h.N : 0);
        inv_w = take(cosines ? 4 * h.V * h.subcenters : 0);
        most = take(cosines ? 4 * kNormBlocks : 0);
        bytes = at;
    }
};

// Tile shapes: classes by rows of the logits, channels by rows (dx) or weight rows (dW) of the products.
using Few = Shape<1, 2, 4, 1, 4>;             // 64 x 32
using Batch = Shape<2, 4, 2, 2, 3>;           // 64 x 128
using Many = Shape<4, 4, 2, 2, 2>;            // 128 x 128
using Wide = Shape<6, 4, 2, 2, 2>;            // 192 x 128
using Vast = Shape<8, 4, 2, 4, 2>;            // 256 x 256

enum Pick { kFew, kBatch, kMany, kWide, kVast };
struct Tiling {
    Pick pick;
    int bm, bn;
    int wn;                                   // waves along the rows
    int side;                                 // weight rows of a class side by side in the tile (of whose classes bm is the number)
    Tiling(Pick p = kFew, int rows = 1) : pick(p), side(rows) { bm = p == kVast ? 256 : p == kWide ? 192 : p == kMany ? 128 : 64, bn = p == kVast ? 256 : p == kFew ? 32 : 128, wn = p == kVast ? 4 : p == kFew ? 1 : 2, bm /= rows; }
    int64_t tiles(int64_t m, int64_t n) const { return (m + bm - 1) / bm * ((n + bn - 1) / bn); }
};
struct Plan {
    Tiling logits, back;                      // of the forward, of the backward
    int64_t m_tiles;
    // backward: ranges of classes, and within each, batches of rows
    int64_t plane;                            // columns to a sub-centre: a range's classes, rounded up to whole steps
    int64_t ranges, rows, batches;
    bool dw_at_once() const { return dw_splits == 1 && batches == 1; }        // else in parts
    int64_t together;                         // ranges whose parts are put together at once
    Tiling dx, dw;
    int dx_splits, dx_per, dw_splits, dw_per;
};
// Bytes of dW's parts that are kept for a launch that puts them together (behind each range by itself: backwards of 16384 x 32768 of 256 channels
// 1192 -> 1222 us, 40000 x 30000 of 128 2015 -> 2080).
constexpr int64_t kMostParts = 128ll << 20;
constexpr int64_t kMostDz = 256ll << 20;      // bytes of dz: what the last level of cache holds (64 MB: +10 to 25 %, 1 GB: 0 to +2 %)

// How long a launch of `first` workgroups of `first_steps` and then `second` of `second_steps` takes, in us: CUs hold one workgroup
// of 256 x 256 or two smaller ones, and take the next as they get free.  What a step of 64 and the rest of a tile take is
// fitted to forwards of 4096 x 32768 logits with 64, 256 and 1024 channels (64 x 128: 94, 143, 358 us; 128 x 128: 64, 101, 263; 192 x 128: 56, 95,
// 255; 256 x 256: 64, 99, 240), that is 990, 1280, 1340 and 1460 TFLOP/s between the ends.  The model also orders what does
// not fill a round: 1024 x 8000, 512 channels 24, 20, 23 and 25 us; 128 x 20000, 1024 channels 21, 24, 25, 33; 300 x 5000, 256 channels 15, 15, 17, 20.
// (It is not right everywhere: 2000 x 2000, 1000 channels take 26 us in the tiles that it picks, 64 x 128, and 24 in 128 x 128.)
struct Cost {
    double step, rest;
    int64_t slots;
};
inline Cost cost_of(Pick p) {
    switch (p) {
        case kMany: return {0.84, 3.0, 512};
        case kWide: return {1.2, 3.5, 512};
        case kVast: return {1.47, 6.0, 256};
        default: return {0.55, 2.55, 512};
    }
}
inline double time_of(Pick p, int64_t first, int64_t first_steps, int64_t second = 0, int64_t second_steps = 0, double more = 0.) {
    const Cost c = cost_of(p);
    const double a = first_steps * c.step + c.rest + more, b = second_steps * c.step + c.rest + more;
    const int64_t rounds = first / c.slots, over = first % c.slots;
    if (!second) return (rounds + (over > 0)) * a;
    double busy[2] = {(rounds + 1) * a, rounds * a};
    const int64_t wide[2] = {over, c.slots - over};
    for (int64_t left = second; left > 0;) {
        const int next = over && busy[0] < busy[1] ? 0 : 1;
        left -= wide[next];
        busy[next] += b;
    }
    return over ? std::max(busy[0], busy[1]) : busy[1];
}
inline Plan plan_of(const na1d_head &h) {
    Plan p{};
    // Logits.  The backward of a margin sums over its tile's classes: there is no room for that in the largest tiles.  Two, three or four
    // weight rows to a class come side by side in the tile whose waves they divide; otherwise they are worked on one after the other.
    const int64_t steps = ceil_div<int64_t>(h.D, kStep);
    auto shortest = [&](Pick largest) {
        Pick best = kBatch;
        double least = 1e30;
        for (const Pick pick : {kBatch, kMany, kWide, kVast}) {
            const double t = time_of(pick, Tiling(pick).tiles(h.V, h.N), steps);
            if (pick <= largest && t < least) best = pick, least = t;
        }
        return Tiling(best);
    };
    // (Unless that takes 2^24 workgroups, as 2^36 cosines of 4 rows do: a launch has less than 2^32 threads.)
    const Tiling side(h.subcenters == 3 ? kWide : kMany, h.subcenters);
    const bool fits_side = h.subcenters >= 2 && h.subcenters <= 4 && side.tiles(h.V, h.N) < 1 << 24;
    p.logits = h.N <= 32 ? Tiling(kFew) : fits_side ? side : shortest(h.subcenters > 1 ? kBatch : kVast);
    p.back = h.N > 32 && h.kind == NA1D_HEAD_MARGIN && h.subcenters == 1 ? shortest(kWide) : p.logits;
    p.m_tiles = ceil_div<int64_t>(h.V, p.logits.bm);
    const int64_t fits = std::min<int64_t>(kMostDz / (2 * h.N * h.subcenters), (1 << 20) / h.subcenters);
    p.plane = std::max<int64_t>(fits / 256 * 256, 256);
    p.ranges = ceil_div(h.V, p.plane);
    p.plane = std::min(round_up(h.V, kStep), round_up(ceil_div(h.V, p.ranges), 256));         // ranges alike
    p.ranges = ceil_div(h.V, p.plane);
    // More than 2^19 rows (times sub-centres) do not fit with 256 classes, and with fewer dx would be read and written in fp32 all the more often. What
    // takes more than four times the room, as only margins' can, goes in batches of rows, alike too: dW's sums are then read and written for each
    // (10^6 x 10000 of 128 channels, 512 MB: 29.2 ms, in two batches 30.4; 40000 x 2000 of 40 rows and 64 channels, 820 MB: 6.8 and 7.9).
    p.batches = ceil_div<int64_t>(2 * h.N * h.subcenters * p.plane, 4 * kMostDz);
    p.rows = p.batches > 1 ? round_up(ceil_div(h.N, p.batches), 256) : h.N;
    p.batches = ceil_div(h.N, p.rows);
    // Products: the tiles and splits (of 4, 8 or 16 steps at least) that take least, with what the sums of splits cost in memory at 4 TB/s and in
    // waiting.  Against splits of 4 steps whatever they cost (whole backwards): 999 x 9973 of 136 channels 42 -> 35 us, 128 x 20000 of
    // 1024 55 -> 47, 128 x 17982 of 192 23 -> 19.
    auto split = [&](int64_t tiles, int64_t length, int64_t most, int64_t shortest_split, int &splits, int &per) {
        const int64_t all = ceil_div<int64_t>(length, kStep), want = std::max<int64_t>(1, std::min<int64_t>(most / tiles, all / shortest_split));
        per = (int)(ceil_div(all, want) * kStep);
        splits = (int)ceil_div<int64_t>(length, per);
    };
    double least = 1e30;
    for (const Pick pick : {kBatch, kMany, kWide, kVast}) for (const int64_t shortest_split : {4, 8, 16}) {
        Plan q = p;
        q.dx = Tiling(h.N <= 32 ? kFew : pick), q.dw = Tiling(pick);
        const int64_t dx_tiles = q.dx.tiles(h.D, p.rows), dw_tiles = h.subcenters * q.dw.tiles(h.D, q.plane), most = cost_of(pick).slots;
        split(dx_tiles, q.plane, most, shortest_split, q.dx_splits, q.dx_per);
        split(dw_tiles, p.rows, most, shortest_split, q.dw_splits, q.dw_per);
        const double fold = (8. * q.dx_splits * p.rows * h.D + (q.dw_splits > 1 ? 8. * q.dw_splits * h.subcenters * q.plane * h.D : 0.)) / 4.0e6;
        const double t = fold + 0.05 * q.dx_splits + time_of(pick, dx_tiles * q.dx_splits, (int64_t)h.subcenters * q.dx_per / kStep, dw_tiles * q.dw_splits, q.dw_per / kStep, 2.);          // whose ends store more
        if (t < least && (h.N > 32 || pick <= kMany)) p = q, least = t;
    }
    p.together = std::max<int64_t>(1, std::min(p.ranges, kMostParts / (4 * p.plane * h.subcenters * h.D * p.dw_splits)));
    return p;
}
struct ForwardScratch {
    int64_t part, rows, at, bytes;
    ForwardScratch(const na1d_head &h, const Plan &p) {
        part = 0;
        rows = round_up(p.m_tiles * h.N * (int64_t)sizeof(f32x2), 256);
        at = rows + round_up(4 * h.N, 256);
        bytes = at + round_up(h.N * (int64_t)sizeof(f32x2), 256);
    }
};
struct BackwardScratch {
    int64_t most, dz, dx, dw, cols, bytes;
    BackwardScratch(const na1d_head &h, const Plan &p) {
        int64_t at = 0;
        auto take = [&](int64_t n) { const int64_t q = at; at += round_up(n, 256); return q; };
        most = take(16);
        dz = take(2 * p.rows * h.subcenters * p.plane);
        dx = take(4 * h.N * h.D * p.dx_splits);
        dw = take(p.dw_at_once() ? 0 : 4 * p.together * p.plane * h.subcenters * h.D * p.dw_splits);
        cols = take(h.kind == NA1D_HEAD_MARGIN && p.dw_at_once() ? 4 * ceil_div<int64_t>(h.N, p.back.bn) * p.back.wn * h.subcenters * p.plane : 0);
        bytes = at;
    }
};

#define NA1D_TRY(x)                      \
    do {                                 \
        const int st_ = (x);             \
        if (st_ != NA1D_OK) return st_;  \
    } while (0)

// A kernel's limit of LDS is raised once on every device.
template <auto KERNEL, class... A> int launch(unsigned grid, unsigned block, size_t lds, hipStream_t s, const A &...a) {
    static std::atomic<uint64_t> raised{0};
    int device = 0;
    if (lds > 64 * 1024 && (hipGetDevice(&device) != hipSuccess || device > 63 || !(raised.load(std::memory_order_relaxed) >> device & 1))) {
        if (!allow_lds(KERNEL, lds)) return NA1D_ERR_LAUNCH;
        if (device <= 63) raised.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    KERNEL<<<grid, block, lds, s>>>(a...);
    return launch_status();
}
template <class DT, class S, bool BACK> int launch_logits_of(const na1d_head &h, const Tiling &t, const Logits &a, hipStream_t s) {
    const unsigned grid = (unsigned)(a.m_tiles * a.n_tiles);
    if (h.kind != NA1D_HEAD_MARGIN) return launch<logits_kernel<DT, S, false, 0, BACK>>(grid, S::kThreadsOf, S::kLds, s, a);
    if constexpr (!BACK || S::MT * S::NT <= 24)
        if (h.subcenters == 1) return launch<logits_kernel<DT, S, true, 0, BACK>>(grid, S::kThreadsOf, S::kLds, s, a);
    if constexpr (S::MT == 4) {
        if (t.side == 2) return launch<logits_kernel<DT, S, true, 2, BACK>>(grid, S::kThreadsOf, S::kLds, s, a);
        if (t.side == 4) return launch<logits_kernel<DT, S, true, 4, BACK>>(grid, S::kThreadsOf, S::kLds, s, a);
    }
    if constexpr (S::MT == 6)
        if (t.side == 3) return launch<logits_kernel<DT, S, true, 3, BACK>>(grid, S::kThreadsOf, S::kLds, s, a);
    if constexpr (S::MT <= 2)
        if (t.side == 1) return launch<logits_kernel<DT, S, true, 1, BACK>>(grid, S::kThreadsOf, S::kLds, s, a);
    return NA1D_ERR_UNSUPPORTED;
}
template <class DT, bool BACK> int launch_logits(const na1d_head &h, const Tiling &t, Logits a, hipStream_t s) {
    a.m_tiles = (int)ceil_div<int64_t>(BACK ? round_up(a.classes, kStep) : a.classes, t.bm);           // dz: to the end of its last step
    a.n_tiles = ceil_div(a.h.N, t.bn);
    switch (t.pick) {
        case kFew: return launch_logits_of<DT, Few, BACK>(h, t, a, s);
        case kBatch: return launch_logits_of<DT, Batch, BACK>(h, t, a, s);
        case kMany: return launch_logits_of<DT, Many, BACK>(h, t, a, s);
        case kWide: return launch_logits_of<DT, Wide, BACK>(h, t, a, s);
        default: return launch_logits_of<DT, Vast, BACK>(h, t, a, s);
    }
}
template <class DT, class SX, class SW> int launch_products_of(const Product &dx, const Product &dw, hipStream_t s) {
    const uint32_t nx = (uint32_t)((int64_t)dx.m_tiles * dx.n_tiles * dx.splits), nw = (uint32_t)((int64_t)dw.m_tiles * dw.n_tiles * dw.splits);
    return launch<products_kernel<DT, SX, SW>>(nx + nw, SX::kThreadsOf, std::max(SX::kLds, SW::kLds), s, dx, dw, nx, nw);
}
template <class DT> int launch_products(const Plan &p, const Product &dx, const Product &dw, hipStream_t s) {
    if (p.dx.pick == kWide) return launch_products_of<DT, Wide, Wide>(dx, dw, s);
    if (p.dx.pick == kVast) return launch_products_of<DT, Vast, Vast>(dx, dw, s);
    if (p.dx.pick == kFew) return p.dw.pick == kBatch ? launch_products_of<DT, Few, Batch>(dx, dw, s) : launch_products_of<DT, Few, Many>(dx, dw, s);
    return p.dw.pick == kBatch ? launch_products_of<DT, Batch, Batch>(dx, dw, s) : launch_products_of<DT, Many, Many>(dx, dw, s);      // both by the channels
}
inline Head head_of(const na1d_head &h, const void *x, const void *w, const char *saved, const Saved &o) {
    const bool cosines = h.kind == NA1D_HEAD_MARGIN;
    const float scale = h.kind == NA1D_HEAD_TEACHER ? 1.f / h.scale : h.scale;             // a teacher's is the temperature
    return Head{(const char *)x, (const char *)w, 2 * h.x_stride, 2 * h.w_stride, (int)h.N, (int)h.V, (int)h.D, h.subcenters, scale * kLog2e,
                cosines ? reinterpret_cast<const float *>(saved + o.inv_x) : nullptr, cosines ? reinterpret_cast<const float *>(saved + o.inv_w) : nullptr};
}

template <class DT>
int forward(const na1d_head &h, float *loss, uint8_t *hits, const void *x, const void *w, const void *ids, const void *teacher, char *saved, char *ws, hipStream_t s) {
    const Saved o(h);
    const Plan p = plan_of(h);
    const ForwardScratch f(h, p);
    const bool cosines = h.kind == NA1D_HEAD_MARGIN, teaches = h.kind == NA1D_HEAD_TEACHER;
    Logits a{};
    a.h = head_of(h, x, w, saved, o);
    if (cosines) {
        norms_kernel<DT><<<kNormBlocks, 256, 0, s>>>(reinterpret_cast<float *>(saved + o.inv_x), reinterpret_cast<float *>(saved + o.inv_w),
                                                     reinterpret_cast<float *>(saved + o.most), a.h.x, a.h.w, a.h.x_pitch, a.h.w_pitch, h.N, h.V * h.subcenters, (int)h.D);
        NA1D_TRY(launch_status());
    }
    a.classes = (int)h.V;
    a.part = reinterpret_cast<f32x2 *>(ws + f.part);
    a.ids = teaches ? nullptr : ids, a.ids_wide = h.ids_64, a.at = reinterpret_cast<f32x2 *>(ws + f.at);
    NA1D_TRY((launch_logits<DT, false>(h, p.logits, a, s)));
    Finish e{};
    e.h = a.h, e.part = a.part, e.at = a.at, e.m_tiles = (int)p.m_tiles;
    // Rows to a workgroup: more read the tiles' results in longer pieces, fewer leave more of them at work.  A teacher's, whole forwards in
    // us with 1, 2 and 4: 1000 rows of 16 entries 23, 25, 30; 2000 of 100 38, 35, 44; 10182 of 84 72, 66, 60; 7433 of 4 69, 53, 46.
    e.rows = teaches ? (h.N >= 4096 ? 4 : h.N >= 1536 ? 2 : 1) : h.N >= 4096 ? 16 : h.N >= 1024 ? 4 : 1;
    e.ids = ids, e.ids_wide = h.ids_64, e.top = teaches ? h.top : 0, e.teacher = teacher, e.teacher_type = h.teacher_type;
    e.ignore = h.ignore_index, e.cosines = cosines, e.temperature = h.scale;
    e.cos_m = (float)cos(h.margin), e.sin_m = (float)sin(h.margin), e.threshold = (float)cos(M_PI - h.margin), e.drop = (float)(sin(M_PI - h.margin) * h.margin);
    e.stats = reinterpret_cast<RowStat *>(saved + o.stats), e.coeff = reinterpret_cast<float *>(saved + o.coeff);
    float *rows = reinterpret_cast<float *>(ws + f.rows);
    e.loss = h.reduction == NA1D_HEAD_NONE ? loss : rows;
    e.hits = hits;
    const size_t lds = kFinishThreads * sizeof(f32x2) + 64 + 12 * (size_t)e.rows * round_up(e.top, 4);
    NA1D_TRY(launch<finish_kernel<DT>>((unsigned)ceil_div<int64_t>(h.N, e.rows), kFinishThreads, lds, s, e));
    if (h.reduction == NA1D_HEAD_NONE) return NA1D_OK;
    float *count = reinterpret_cast<float *>(saved + o.count);
    return launch<reduce_kernel>(1, 1024, 0, s, Reduce{loss, count, count + 1, rows, nullptr, a.h.inv_x, a.h.inv_w, cosines ? reinterpret_cast<const float *>(saved + o.most) : nullptr,
                                                       e.stats, (int)h.N, h.subcenters, h.reduction == NA1D_HEAD_MEAN});
}

template <class DT>
int backward(const na1d_head &h, char *dx, char *dw, const float *dloss, const void *x, const void *w, const void *ids, const char *saved, char *ws, hipStream_t s) {
    const Saved o(h);
    const Plan p = plan_of(h);
    const BackwardScratch b(h, p);
    const bool cosines = h.kind == NA1D_HEAD_MARGIN;
    const RowStat *stats = reinterpret_cast<const RowStat *>(saved + o.stats);
    const float *most_w = cosines ? reinterpret_cast<const float *>(saved + o.most) : nullptr;
    Logits a{};
    a.h = head_of(h, x, w, saved, o);
    Upstream up{};
    up.dloss = dloss, up.factor = h.scale, up.mean = h.reduction == NA1D_HEAD_MEAN;           // a teacher's: temperature^2 / temperature
    if (h.reduction == NA1D_HEAD_NONE) {
        up.most = reinterpret_cast<const float *>(ws + b.most);
        NA1D_TRY(launch<reduce_kernel>(1, 1024, 0, s, Reduce{nullptr, nullptr, reinterpret_cast<float *>(ws + b.most), nullptr, dloss, a.h.inv_x, a.h.inv_w, most_w, stats, (int)h.N, h.subcenters, 0}));
    } else {
        up.count = reinterpret_cast<const float *>(saved + o.count), up.most = up.count + 1;
    }
    a.up = up, a.dz = ws + b.dz, a.plane = p.plane;
    a.col_part = cosines && dw && p.dw_at_once() ? reinterpret_cast<float *>(ws + b.cols) : nullptr;
    Product g{};
    g.dz = a.dz, g.plane = p.plane, g.D = (int)h.D, g.subs = h.subcenters, g.up = up;
    // (Of at most 2^22 rows, those of dx or of kMostParts: a launch has less than 2^32 threads.)
    auto fold = [&](char *out, int64_t part, int64_t stride, int64_t rows, int splits, const char *own, int64_t own_pitch, const float *inv) {
        const Fold f{out, reinterpret_cast<const float *>(ws + part), stride, rows, splits, (int)h.D, up, cosines ? own : nullptr, own_pitch, inv};
        if (splits >= 32 && rows <= 512) return launch<fold_kernel<DT, 16>>((unsigned)rows, 1024, 0, s, f);
        return splits >= 8 ? launch<fold_kernel<DT, 4>>((unsigned)rows, 256, 0, s, f) : launch<fold_kernel<DT, 1>>((unsigned)ceil_div<int64_t>(rows, 4), 256, 0, s, f);
    };
    const int64_t dw_stride = p.together * p.plane * h.subcenters * h.D;
    for (int64_t range = 0; range < p.ranges; ++range) {
        a.class0 = g.class0 = (int)(range * p.plane);
        a.classes = g.classes = (int)std::min(p.plane, h.V - a.class0);
        g.columns = (int)round_up(a.classes, kStep);
        const int64_t first = range / p.together * p.together * p.plane;                      // class of the parts
        for (int64_t batch = 0; batch < p.batches; ++batch) {
            const int64_t r0 = batch * p.rows;
            const Head whole = a.h;
            a.h.N = g.N = (int)std::min(p.rows, h.N - r0);
            a.h.x += r0 * a.h.x_pitch;
            if (cosines) a.h.inv_x += r0;                                                     // (no others come in batches)
            a.stats = stats + r0;
            a.up = up;
            if (!up.count) a.up.dloss += r0;                                                  // of every row
            NA1D_TRY((launch_logits<DT, true>(h, p.back, a, s)));
            if (h.kind == NA1D_HEAD_TEACHER) {
                entries_kernel<DT><<<(unsigned)ceil_div<int64_t>(h.N * h.top, 256), 256, 0, s>>>((uint16_t *)a.dz, reinterpret_cast<const float *>(saved + o.coeff), stats,
                                                                                                 up, ids, h.ids_64, (int)h.N, h.top, a.class0, a.classes, p.plane);
                NA1D_TRY(launch_status());
            }
            Product gx = g, gw = g;                                                           // what is not asked for has no workgroups
            if (dx) {
                gx.other = a.h.w, gx.other_pitch = a.h.w_pitch;
                gx.m_tiles = (int)ceil_div<int64_t>(h.D, p.dx.bm), gx.n_tiles = (int)ceil_div<int64_t>(g.N, p.dx.bn), gx.splits = p.dx_splits, gx.per = p.dx_per;
                gx.part = reinterpret_cast<float *>(ws + b.dx) + r0 * h.D, gx.part_stride = h.N * h.D, gx.add = range > 0;
            }
            if (dw) {
                gw.other = a.h.x, gw.other_pitch = a.h.x_pitch;
                gw.m_tiles = (int)ceil_div<int64_t>(h.D, p.dw.bm), gw.n_tiles = (int)(h.subcenters * ceil_div(g.columns, p.dw.bn)), gw.splits = p.dw_splits, gw.per = p.dw_per;
                gw.part = reinterpret_cast<float *>(ws + b.dw) + (a.class0 - first) * h.subcenters * h.D, gw.part_stride = dw_stride, gw.add = batch > 0, gw.out = p.dw_at_once() ? dw : nullptr;
                gw.w = cosines ? a.h.w : nullptr, gw.w_pitch = a.h.w_pitch, gw.inv_w = a.h.inv_w, gw.col_part = a.col_part, gw.col_parts = (int)ceil_div<int64_t>(h.N, p.back.bn) * p.back.wn;
            }
            NA1D_TRY(launch_products<DT>(p, gx, gw, s));
            a.h = whole;
        }
        if (dw && !p.dw_at_once() && ((range + 1) % p.together == 0 || range + 1 == p.ranges)) {
            const int64_t w0 = first * h.subcenters, rows = (a.class0 + a.classes - first) * h.subcenters;
            NA1D_TRY(fold(dw + 2 * w0 * h.D, b.dw, dw_stride, rows, p.dw_splits, a.h.w + w0 * a.h.w_pitch, a.h.w_pitch, cosines ? a.h.inv_w + w0 : nullptr));
        }
    }
    if (dx) NA1D_TRY(fold(dx, b.dx, h.N * h.D, h.N, p.dx_splits, a.h.x, a.h.x_pitch, a.h.inv_x));
    return NA1D_OK;
}

int64_t saved_bytes(const na1d_head &h) { return Saved(h).bytes; }
int64_t scratch_bytes(const na1d_head &h, bool back) {
    const Plan p = plan_of(h);
    return back ? BackwardScratch(h, p).bytes : ForwardScratch(h, p).bytes;
}
int run_forward(const na1d_head &h, float *loss, uint8_t *hits, const void *x, const void *w, const void *ids, const void *teacher, void *saved, void *ws,
                hipStream_t s) {
    return h.dtype == NA1D_BF16 ? forward<BF16>(h, loss, hits, x, w, ids, teacher, (char *)saved, (char *)ws, s)
                                : forward<FP16>(h, loss, hits, x, w, ids, teacher, (char *)saved, (char *)ws, s);
}
int run_backward(const na1d_head &h, void *dx, void *dw, const float *dloss, const void *x, const void *w, const void *ids, const void *saved, void *ws, hipStream_t s) {
    return h.dtype == NA1D_BF16 ? backward<BF16>(h, (char *)dx, (char *)dw, dloss, x, w, ids, (const char *)saved, (char *)ws, s)
                                : backward<FP16>(h, (char *)dx, (char *)dw, dloss, x, w, ids, (const char *)saved, (char *)ws, s);
}

}  // namespace loss
}  // namespace na1d
