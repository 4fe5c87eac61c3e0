// Causal attention with a sliding window of any length and a few first tokens that stay visible (sinks), forward and backward, on the
// matrix cores (gfx950):
//   P = softmax over the visible keys of q k^T * scale,  O = P v;   query t sees key u where u <= t and (t - u < window or u < sinks)
// Queries have `group` heads to every head of keys and values.  Built from the tile machinery of na1d_mfma_core.h, like the dense
// attention of na1d_global.hip: S^T tiles of 16 keys x 16 queries, an online softmax whose row statistics are lane-local up to a
// reduction over the four lane groups, and the rounded probabilities fed straight back as the B operand of O^T += V^T P^T.
//
// A workgroup of the forward and of dQ owns a strip of one head's queries and walks the keys in chunks of 32 that its four waves share
// through LDS: the chunks that hold sinks, then those that the strip's windows reach.  A workgroup of dK and dV owns a strip of
// one key head's rows and walks the queries of all the heads of its group.  A chunk that all rows of a wave see whole needs no mask, one that
// none of them sees is passed over by that wave.
//
// Rows from a sample's t_valid on do not exist: they are read as zeros whatever they hold (the buffer resources end there), and
// their outputs and gradients are zeros.
#include <type_traits>

#include "na1d_mfma_core.h"

namespace na1d {
namespace mfma {
namespace {

constexpr int kChunkTiles = 4, kChunkRows = 16 * kChunkTiles;      // queries that dK and dV take at a time, and rows of a strip (twice that in large forwards)
static_assert(kChunkTiles == kWaves, "row constants of a chunk are loaded by one wave to a tile");
// Keys that the forward and dQ take at a time.  64 of them cost registers and LDS that another wave to a SIMD can have: forward of 16 x 16 x 1000, 64 channels,
// window 128, 46.5 -> 43 us, 2 x 16 x 8192, 128 channels, window 1024, 191 -> 177.
constexpr int kKeyTiles = 2, kKeyRows = 16 * kKeyTiles;
constexpr float kNoMaximum = -3.4e38f;      // where a row's running maximum starts: finite, so that a chunk which a row does not see leaves it alone

struct SinkRows {               // one tensor: bytes from one sample, head, row to the next
    int64_t sample, head;
    int pitch;
};
struct SinkArgs {
    int T, H, K, group, strips, window, sinks, width;      // width: bytes of a row
    float scale;
    SinkRows q, k, v, o;        // o: out and dout, and dq
    SinkRows dkv;               // dk and dv
    // dK and dV (see there): strips of all heads up to `whole` have a workgroup each, the others `parts`; strips that hold sinks have `far` more
    int whole, parts, sink_strips, sink_rows, far;
};

struct SinkItem {
    uint32_t sample, kv, g;
    int strip;
};
// A value that is the same in all lanes, in a scalar register (divisions and loads leave it in vector registers, where buffer resources cannot start).
__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// Heads of a group run side by side, then strips: what runs together on an XCD reads the same keys.
__device__ inline SinkItem sink_item(uint32_t wg, uint32_t items, const SinkArgs &a) {
    const uint32_t lin = xcd_item(wg, items), rest = uniform(lin / (uint32_t)a.group), head = uniform(rest / (uint32_t)a.strips);
    SinkItem i;
    i.g = lin - rest * a.group;
    i.strip = (int)(rest - head * a.strips);
    i.sample = uniform(head / (uint32_t)a.K);
    i.kv = head - i.sample * a.K;
    return i;
}

// Chunks of keys that rows row0 .. row1 meet: those of the sinks, [0, sink_end), and those of the windows, [from, end).
struct KeyChunks {
    int sink_end, from, end;
    __device__ inline KeyChunks(int row0, int row1, int tv, const SinkArgs &a) {
        const int last = min(row1, tv - 1);
        end = last < row0 ? 0 : last / kKeyRows + 1;                   // nothing for a strip without a valid row
        from = max(0, row0 - a.window + 1) / kKeyRows;
        sink_end = min((a.sinks + kKeyRows - 1) / kKeyRows, end);
        from = min(max(from, sink_end), end);
    }
    __device__ inline int first() const { return sink_end > 0 ? 0 : from; }
    __device__ inline int after(int c) const { return c + 1 == sink_end ? from : c + 1; }
};
enum Sight { kNothing, kPart, kAll };
// What queries q0 .. q1 see of keys k0 .. k1.
__device__ inline Sight sight(int q0, int q1, int k0, int k1, const SinkArgs &a) {
    if (k0 > q1 || (k0 >= a.sinks && q0 - k1 >= a.window)) return kNothing;
    return k1 <= q0 && (k1 < a.sinks || q1 - k0 < a.window) ? kAll : kPart;
}

// The same for a wave's queries q0 .. q1 and chunks of keys by their number, worked out once: a chunk's turn is a chain of instructions, scalar ones among them.
struct KeySight {
    int last, sinks_end, passed, below, all_sinks, near;
    __device__ inline KeySight(int q0, int q1, int tv, const SinkArgs &a)
        : last(q0 < tv ? q1 / kKeyRows : -1), sinks_end((a.sinks + kKeyRows - 1) / kKeyRows), passed(floored(q0 - a.window - (kKeyRows - 1))), below(floored(q0 - (kKeyRows - 1))),
          all_sinks(floored(a.sinks - kKeyRows)), near(floored(q1 - a.window) + 1) {}
    __device__ static inline int floored(int x) { return x >> 5; }
    __device__ inline Sight of(int c) const {
        if (c > last || (c >= sinks_end && c <= passed)) return kNothing;
        return c <= below && (c <= all_sinks || c >= near) ? kAll : kPart;
    }
};
static_assert(kKeyRows == 32, "floored()");

// `rows` rows (0 or more) of a tensor from row `row` on as a buffer resource: at most a strip of them, so that its bytes fit 31 bits wherever it lies.
__device__ inline Rsrc rows_of(const void *base, int row, int rows, int pitch) {
    const uint64_t at = (uint64_t)base + (int64_t)row * pitch;
    return make_rsrc((const void *)((uint64_t)(uint32_t)uniform((int)(at >> 32)) << 32 | (uint32_t)uniform((int)at)), uniform(rows) * pitch);
}

// What outputs lose in rounding, for the backward: delta = rowsum(dO * O) is taken away from every dP of a row, and with O as it is stored, half a step off, that
// alone made dQ and dK 3.5e-3 (bf16) and 4e-4 (fp16) wrong, as a norm; all else together 2e-3 and 2e-4.  As integers, an fp32 value and the fp32 value of its rounding are
// apart by half a step of bf16 or fp16 at most, 2^15 or 2^12: a signed byte of that, 2^8 or 2^5 each and rounded down, leaves 2^-15 or 2^-18 of the value at most.  (fp16 below
// its normal range has larger steps: there the byte ends at its range.)  The bytes of a tile of 16 rows lie as dQ's waves read them: channels 32 s + 8 g of row n in the eight bytes of lane
// 16 g + n of step s (16 channels: four bytes of a lane).
template <int C> constexpr int kRestBytes = 16 * C;      // of a tile
template <class DT> constexpr int kRestShift = DT::tag == NA1D_BF16 ? 8 : 5;
template <class DT> __device__ inline uint32_t bits_of_half(uint32_t pair, int i) {      // of the fp32 value of half `i` of a pair
    const f32x2 x = unpack2<DT>(pair);
    return __float_as_uint(i ? x.y : x.x);
}
// Four products' roundings `w` and the bytes they lack.
template <class DT> __device__ inline uint32_t rest_of(f32x4 x, float f, u32x2 w) {
    uint32_t b[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int32_t apart = (int32_t)(__float_as_uint(x[r] * f) - bits_of_half<DT>(w[r / 2], r & 1)) >> kRestShift<DT>;
        b[r] = (uint32_t)max(-128, min(127, apart)) & 0xffu;
    }
    return b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
}
// Half `i` of a pair and its byte, byte `j` of `rest`.
template <class DT> __device__ inline float with_rest(uint32_t pair, int i, uint32_t rest, int j) {
    return __uint_as_float(bits_of_half<DT>(pair, i) + (uint32_t)((int32_t)(rest << (24 - 8 * j)) >> 24 << kRestShift<DT>));
}
// rowsum over this lane's channels of a row of dO and one of O
template <class DT, int C> __device__ inline float dot_whole(const RowOperand<C> &a, const RowOperand<C> &o, const char *rest, int lane) {
    float acc = 0.f;
    auto add = [&](uint32_t x, uint32_t y, uint32_t b, int j) {
        const f32x2 d = unpack2<DT>(x);
        acc = __builtin_fmaf(d.x, with_rest<DT>(y, 0, b, j), __builtin_fmaf(d.y, with_rest<DT>(y, 1, b, j + 1), acc));
    };
#pragma unroll
    for (int s = 0; s < RowOperand<C>::k32; ++s) {
        const u32x2 b = *reinterpret_cast<const u32x2 *>(rest + s * 512 + lane * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) add(a.w32[s][i], o.w32[s][i], b[i / 2], 2 * (i & 1));
    }
    if (RowOperand<C>::k16) {
        const uint32_t b = *reinterpret_cast<const uint32_t *>(rest + lane * 4);
        add(a.w16[0][0], o.w16[0][0], b, 0);
        add(a.w16[0][1], o.w16[0][1], b, 2);
    }
    return acc;
}
template <int C> __device__ inline void store_rest(char *rest, const uint32_t (&b)[C / 16], int lane) {
    if constexpr (C == 16) {
        *reinterpret_cast<uint32_t *>(rest + lane * 4) = b[0];
    } else {
        const int g = lane >> 4, to = (lane & 15) + 16 * (g == 1 ? 2 : g == 2 ? 1 : g);
#pragma unroll
        for (int s = 0; s < C / 32; ++s) {      // even groups get the first tile's eight channels, odd ones the second's
            const u32x2 both = __builtin_amdgcn_permlane16_swap(b[2 * s], b[2 * s + 1], false, false);
            *reinterpret_cast<u32x2 *>(rest + s * 512 + to * 8) = both;
        }
    }
}

// What a wave has loaded for good is here before its loop: the compiler, which does not know of the loads that write LDS, would wait for it inside, where the chunk to come is on
// its way, and so for that.
template <int C> __device__ inline void settle_rows(RowOperand<C> &o) {
#pragma unroll
    for (int s = 0; s < RowOperand<C>::k32; ++s) settle(o.w32[s]);
    if (RowOperand<C>::k16) settle(o.w16[0]);
}
// Two values as a pair of 16-bit numbers each: the roundings, and those of what these lost.  A row's dS sum to 0, so what all keys have in common drops out of dQ (and of dK
// what all queries have), but not out of roundings of dS: they go into the products twice, and so does P into dV's.  As norms against 64 bits, 2 x 16 x 8192 rows, bf16, 16 sinks:
// dQ 3.2e-3 -> 2.1e-3, dK and dV 2.4e-3 -> 1.7e-3, where the rounding of the result alone is 1.7e-3.  It cost 280 us and not 240 (dQ) and 460 and not 405 (dK and
// dV) there, at 128 channels, 52 and 48, 64 and 61 for 16 x 16 x 1000 rows of 64 channels, window 128.
template <class DT> __device__ inline void pack_twice(float x, float y, uint32_t &w, uint32_t &rest) {
    w = Mma<DT>::pack(x, y);
    const f32x2 there = unpack2<DT>(w);
    rest = Mma<DT>::pack(x - there.x, y - there.y);
}

// fp16 holds 2^-24 to 65504, and a backward's P and dS may be anywhere: small beside one key that takes nearly all of a row or with a small dO, beyond it with a large one.  Both count
// 2^kBackLift times where they are rounded (of small ones 2^-35 is lost at most, which their sums of products do not see beside a result's own 2^-25), and dS less than that where it
// would pass 2^15: dQ's kernel takes a row down, with what it has summed up, when it meets such a value, and leaves the largest of every tile of rows for dK's and dV's, which take P and
// dS down by the largest that they will meet (a P is then off by 2^-40 of that).  As norms, 4096 tokens of 64 channels, dO of 2^-12 and 2^-16: dQ 7.8e-4 and 7.5e-3 -> 2.5e-4 and
// 1.0e-3, where the results' rounding alone is 2.1e-4 and 1.0e-3.  (16 x 16 x 1000 rows of 64 channels, fp16, dQ: 49 -> 50.5 us, dK and dV 61 -> 63; these took 64 to 66 looking for
// large values themselves, or taking down on the way what they had summed up.)
template <int CTRL> __device__ inline float max_with(float x) {
    return __builtin_fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CTRL, 0xf, 0xf, true)));
}
// Over all lanes: pairs, fours, halves of 16 lanes in reverse, 16 in reverse, then the four groups.
__device__ inline float wave_max(float x) { return xor_max(max_with<0x140>(max_with<0x141>(max_with<0x4e>(max_with<0xb1>(x))))); }
template <class DT> constexpr bool kNarrow = DT::tag == NA1D_FP16;
template <class DT> constexpr int kBackLift = kNarrow<DT> ? 10 : 0;
constexpr float kTooLarge = 32768.f;        // and what is, is taken down to between 2^14 and 2^15
__device__ inline int too_much(float high) { return high > kTooLarge && high < __builtin_inff() ? __builtin_amdgcn_frexp_expf(high) - 15 : 0; }

// =============================================================================
// Forward
// =============================================================================
// What bounds it: with long windows the matrix cores and what a softmax takes of the vector unit, which wait for each other (2 x 16 x 8192 rows of 128 channels, 4 key heads, window 1024:
// 170 us, 0.77 PFLOP/s of what the mask leaves, matrix cores busy 0.44 of the time; 32 x 16384 over 8, window 2048: 520 us, 1.0 PFLOP/s, 0.53), with short ones memory (16 x 16 x 1000 rows of
// 64 channels, window 128: 33 us, 153 MB behind the L2s, 4.6 TB/s), with few rows a chunk's turn, a chain of
// dependent instructions (4 x 300 rows: 6.7 us; a third chunk on its way does nothing for them).
template <class DT, int C, int QT>
__global__ void __launch_bounds__(kThreads, 3)
sink_fwd_kernel(char *__restrict__ out, float *__restrict__ lse, char *__restrict__ rest, const char *__restrict__ q, const char *__restrict__ k, const char *__restrict__ v,
                const int32_t *__restrict__ t_valid, uint32_t items, SinkArgs a) {
    constexpr int CT = C / 16, CS = kStaged<C>, kStep = region_bytes<CS>(kKeyTiles);
    using LL = Lds<CS>;
    extern __shared__ __attribute__((aligned(16))) char smem[];          // 4 * kStep bytes: K and V of two chunks
    LDS_PTR(char) kv_lds = (LDS_PTR(char))smem;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    __builtin_assume(wave >= 0 && wave < kWaves);
    const int g = lane >> 4, n = lane & 15;
    const SinkItem it = sink_item(blockIdx.x, items, a);
    const int head = it.kv * a.group + it.g, T = a.T, width = a.width;
    int tv = T;
    if (t_valid) tv = uniform(max(0, min(T, t_valid[it.sample])));
    const int row0 = it.strip * (kChunkRows * QT), row_end = min(T, row0 + kChunkRows * QT);
    const char *kb = k + it.sample * a.k.sample + it.kv * a.k.head, *vb = v + it.sample * a.v.sample + it.kv * a.v.head;
    const int k_lane = direct_lane_offset<CS>(wave, lane, a.k.pitch, width), v_lane = direct_lane_offset<CS>(wave, lane, a.v.pitch, width);
    auto stage = [&](int c, LDS_PTR(char) to) {
        const int rows = min(kKeyRows, tv - c * kKeyRows);
        stage_direct<CS, kKeyTiles, kReadShared>(rows_of(kb, c * kKeyRows, rows, a.k.pitch), 0, to, kKeyTiles, wave, k_lane, a.k.pitch);
        stage_direct<CS, kKeyTiles, kReadShared>(rows_of(vb, c * kKeyRows, rows, a.v.pitch), 0, to + kStep, kKeyTiles, wave, v_lane, a.v.pitch);
    };
    const KeyChunks chunks(row0, row_end - 1, tv, a);
    int c = chunks.first();
    if (c < chunks.end) stage(c, kv_lds);
    const int own = 16 * QT * wave, w0 = row0 + own, w1 = w0 + 16 * QT - 1;      // this wave's rows
    const Rsrc qs = rows_of(q + it.sample * a.q.sample + head * a.q.head, row0, max(0, min(row_end, tv) - row0), a.q.pitch);
    RowOperand<C> qop[QT];
#pragma unroll
    for (int h = 0; h < QT; ++h) load_rows<C, kReadOnce>(qop[h], qs, (own + 16 * h) * a.q.pitch, a.q.pitch, width, lane);
    const float scale2 = a.scale * kLog2e;               // the scale is positive: checked at the C boundary

    RowLane<C, CS> row_lane;
    TrLane<C, CS> tr_lane;
    row_lane.init(0, lane);
    tr_lane.init(0, lane);
    constexpr float kSlack = 6.f;
    float m[QT];
    f32x4 o[QT][CT], lsum[QT];                            // lsum: the row sum, in every register
#pragma unroll
    for (int h = 0; h < QT; ++h) {
        m[h] = kNoMaximum;
        lsum[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) o[h][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const KeySight sees(w0, w1, tv, a);
#pragma unroll
    for (int h = 0; h < QT; ++h) settle_rows<C>(qop[h]);
    int at = 0;                                           // byte offset of the chunk's pair of regions: 0 or 2 * kStep
    while (c < chunks.end) {
        wait_direct();
        barrier_lds();      // this chunk has landed, and every wave is done with the one before, whose regions the next takes
        const int next = chunks.after(c), k0 = c * kKeyRows;
        if (next < chunks.end) stage(next, kv_lds + (at ^ 2 * kStep));
        LDS_PTR(char) k_lds = kv_lds + at;
        LDS_PTR(char) v_lds = k_lds + kStep;
        at ^= 2 * kStep;
        c = next;
        const Sight see = sees.of(k0 / kKeyRows);
        if (see == kNothing) continue;
        f32x4 s[QT][kKeyTiles];
#pragma unroll
        for (int kt = 0; kt < kKeyTiles; ++kt) {
            RowOperand<C> kop;
            read_rows<C, CS>(kop, k_lds + kt * LL::kTileBytes, row_lane);
#pragma unroll
            for (int h = 0; h < QT; ++h) s[h][kt] = dot_rows_mma<DT, C>(kop, qop[h]);
        }
        if (see == kPart) {
#pragma unroll
            for (int h = 0; h < QT; ++h) {
                const int row = w0 + 16 * h + n, d = row - k0 - 4 * g, stay = min(a.sinks, row + 1) - k0 - 4 * g;
#pragma unroll
                for (int kt = 0; kt < kKeyTiles; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!((uint32_t)(d - 16 * kt - r) < (uint32_t)a.window || 16 * kt + r < stay)) s[h][kt][r] = kNegInf;
            }
        }
        u32x4 pp[QT][kKeyTiles / 2];          // probabilities of two key tiles: the B operand of a 32-deep product
#pragma unroll
        for (int h = 0; h < QT; ++h) {
            float mc = kNegInf;
#pragma unroll
            for (int kt = 0; kt < kKeyTiles; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) mc = __builtin_fmaxf(mc, s[h][kt][r]);
            mc = xor_max(mc) * scale2;
            // The reference point of the exponentials moves only when a row's maximum has outgrown it by more than
            // kSlack (probabilities then stay below 2^kSlack, which every format here holds, also 2^kLift times that): most
            // chunks leave the accumulators as they are.
            if (__builtin_amdgcn_ballot_w64(mc > m[h] + kSlack)) {
                const float m_new = max2(m[h], reference_of<DT>(mc));
                const float alpha = __builtin_amdgcn_exp2f(m[h] - m_new);
                m[h] = m_new;
                lsum[h] *= alpha;
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) o[h][ct] *= alpha;
            }
            const float ref = kLift<DT> - m[h];
#pragma unroll
            for (int kt = 0; kt < kKeyTiles; ++kt) {
                float p[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][kt][r], scale2, ref));
                pp[h][kt / 2][2 * (kt & 1)] = Mma<DT>::pack(p[0], p[1]);
                pp[h][kt / 2][2 * (kt & 1) + 1] = Mma<DT>::pack(p[2], p[3]);
            }
        }
        // O^T += V^T P^T over two key tiles at a time; the row sums come from the same instruction with ones in place of V^T.
#pragma unroll
        for (int kt = 0; kt < kKeyTiles; kt += 2) {
            LDS_PTR(char) blk = v_lds + kt * LL::kTileBytes;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const u32x2 v0 = read_tr(blk + tr_lane.off[ct]), v1 = read_tr(blk + LL::kTileBytes + tr_lane.off[ct]);
                const u32x4 vv = {v0.x, v0.y, v1.x, v1.y};
#pragma unroll
                for (int h = 0; h < QT; ++h) o[h][ct] = Mma<DT>::k32(vv, pp[h][kt / 2], o[h][ct]);
            }
            const uint32_t one = Mma<DT>::pack(1.f, 1.f);
            const u32x4 ones = {one, one, one, one};
#pragma unroll
            for (int h = 0; h < QT; ++h) lsum[h] = Mma<DT>::k32(ones, pp[h][kt / 2], lsum[h]);
        }
    }
    const Rsrc os = rows_of(out + it.sample * a.o.sample + head * a.o.head, row0, row_end - row0, a.o.pitch);
    const Rsrc ls = make_rsrc(lse ? lse + ((int64_t)it.sample * a.H + head) * T + row0 : nullptr, lse ? (row_end - row0) * 4 : 0);
#pragma unroll
    for (int h = 0; h < QT; ++h) {
        const int at_row = own + 16 * h + n;
        const bool valid = row0 + at_row < tv;
        const float l = lsum[h][0], inv = __builtin_amdgcn_rcpf(l);
        u32x2 ow[CT];
        uint32_t rw[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            ow[ct] = pack_acc<DT>(o[h][ct], inv);
            rw[ct] = rest_of<DT>(o[h][ct], inv, ow[ct]);
            if (!valid) ow[ct] = u32x2{0u, 0u}, rw[ct] = 0u;
        }
        if (rest && w0 + 16 * h < T)
            store_rest<C>(rest + (((int64_t)it.sample * a.H + head) * ((T + 15) / 16) + (w0 / 16 + h)) * kRestBytes<C>, rw, lane);
        store_tile<C>(os, at_row * a.o.pitch, ow, g, stores_whole_lines(a.o.pitch, C, 0), width);   // rows past T are dropped
        // log2 of the row's sum of exponentials; 0 for a row that does not exist, whose q and dO the backward reads as zeros
        if (g == 0) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(valid ? (m[h] - kLift<DT>) + __builtin_amdgcn_logf(l) : 0.f), ls, at_row * 4, 0, 0);
    }
}

// =============================================================================
// Backward, query side: delta = rowsum(dO * O) and dQ = scale * dS K,  dS = P (dO V^T - delta)
// =============================================================================
// What bounds it is LDS, 24 KB of operands to a wave and 32 keys, and the matrix cores (both busy 0.6 of the time at 2 x 16 x 8192 rows of 128, window 1024, 254 to 272 us).  Two tiles of 16 queries to a wave, as in the forward, halve that, but 228 registers leave two waves to a SIMD and
// not four, and the launches are half as many workgroups: 2 x 16 x 8192, 128 channels, window 1024, took 310 us and not 280; 16 x 16 x 1000, 64 channels, window 128, took
// 57 and not 48, 5 x 10 x 777, 96 channels, window 100, 24 and not 17.5 (these two before dS went into the product twice).
template <class DT, int C>
__global__ void __launch_bounds__(kThreads)
sink_dq_kernel(char *__restrict__ dq, float *__restrict__ delta, float *__restrict__ largest, const char *__restrict__ q, const char *__restrict__ k, const char *__restrict__ v,
               const char *__restrict__ out, const char *__restrict__ dout, const float *__restrict__ lse, const char *__restrict__ rest, const int32_t *__restrict__ t_valid,
               uint32_t items, SinkArgs a) {
    constexpr int CT = C / 16, CS = kStaged<C>, kStep = region_bytes<CS>(kKeyTiles);
    using LL = Lds<CS>;
    extern __shared__ __attribute__((aligned(16))) char smem[];          // 4 * kStep bytes
    LDS_PTR(char) kv_lds = (LDS_PTR(char))smem;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    __builtin_assume(wave >= 0 && wave < kWaves);
    const int g = lane >> 4, n = lane & 15;
    const SinkItem it = sink_item(blockIdx.x, items, a);
    const int head = it.kv * a.group + it.g, T = a.T, width = a.width;
    int tv = T;
    if (t_valid) tv = uniform(max(0, min(T, t_valid[it.sample])));
    const int row0 = it.strip * kChunkRows, row_end = min(T, row0 + kChunkRows);
    const char *kb = k + it.sample * a.k.sample + it.kv * a.k.head, *vb = v + it.sample * a.v.sample + it.kv * a.v.head;
    const int k_lane = direct_lane_offset<CS>(wave, lane, a.k.pitch, width), v_lane = direct_lane_offset<CS>(wave, lane, a.v.pitch, width);
    auto stage = [&](int c, LDS_PTR(char) to) {
        const int rows = min(kKeyRows, tv - c * kKeyRows);
        stage_direct<CS, kKeyTiles, kReadShared>(rows_of(kb, c * kKeyRows, rows, a.k.pitch), 0, to, kKeyTiles, wave, k_lane, a.k.pitch);
        stage_direct<CS, kKeyTiles, kReadShared>(rows_of(vb, c * kKeyRows, rows, a.v.pitch), 0, to + kStep, kKeyTiles, wave, v_lane, a.v.pitch);
    };
    const KeyChunks chunks(row0, row_end - 1, tv, a);
    int c = chunks.first();
    if (c < chunks.end) stage(c, kv_lds);
    const int own = 16 * wave, w0 = row0 + own, w1 = w0 + 15;
    const int64_t o_off = it.sample * a.o.sample + head * a.o.head, stat = ((int64_t)it.sample * a.H + head) * T + row0;
    const int valid_rows = max(0, min(row_end, tv) - row0);
    const Rsrc qs = rows_of(q + it.sample * a.q.sample + head * a.q.head, row0, valid_rows, a.q.pitch);
    const Rsrc os = rows_of(out + o_off, row0, valid_rows, a.o.pitch), gs = rows_of(dout + o_off, row0, valid_rows, a.o.pitch);
    const Rsrc ls = make_rsrc(lse + stat, (row_end - row0) * 4), ds = make_rsrc(delta + stat, (row_end - row0) * 4);
    RowOperand<C> qop, gop, oop;
    load_rows<C, kReadShared>(qop, qs, own * a.q.pitch, a.q.pitch, width, lane);
    load_rows<C, kReadShared>(gop, gs, own * a.o.pitch, a.o.pitch, width, lane);
    load_rows<C, kReadOnce>(oop, os, own * a.o.pitch, a.o.pitch, width, lane);
    float ref = -__uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ls, (own + n) * 4, 0, 0));      // minus the row's log2 of its sum
    const float scale2 = a.scale * kLog2e;
    RowLane<C, CS> row_lane;
    TrLane<C, CS> tr_lane;
    row_lane.init(0, lane);
    tr_lane.init(0, lane);
    const int tile = min(w0 / 16, (T - 1) / 16);          // a tile past the last reads the last's bytes, with zeros for dO
    const char *bytes = rest + (((int64_t)it.sample * a.H + head) * ((T + 15) / 16) + tile) * kRestBytes<C>;
    const float dl = xor_sum(dot_whole<DT, C>(gop, oop, bytes, lane));      // lane (n, g) holds a quarter of row n's channels
    if (g == 0) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(dl), ds, (own + n) * 4, 0, 0);
    const f32x4 minus_dl = {-dl, -dl, -dl, -dl};          // the product dO . V^T starts at minus delta
    f32x4 acc[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) acc[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    const KeySight sees(w0, w1, tv, a);
    settle_rows<C>(qop), settle_rows<C>(gop), settle(ref);
    ref += kBackLift<DT>;
    int less = 0;                                         // what this row's dS has been taken down by: 2^less
    float most = 0.f;                                     // the largest of this lane's
    int at = 0;
    while (c < chunks.end) {
        wait_direct();
        barrier_lds();
        const int next = chunks.after(c), k0 = c * kKeyRows;
        if (next < chunks.end) stage(next, kv_lds + (at ^ 2 * kStep));
        LDS_PTR(char) k_lds = kv_lds + at;
        LDS_PTR(char) v_lds = k_lds + kStep;
        at ^= 2 * kStep;
        c = next;
        const Sight see = sees.of(k0 / kKeyRows);
        if (see == kNothing) continue;
#pragma unroll
        for (int kt = 0; kt < kKeyTiles; kt += 2) {
            float dsv[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                RowOperand<C> kop, vop;
                read_rows<C, CS>(kop, k_lds + (kt + j) * LL::kTileBytes, row_lane);
                read_rows<C, CS>(vop, v_lds + (kt + j) * LL::kTileBytes, row_lane);
                const f32x4 s = dot_rows_mma<DT, C>(kop, qop);
                const f32x4 dp = dot_rows_mma<DT, C>(vop, gop, minus_dl);
                float p[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale2, ref));
                if (see == kPart) {
                    const int row = w0 + n, d = row - k0 - 4 * g - 16 * (kt + j), stay = min(a.sinks, row + 1) - k0 - 4 * g - 16 * (kt + j);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!((uint32_t)(d - r) < (uint32_t)a.window || r < stay)) p[r] = 0.f;
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) dsv[4 * j + r] = p[r] * dp[r];
            }
            if constexpr (kNarrow<DT>) {
#pragma unroll
                for (int i = 0; i < 8; ++i) most = __builtin_fmaxf(most, __builtin_fabsf(dsv[i]));
                if (__builtin_amdgcn_ballot_w64(most > kTooLarge)) {
                    const int more = too_much(xor_max(most));       // of the four lanes that share the row
                    const float by = __builtin_amdgcn_ldexpf(1.f, -more);
                    less += more, ref -= (float)more, most *= by;
#pragma unroll
                    for (int i = 0; i < 8; ++i) dsv[i] *= by;
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) acc[ct] *= by;
                }
            }
            u32x4 db, rb;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w, r;
                pack_twice<DT>(dsv[2 * i], dsv[2 * i + 1], w, r);
                db[i] = w, rb[i] = r;
            }
            LDS_PTR(char) blk = k_lds + kt * LL::kTileBytes;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const u32x2 k0t = read_tr(blk + tr_lane.off[ct]), k1t = read_tr(blk + LL::kTileBytes + tr_lane.off[ct]);
                const u32x4 kk = {k0t.x, k0t.y, k1t.x, k1t.y};
                acc[ct] = Mma<DT>::k32(kk, db, acc[ct]);
                acc[ct] = Mma<DT>::k32(kk, rb, acc[ct]);
            }
        }
    }
    const Rsrc dqs = rows_of(dq + o_off, row0, row_end - row0, a.o.pitch);
    if constexpr (kNarrow<DT>) {
        most = wave_max(__builtin_amdgcn_ldexpf(most, less - kBackLift<DT>));
        if (lane == 0) largest[(((int64_t)it.sample * a.H + head) * a.strips + it.strip) * kWaves + wave] = most;
    }
    const float back = __builtin_amdgcn_ldexpf(a.scale, less - kBackLift<DT>);
    u32x2 qw[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        qw[ct] = pack_acc<DT>(acc[ct], back);
        if (w0 + n >= tv) qw[ct] = u32x2{0u, 0u};
    }
    store_tile<C>(dqs, (own + n) * a.o.pitch, qw, g, stores_whole_lines(a.o.pitch, C, 0), width);
}

// =============================================================================
// Backward, key side: dV = P^T dO and dK = scale * dS^T Q, summed over the heads of the group
// =============================================================================
// A workgroup owns a strip of 64 keys, a tile of them to a wave, whose K and V rows stay in registers, and walks units of (head of the group, chunk
// of 64 queries): Q and dO through LDS, double-buffered.  The score product is taken with Q and K swapped, so that P and dS come out as B operands.
// What bounds it is LDS, 64 KB of operands to a wave and unit (busy 0.54 of the time), beside the matrix cores (0.49) and the waits of two waves to a SIMD for each other's: 2 x 8192 rows, 16
// heads of 128 over 4, window 1024: 425 to 460 us; 16 x 16 x 1000 rows of 64, window 128: 60 us, 289 MB behind the L2s, 4.8 TB/s.  Two tiles of keys to a wave would halve what LDS gives,
// and need 308 registers at 128 channels, so one wave to a SIMD: 510 us in place of 435 then, and at 64 channels 81 in place of 60.
//
// A launch ends when its last workgroup does, so it is cut to fit the card: strips beyond a whole number of rounds of it are shared by `parts` workgroups
// each.  Sinks are seen by all queries behind them, other keys by a window of them: the queries that see of a strip nothing but its sinks are left to
// `far` workgroups.  What several workgroups have a share in they leave in fp32 in `partial`, and sink_join_kernel adds it up in a fixed order.
struct Partial {                // floats from the start of `partial`: [parts of a shared strip][dk, dv][64][C], and twice [..][dk, dv][sink_rows][C]
    int64_t shared, near, far;
};
template <int C> __device__ inline Partial partial_of(int64_t strip_id, int part, int64_t sink_strip, int far, int64_t heads, const SinkArgs &a) {
    const int64_t shared_size = (heads * a.strips - a.whole) * a.parts * (2 * kChunkRows * C), slot = 2 * a.sink_rows * C;
    return Partial{((strip_id - a.whole) * a.parts + part) * (2 * kChunkRows * C), shared_size + sink_strip * slot,
                   shared_size + (heads * a.sink_strips + sink_strip * a.far + far) * slot};
}
template <class DT, int C>
__global__ void __launch_bounds__(kThreads)
sink_dkv_kernel(char *__restrict__ dk, char *__restrict__ dv, float *__restrict__ partial, const char *__restrict__ q, const char *__restrict__ k,
                const char *__restrict__ v, const char *__restrict__ dout, const float *__restrict__ lse, const float *__restrict__ delta, const float *__restrict__ largest,
                const int32_t *__restrict__ t_valid, uint32_t rest, uint32_t heads, SinkArgs a) {
    constexpr int CT = C / 16, CS = kStaged<C>, kStep = region_bytes<CS>(kChunkTiles), kBuf = 2 * kStep + 2 * kChunkRows * 4;
    using LL = Lds<CS>;
    extern __shared__ __attribute__((aligned(16))) char smem[];          // 2 * kBuf bytes: Q, dO and the rows' constants of two chunks
    LDS_PTR(char) buf_lds = (LDS_PTR(char))smem;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    __builtin_assume(wave >= 0 && wave < kWaves);
    const int g = lane >> 4, n = lane & 15;
    // strips with a workgroup of their own; then (`rest` of them) the parts of the others, and the far workgroups
    uint32_t strip_id, part = 0, each = 1, head, strip;
    bool far = false;
    if (blockIdx.x < (uint32_t)a.whole) {
        strip_id = xcd_item(blockIdx.x, a.whole);
    } else {
        const uint32_t lin = xcd_item(blockIdx.x - a.whole, rest), shared = (heads * a.strips - a.whole) * a.parts;
        far = lin >= shared;
        each = far ? a.far : a.parts;
        const uint32_t i = far ? lin - shared : lin;
        strip_id = uniform(i / each);
        part = i - strip_id * each;
        if (!far) strip_id += a.whole;
    }
    head = uniform(strip_id / (uint32_t)(far ? a.sink_strips : a.strips));
    strip = strip_id - head * (far ? a.sink_strips : a.strips);
    const uint32_t sample = uniform(head / (uint32_t)a.K), kv = head - sample * a.K;
    const int T = a.T, width = a.width;
    int tv = T;
    if (t_valid) tv = uniform(max(0, min(T, t_valid[sample])));
    const int row0 = strip * kChunkRows, row_end = min(T, row0 + kChunkRows);
    // chunks of queries that see something of the strip: [c_from, c_near) its windows, [c_near, c_end) its sinks
    const int last_key = min(row_end, tv) - 1;
    int c_from = row0 / kChunkRows, c_end = c_from;
    if (last_key >= row0) {
        const int chunks = (tv - 1) / kChunkRows + 1, near = (int)min((int64_t)chunks, ((int64_t)last_key + a.window - 1) / kChunkRows + 1);
        if (far) {
            c_from = near, c_end = chunks;
        } else {
            c_end = row0 < a.sinks && !a.far ? chunks : near;
        }
    }
    const int nc = c_end - c_from, units = nc * a.group, u_end = uniform((int)((int64_t)units * (part + 1) / each));
    int u = uniform((int)((int64_t)units * part / each));
    const int hg = nc ? uniform(u / nc) : 0;
    int c = nc ? c_from + u - hg * nc : 0;

    const int q_lane = direct_lane_offset<CS>(wave, lane, a.q.pitch, width), g_lane = direct_lane_offset<CS>(wave, lane, a.o.pitch, width);
    const char *qb = q + sample * a.q.sample, *gb = dout + sample * a.o.sample;
    float row_lse, row_delta;                             // of row 16 * wave + n of the chunk in flight
    // of the head at hand: where it begins, and its rows' constants
    const int first_head = kv * a.group + hg;
    const char *qh = qb + first_head * a.q.head, *gh = gb + first_head * a.o.head;
    const float *lse_h = lse + ((int64_t)sample * a.H + first_head) * T, *delta_h = delta + ((int64_t)sample * a.H + first_head) * T;
    auto stage = [&](int c_, LDS_PTR(char) to) {
        const int r0 = c_ * kChunkRows, rows = min(kChunkRows, tv - r0);
        stage_direct<CS, kChunkTiles, kReadShared>(rows_of(qh, r0, rows, a.q.pitch), 0, to, kChunkTiles, wave, q_lane, a.q.pitch);
        stage_direct<CS, kChunkTiles, kReadShared>(rows_of(gh, r0, rows, a.o.pitch), 0, to + kStep, kChunkTiles, wave, g_lane, a.o.pitch);
        const Rsrc ls = rows_of(lse_h, r0, rows, 4), ds = rows_of(delta_h, r0, rows, 4);
        row_lse = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ls, (16 * wave + n) * 4, 0, 0));
        row_delta = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ds, (16 * wave + n) * 4, 0, 0));
    };
    if (u < u_end) stage(c, buf_lds);
    const int own = 16 * wave, w0 = row0 + own, w1 = w0 + 15, key = w0 + n;
    const Rsrc ks = rows_of(k + sample * a.k.sample + kv * a.k.head, row0, max(0, last_key + 1 - row0), a.k.pitch);
    const Rsrc vs = rows_of(v + sample * a.v.sample + kv * a.v.head, row0, max(0, last_key + 1 - row0), a.v.pitch);
    RowOperand<C> kop, vop;
    load_rows<C, kReadShared>(kop, ks, own * a.k.pitch, a.k.pitch, width, lane);
    load_rows<C, kReadShared>(vop, vs, own * a.v.pitch, a.v.pitch, width, lane);
    const float scale2 = a.scale * kLog2e;
    const uint32_t reach = key < a.sinks ? 0x7fffffffu : (uint32_t)a.window;
    RowLane<C, CS> row_lane;
    TrLane<C, CS> tr_lane;
    row_lane.init(0, lane);
    tr_lane.init(0, lane);
    f32x4 acck[CT], accv[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) acck[ct] = accv[ct] = f32x4{0.f, 0.f, 0.f, 0.f};

    // P and dS are taken down by 2^less, by the largest dS of all units: a lane has every 64th of them
    int less = 0;
    auto largest_of = [&](int i) {
        const int h = i / nc;
        const f32x4 x = *reinterpret_cast<const f32x4 *>(largest + (((int64_t)sample * a.H + kv * a.group + h) * a.strips + c_from + i - h * nc) * kWaves);
        return __builtin_fmaxf(__builtin_fmaxf(x[0], x[1]), __builtin_fmaxf(x[2], x[3]));
    };
    float high = 0.f;
    if (kNarrow<DT> && u + lane < u_end) high = largest_of(u + lane);
    settle_rows<C>(kop), settle_rows<C>(vop);
    if constexpr (kNarrow<DT>) {
        for (int i = u + lane + 64; i < u_end; i += 64) high = __builtin_fmaxf(high, largest_of(i));
        less = uniform(too_much(__builtin_amdgcn_ldexpf(wave_max(high), kBackLift<DT>)));
    }
    int at = 0;
    for (; u < u_end; ++u) {
        wait_direct();
        {
            // rows past tv: q and dO are zeros there, and so are these
            const float constant = g == 0 ? (float)(kBackLift<DT> - less) - row_lse : -row_delta;
            if (g < 2) *reinterpret_cast<LDS_PTR(float)>(buf_lds + at + 2 * kStep + (g * kChunkRows + 16 * wave + n) * 4) = constant;
        }
        barrier_lds();
        const int q0 = c * kChunkRows;
        if (++c == c_end) c = c_from, qh += a.q.head, gh += a.o.head, lse_h += T, delta_h += T;
        if (u + 1 < u_end) stage(c, buf_lds + (kBuf - at));
        LDS_PTR(char) q_lds = buf_lds + at;
        LDS_PTR(char) g_lds = q_lds + kStep;
        LDS_PTR(char) ref_lds = q_lds + 2 * kStep + 16 * g;
        at = kBuf - at;
        const Sight see = w0 < tv ? sight(q0, q0 + kChunkRows - 1, w0, w1, a) : kNothing;
        if (see == kNothing) continue;
#pragma unroll
        for (int qi = 0; qi < kChunkTiles; qi += 2) {
            u32x4 pb, db, pr, dr;
            float dsv[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                RowOperand<C> qop, gop;
                read_rows<C, CS>(qop, q_lds + (qi + j) * LL::kTileBytes, row_lane);
                read_rows<C, CS>(gop, g_lds + (qi + j) * LL::kTileBytes, row_lane);
                const f32x4 ref = *reinterpret_cast<LDS_PTR(f32x4)>(ref_lds + 64 * (qi + j));
                const f32x4 del4 = *reinterpret_cast<LDS_PTR(f32x4)>(ref_lds + kChunkRows * 4 + 64 * (qi + j));
                const f32x4 s = dot_rows_mma<DT, C>(qop, kop);        // [query 4g+r][key n]
                const f32x4 dp = dot_rows_mma<DT, C>(gop, vop, del4);
                float p[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale2, ref[r]));
                if (see == kPart) {
                    const int d = q0 + 16 * (qi + j) + 4 * g - key;      // query 4g less the key
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!((uint32_t)(d + r) < reach)) p[r] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t w, r;
                    pack_twice<DT>(p[2 * i], p[2 * i + 1], w, r);
                    pb[2 * j + i] = w, pr[2 * j + i] = r;
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) dsv[4 * j + r] = p[r] * dp[r];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w, r;
                pack_twice<DT>(dsv[2 * i], dsv[2 * i + 1], w, r);
                db[i] = w, dr[i] = r;
            }
            LDS_PTR(char) qtile = q_lds + qi * LL::kTileBytes;
            LDS_PTR(char) gtile = g_lds + qi * LL::kTileBytes;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const u32x2 g0 = read_tr(gtile + tr_lane.off[ct]), g1 = read_tr(gtile + LL::kTileBytes + tr_lane.off[ct]);
                const u32x2 q0t = read_tr(qtile + tr_lane.off[ct]), q1t = read_tr(qtile + LL::kTileBytes + tr_lane.off[ct]);
                const u32x4 gg = {g0.x, g0.y, g1.x, g1.y}, qq = {q0t.x, q0t.y, q1t.x, q1t.y};
                accv[ct] = Mma<DT>::k32(gg, pb, accv[ct]);
                acck[ct] = Mma<DT>::k32(qq, db, acck[ct]);
                accv[ct] = Mma<DT>::k32(gg, pr, accv[ct]);
                acck[ct] = Mma<DT>::k32(qq, dr, acck[ct]);
            }
        }
    }
    const float back = __builtin_amdgcn_ldexpf(1.f, less - kBackLift<DT>);
    const bool shared = !far && strip_id >= (uint32_t)a.whole, sinking = a.far && w0 < a.sinks;
    if (shared || far || sinking) {
        if (far && !sinking) return;
        const Partial at_ = partial_of<C>(strip_id, part, (int64_t)head * a.sink_strips + strip, part, heads, a);
        const int rows = shared ? kChunkRows : a.sink_rows;
        float *to = partial + (shared ? at_.shared : far ? at_.far : at_.near) + (own + n) * C + 4 * g;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            *reinterpret_cast<f32x4 *>(to + 16 * ct) = acck[ct] * back;
            *reinterpret_cast<f32x4 *>(to + rows * C + 16 * ct) = accv[ct] * back;
        }
        return;
    }
    const int64_t off = sample * a.dkv.sample + kv * a.dkv.head;
    const Rsrc dks = rows_of(dk + off, row0, row_end - row0, a.dkv.pitch), dvs = rows_of(dv + off, row0, row_end - row0, a.dkv.pitch);
    const bool stream = stores_whole_lines(a.dkv.pitch, C, 0);
    u32x2 kw[CT], vw[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        kw[ct] = pack_acc<DT>(acck[ct], a.scale * back);
        vw[ct] = pack_acc<DT>(accv[ct], back);
        if (key >= tv) kw[ct] = vw[ct] = u32x2{0u, 0u};
    }
    store_tile<C>(dks, (own + n) * a.dkv.pitch, kw, g, stream, width);      // rows past T are dropped
    store_tile<C>(dvs, (own + n) * a.dkv.pitch, vw, g, stream, width);
}

// Rows of dK and dV that several workgroups have a share in: strips in parts, and the tiles with sinks of the others.  Four channels of a row to a thread.
template <class DT, int C>
__global__ void __launch_bounds__(kThreads)
sink_join_kernel(char *__restrict__ dk, char *__restrict__ dv, const float *__restrict__ partial, const int32_t *__restrict__ t_valid, uint32_t heads, SinkArgs a) {
    constexpr int kQuads = C / 4;
    constexpr uint32_t kBlocks = (kChunkRows * kQuads + kThreads - 1) / kThreads;     // workgroups to a strip
    const uint32_t block = blockIdx.x % kBlocks, unit = blockIdx.x / kBlocks, shared = heads * a.strips - a.whole;
    const int i = block * kThreads + threadIdx.x, r = i / kQuads, ch = (i % kQuads) * 4;
    // the strips in parts, then those with sinks (which may be among them)
    uint32_t head, strip;
    if (unit < shared) {
        head = (a.whole + unit) / (uint32_t)a.strips, strip = a.whole + unit - head * a.strips;
    } else {
        head = (unit - shared) / (uint32_t)a.sink_strips, strip = unit - shared - head * a.sink_strips;
    }
    const uint32_t strip_id = head * a.strips + strip;
    const bool in_parts = strip_id >= (uint32_t)a.whole, sinking = a.far && strip < (uint32_t)a.sink_strips && r < a.sink_rows && (int)(strip * kChunkRows) + (r & ~15) < a.sinks;
    const int row = strip * kChunkRows + r;
    if (i >= kChunkRows * kQuads || row >= a.T || 2 * ch >= a.width || (unit >= shared && (in_parts || !sinking))) return;
    f32x4 sk = {0.f, 0.f, 0.f, 0.f}, sv = sk;
    auto add = [&](int64_t from, int rows) {
        sk += *reinterpret_cast<const f32x4 *>(partial + from + r * C + ch);
        sv += *reinterpret_cast<const f32x4 *>(partial + from + (rows + r) * C + ch);
    };
    const int64_t sink_strip = (int64_t)head * a.sink_strips + strip;
    if (in_parts) {
#pragma unroll 4
        for (int p = 0; p < a.parts; ++p) add(partial_of<C>(strip_id, p, sink_strip, 0, heads, a).shared, kChunkRows);
    } else {
        add(partial_of<C>(strip_id, 0, sink_strip, 0, heads, a).near, a.sink_rows);
    }
    if (sinking) {
#pragma unroll 8
        for (int f = 0; f < a.far; ++f) add(partial_of<C>(strip_id, 0, sink_strip, f, heads, a).far, a.sink_rows);
    }
    u32x2 kw = pack_acc<DT>(sk, a.scale), vw = pack_acc<DT>(sv, 1.f);
    const uint32_t sample = head / (uint32_t)a.K, kv = head - sample * a.K;
    if (t_valid && row >= t_valid[sample]) kw = vw = u32x2{0u, 0u};
    const int64_t off = sample * a.dkv.sample + kv * a.dkv.head + (int64_t)row * a.dkv.pitch + 2 * ch;
    *reinterpret_cast<u32x2 *>(dk + off) = kw;
    *reinterpret_cast<u32x2 *>(dv + off) = vw;
}

// ----------------------------------------------------------------------------- launchers
// The forward takes two tiles of 16 queries to a wave, strips of 128, where there are many of those and windows are long: each operand read from LDS then feeds
// two products (window 2048, 16384 tokens, 32 heads of 128: 669 us and not 764; 8192 tokens, 2 x 16 heads of 32, window 1024: 88 and 102).  Fewer workgroups
// are better off as twice as many (4096 tokens, 16 heads of 128, window 1024: 52.7 us and not 53.4; 6 x 12 x 1237, 72 channels, window 333: 23 and 27), and
// windows of a few chunks spend their time on what the strip has to load and store (16 x 16 x 1000, 64 channels, window 128: 39.8 and 43).
bool two_tiles(const na1d_sink &h) { return h.N * h.heads * ((h.T + 127) / 128) >= 1024 && std::min(h.window, h.T) >= 256; }

SinkArgs sink_args(const na1d_sink &h, int tiles) {
    SinkArgs a{};
    const int64_t rows = kChunkRows * tiles;
    a.T = (int)h.T, a.H = h.heads, a.K = h.kv_heads, a.group = h.heads / h.kv_heads, a.strips = (int)((h.T + rows - 1) / rows);
    a.window = (int)std::min(h.window, h.T), a.sinks = (int)std::min(h.sinks, h.T), a.width = 2 * h.head_dim, a.scale = h.scale;
    auto strided = [](const int64_t (&s)[3]) { return SinkRows{2 * s[0], 2 * s[1], (int)(2 * s[2])}; };
    auto packed = [&](int heads) { return SinkRows{2 * h.T * heads * h.head_dim, 2 * h.head_dim, 2 * heads * h.head_dim}; };
    a.q = strided(h.q_strides), a.k = strided(h.k_strides), a.v = strided(h.v_strides), a.o = packed(h.heads), a.dkv = packed(h.kv_heads);
    return a;
}
// How dK and dV are cut into workgroups (see sink_dkv_kernel).
struct KeyPlan {
    SinkArgs a;
    int64_t heads, rest, floats, joined;      // rest: workgroups beside the strips' own; floats of partial sums; strips that are joined
};
KeyPlan key_plan(const na1d_sink &h) {
    KeyPlan p{};
    SinkArgs &a = p.a;
    a = sink_args(h, 1);
    p.heads = h.N * h.kv_heads;
    const int C = channels_of(h.head_dim);
    const int64_t strips = p.heads * a.strips, round = 256 * (C >= 96 ? 2 : C == 64 ? 4 : 6);      // workgroups that the card holds at once
    const int64_t chunks = a.strips, near = std::min<int64_t>(chunks, (a.window + kChunkRows - 2) / kChunkRows + 1), units = near * a.group;      // a strip's
    const int64_t over = strips % round;
    a.parts = 1;
    if (over > 0 && over <= round / 2) a.parts = (int)std::max<int64_t>(1, std::min<int64_t>({round / over, units / 4, 16}));
    a.whole = (int)std::min<int64_t>(strips - (a.parts > 1 ? over : 0), INT32_MAX);
    a.sink_strips = (int)((a.sinks + kChunkRows - 1) / kChunkRows);
    a.sink_rows = std::min(kChunkRows, (a.sinks + 15) / 16 * 16);
    // far workgroups are as many as there are CUs, or have as many units as the others where that makes more of them; from a thousand strips with sinks on
    // there are enough of those as they are
    const int64_t sinking = p.heads * a.sink_strips, beyond = chunks - near;
    if (sinking > 0 && sinking < 1024 && beyond > 0)
        a.far = (int)std::max<int64_t>(1, std::min<int64_t>({std::max((beyond + near - 1) / near, 256 / sinking), 1024 / sinking, beyond * a.group / 4}));
    const int64_t shared = strips - a.whole;
    p.rest = shared * a.parts + sinking * a.far;
    p.floats = shared * a.parts * (2 * kChunkRows * (int64_t)C) + (a.far ? sinking * (1 + a.far) * (2 * a.sink_rows * (int64_t)C) : 0);
    p.joined = shared + (a.far ? sinking : 0);
    return p;
}
int64_t lse_floats(const na1d_sink &h) { return (h.N * h.heads * h.T + 3) / 4 * 4; }
int64_t largest_floats(const na1d_sink &h) { return h.dtype == NA1D_FP16 ? h.N * h.heads * ((h.T + kChunkRows - 1) / kChunkRows) * kWaves : 0; }

template <class DT, int C>
int launch_sink_fwd(const na1d_sink &h, void *out, float *saved, const void *q, const void *k, const void *v, const int32_t *t_valid, hipStream_t s) {
    const bool two = two_tiles(h);
    const SinkArgs a = sink_args(h, two ? 2 : 1);
    const int64_t items = h.N * h.heads * a.strips;
    if (!launchable(items)) return NA1D_ERR_UNSUPPORTED;
    const size_t lds = 4 * (size_t)region_bytes<kStaged<C>>(kKeyTiles);
    auto go = [&](auto kern) {
        if (!allow_lds(kern, lds)) return (int)NA1D_ERR_LAUNCH;
        note_kernel_as("sink_fwd_kernel<%s, %d, %d>", DT::tag == NA1D_BF16 ? "BF16" : "FP16", C, two ? 2 : 1);
        launch_kernel(kern, (unsigned)items, lds, s, (char *)out, saved, saved ? (char *)(saved + lse_floats(h)) : nullptr, (const char *)q, (const char *)k,
                      (const char *)v, t_valid, (uint32_t)items, a);
        return launch_status();
    };
    return two ? go(sink_fwd_kernel<DT, C, 2>) : go(sink_fwd_kernel<DT, C, 1>);
}

template <class DT, int C>
int launch_sink_bwd(const na1d_sink &h, void *dq, void *dk, void *dv, const void *q, const void *k, const void *v, const void *out, const void *dout,
                    const float *saved, const int32_t *t_valid, float *ws, hipStream_t s) {
    const SinkArgs a = sink_args(h, 1);
    const KeyPlan p = key_plan(h);
    const int64_t items = h.N * h.heads * a.strips, key_items = p.a.whole + p.rest, join_items = p.joined * ((kChunkRows * (C / 4) + kThreads - 1) / kThreads);
    if (!launchable(items) || !launchable(p.heads * p.a.strips) || !launchable(key_items) || !launchable(join_items)) return NA1D_ERR_UNSUPPORTED;
    float *const delta = ws, *const largest = ws + lse_floats(h), *const partial = largest + largest_floats(h);
    constexpr size_t dq_lds = 4 * (size_t)region_bytes<kStaged<C>>(kKeyTiles), dkv_lds = 2 * (2 * (size_t)region_bytes<kStaged<C>>(kChunkTiles) + 2 * kChunkRows * sizeof(float));
    if (!allow_lds(sink_dq_kernel<DT, C>, dq_lds) || !allow_lds(sink_dkv_kernel<DT, C>, dkv_lds)) return NA1D_ERR_LAUNCH;
    note_kernel_as("sink_dq_kernel + sink_dkv_kernel<%s, %d>", DT::tag == NA1D_BF16 ? "BF16" : "FP16", C);
    launch_kernel_span(1, sink_dq_kernel<DT, C>, (unsigned)items, (unsigned)kThreads, dq_lds, s, (char *)dq, delta, largest, (const char *)q, (const char *)k, (const char *)v, (const char *)out,
                       (const char *)dout, saved, (const char *)(saved + lse_floats(h)), t_valid, (uint32_t)items, a);
    launch_kernel_span(p.joined ? 0 : 2, sink_dkv_kernel<DT, C>, (unsigned)key_items, (unsigned)kThreads, dkv_lds, s, (char *)dk, (char *)dv, partial, (const char *)q,
                       (const char *)k, (const char *)v, (const char *)dout, saved, (const float *)delta, (const float *)largest, t_valid, (uint32_t)p.rest, (uint32_t)p.heads, p.a);
    if (p.joined)
        launch_kernel_span(2, sink_join_kernel<DT, C>, (unsigned)join_items, (unsigned)kThreads, 0, s, (char *)dk, (char *)dv, (const float *)partial, t_valid,
                           (uint32_t)p.heads, p.a);
    return launch_status();
}

template <class F> int by_width(const na1d_sink &h, F run) {
    auto typed = [&](auto dt) {
        switch (channels_of(h.head_dim)) {
            case 16: return run(dt, std::integral_constant<int, 16>());
            case 32: return run(dt, std::integral_constant<int, 32>());
            case 64: return run(dt, std::integral_constant<int, 64>());
            case 96: return run(dt, std::integral_constant<int, 96>());
            case 128: return run(dt, std::integral_constant<int, 128>());
        }
        return (int)NA1D_ERR_UNSUPPORTED;
    };
    return h.dtype == NA1D_BF16 ? typed(BF16()) : typed(FP16());
}

}  // namespace

int64_t sink_saved_bytes(const na1d_sink &h) {
    return 4 * lse_floats(h) + h.N * h.heads * ((h.T + 15) / 16) * 16 * channels_of(h.head_dim);
}
int64_t sink_bwd_workspace_bytes(const na1d_sink &h) {
    return 4 * (lse_floats(h) + largest_floats(h) + key_plan(h).floats);
}

int sink_fwd(const na1d_sink &h, void *out, float *saved, const void *q, const void *k, const void *v, const int32_t *t_valid, hipStream_t s) {
    return by_width(h, [&](auto dt, auto c) { return launch_sink_fwd<decltype(dt), decltype(c)::value>(h, out, saved, q, k, v, t_valid, s); });
}

int sink_bwd(const na1d_sink &h, void *dq, void *dk, void *dv, const void *q, const void *k, const void *v, const void *out, const void *dout, const float *saved,
             const int32_t *t_valid, float *ws, hipStream_t s) {
    return by_width(h, [&](auto dt, auto c) { return launch_sink_bwd<decltype(dt), decltype(c)::value>(h, dq, dk, dv, q, k, v, out, dout, saved, t_valid, ws, s); });
}

}  // namespace mfma
}  // namespace na1d
