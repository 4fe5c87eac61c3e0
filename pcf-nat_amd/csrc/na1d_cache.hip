// Attention of a few tokens over a cache that holds what a causal window with sinks can see (na1d_sink.hip has whole sequences), with its rows
// in 16 bits or in 4, and what goes with such a cache (gfx950): storing tokens, and reading rows back.
//
// Position p of a sequence is in row p where p < sinks, else in row sinks + (p - sinks) mod ring, ring = capacity - sinks.  The keys that a call's
// tokens see are numbered 0 .. total - 1: the sinks that lie before the window of the first of them, then the positions from there on.
//
// A workgroup has one head of keys of one sequence, 16 to 64 rows of queries (a token's heads of the group, then the next token's) and a share of
// the keys.  What bounds these kernels is memory: every byte of the cache is used for a handful of queries.  So each wave walks its own units of
// keys and keeps the next one in flight, straight into a part of LDS of its own: no barriers, and every wave's loads overlap all other work.  The
// waves join their sums at the end, workgroups that share a head's keys through memory (cache_join_kernel).
//
// 4 bits: a row is codes c, two to a byte, with its least value and the step from one code to the next: x = low + step c.  Both products take the
// codes as they are, exact in 16 bits:
//   q . k = step (q . (16 + c)) + (low - 16 step) sum(q),   sum p v = sum (p step)(16 + c) - 23.5 sum (p step) + sum p (low + 7.5 step)
// where 16 + c costs two instructions for two codes: the code's bits shifted and put into the mantissa of 16.  (p step) is rounded to 16 bits, all else is
// exact or fp32; with 16 for 23.5 and low for the middle of the row's range that rounding would weigh up to 15 steps in place of 7.5.  In fp16, where p may be
// 2^6 and a step anything from 2^-24 to 2^13, steps count times a power of two that a wave chooses by the largest it has met.
#include <type_traits>

#include "na1d_mfma_core.h"

namespace na1d {
namespace mfma {
namespace {

constexpr float kNoMaximum = -3.4e38f;      // where a row's running maximum starts: finite, so that keys which a row does not see leave it alone
constexpr int kLatest = 1 << 30;            // a sequence that has seen more is taken as idle

struct Rows {                   // one tensor [N, T, heads, C]: bytes from one sample, head, token to the next
    int64_t sample, head, row;
};
struct CacheArgs {
    int K, group, fresh, rows, blocks, splits;      // fresh: tokens of the call; rows of queries to a key head: fresh * group, in `blocks` blocks
    int window, sinks, ring, width;                 // width: bytes of a row in 16 bits
    int stored;                                     // tokens that this call puts into the cache: fresh, or 0
    float scale;
    Rows q, k, v;
    int64_t slice, ranges;      // bytes of a head's rows, and of their ranges
};

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// What a call's tokens see of one sequence.
struct Seen {
    int total, apart, from, end, first;      // `apart` sinks, then the positions from .. end - 1, the first of them in ring row `first`
    int ring, sinks;
    __device__ inline Seen(int len, const CacheArgs &a) {
        ring = a.ring, sinks = a.sinks;
        const bool idle = len < 0 || len > kLatest;
        end = idle ? 0 : len + a.stored;
        from = max(0, end - a.fresh - a.window + 1);
        apart = min(sinks, from);
        total = apart + end - from;
        // (positions that follow the sinks directly have not come round the ring)
        first = from >= sinks ? (from - sinks) % ring : from - sinks;
    }
    __device__ inline int position(int i) const { return i < apart ? i : from + (i - apart); }
    __device__ inline int row(int i) const {
        int r = first + (i - apart);
        if (r >= ring) r -= ring;
        return i < apart ? i : sinks + r;
    }
};
__device__ inline int row_of(int position, int sinks, int ring) { return position < sinks ? position : sinks + (position - sinks) % ring; }

// Keys i0 .. i1 - 1 of a share: the call's own tokens all belong to the last one, which stores them if they are not in the cache.
__device__ inline void share_of(int split, int splits, int unit, const Seen &s, int fresh, int &i0, int &i1) {
    const int units = max(0, s.total - fresh) / unit;
    i0 = unit * (int)((int64_t)units * split / splits);
    i1 = split + 1 == splits ? s.total : unit * (int)((int64_t)units * (split + 1) / splits);
}

// ------------------------------------------------------------------------------------------------ rows in 4 bits
// One row by as many lanes as have eight of its channels each (4, 8 or 16, from a multiple of that on; `there`: this lane has some): their codes, and the row's
// step and least value.  The step is rounded to the rows' type; the codes are of the step as it is stored.
template <int CTRL> __device__ inline float from_lane(float x) { return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CTRL, 0xf, 0xf, true)); }
template <class DT> __device__ inline uint32_t quantized(const Chunk8 &c, bool there, int lanes, uint32_t &range) {
    float x[8];
    unpack8<DT>(c, x);
    float low = __builtin_inff(), high = -__builtin_inff();
    if (there) {
#pragma unroll
        for (int i = 0; i < 8; ++i) low = __builtin_fminf(low, x[i]), high = __builtin_fmaxf(high, x[i]);
    }
    auto meet = [&](float l, float h) { low = __builtin_fminf(low, l), high = __builtin_fmaxf(high, h); };
    meet(from_lane<0xb1>(low), from_lane<0xb1>(high));           // lanes 1, 0, 3, 2 of four
    meet(from_lane<0x4e>(low), from_lane<0x4e>(high));           // lanes 2, 3, 0, 1
    if (lanes > 4) meet(from_lane<0x141>(low), from_lane<0x141>(high));       // eight lanes in reverse
    if (lanes > 8) meet(from_lane<0x140>(low), from_lane<0x140>(high));       // sixteen
    const uint16_t step16 = DT::from_f32((high - low) / 15.f);
    const float step = DT::to_f32(step16);
    range = step16 | (uint32_t)DT::from_f32(low) << 16;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (step > 0.f ? (uint32_t)__builtin_fminf(__builtin_fmaxf(__builtin_rintf((x[i] - low) / step), 0.f), 15.f) : 0u) << (4 * i);
    return w;
}

// Tokens into the cache: lane `part` of those that a row has (8 channels each) stores its own.
__device__ inline int lanes_to_row(int width) { return width <= 64 ? 4 : width <= 128 ? 8 : 16; }      // width: of 16-bit rows, bytes
template <class DT, int BITS>
__device__ inline void store_token(char *cache, char *ranges, int row, const char *x, int width, int part, int lanes) {
    const bool there = part * 16 < width;
    Chunk8 c = {{0u, 0u, 0u, 0u}};
    if (there) c = *reinterpret_cast<const Chunk8 *>(x + part * 16);
    if constexpr (BITS == 16) {
        if (there) *reinterpret_cast<Chunk8 *>(cache + (int64_t)row * width + part * 16) = c;
    } else {
        uint32_t range;
        const uint32_t w = quantized<DT>(c, there, lanes, range);
        if (there) *reinterpret_cast<uint32_t *>(cache + (int64_t)row * (width / 4) + part * 4) = w;
        if (part == 0) *reinterpret_cast<uint32_t *>(ranges + (int64_t)row * 4) = range;
    }
}
// Tokens of sample n at positions lengths[n] on: those that a later token can see, sinks and the last `ring` ones.  In 4 bits what bounds it is the vector unit: eight
// divisions to a lane, since a code is a quotient's rounding (8 streams of up to 5000 tokens, 8 heads of 128: 32 us, 89 MB); with reciprocals, or two tokens at a time, 35 to 40.
template <class DT, int BITS>
__global__ void __launch_bounds__(kThreads)
cache_append_kernel(char *__restrict__ kc, char *__restrict__ vc, char *__restrict__ kr, char *__restrict__ vr, const char *__restrict__ k, const char *__restrict__ v,
                    const int32_t *__restrict__ lengths, const int32_t *__restrict__ t_valid, int T, int blocks, CacheArgs a) {
    const uint32_t head = uniform(blockIdx.x / (uint32_t)blocks), sample = uniform(head / (uint32_t)a.K), kv = head - sample * a.K;
    const int block = (int)(blockIdx.x - head * blocks), start = lengths ? lengths[sample] : 0;
    const int tv = t_valid ? max(0, min(T, t_valid[sample])) : T;
    if (start < 0 || start > kLatest) return;
    const int lanes = lanes_to_row(a.width), part = threadIdx.x & (lanes - 1), slot = (int)((uint32_t)threadIdx.x / (uint32_t)lanes), slots = kThreads / lanes;
    const char *kx = k + sample * a.k.sample + kv * a.k.head, *vx = v + sample * a.v.sample + kv * a.v.head;
    kc += head * a.slice, vc += head * a.slice, kr += head * a.ranges, vr += head * a.ranges;
    // the last `ring` tokens, and before them those that are sinks
    const int tail = max(0, tv - a.ring), early = max(0, min(tail, a.sinks - start)), count = early + tv - tail;
    for (int j = block * slots + slot; j < count; j += blocks * slots) {
        const int t = j < early ? j : tail + (j - early), row = row_of(start + t, a.sinks, a.ring);
        store_token<DT, BITS>(kc, kr, row, kx + t * a.k.row, a.width, part, lanes);
        store_token<DT, BITS>(vc, vr, row, vx + t * a.v.row, a.width, part, lanes);
    }
}
// Rows as the values that they stand for, or the type's largest number where a step that was rounded up leads beyond it (an fp16 row of -65504 .. 65504 has steps of 8736): eight channels
// to a thread (8 x 8 x 4010 rows of 128: 16 us, 84 MB, 5.2 TB/s).
template <class DT> constexpr float kLargest = DT::tag == NA1D_BF16 ? 0x1.fep127f : 65504.f;
template <class DT>
__global__ void __launch_bounds__(kThreads) cache_rows_kernel(char *__restrict__ out, const char *__restrict__ codes, const char *__restrict__ ranges, int64_t words, int per_row) {
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < words; i += (int64_t)gridDim.x * kThreads) {
        const uint32_t w = reinterpret_cast<const uint32_t *>(codes)[i], range = reinterpret_cast<const uint32_t *>(ranges)[i / per_row];
        const float step = DT::to_f32((uint16_t)(range & 0xffffu)), low = DT::to_f32((uint16_t)(range >> 16));
        float x[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) x[c] = __builtin_fminf(__builtin_fmaf((float)(w >> (4 * c) & 15u), step, low), kLargest<DT>);      // the product is exact
        reinterpret_cast<Chunk8 *>(out)[i] = pack8<DT>(x);
    }
}

// ------------------------------------------------------------------------------------------------ attention
// What a wave has of its rows of queries: lane (n, g) channels 16 ct + 4 g .. + 3 of row n of every tile.
template <int C, int QT> struct Sums {
    float m[QT], l[QT];         // l: this lane's part of the row's sum
    f32x4 o[QT][C / 16];
    __device__ inline void clear() {
#pragma unroll
        for (int h = 0; h < QT; ++h) {
            m[h] = kNoMaximum, l[h] = 0.f;
#pragma unroll
            for (int ct = 0; ct < C / 16; ++ct) o[h][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // `high`: a row's largest score of the unit at hand.  The reference of its exponentials moves only when that has outgrown it by more than
    // kSlack (probabilities stay below 2^kSlack, which every format here holds, also 2^kLift times that).
    __device__ inline float move(int h, float high) {
        constexpr float kSlack = 6.f;
        float alpha = 1.f;
        if (__builtin_amdgcn_ballot_w64(high > m[h] + kSlack)) {
            const float m_new = max2(m[h], high);
            alpha = __builtin_amdgcn_exp2f(m[h] - m_new);
            m[h] = m_new;
            l[h] *= alpha;
#pragma unroll
            for (int ct = 0; ct < C / 16; ++ct) o[h][ct] *= alpha;
        }
        return alpha;
    }
};
template <int C, int QT> constexpr int kJoinRow = C + 4;      // floats: rows of the waves' sums in LDS, apart from each other's banks
template <int C, int QT, int NW> constexpr int kJoinBytes = NW * 16 * QT * (kJoinRow<C, QT> + 2) * 4;

// The waves' sums together: to the output, or (several shares) to memory.
template <class DT, int C, int QT, int NW>
__device__ inline void join_waves(const Sums<C, QT> &s, char *smem, char *out, float *partial, uint32_t head, uint32_t sample, uint32_t kv, int block, int split, int wave, int lane,
                                  const CacheArgs &a) {
    constexpr int kRows = 16 * QT, kQuads = C / 4, kRow = kJoinRow<C, QT>;
    float *rows = reinterpret_cast<float *>(smem), *stats = rows + NW * kRows * kRow;
    const int g = lane >> 4, n = lane & 15;
    __syncthreads();            // the waves are done with what they staged
#pragma unroll
    for (int h = 0; h < QT; ++h) {
        const float l = xor_sum(s.l[h]);
        const int r = wave * kRows + 16 * h + n;
#pragma unroll
        for (int ct = 0; ct < C / 16; ++ct) *reinterpret_cast<f32x4 *>(rows + r * kRow + 16 * ct + 4 * g) = s.o[h][ct];
        if (g == 0) stats[2 * r] = s.m[h], stats[2 * r + 1] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * kQuads; i += 64 * NW) {
        const int r = i / kQuads, ch = (i % kQuads) * 4, row = block * kRows + r;
        if (row >= a.rows || 2 * ch >= a.width) continue;
        float m = kNoMaximum, l = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) m = __builtin_fmaxf(m, stats[2 * (w * kRows + r)]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(stats[2 * (w * kRows + r)] - m);
            l = __builtin_fmaf(stats[2 * (w * kRows + r) + 1], f, l);
            o += *reinterpret_cast<const f32x4 *>(rows + (w * kRows + r) * kRow + ch) * f;
        }
        if (a.splits > 1) {
            const int64_t to = ((int64_t)(head * a.blocks + block) * a.splits + split) * kRows + r;
            *reinterpret_cast<f32x4 *>(partial + to * (C + 4) + ch) = o;
            if (ch == 0) partial[to * (C + 4) + C] = m, partial[to * (C + 4) + C + 1] = l;
        } else {
            const int token = row / a.group, gi = row - token * a.group;
            const int64_t at = (((int64_t)sample * a.fresh + token) * a.K * a.group + kv * a.group + gi) * a.width + 2 * ch;
            *reinterpret_cast<u32x2 *>(out + at) = l > 0.f ? pack_acc<DT>(o, 1.f / l) : u32x2{0u, 0u};
        }
    }
}
// The shares of a head's keys, in a fixed order: four channels of a row to a thread, and eight shares on their way together (2 to 4 us, of which little is work).
template <class DT, int C, int QT>
__global__ void __launch_bounds__(kThreads) cache_join_kernel(char *__restrict__ out, const float *__restrict__ partial, uint32_t quads, CacheArgs a) {
    constexpr int kRows = 16 * QT, kAtOnce = 8;
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;      // (shares are many only where heads are few: 32 bits hold these)
    if (i >= quads) return;
    const uint32_t per_row = a.width / 8, hr = i / per_row, head = hr / (uint32_t)a.rows, row = hr - head * a.rows, sample = head / (uint32_t)a.K, kv = head - sample * a.K;
    const uint32_t ch = (i - hr * per_row) * 4, block = row / kRows;
    const float *from = partial + (((int64_t)(head * a.blocks + block) * a.splits) * kRows + row - block * kRows) * (C + 4);
    float m = kNoMaximum, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; s += kAtOnce) {
        float ms[kAtOnce], ls[kAtOnce], high = m;
        f32x4 os[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const float *x = from + (int64_t)min(s + j, a.splits - 1) * (kRows * (C + 4));
            ms[j] = x[C], ls[j] = x[C + 1], os[j] = *reinterpret_cast<const f32x4 *>(x + ch);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) high = __builtin_fmaxf(high, ms[j]);      // (one share twice at the end: the same maximum)
        const float alpha = __builtin_amdgcn_exp2f(m - high);
        m = high, l *= alpha, o *= alpha;
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const float f = s + j < a.splits ? __builtin_amdgcn_exp2f(ms[j] - m) : 0.f;
            l = __builtin_fmaf(ls[j], f, l);
            o += os[j] * f;
        }
    }
    const uint32_t token = row / (uint32_t)a.group, gi = row - token * a.group;
    const int64_t at = (((int64_t)sample * a.fresh + token) * a.K * a.group + kv * a.group + gi) * a.width + 2 * ch;
    *reinterpret_cast<u32x2 *>(out + at) = l > 0.f ? pack_acc<DT>(o, 1.f / l) : u32x2{0u, 0u};
}

// What is the same in both kernels.
struct Place {
    uint32_t head, sample, kv;
    int block, split;
    __device__ inline Place(uint32_t items, const CacheArgs &a) {
        const uint32_t lin = xcd_item(blockIdx.x, items), hb = uniform(lin / (uint32_t)a.splits);
        split = (int)(lin - hb * a.splits);
        head = uniform(hb / (uint32_t)a.blocks);
        block = (int)(hb - head * a.blocks);
        sample = uniform(head / (uint32_t)a.K);
        kv = head - sample * a.K;
    }
};
// The last share stores the call's tokens.  (Workgroups of other blocks of queries store the same.)
template <class DT, int BITS, int NW>
__device__ inline void store_fresh(char *kc, char *vc, char *kr, char *vr, const char *k, const char *v, const Place &p, const Seen &seen, const CacheArgs &a) {
    if (!a.stored || p.split + 1 < a.splits || seen.total == 0) return;
    const int lanes = lanes_to_row(a.width), part = threadIdx.x & (lanes - 1);
    for (int j = (int)((uint32_t)threadIdx.x / (uint32_t)lanes); j < 2 * a.stored; j += 64 * NW / lanes) {
        const int t = j >> 1, row = row_of(seen.end - a.stored + t, a.sinks, a.ring);
        const bool second = j & 1;
        const Rows &from = second ? a.v : a.k;
        store_token<DT, BITS>((second ? vc : kc) + p.head * a.slice, (second ? vr : kr) + p.head * a.ranges, row,
                              (second ? v : k) + p.sample * from.sample + p.kv * from.head + t * from.row, a.width, part, lanes);
    }
}
// Rows n of the tiles of a block of queries: where they are, and when.
struct QueryRow {
    int64_t at;
    int position;               // -1: no such row
    __device__ inline QueryRow(int row, const Place &p, const Seen &seen, const CacheArgs &a) {
        const int token = row / a.group;
        position = row < a.rows ? seen.end - a.fresh + token : -1;
        at = p.sample * a.q.sample + (p.kv * a.group + row - token * a.group) * a.q.head + token * a.q.row;
    }
};

// A wave's loads that write LDS directly and are still on their way: all but the newest COUNT have landed.
template <int COUNT> __device__ inline void wait_all_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COUNT) : "memory"); }
// LDS reads of the unit before have returned: its place may be written again.
__device__ inline void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// =============================================================================
// Rows in 16 bits: units of 32 keys
// =============================================================================
// One load that writes LDS directly, from anywhere: lane l's 16 bytes land at lds + 16 * l.  As load_to_lds(), unknown to the compiler.
__device__ inline void load_from(const char *p, LDS_PTR(char) lds) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>(lds));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(p) : "memory");
}
// The same from `offset` bytes behind a place that is the same in all lanes.
__device__ inline void load_behind(const char *p, int offset, LDS_PTR(char) lds) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>(lds));
    const uint64_t base = (uint64_t)(uint32_t)uniform((int)((uint64_t)p >> 32)) << 32 | (uint32_t)uniform((int)(uint64_t)p);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(offset), "s"(base) : "memory");
}
// 64 streams, 32 heads over 8 of 128 channels, 4100 keys: 178 us, 1.08 GB, 6.0 TB/s, more than a copy reaches.  A key's row is in the cache, or with the call's tokens: a step does not wait for its own stores.  Past the share's last key that one is loaded again, and
// past a row's channels its first ones: finite, and met by probabilities and queries of zero.
template <class DT, int C, int QT, int NW>
__global__ void __launch_bounds__(64 * NW)
cache_attend_kernel(char *__restrict__ out, float *__restrict__ partial, const char *__restrict__ q, const char *__restrict__ k, const char *__restrict__ v,
                    char *kc, char *vc, const int32_t *__restrict__ lengths, uint32_t items, CacheArgs a) {
    constexpr int CS = kStaged<C>;
    using LL = Lds<CS>;
    constexpr int CT = C / 16, kUnit = 32, kRegion = region_bytes<CS>(2), kStage = 2 * kRegion, kLoads = kStage / kChunk, kChunkKeys = kChunk / LL::kRowBytes;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, n = lane & 15;
    LDS_PTR(char) mine = (LDS_PTR(char))smem + wave * 2 * kStage;
    const Place p(items, a);
    const Seen seen(uniform(lengths[p.sample]), a);
    int i0, i1;
    share_of(p.split, a.splits, kUnit, seen, a.fresh, i0, i1);

    RowOperand<C> qop[QT];
    int when[QT];
#pragma unroll
    for (int h = 0; h < QT; ++h) {
        const QueryRow r(16 * (QT * p.block + h) + n, p, seen, a);
        when[h] = r.position;
#pragma unroll
        for (int s = 0; s < RowOperand<C>::k32; ++s)
            qop[h].w32[s] = r.position >= 0 && 64 * s + 16 * g < a.width ? *reinterpret_cast<const u32x4 *>(q + r.at + 64 * s + 16 * g) : u32x4{0u, 0u, 0u, 0u};
        if (RowOperand<C>::k16)
            qop[h].w16[0] = r.position >= 0 && 8 * g < a.width ? *reinterpret_cast<const u32x2 *>(q + r.at + 8 * g) : u32x2{0u, 0u};
    }
    const char *ks = kc + p.head * a.slice, *vs = vc + p.head * a.slice;
    const char *kx = k + p.sample * a.k.sample + p.kv * a.k.head, *vx = v + p.sample * a.v.sample + p.kv * a.v.head;
    const int old = seen.total - a.stored;
    auto stage = [&](int i, LDS_PTR(char) to) {
        int row0 = seen.first + (i - seen.apart);
        if (row0 >= seen.ring) row0 -= seen.ring;
        if (i >= seen.apart && i + kUnit <= min(i1, old) && row0 + kUnit <= seen.ring) {      // rows of the cache, one behind the other
            const int64_t base = (int64_t)(seen.sinks + row0) * a.width;
#pragma unroll
            for (int c = 0; c < kRegion / kChunk; ++c) {
                const int r = c * kChunkKeys + lane / LL::kUnits, unit = (lane % LL::kUnits) ^ LL::swz(r), offset = r * a.width + (unit * 16 < a.width ? unit * 16 : 0);
                load_behind(ks + base, offset, to + c * kChunk);
                load_behind(vs + base, offset, to + kRegion + c * kChunk);
            }
            return;
        }
#pragma unroll
        for (int c = 0; c < kRegion / kChunk; ++c) {
            const int r = c * kChunkKeys + lane / LL::kUnits, unit = (lane % LL::kUnits) ^ LL::swz(r), key = min(i + r, i1 - 1);
            const int byte = unit * 16 < a.width ? unit * 16 : 0;
            const int64_t at = (int64_t)seen.row(key) * a.width + byte;
            const bool fresh = key >= old;
            load_from(fresh ? kx + (key - old) * a.k.row + byte : ks + at, to + c * kChunk);
            load_from(fresh ? vx + (key - old) * a.v.row + byte : vs + at, to + kRegion + c * kChunk);
        }
    };
    RowLane<C, CS> row_lane;
    TrLane<C, CS> tr_lane;
    row_lane.init(0, lane);
    tr_lane.init(0, lane);
    const float scale2 = a.scale * kLog2e;
    Sums<C, QT> sums;
    sums.clear();
    int at = 0;
    int i = i0 + kUnit * wave;
    if (i < i1) stage(i, mine);
#pragma unroll
    for (int h = 0; h < QT; ++h) {          // the queries are here before the next unit is asked for: waiting for them later would wait for that as well
#pragma unroll
        for (int s = 0; s < RowOperand<C>::k32; ++s) settle(qop[h].w32[s]);
        if (RowOperand<C>::k16) settle(qop[h].w16[0]);
    }
    store_fresh<DT, 16, NW>(kc, vc, nullptr, nullptr, k, v, p, seen, a);
    for (; i < i1; i += kUnit * NW, at ^= kStage) {
        reads_done();
        if (i + kUnit * NW < i1) {
            stage(i + kUnit * NW, mine + (at ^ kStage));
            wait_all_but<kLoads>();
        } else {
            wait_direct();
        }
        LDS_PTR(char) k_lds = mine + at;
        LDS_PTR(char) v_lds = k_lds + kRegion;
        f32x4 s[QT][2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            RowOperand<C> kop;
            read_rows<C, CS>(kop, k_lds + kt * LL::kTileBytes, row_lane);
#pragma unroll
            for (int h = 0; h < QT; ++h) s[h][kt] = dot_rows_mma<DT, C>(kop, qop[h]);
        }
        const bool ends = i + kUnit > i1;
        u32x4 pp[QT];
#pragma unroll
        for (int h = 0; h < QT; ++h) {
            if (ends || a.fresh > 1) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = i + 16 * kt + 4 * g + r, behind = when[h] - seen.position(key);
                        if (!(key < i1 && behind >= 0 && (behind < a.window || key < seen.apart || seen.position(key) < a.sinks))) s[h][kt][r] = kNegInf;
                    }
            }
            float high = kNegInf;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) high = __builtin_fmaxf(high, s[h][kt][r]);
            sums.move(h, reference_of<DT>(xor_max(high) * scale2));
            const float ref = kLift<DT> - sums.m[h];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                float e[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][kt][r], scale2, ref));
                sums.l[h] += (e[0] + e[1]) + (e[2] + e[3]);
                pp[h][2 * kt] = Mma<DT>::pack(e[0], e[1]);
                pp[h][2 * kt + 1] = Mma<DT>::pack(e[2], e[3]);
            }
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const u32x2 v0 = read_tr(v_lds + tr_lane.off[ct]), v1 = read_tr(v_lds + LL::kTileBytes + tr_lane.off[ct]);
            const u32x4 vv = {v0.x, v0.y, v1.x, v1.y};
#pragma unroll
            for (int h = 0; h < QT; ++h) sums.o[h][ct] = Mma<DT>::k32(vv, pp[h], sums.o[h][ct]);
        }
    }
    join_waves<DT, C, QT, NW>(sums, smem, out, partial, p.head, p.sample, p.kv, p.block, p.split, wave, lane, a);
}

// =============================================================================
// Rows in 4 bits: units of 64 keys
// =============================================================================
// 64 streams, 32 heads over 8 of 128 channels, 8196 keys: 113 us, 572 MB, 5.1 TB/s.  What keeps it from the 6.0 of 16 bits is the vector unit: codes into values, and a softmax of
// 16 rows where a group has four, about 550 instructions to a unit of 8.7 KB.
// Values 16 + c of the eight codes of a word, channels (or keys) 0, 4, 1, 5, 2, 6, 3, 7 of it: codes four apart share a register.
template <class DT> __device__ inline u32x4 of_codes(uint32_t w) {
    if constexpr (DT::tag == NA1D_BF16) {       // 16 (1 + c / 16): c at bit 3 of seven
        constexpr uint32_t m = 0x00780078u, one = 0x41804180u;
        return u32x4{(w << 3 & m) | one, (w >> 1 & m) | one, (w >> 5 & m) | one, (w >> 9 & m) | one};
    } else {                                    // c at bit 6 of ten
        constexpr uint32_t m = 0x03c003c0u, one = 0x4c004c00u;
        return u32x4{(w << 6 & m) | one, (w << 2 & m) | one, (w >> 2 & m) | one, (w >> 6 & m) | one};
    }
}
// Eight 16-bit values in the order in which of_codes() has its own.
__device__ inline u32x4 in_code_order(u32x4 x) {
    auto low = [](uint32_t a, uint32_t b) { return (a & 0xffffu) | b << 16; };
    auto high = [](uint32_t a, uint32_t b) { return a >> 16 | (b & 0xffff0000u); };
    return u32x4{low(x[0], x[2]), high(x[0], x[2]), low(x[1], x[3]), high(x[1], x[3])};
}
// The product of two tiles of keys with V takes them where ds_read_b64_tr_b4 leaves them: lane (n, g) gets channel n of the 16 keys 16 g .., the first
// eight for one product, the others for the next.  Row m = 4 g' + r of score tile kt leaves its scores in lanes of group g', register r; so that
// row has to be the key that those lanes' register stands for in the product with V (in the order of of_codes()): the tiles of keys are staged in this order.
__device__ inline int key_of_row(int row) {
    const int kt = row >> 4, g = (row >> 2) & 3, r = row & 3;
    return 16 * g + 8 * (kt >> 1) + 2 * (kt & 1) + (r >> 1) + 4 * (r & 1);
}
template <class DT, int C, int QT, int NW>
__global__ void __launch_bounds__(64 * NW)
cache_attend4_kernel(char *__restrict__ out, float *__restrict__ partial, const char *__restrict__ q, const char *__restrict__ k, const char *__restrict__ v,
                     char *kc, char *vc, char *kr, char *vr, const int32_t *__restrict__ lengths, uint32_t items, CacheArgs a) {
    constexpr int CT = C / 16, S = C / 32, kUnit = 64, kRow = C / 2, kUnits = kRow / 16;
    constexpr int kCodes = kUnit * kRow, kRanges = kUnit * 4, kStage = 2 * (kCodes + kRanges), kLoads = 2 * (kCodes / kChunk + 1);
    static_assert(C % 32 == 0 && kCodes % kChunk == 0, "whole chunks");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, n = lane & 15;
    LDS_PTR(char) mine = (LDS_PTR(char))smem + wave * 2 * kStage;
    const Place p(items, a);
    const Seen seen(uniform(lengths[p.sample]), a);
    store_fresh<DT, 4, NW>(kc, vc, kr, vr, k, v, p, seen, a);
    if (a.stored) __syncthreads();      // the call's tokens are read back as the cache holds them
    int i0, i1;
    share_of(p.split, a.splits, kUnit, seen, a.fresh, i0, i1);
    const Rsrc ks = make_rsrc(kc + p.head * a.slice, (int)a.slice), vs = make_rsrc(vc + p.head * a.slice, (int)a.slice);
    const Rsrc krs = make_rsrc(kr + p.head * a.ranges, (int)a.ranges), vrs = make_rsrc(vr + p.head * a.ranges, (int)a.ranges);

    // Queries: lane (n, g) has channels (C / 4) g + 8 s .. + 7 of row n for step s, where its words of a row of codes are.
    u32x4 qop[QT][S];
    int when[QT];
    float qsum[QT];
#pragma unroll
    for (int h = 0; h < QT; ++h) {
        const QueryRow r(16 * (QT * p.block + h) + n, p, seen, a);
        when[h] = r.position;
#pragma unroll
        for (int s = 0; s < S; ++s) qop[h][s] = r.position >= 0 ? *reinterpret_cast<const u32x4 *>(q + r.at + (C / 2) * g + 16 * s) : u32x4{0u, 0u, 0u, 0u};
    }
    // Rows have their 16-byte units swapped about so that the 16 rows a read takes a unit of lie in distinct banks
    auto swz = [](int row) { return kUnits == 4 ? row >> 2 & 3 : kUnits == 2 ? row >> 3 & 1 : 0; };
    auto stage = [&](int i, LDS_PTR(char) to) {
        int row0 = seen.first + (i - seen.apart);
        if (row0 >= seen.ring) row0 -= seen.ring;
        if (i >= seen.apart && i + kUnit <= i1 && row0 + kUnit <= seen.ring) {      // rows one behind the other: what a lane adds to the first's place stays the same
            row0 += seen.sinks;
#pragma unroll
            for (int c = 0; c < kCodes / kChunk; ++c) {
                const int u = 64 * c + lane, r = u / kUnits, at = ((u % kUnits) ^ swz(r)) * 16;
                load_to_lds<16, kReadShared>(ks, to + c * kChunk, row0 * kRow + (key_of_row(r) * kRow + at));
                load_to_lds<16, kReadShared>(vs, to + kCodes + c * kChunk, row0 * kRow + (r * kRow + at));
            }
            load_to_lds<4, kReadShared>(krs, to + 2 * kCodes, row0 * 4 + key_of_row(lane) * 4);
            load_to_lds<4, kReadShared>(vrs, to + 2 * kCodes + kRanges, row0 * 4 + key_of_row(lane) * 4);
            return;
        }
#pragma unroll
        for (int c = 0; c < kCodes / kChunk; ++c) {
            const int u = 64 * c + lane, r = u / kUnits, unit = u % kUnits, kkey = i + key_of_row(r), vkey = i + r;
            load_to_lds<16, kReadShared>(ks, to + c * kChunk, kkey < i1 ? seen.row(kkey) * kRow + (unit ^ swz(r)) * 16 : kNowhere);
            load_to_lds<16, kReadShared>(vs, to + kCodes + c * kChunk, vkey < i1 ? seen.row(vkey) * kRow + (unit ^ swz(r)) * 16 : kNowhere);
        }
        const int key = i + key_of_row(lane), at = key < i1 ? seen.row(key) * 4 : kNowhere;
        load_to_lds<4, kReadShared>(krs, to + 2 * kCodes, at);
        load_to_lds<4, kReadShared>(vrs, to + 2 * kCodes + kRanges, at);
    };
    const int k_off = n * kRow + ((((kRow / 4) * g >> 4) ^ swz(n)) << 4 | ((kRow / 4) * g & 15));      // of this lane's row n, channels (C / 4) g ..
    int v_off[CT];              // of this lane's row 16 g + n, channels 16 ct ..
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) v_off[ct] = (16 * g + n) * kRow + (((ct >> 1) ^ swz(16 * g + n)) << 4 | (ct & 1) << 3);
    const float scale2 = a.scale * kLog2e;
    Sums<C, QT> sums;
    sums.clear();
    f32x4 steps[QT];            // sum of (p step), as rounded
    float mids[QT];             // this lane's part of sum p (low + 7.5 step)
#pragma unroll
    for (int h = 0; h < QT; ++h) steps[h] = f32x4{0.f, 0.f, 0.f, 0.f}, mids[h] = 0.f;
    // fp16: steps, and with them `o` and `steps`, count times 2^up.  The largest step is between 2^7 and 2^9 then: 2^15 with a p of 2^6, while a key is off by 2^-32 of it at most where
    // its product is below fp16's normal range (as they were, products of steps above 1000 were infinite, and those of shares of 2^-12 with steps of 2^-11 a tenth off).
    constexpr bool kLifts = DT::tag == NA1D_FP16;
    int up = 31;                // has the least step there
    int at = 0;
    int i = i0 + kUnit * wave;
    if (i < i1) stage(i, mine);
#pragma unroll
    for (int h = 0; h < QT; ++h) {
        float sum = 0.f;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            qop[h][s] = in_code_order(qop[h][s]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x2 x = unpack2<DT>(qop[h][s][j]);
                sum += x.x + x.y;
            }
            settle(qop[h][s]);
        }
        qsum[h] = xor_sum(sum) * scale2;
    }
    for (; i < i1; i += kUnit * NW, at ^= kStage) {
        reads_done();
        if (i + kUnit * NW < i1) {
            stage(i + kUnit * NW, mine + (at ^ kStage));
            wait_all_but<kLoads>();
        } else {
            wait_direct();
        }
        LDS_PTR(char) k_lds = mine + at;
        LDS_PTR(char) v_lds = k_lds + kCodes;
        LDS_PTR(char) r_lds = v_lds + kCodes;
        // What goes with a key, worked out by one lane for all: in the place of the ranges first K's numbers, then V's (the wave's own accesses stay in order, and all are of 32-bit integers).
        const f32x2 of_k = unpack2<DT>(*reinterpret_cast<LDS_PTR(uint32_t)>(r_lds + 4 * lane)), of_v = unpack2<DT>(*reinterpret_cast<LDS_PTR(uint32_t)>(r_lds + kRanges + 4 * lane));
        float v_step = of_v.x;
        if constexpr (kLifts) {
            if (__builtin_amdgcn_ballot_w64(__builtin_amdgcn_ldexpf(v_step, up) > 512.f)) {
                float most = v_step;
#pragma unroll
                for (int d = 1; d < 64; d *= 2) most = __builtin_fmaxf(most, __shfl_xor(most, d));
                const int now = uniform(8 - __builtin_amdgcn_frexp_expf(most));       // between 2^7 and 2^8
                const float by = __builtin_amdgcn_ldexpf(1.f, now - up);
                up = now;
#pragma unroll
                for (int h = 0; h < QT; ++h) {
                    steps[h] *= by;
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) sums.o[h][ct] *= by;
                }
            }
            v_step = __builtin_amdgcn_ldexpf(v_step, up);
        }
        auto share = [&](float x, float y) {
            *reinterpret_cast<LDS_PTR(uint32_t)>(r_lds + 4 * lane) = __float_as_uint(x);
            *reinterpret_cast<LDS_PTR(uint32_t)>(r_lds + kRanges + 4 * lane) = __float_as_uint(y);
        };
        auto shared = [&](int which, int kt) { return __builtin_bit_cast(f32x4, *reinterpret_cast<LDS_PTR(u32x4)>(r_lds + which * kRanges + 64 * kt + 16 * g)); };
        share(of_k.x * scale2, __builtin_fmaf(-16.f, of_k.x, of_k.y));
        f32x4 z[QT][4];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            uint32_t w[S];
#pragma unroll
            for (int s = 0; s < S; ++s) w[s] = *reinterpret_cast<LDS_PTR(uint32_t)>(k_lds + 16 * kt * kRow + k_off + 4 * s);
#pragma unroll
            for (int h = 0; h < QT; ++h) z[h][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const u32x4 kop = of_codes<DT>(w[s]);
#pragma unroll
                for (int h = 0; h < QT; ++h) z[h][kt] = Mma<DT>::k32(kop, qop[h][s], z[h][kt]);
            }
            const f32x4 by = shared(0, kt), and_ = shared(1, kt);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int h = 0; h < QT; ++h) z[h][kt][r] = __builtin_fmaf(z[h][kt][r], by[r], and_[r] * qsum[h]);
        }
        share(v_step, __builtin_fmaf(7.5f, of_v.x, of_v.y));
        const bool ends = i + kUnit > i1;
        u32x4 pp[QT][2];
#pragma unroll
        for (int h = 0; h < QT; ++h) {
            if (ends || a.fresh > 1) {
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = i + key_of_row(16 * kt + 4 * g + r), behind = when[h] - seen.position(key);
                        if (!(key < i1 && behind >= 0 && (behind < a.window || key < seen.apart || seen.position(key) < a.sinks))) z[h][kt][r] = kNegInf;
                    }
            }
            float high = kNegInf;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) high = __builtin_fmaxf(high, z[h][kt][r]);
            const float alpha = sums.move(h, xor_max(high));
            steps[h] *= alpha;
            mids[h] *= alpha;
            const float m = sums.m[h];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                const f32x4 step = shared(0, kt), mid = shared(1, kt);
                float e[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    e[r] = __builtin_amdgcn_exp2f(z[h][kt][r] - m);
                    sums.l[h] += e[r];
                    mids[h] = __builtin_fmaf(e[r], mid[r], mids[h]);
                    e[r] *= step[r];
                }
                pp[h][kt >> 1][2 * (kt & 1)] = Mma<DT>::pack(e[0], e[1]);
                pp[h][kt >> 1][2 * (kt & 1) + 1] = Mma<DT>::pack(e[2], e[3]);
            }
        }
        const uint32_t one = Mma<DT>::pack(1.f, 1.f);
        const u32x4 ones = {one, one, one, one};
#pragma unroll
        for (int h = 0; h < QT; ++h) {
            steps[h] = Mma<DT>::k32(ones, pp[h][0], steps[h]);
            steps[h] = Mma<DT>::k32(ones, pp[h][1], steps[h]);
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            typedef int i32x2 __attribute__((ext_vector_type(2)));
            const i32x2 w = __builtin_amdgcn_ds_read_tr4_b64_v2i32(reinterpret_cast<LDS_PTR(i32x2)>(v_lds + v_off[ct]));
            const u32x4 v0 = of_codes<DT>((uint32_t)w.x), v1 = of_codes<DT>((uint32_t)w.y);
#pragma unroll
            for (int h = 0; h < QT; ++h) {
                sums.o[h][ct] = Mma<DT>::k32(v0, pp[h][0], sums.o[h][ct]);
                sums.o[h][ct] = Mma<DT>::k32(v1, pp[h][1], sums.o[h][ct]);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < QT; ++h) {
        const float down = kLifts ? __builtin_amdgcn_ldexpf(1.f, -up) : 1.f, extra = __builtin_fmaf(-23.5f * down, steps[h][0], xor_sum(mids[h]));
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums.o[h][ct][r] = __builtin_fmaf(sums.o[h][ct][r], down, extra);
    }
    join_waves<DT, C, QT, NW>(sums, smem, out, partial, p.head, p.sample, p.kv, p.block, p.split, wave, lane, a);
}

// ----------------------------------------------------------------------------- launchers
constexpr int kFewWaves = kWaves;
// Bytes of LDS that a wave stages into, and the most waves of a workgroup that find room.
constexpr int staged_bytes(int C, bool four) { return four ? 2 * 2 * (64 * (C / 2) + 64 * 4) : 2 * 2 * (C <= 16 ? kChunk : 64 * (C == 96 ? 128 : C)); }
constexpr int most_waves(int C, bool four) { return four || staged_bytes(C, four) > 20480 ? kFewWaves : staged_bytes(C, four) > 10240 ? 8 : 16; }
int width_of(const na1d_sink_cache &c) { return channels_of(c.head_dim); }

struct CachePlan {
    int tiles, waves;
    CacheArgs a;
    int64_t items;
};
// Blocks of 16, 32 or 64 rows of queries.  16-bit rows of up to 64 channels: where the card is not full with a workgroup to every head of keys, and a large one gets through them with at most
// kSerial units to a wave, that one has them all, and a launch less.  With one and with shares, us of a captured step over 1024 and 2048 keys, 16 heads: 5.7 and 6.3, 6.7 and 6.2 (16
// channels), 5.9 and 6.8, 7.1 and 6.8 (32), 6.5 and 7.3, 8.2 and 7.5 (64: the second are eight units to a wave); 256 heads: 6.2 and 8.4, 7.4 and 9.8 (16), 6.5 and 9.2, 13.2 and 16.0 (32), 14.2 and 16.4 (64,
// 1024 keys).  (Rows in 4 bits, whose units take longer: 15.6 us in one workgroup of 16 waves to a head, 8.7 and 4.9 in shares, for 5 streams of 2 heads of 64, 2008 keys.)
// Otherwise workgroups of four waves, as many to a head as occupy the card in whole rounds, with two units of keys to a wave at least, one in 4 bits.
constexpr int kSerial = 5;
CachePlan cache_plan(const na1d_sink_cache &c, int64_t fresh, int heads, int64_t window) {
    CachePlan p{};
    CacheArgs &a = p.a;
    a.K = c.kv_heads, a.group = heads / c.kv_heads, a.fresh = (int)fresh, a.rows = (int)(fresh * a.group);
    p.tiles = a.rows <= 16 ? 1 : a.rows <= 32 ? 2 : 4;
    a.blocks = (a.rows + 16 * p.tiles - 1) / (16 * p.tiles);
    a.window = (int)window, a.sinks = (int)c.sinks, a.ring = (int)(c.capacity - c.sinks), a.width = 2 * c.head_dim;
    const bool four = c.bits == 4;
    const int C = width_of(c), unit = four ? 64 : 32, wide = most_waves(C, four);
    const int64_t most = std::min(c.capacity, c.sinks + window + fresh - 1), heads_blocks = c.N * c.kv_heads * a.blocks;
    p.waves = kFewWaves, a.splits = 1;
    if (p.tiles == 1 && wide > kFewWaves && heads_blocks <= 256 && most <= (int64_t)kSerial * unit * wide) {
        p.waves = wide;
    } else {
        const int64_t slots = 256 * std::min(4, 160 * 1024 / (kFewWaves * staged_bytes(C, four))), longest = std::max<int64_t>(1, most / ((four ? 1 : 2) * unit * kFewWaves));
        auto wasted = [&](int64_t s) { return heads_blocks * s % slots ? slots - heads_blocks * s % slots : 0; };      // of the last round
        int64_t s = std::max<int64_t>(1, slots / std::max<int64_t>(1, heads_blocks));
        if (heads_blocks > slots / 2)
            for (s = 1; s < 4 && wasted(s) * 10 > heads_blocks * s; ++s) {}
        a.splits = (int)std::min<int64_t>({s, longest, 256});
    }
    a.slice = c.capacity * (four ? c.head_dim / 2 : 2 * c.head_dim);
    a.ranges = four ? c.capacity * 4 : 0;
    p.items = heads_blocks * a.splits;
    return p;
}
Rows rows_by(const int64_t *s) { return Rows{2 * s[0], 2 * s[1], 2 * s[2]}; }

template <class DT, int C, int QT, int NW, bool FOUR>
int launch_attend(const na1d_sink_cache &c, const CachePlan &p, void *out, const void *q, const void *k, const void *v, const int32_t *lengths, float *ws, hipStream_t s) {
    constexpr size_t staged = (size_t)NW * staged_bytes(C, FOUR);
    constexpr size_t lds = staged > (size_t)kJoinBytes<C, QT, NW> ? staged : (size_t)kJoinBytes<C, QT, NW>;
    static_assert(lds <= 160 * 1024, "a CU's LDS");
    const char *dt = DT::tag == NA1D_BF16 ? "BF16" : "FP16";
    const bool joins = p.a.splits > 1;
    if constexpr (FOUR) {
        if (!allow_lds(cache_attend4_kernel<DT, C, QT, NW>, lds)) return NA1D_ERR_LAUNCH;
        note_kernel_as("cache_attend4_kernel<%s, %d, %d, %d>", dt, C, QT, NW);
        launch_kernel_span(joins ? 1 : 3, cache_attend4_kernel<DT, C, QT, NW>, (unsigned)p.items, 64u * NW, lds, s, (char *)out, ws, (const char *)q, (const char *)k,
                           (const char *)v, (char *)c.k, (char *)c.v, (char *)c.k_ranges, (char *)c.v_ranges, lengths, (uint32_t)p.items, p.a);
    } else {
        if (!allow_lds(cache_attend_kernel<DT, C, QT, NW>, lds)) return NA1D_ERR_LAUNCH;
        note_kernel_as("cache_attend_kernel<%s, %d, %d, %d>", dt, C, QT, NW);
        launch_kernel_span(joins ? 1 : 3, cache_attend_kernel<DT, C, QT, NW>, (unsigned)p.items, 64u * NW, lds, s, (char *)out, ws, (const char *)q, (const char *)k,
                           (const char *)v, (char *)c.k, (char *)c.v, lengths, (uint32_t)p.items, p.a);
    }
    if (joins) {
        const int64_t quads = c.N * c.kv_heads * (int64_t)p.a.rows * (p.a.width / 8);
        launch_kernel_span(2, cache_join_kernel<DT, C, QT>, (unsigned)((quads + kThreads - 1) / kThreads), (unsigned)kThreads, 0, s, (char *)out, (const float *)ws, (uint32_t)quads, p.a);
    }
    return launch_status();
}
template <class DT, int C, bool FOUR, class... A> int launch_tiles(const na1d_sink_cache &c, const CachePlan &p, A... args) {
    if constexpr (most_waves(C, FOUR) > kFewWaves)
        if (p.waves > kFewWaves) return launch_attend<DT, C, 1, most_waves(C, FOUR), FOUR>(c, p, args...);
    if (p.tiles == 1) return launch_attend<DT, C, 1, kFewWaves, FOUR>(c, p, args...);
    return p.tiles == 2 ? launch_attend<DT, C, 2, kFewWaves, FOUR>(c, p, args...) : launch_attend<DT, C, 4, kFewWaves, FOUR>(c, p, args...);
}
template <class DT, class... A> int launch_width(const na1d_sink_cache &c, const CachePlan &p, A... args) {
    const bool four = c.bits == 4;
    switch (width_of(c)) {
        case 16: return launch_tiles<DT, 16, false>(c, p, args...);
        case 32: return four ? launch_tiles<DT, 32, true>(c, p, args...) : launch_tiles<DT, 32, false>(c, p, args...);
        case 64: return four ? launch_tiles<DT, 64, true>(c, p, args...) : launch_tiles<DT, 64, false>(c, p, args...);
        case 96: return four ? launch_tiles<DT, 96, true>(c, p, args...) : launch_tiles<DT, 96, false>(c, p, args...);
        case 128: return four ? launch_tiles<DT, 128, true>(c, p, args...) : launch_tiles<DT, 128, false>(c, p, args...);
    }
    return NA1D_ERR_UNSUPPORTED;
}

}  // namespace

int64_t cache_attend_workspace_bytes(const na1d_sink_cache &c, int64_t fresh, int heads, int64_t window) {
    const CachePlan p = cache_plan(c, fresh, heads, window);
    return p.a.splits > 1 ? p.items * 16 * p.tiles * (width_of(c) + 4) * 4 : 0;
}
int cache_attend(const na1d_sink_cache &c, void *out, const void *q, const void *k, const void *v, const int64_t *q_strides, const int64_t *k_strides, const int64_t *v_strides,
                 const int32_t *lengths, int64_t fresh, int heads, int64_t window, float scale, float *ws, hipStream_t s) {
    CachePlan p = cache_plan(c, fresh, heads, window);
    if (!launchable(p.items, 64 * p.waves)) return NA1D_ERR_UNSUPPORTED;
    p.a.scale = scale, p.a.q = rows_by(q_strides);
    if (k) p.a.k = rows_by(k_strides), p.a.v = rows_by(v_strides), p.a.stored = p.a.fresh;
    return c.dtype == NA1D_BF16 ? launch_width<BF16>(c, p, out, q, k, v, lengths, ws, s) : launch_width<FP16>(c, p, out, q, k, v, lengths, ws, s);
}
int cache_append(const na1d_sink_cache &c, const void *k, const void *v, const int64_t *k_strides, const int64_t *v_strides, const int32_t *lengths, const int32_t *t_valid, int64_t T,
                 hipStream_t s) {
    CachePlan p = cache_plan(c, 1, c.kv_heads, 1);
    p.a.k = rows_by(k_strides), p.a.v = rows_by(v_strides);
    // workgroups fill the card eight times, where there are so many tokens
    const int64_t heads = c.N * c.kv_heads, tokens = std::min(T, c.capacity), slots = kThreads / (c.head_dim <= 32 ? 4 : c.head_dim <= 64 ? 8 : 16);
    const int64_t blocks = std::max<int64_t>(1, std::min((tokens + slots - 1) / slots, 16384 / heads));
    if (!launchable(heads * blocks)) return NA1D_ERR_UNSUPPORTED;
    auto go = [&](auto kern) {
        launch_kernel(kern, (unsigned)(heads * blocks), 0, s, (char *)c.k, (char *)c.v, (char *)c.k_ranges, (char *)c.v_ranges, (const char *)k, (const char *)v, lengths, t_valid,
                      (int)T, (int)blocks, p.a);
        return launch_status();
    };
    if (c.dtype == NA1D_BF16) return c.bits == 4 ? go(cache_append_kernel<BF16, 4>) : go(cache_append_kernel<BF16, 16>);
    return c.bits == 4 ? go(cache_append_kernel<FP16, 4>) : go(cache_append_kernel<FP16, 16>);
}
int cache_rows(void *out, const void *codes, const void *ranges, int64_t rows, int head_dim, int dtype, hipStream_t s) {
    const int per_row = head_dim / 8;
    const int64_t words = rows * per_row;
    const unsigned grid = (unsigned)std::min<int64_t>((words + kThreads - 1) / kThreads, 1 << 20);
    auto go = [&](auto kern) {
        launch_kernel(kern, grid, 0, s, (char *)out, (const char *)codes, (const char *)ranges, words, per_row);
        return launch_status();
    };
    return dtype == NA1D_BF16 ? go(cache_rows_kernel<BF16>) : go(cache_rows_kernel<FP16>);
}

}  // namespace mfma
}  // namespace na1d
