// Rotation of heads by their positions, alone and on the way into a paged
// cache.
//
// Pair j of a head's first 2 `half` dimensions, (x_a, x_b) = (x_2j, x_2j+1)
// (neighbours) or (x_j, x_j+half), becomes magnitude times
//   (x_a cos p - x_b sin p, x_b cos p + x_a sin p),  p = position * frequency_j;
// the dimensions behind stay.  A frequency comes as the part of a turn per
// position in units of 2^-64, so that position * step modulo 2^64 is the angle
// modulo a turn, exactly, however far the position: an FP32 product of a
// position of 10^6 and a frequency is off by 0.06 rad.  The axis of a pair's
// position (0..3) stands in the step's two lowest bits; they and the rounding to
// 2^-62 put the step up to 1.25 * 2^-62 turns a position off its frequency.
//
// A lane holds 8 pairs of a head, so D / 16 lanes hold a head, whatever the
// pairing: a head's sum of squares is a butterfly over them, its rotation stays
// in a lane, and both halves of the pairs are 16-byte accesses.  Everything
// between a value's load and its store is FP32, with one rounding at the end.
#include <algorithm>
#include <type_traits>

#include "device.hpp"
#include "rotate.hpp"

namespace fp8lin {
namespace {

constexpr int kThreads = 256, kPairs = 8;

// Workgroups beyond 2^20 (a grid's dimension stays below 2^32 threads) go into
// the grid's second dimension.
constexpr int kGridBits = 20;
__device__ __forceinline__ int64_t group_index() { return ((int64_t)blockIdx.y << kGridBits) + blockIdx.x; }
dim3 grid_of(int64_t groups) {
    const int64_t x = (int64_t)1 << kGridBits;
    return groups <= x ? dim3((unsigned)groups) : dim3((unsigned)x, (unsigned)((groups + x - 1) / x));
}

typedef u32x4 __attribute__((aligned(2))) u32x4_any;  // gfx950 takes unaligned global accesses

// cos and sin of 2 pi phase / 2^64: the nearest quarter turn, then the series
// of the rest, |r| <= pi / 4, to r^8 and r^9 (next terms 2.5e-8 and 2e-9).  r is off
// by up to 2^-26 turns: the phase's upper 32 bits (2^-32), their FP32 (2^-28), the
// constant's rounding (2^-28) and the product's (2^-27.6).
__device__ __forceinline__ void cos_sin(uint64_t phase, float& c, float& s) {
    const uint32_t turn = (uint32_t)(phase >> 32), quarter = (turn + 0x20000000u) >> 30;
    const float r = (float)(int32_t)(turn - (quarter << 30)) * (float)(6.283185307179586 / 4294967296.0), z = r * r;
    const float rs = r + r * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
    const float rc = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320))));
    const float x = quarter & 1 ? rs : rc, y = quarter & 1 ? rc : rs;
    c = (quarter + 1) & 2 ? -x : x;
    s = quarter & 2 ? -y : y;
}

// A lane's 8 pairs, j0 .. j0 + 7 of a head's D / 2.  Behind the rotated ones, in
// the halves' layout, (half + j, D / 2 + j) make pairs too, which are not
// turned.  In kHalves and kNeighbours a lane's values are two times 8 side by
// side (D in multiples of 16, half of 8); kAny takes them one by one.
enum Layout { kHalves, kNeighbours, kAny };
struct Lane {
    int j0, a, b;  // first dimensions of the two times 8
};
__device__ __forceinline__ Lane lane_of(int j0, int half, int D, bool neighbours) {
    if (neighbours) return Lane{j0, 2 * j0, 2 * j0 + 8};
    return j0 < half ? Lane{j0, j0, j0 + half} : Lane{j0, j0 + half, j0 + D / 2};
}
__device__ __forceinline__ void sides(int j, int half, int D, bool neighbours, int& a, int& b) {
    a = neighbours ? 2 * j : j < half ? j : j + half;
    b = neighbours ? 2 * j + 1 : j < half ? j + half : j + D / 2;
}

struct Packed {
    u32x4 a, b;  // 8 values each, as they lie in memory; kAny: pair by pair
};
template <int LAYOUT>
__device__ __forceinline__ Packed load_pairs(const uint16_t* row, const Lane& l, int half, int D, bool neighbours) {
    Packed p{{0, 0, 0, 0}, {0, 0, 0, 0}};
    if constexpr (LAYOUT != kAny) {
        p.a = *reinterpret_cast<const u32x4_any*>(row + l.a);
        p.b = *reinterpret_cast<const u32x4_any*>(row + l.b);
    } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
            if (l.j0 + i < D / 2) {
                int a, b;
                sides(l.j0 + i, half, D, neighbours, a, b);
                p.a[i / 2] |= (uint32_t)row[a] << (16 * (i & 1));
                p.b[i / 2] |= (uint32_t)row[b] << (16 * (i & 1));
            }
    }
    return p;
}
// The values by pair.
template <int LAYOUT>
__device__ __forceinline__ void unpack(const Packed& p, float (&a)[kPairs], float (&b)[kPairs]) {
    auto value = [](const u32x4& w, int i) { return bf16_bits_to_f32((w[i / 2] >> (16 * (i & 1))) & 0xffffu); };
    if constexpr (LAYOUT == kNeighbours) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const u32x4& w = i < 4 ? p.a : p.b;
            a[i] = value(w, 2 * (i & 3));
            b[i] = value(w, 2 * (i & 3) + 1);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            a[i] = value(p.a, i);
            b[i] = value(p.b, i);
        }
    }
}

template <int LAYOUT>
__device__ __forceinline__ void store_bf16(uint16_t* row, const Lane& l, int half, int D, bool neighbours,
                                           const float (&a)[kPairs], const float (&b)[kPairs]) {
    if constexpr (LAYOUT != kAny) {
        u32x4 x, y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = LAYOUT == kNeighbours ? pack_bf16x2(f32x2{a[i], b[i]}) : pack_bf16x2(f32x2{a[2 * i], a[2 * i + 1]});
            y[i] = LAYOUT == kNeighbours ? pack_bf16x2(f32x2{a[4 + i], b[4 + i]}) : pack_bf16x2(f32x2{b[2 * i], b[2 * i + 1]});
        }
        *reinterpret_cast<u32x4_any*>(row + l.a) = x;
        *reinterpret_cast<u32x4_any*>(row + l.b) = y;
    } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
            if (l.j0 + i < D / 2) {
                int ia, ib;
                sides(l.j0 + i, half, D, neighbours, ia, ib);
                row[ia] = f32_to_bf16_bits(a[i]);
                row[ib] = f32_to_bf16_bits(b[i]);
            }
    }
}

// E4M3FN of values within +-448, to nearest even; NaN stays NaN.
__device__ __forceinline__ float cut(float v) { return v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f); }
__device__ __forceinline__ void cut_pairs(float (&a)[kPairs], float (&b)[kPairs]) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        a[i] = cut(a[i]);
        b[i] = cut(b[i]);
    }
}
__device__ __forceinline__ uint32_t codes4(float x, float y, float z, float w) {
    const int p = __builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z, w, p, true);
}
template <int LAYOUT>
__device__ __forceinline__ void store_codes(uint8_t* row, const Lane& l, int half, int D, bool neighbours,
                                            const float (&a)[kPairs], const float (&b)[kPairs]) {
    if constexpr (LAYOUT != kAny) {
        u32x2 x, y;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = LAYOUT == kNeighbours ? codes4(a[2 * i], b[2 * i], a[2 * i + 1], b[2 * i + 1]) : codes4(a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]);
            y[i] = LAYOUT == kNeighbours ? codes4(a[4 + 2 * i], b[4 + 2 * i], a[5 + 2 * i], b[5 + 2 * i])
                              : codes4(b[4 * i], b[4 * i + 1], b[4 * i + 2], b[4 * i + 3]);
        }
        *reinterpret_cast<u32x2*>(row + l.a) = x;
        *reinterpret_cast<u32x2*>(row + l.b) = y;
    } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
            if (l.j0 + i < D / 2) {
                int ia, ib;
                sides(l.j0 + i, half, D, neighbours, ia, ib);
                const uint32_t w = codes4(a[i], b[i], 0.0f, 0.0f);
                row[ia] = (uint8_t)w;
                row[ib] = (uint8_t)(w >> 8);
            }
    }
}

// A token and its position on the first axis (the others' are read where a pair takes them).
struct Place {
    int64_t t;
    uint64_t at;
};
__device__ __forceinline__ Place place_of(const Rotation& r, int64_t t) {
    return Place{t, r.steps ? (uint64_t)r.positions[t] : 0};
}
// A token's turns in LDS: its cosines and sines times the magnitude, and of 8
// pairs that the rotated ones end in (1, 0) for the rest, which nothing takes.
__host__ __device__ __forceinline__ int turns_of(int half) { return (half + kPairs - 1) & ~(kPairs - 1); }
// By `lanes` lanes of a wave (lane l of them): each computes every lanes-th, as one is
// some 40 instructions and every lane of the heads needs 8.  The lanes of a wave
// run together: what they read back needs no barrier.
__device__ __forceinline__ void fill_turns(const Rotation& r, const uint64_t* steps, const Place& p, f32x2* turns, int l, int lanes) {
    if (!r.steps) return;
    const int n = turns_of(r.half);
    for (int j = l; j < n; j += lanes) {
        f32x2 turn = {1.0f, 0.0f};
        if (j < r.half) {
            const uint64_t step = steps[j];
            uint64_t at = p.at;
            if (r.axes > 1) at = (uint64_t)r.positions[(int64_t)min((int)step & 3, r.axes - 1) * r.axis + p.t];
            float c, z;
            cos_sin(at * step, c, z);
            turn = f32x2{c * r.magnitude, z * r.magnitude * r.sign};
        }
        turns[j] = turn;
    }
    __builtin_amdgcn_wave_barrier();
}
// The lane's pairs, turned; those behind the rotated ones stay as they are: chosen,
// not multiplied by (1, 0), as 0 times an infinity is NaN.  In kHalves no lane has both.
template <int LAYOUT>
__device__ __forceinline__ void rotate_pairs(const Rotation& r, const f32x2* turns, int j0, float (&a)[kPairs], float (&b)[kPairs]) {
    if (!r.steps || j0 >= r.half) return;
    const int turned = LAYOUT == kHalves ? kPairs : r.half - j0;
#pragma unroll
    for (int i = 0; i < kPairs; i += 2) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(turns + j0 + i);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float x = a[i + k], y = b[i + k], c = t[2 * k], z = t[2 * k + 1];
            a[i + k] = i + k < turned ? x * c - y * z : x;
            b[i + k] = i + k < turned ? y * c + x * z : y;
        }
    }
}

// A value of the lane's neighbour, by the vector unit: the lane 1 or 2 off in its
// 4, the lane's mirror image in its 8 or 16.  Sums and maxima of 4 (8) lanes that
// hold the same are those of the 4 (8) beside them.
template <int CONTROL>
__device__ __forceinline__ float across(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CONTROL, 0xf, 0xf, true));
}
template <class OP>
__device__ __forceinline__ float over_lanes(float v, int lanes, OP op) {
    if (lanes > 1) v = op(v, across<0xb1>(v));
    if (lanes > 2) v = op(v, across<0x4e>(v));
    if (lanes > 4) v = op(v, across<0x141>(v));
    if (lanes > 8) v = op(v, across<0x140>(v));
    if (lanes > 16) v = op(v, __shfl_xor(v, 16, 64));
    if (lanes > 32) v = op(v, __shfl_xor(v, 32, 64));
    return v;
}

// The lane's factors of the norm, center + weight.
__device__ __forceinline__ void add_center(float (&a)[kPairs], float (&b)[kPairs], float center) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        a[i] += center;
        b[i] += center;
    }
}
// x / sqrt(mean(x^2) + eps) times the factors, over the `lanes` lanes of a head
// (all of the wave's take part); a head without a norm is multiplied by 1.
__device__ __forceinline__ void norm_pairs(float (&a)[kPairs], float (&b)[kPairs], const float (&wa)[kPairs],
                                           const float (&wb)[kPairs], int lanes, int D, float eps, bool normed = true) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) sum += a[i] * a[i] + b[i] * b[i];
    sum = over_lanes(sum, lanes, [](float x, float y) { return x + y; });
    const float inv = normed ? __builtin_amdgcn_rsqf(sum / (float)D + eps) : 1.0f;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        a[i] *= inv * wa[i];
        b[i] *= inv * wb[i];
    }
}

// ---- rotation alone -----------------------------------------------------------
//
// A wave takes a token and ITERS times 64 / lanes of its heads, all loads in
// flight together; the heads share the token's cosines and sines.

template <int LAYOUT, int ITERS>
__global__ __launch_bounds__(kThreads) void rotate_kernel(Rotate a, int lane_bits, int chunks) {
    const int lane = threadIdx.x & 63, lanes = 1 << lane_bits, l = lane & (lanes - 1), g = lane >> lane_bits, per = 64 >> lane_bits;
    // a workgroup: 4 tokens, one of `chunks` parts of their heads
    const int64_t group = group_index(), tokens = group / chunks;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), first = (int)(group - tokens * chunks) * ITERS * per + g;
    const int64_t t = tokens * (kThreads / 64) + wave;
    if (t >= a.T) return;
    const bool nb = a.r.neighbours;
    const int half = a.r.half, D = a.D;
    const Lane at = lane_of(kPairs * l, half, D, nb);
    const bool live = at.j0 < D / 2;
    extern __shared__ __align__(16) uint8_t lds[];
    f32x2* turns = reinterpret_cast<f32x2*>(lds) + wave * turns_of(half);
    const Place place = place_of(a.r, t);
    const uint16_t* x = a.x.x + t * a.x.tok;
    uint16_t* y = a.y + t * a.y_tok;
    Packed p[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
        if (live && first + i * per < a.x.n) p[i] = load_pairs<LAYOUT>(x + (first + i * per) * a.x.head, at, half, D, nb);
    fill_turns(a.r, a.r.steps, place, turns, lane, 64);
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int h = first + i * per;
        if (!live || h >= a.x.n) break;
        float u[kPairs], v[kPairs];
        unpack<LAYOUT>(p[i], u, v);
        rotate_pairs<LAYOUT>(a.r, turns, at.j0, u, v);
        store_bf16<LAYOUT>(y + h * a.y_head, at, half, D, nb, u, v);
    }
}

// ---- rotation on the way into the cache -----------------------------------------

enum Mode { kBf16, kHeads, kBlocks };

// Token t's rows, ITERS times 64 / lanes of them: its query heads, and (but in
// kBlocks) its keys and values.
template <int MODE, int LAYOUT, int ITERS>
__device__ __forceinline__ void append_rows(const RotateAppend& a, int lane_bits, int chunk, int64_t t, f32x2* turns) {
    const int lane = threadIdx.x & 63, lanes = 1 << lane_bits, l = lane & (lanes - 1), g = lane >> lane_bits, per = 64 >> lane_bits;
    if (t >= a.T) return;
    const bool nb = a.r.neighbours;
    const int half = a.r.half, D = a.D, rows = a.q.n + (MODE == kBlocks ? 0 : 2 * a.k.n), first = chunk * ITERS * per + g;
    const Lane at = lane_of(kPairs * l, half, D, nb);
    const bool live = at.j0 < D / 2;
    auto kind_of = [&](int row, bool& is_q, bool& is_v, int& h) {
        is_q = MODE == kBlocks || row < a.q.n;
        is_v = !is_q && row >= a.q.n + a.k.n;
        h = is_q ? row : is_v ? row - a.q.n - a.k.n : row - a.q.n;
    };
    // member by member: a reference to one of the records would put them into memory
    auto pick = [](bool is_q, bool is_v, auto q, auto k, auto v) { return MODE == kBlocks || is_q ? q : is_v ? v : k; };
    const uint16_t *qt = a.q.x + t * a.q.tok, *kt = a.k.x + t * a.k.tok, *vt = a.v.x + t * a.v.tok;
    Packed p[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int row = first + i * per;
        bool is_q, is_v;
        int h;
        kind_of(row, is_q, is_v, h);
        p[i] = Packed{{0, 0, 0, 0}, {0, 0, 0, 0}};
        if (live && row < rows) p[i] = load_pairs<LAYOUT>(pick(is_q, is_v, qt, kt, vt) + h * pick(is_q, is_v, a.q.head, a.k.head, a.v.head), at, half, D, nb);
    }
    const int64_t slot = MODE == kBlocks ? -1 : a.slots[t];
    const Place place = place_of(a.r, t);
    float qx[kPairs] = {}, qy[kPairs] = {}, kx[kPairs] = {}, ky[kPairs] = {};
    if (a.q_norm && live) unpack<LAYOUT>(load_pairs<LAYOUT>(a.q_norm, at, half, D, nb), qx, qy);
    if (MODE != kBlocks && a.k_norm && live) unpack<LAYOUT>(load_pairs<LAYOUT>(a.k_norm, at, half, D, nb), kx, ky);
    add_center(qx, qy, a.center);
    add_center(kx, ky, a.center);
    fill_turns(a.r, a.r.steps, place, turns, lane, 64);
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int row = first + i * per;
        if (first - g + i * per >= rows) break;  // of the whole wave
        bool is_q, is_v;
        int h;
        kind_of(row, is_q, is_v, h);
        float x[kPairs], y[kPairs];
        unpack<LAYOUT>(p[i], x, y);
        if (a.q_norm || (MODE != kBlocks && a.k_norm)) {
            // all lanes: those of a head agree on whether it is normed
            const bool normed = is_q ? a.q_norm != nullptr : !is_v && a.k_norm;
            float wx[kPairs], wy[kPairs];
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                wx[k] = !normed ? 1.0f : is_q ? qx[k] : kx[k];
                wy[k] = !normed ? 1.0f : is_q ? qy[k] : ky[k];
            }
            norm_pairs(x, y, wx, wy, lanes, D, a.eps, normed);
        }
        if (!live || row >= rows) continue;
        if (!is_v) rotate_pairs<LAYOUT>(a.r, turns, at.j0, x, y);
        if (is_q) {
            store_bf16<LAYOUT>(a.y + t * a.y_tok + h * a.y_head, at, half, D, nb, x, y);
            continue;
        }
        if constexpr (MODE != kBlocks) {
            if (slot < 0 || slot >= a.limit) continue;
            const int64_t page = slot >> a.page_bits, in_page = slot & (((int64_t)1 << a.page_bits) - 1);
            const int64_t dst = is_v ? page * a.vc.page + in_page * a.vc.slot + h * a.vc.head : page * a.kc.page + in_page * a.kc.slot + h * a.kc.head;
            void* const to = const_cast<void*>(is_v ? a.vc.data : a.kc.data);
            if constexpr (MODE == kHeads) {
                // an IEEE division, as paged_append's
                const float s = is_v ? a.v_scale[h] : a.k_scale[h];
#pragma unroll
                for (int k = 0; k < kPairs; ++k) {
                    x[k] /= s;
                    y[k] /= s;
                }
                cut_pairs(x, y);
                store_codes<LAYOUT>(static_cast<uint8_t*>(to) + dst, at, half, D, nb, x, y);
            } else {
                store_bf16<LAYOUT>(static_cast<uint16_t*>(to) + dst, at, half, D, nb, x, y);
            }
        }
    }
}

// The exponent byte of the least 2^e with top <= 448 2^e, e from -120 (so that
// its reciprocal and every code times it are normal numbers) to 119 (so that
// they stay below 2^128).
constexpr int kMinPower = 7, kMaxPower = 246;
__device__ __forceinline__ int block_power(float top) {
    const uint32_t u = __builtin_bit_cast(uint32_t, top);
    return min(max((int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u), kMinPower), kMaxPower);
}
__device__ __forceinline__ float power_of(int exponent) {  // 2^(exponent - 127), 0 below
    return __builtin_bit_cast(float, exponent > 0 ? (uint32_t)exponent << 23 : 0u);
}

// What a workgroup that appends runs has in LDS: the slots and (first axis)
// positions of kThreads tokens from the one before its first on; behind that the
// steps, then of `cap` rows in hand their turns and each lane's values as they were
// loaded.
constexpr int kKeep = 4;
struct RunLds {
    int64_t slots[kThreads];
    uint64_t positions[kThreads];
    float tops[4];
    __device__ __forceinline__ uint64_t* steps() { return reinterpret_cast<uint64_t*>(this + 1); }
    __device__ __forceinline__ f32x2* turns(int half) { return reinterpret_cast<f32x2*>(steps() + turns_of(half)); }
    __device__ __forceinline__ u32x4* rows(int half, int cap) { return reinterpret_cast<u32x4*>(turns(half) + cap * turns_of(half)); }
};
// Rows in hand: a block's, of one to kKeep times what the workgroup's lanes hold at once.
__host__ __device__ __forceinline__ int cap_of(int block_bits, int lane_bits) {
    const int once = kThreads >> lane_bits, block = 1 << block_bits;
    return block < once ? once : block < kKeep * once ? block : kKeep * once;
}
// The most: heads of 1024, all of them rotated (16 rows' turns of 512).
constexpr int kMaxLds = 112 * 1024;
int run_lds(int half, int block_bits, int lane_bits) {
    const int cap = cap_of(block_bits, lane_bits);
    return (int)sizeof(RunLds) + 8 * turns_of(half) * (1 + cap) + 32 * kThreads * ((cap >> (8 - lane_bits)) - 1);
}

// The slots of a block that n rows write.
template <class SLOT>
__device__ __forceinline__ void written_slots(SLOT slot_at, int64_t n, int block, uint32_t (&written)[4]) {
#pragma unroll
    for (int w = 0; w < 4; ++w) written[w] = 0;
#pragma unroll 1
    for (int64_t i = 0; i < n; ++i) {
        const int s = (int)(slot_at(i) & (block - 1));
#pragma unroll
        for (int w = 0; w < 4; ++w) written[w] |= s >> 5 == w ? 1u << (s & 31) : 0;
    }
}
// The codes of a block's other slots times f, by `team` lanes, 16 a lane and 4 of
// those in flight.  The blocks of a decode step's requests grow now and then, so
// most steps have some (61 requests, blocks of 64, 2 heads of 256, a call in a graph:
// 7.6 us, and 13 where every block grows; by the lanes of the row alone 200).
__device__ __forceinline__ void grow_block(uint8_t* codes, int64_t slot_stride, int block, int D, float f, const uint32_t (&written)[4], int tid,
                                           int team) {
    constexpr int UN = 4;
    const int per = D / 16, pieces = block * per;
#pragma unroll 1
    for (int p0 = tid; p0 < pieces; p0 += UN * team) {
        u32x4 w[UN];
        u32x4* at[UN];
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const int p = p0 + i * team, s = p / per;
            const uint32_t mask = s < 32 ? written[0] : s < 64 ? written[1] : s < 96 ? written[2] : written[3];
            at[i] = p < pieces && !(mask >> (s & 31) & 1) ? reinterpret_cast<u32x4*>(codes + s * slot_stride + 16 * (p - s * per)) : nullptr;
            if (at[i]) w[i] = *at[i];
        }
#pragma unroll
        for (int i = 0; i < UN; ++i)
            if (at[i]) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x2 lo = fp8x2_to_f32<false>(w[i][k]), hi = fp8x2_to_f32<true>(w[i][k]);
                    w[i][k] = codes4(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
                }
                *at[i] = w[i];
            }
    }
}

// Rows i0 .. i0 + n of the window, all of one block of one head, by the lanes that
// hold a row, by a wave or by the workgroup: their
// largest value gives the block's power of two; where that grows, the block's
// other codes are multiplied; then the rows' codes.
//
// A workgroup has a run's 64 rows or so for itself, a wave per SIMD, so it is
// bound by latency and by its own instructions: its loads go out together, into LDS
// (the registers that would hold them would halve the waves of the queries' rows in the
// same launch), the second pass over the rows computes them again but for their
// turns, and both are one loop's code, as code that runs once comes from L2.
enum Team { kOne, kWave, kAll };
template <int LAYOUT, int TEAM>
__device__ __forceinline__ void append_run(const RotateAppend& a, RunLds& lds, int lane_bits, int64_t window, int i0, int64_t n, int h, bool is_v) {
    const int lanes = 1 << lane_bits, team = TEAM == kAll ? kThreads : TEAM == kWave ? 64 : lanes, tid = threadIdx.x & (team - 1), l = tid & (lanes - 1), g = tid >> lane_bits;
    const int G = team >> lane_bits;
    const bool nb = a.r.neighbours;
    const int half = a.r.half, D = a.D, block = 1 << a.block_bits;
    const Lane at = lane_of(kPairs * l, half, D, nb);
    const bool live = at.j0 < D / 2;
    const int64_t t0 = window + i0, row_stride = is_v ? a.v.tok : a.k.tok;
    const uint16_t* rows = (is_v ? a.v.x + h * a.v.head : a.k.x + h * a.k.head) + t0 * row_stride;
    const uint16_t* norm = is_v ? nullptr : a.k_norm;
    const int all_cap = cap_of(a.block_bits, lane_bits), cap = TEAM == kAll ? all_cap : G;
    f32x2* turns = lds.turns(half) + ((int)threadIdx.x - tid >> lane_bits) * turns_of(half);  // kAll: the first
    u32x4* held = lds.rows(half, all_cap) + threadIdx.x;
    auto slot_at = [&](int64_t i) { return i0 + i < kThreads ? lds.slots[i0 + i] : a.slots[t0 + i]; };
    auto load = [&](int64_t i) __attribute__((always_inline)) {
        Packed p{{0, 0, 0, 0}, {0, 0, 0, 0}};
        if (live && i < n) p = load_pairs<LAYOUT>(rows + i * row_stride, at, half, D, nb);
        return p;
    };
    Packed mine = load(g);
    if constexpr (TEAM == kAll) {
        Packed more[kKeep - 1];
#pragma unroll
        for (int k = 1; k < kKeep; ++k)
            if (k * G < cap) more[k - 1] = load(k * G + g);
#pragma unroll
        for (int k = 1; k < kKeep; ++k)
            if (k * G < cap) {
                held[2 * (k - 1) * kThreads] = more[k - 1].a;
                held[(2 * k - 1) * kThreads] = more[k - 1].b;
            }
    }
    const int64_t slot0 = slot_at(0) >> a.block_bits << a.block_bits, page = slot0 >> a.page_bits, slot_stride = is_v ? a.vc.slot : a.kc.slot;
    const int in_page = (int)(slot0 & (((int64_t)1 << a.page_bits) - 1));
    uint8_t* codes = static_cast<uint8_t*>(const_cast<void*>(is_v ? a.vc.data : a.kc.data)) + page * (is_v ? a.vc.page : a.kc.page) +
                     in_page * slot_stride + h * (is_v ? a.vc.head : a.kc.head);
    uint8_t* byte = (is_v ? a.v_pow : a.k_pow) + ((page << (a.page_bits - a.block_bits)) + (in_page >> a.block_bits)) * a.k.n + h;
    const int old = n ? min((int)*byte, kMaxPower) : 0;
    float wx[kPairs] = {}, wy[kPairs] = {};
    if (norm && live) unpack<LAYOUT>(load_pairs<LAYOUT>(norm, at, half, D, nb), wx, wy);
    add_center(wx, wy, a.center);

    float x[kPairs], y[kPairs], top = 0.0f, factor = 1.0f;
    int power = 0;
    bool fresh = false, odd = false;  // odd: some value does not fit its block's range, infinities are left out of it
    bool any_odd = false;             // of the wave's blocks: the passes are the whole wave's, as it shares the growing
    enum { kLargest, kLargestFinite, kStore };
#pragma unroll 1
    for (int pass = kLargest; pass <= kStore; ++pass) {
        if (pass == kLargestFinite && !any_odd) continue;
        if (pass == kStore) {
            // by the whole wave or workgroup, whosever block it is
            const bool grows = n && !fresh && old < power;
            if constexpr (TEAM == kAll) {
                if (grows) {
                    uint32_t written[4];
                    written_slots(slot_at, n, block, written);
                    grow_block(codes, slot_stride, block, D, power_of(127 + old - power), written, tid, kThreads);
                }
            } else {
                for (uint64_t left = __ballot(grows); left;) {
                    const int from = __builtin_ctzll(left);
                    left &= TEAM == kWave ? 0 : ~(((lanes < 64 ? 1ull << lanes : 0) - 1) << from);
                    const int first = __builtin_amdgcn_readlane(i0, from), rows = __builtin_amdgcn_readlane((int)n, from);
                    const uint64_t to = (uint64_t)(uintptr_t)codes;
                    const uint64_t at0 = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)to, from) |
                                         (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(to >> 32), from) << 32;
                    const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, power_of(127 + old - power)), from));
                    uint32_t written[4];
                    written_slots([&](int64_t i) { return lds.slots[first + i]; }, rows, block, written);
                    grow_block(reinterpret_cast<uint8_t*>(at0), slot_stride, block, D, f, written, threadIdx.x & 63, 64);
                }
            }
        }
#pragma unroll 1
        for (int64_t k = 0; k * G < n; ++k) {
            const int64_t i = k * G + g;
            if (pass == kLargest || n > G) {
                Packed w = mine;
                if (TEAM == kAll && k) w = k * G < cap ? Packed{held[2 * (k - 1) * kThreads], held[(2 * k - 1) * kThreads]} : load(i);
                unpack<LAYOUT>(w, x, y);
                if (!is_v) {
                    if (norm) norm_pairs(x, y, wx, wy, lanes, D, a.eps);
                    f32x2* row = turns + ((int)i & (cap - 1)) * turns_of(half);
                    if (a.r.steps && (pass == kLargest || n > cap)) {
                        const int64_t t = min(t0 + i, a.T - 1);
                        fill_turns(a.r, lds.steps(), Place{t, i0 + i < kThreads ? lds.positions[i0 + i] : (uint64_t)a.r.positions[t]}, row, l, lanes);
                    }
                    rotate_pairs<LAYOUT>(a.r, row, at.j0, x, y);
                }
            }
            if (pass == kLargest) {
                // NaN does not count: by comparisons, as a maximum with a signalling NaN is NaN
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const float u = fabsf(x[j]), v = fabsf(y[j]);
                    top = u > top ? u : top;
                    top = v > top ? v : top;
                }
            } else if (pass == kLargestFinite) {
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const float u = fabsf(x[j]), v = fabsf(y[j]);
                    top = fmaxf(top, odd && u < __builtin_inff() ? u : 0.0f);
                    top = fmaxf(top, odd && v < __builtin_inff() ? v : 0.0f);
                }
            } else if (live && i < n) {
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    x[j] *= factor;
                    y[j] *= factor;
                }
                if (odd) cut_pairs(x, y);
                store_codes<LAYOUT>(codes + (slot_at(i) & (block - 1)) * slot_stride, at, half, D, nb, x, y);
            }
        }
        if (pass == kStore) break;
        if (pass == kLargest)
            for (int64_t i = TEAM == kOne ? 0 : tid; i < n; i += TEAM == kOne ? 1 : team) fresh |= (slot_at(i) & (block - 1)) == 0;
        top = over_lanes(top, TEAM == kOne ? lanes : 64, [](float x, float y) { return fmaxf(x, y); });
        if constexpr (TEAM == kWave) fresh = __any(fresh);
        if constexpr (TEAM == kAll) {
            if ((tid & 63) == 0) lds.tops[tid >> 6] = top;
            fresh = __syncthreads_or(fresh);
#pragma unroll
            for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, lds.tops[w]);
            __syncthreads();
        }
        if (pass == kLargest) {
            odd = top > 448.0f * power_of(kMaxPower);
            any_odd = TEAM == kAll ? odd : __any(odd);
            if (odd) top = 0.0f;
            if (any_odd) continue;
        }
        power = block_power(top);
        if (!fresh) power = max(power, old);
        factor = power_of(254 - power);
    }
    if (tid == 0 && n) *byte = (uint8_t)power;
}

// The runs of one head of the keys or values that begin in the tokens first ..
// last, at most 64: those of one row (a decode step's) by the lanes of a row each,
// those of up to the rows that a wave holds (drafted tokens) by a wave each, the
// others by the workgroup.  A run's end is in the window, as it has
// no more rows than a block has slots, if none comes twice.
template <int LAYOUT>
__device__ __forceinline__ void append_runs(const RotateAppend& a, RunLds& lds, int lane_bits, int64_t first, int64_t last, int unit) {
    constexpr int WORDS = kThreads / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = unit >> 1;
    const bool is_v = unit & 1;
    const int64_t window = first - 1;
    auto block_of = [&](int64_t s) { return s < 0 || s >= a.limit ? -1 : s >> a.block_bits; };
    const bool there = window + tid >= 0 && window + tid < a.T;
    lds.slots[tid] = there ? a.slots[window + tid] : -1;
    if (a.r.steps && !is_v) {
        lds.positions[tid] = there ? (uint64_t)a.r.positions[window + tid] : 0;
        for (int j = tid; j < a.r.half; j += kThreads) lds.steps()[j] = a.r.steps[j];
    }
    __syncthreads();
    // the rows that are of another block than the one before, in every wave
    uint64_t border[WORDS];
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
        const int i = 64 * w + lane;
        border[w] = __ballot(i > 0 && block_of(lds.slots[i]) != block_of(lds.slots[max(i - 1, 0)]));
    }
    // the lane's row, first + lane, at i: the next border behind it
    const int i = lane + 1;
    int end = kThreads;
#pragma unroll
    for (int w = WORDS - 1; w >= 0; --w) {
        const uint64_t behind = 64 * w > i ? border[w] : 64 * w + 63 <= i ? 0 : border[w] & (~0ull << (i - 64 * w + 1));
        if (behind) end = 64 * w + __builtin_ctzll(behind);
    }
    const int rows = end - i, few = 64 >> lane_bits;
    const bool is_border = i < 64 ? border[0] >> i & 1 : border[1] & 1;
    const uint64_t begins = __ballot(first + lane < last && is_border && block_of(lds.slots[i]) >= 0);
    const uint64_t ones = begins & __ballot(rows == 1), waves = begins & __ballot(rows > 1 && rows <= few), all = begins & ~ones & ~waves;
    // in turn over the waves, which grow their blocks one after the other
    uint64_t left = ones;
    for (int skip = (lane >> lane_bits) * WORDS + wave; left && skip; --skip) left &= left - 1;
#pragma unroll 1
    while (__any(left != 0)) {
        const int at = left ? __builtin_ctzll(left) : 0, n = __shfl(rows, at, 64);
        append_run<LAYOUT, kOne>(a, lds, lane_bits, window, at + 1, left ? n : 0, h, is_v);
        for (int skip = kThreads >> lane_bits; left && skip; --skip) left &= left - 1;
    }
    int turn = 0;
#pragma unroll 1
    for (left = waves; left; left &= left - 1, ++turn) {
        const int at = __builtin_ctzll(left);
        if (turn % WORDS == wave) append_run<LAYOUT, kWave>(a, lds, lane_bits, window, at + 1, __builtin_amdgcn_readlane(rows, at), h, is_v);
    }
    if (!all) return;
    __syncthreads();  // the waves' turns are the workgroup's
#pragma unroll 1
    for (left = all; left; left &= left - 1) {
        const int at = __builtin_ctzll(left);
        int64_t n = __builtin_amdgcn_readlane(rows, at);
        if (at + 1 + n == kThreads) {
            const int64_t of = block_of(lds.slots[at + 1]);
            while (first + at + n < a.T && block_of(a.slots[first + at + n]) == of) ++n;
        }
        append_run<LAYOUT, kAll>(a, lds, lane_bits, window, at + 1, n, h, is_v);
    }
}

// The first workgroups take the runs of a head of the keys or values (one of
// `units`) that begin in 2^run_bits tokens; the others 4 tokens' rows, a wave
// each, one of `chunks` parts of them.
template <int MODE, int LAYOUT, int ITERS>
__global__ __launch_bounds__(kThreads) void rotate_append_kernel(RotateAppend a, int lane_bits, int chunks, int units, int run_bits,
                                                             int64_t run_groups) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int64_t group = group_index();
    if constexpr (MODE == kBlocks) {
        if (group < run_groups) {
            const int64_t first = group / units << run_bits;
            append_runs<LAYOUT>(a, *reinterpret_cast<RunLds*>(lds), lane_bits, first, min(first + (1 << run_bits), a.T), (int)(group % units));
            return;
        }
        group -= run_groups;
    }
    const int64_t tokens = group / chunks;
    append_rows<MODE, LAYOUT, ITERS>(a, lane_bits, (int)(group - tokens * chunks), tokens * (kThreads / 64) + wave,
                                     reinterpret_cast<f32x2*>(lds) + wave * turns_of(a.r.half));
}

int lane_bits_of(int D) {
    int bits = 0;
    while ((16 << bits) < D) ++bits;
    return bits;
}
// Heads that a lane has in flight (times 64 / lanes): 4 for heads of 256 alone
// (3913 tokens, 12 heads: 9.9 us, with 1 10.6), where 8191 x 32 heads of 128 take 26 to
// 27 us with any number; with the cache's writes beside them 2 (a mixed batch of
// 13 requests into a BF16 cache: 9.5 us, with 1 11.0, with 4 10.4), and 4 again beside
// runs (a prompt of 3913: 18 us, with 1 24), whose LDS leaves few workgroups a CU.
constexpr int kRotateIters = 4, kRowsIters = 2, kBesideRunsIters = 4;
// Workgroups of runs up to which they take few tokens each.
constexpr int kManyRuns = 256;

template <int ITERS, class F>
hipError_t by_layout(const Rotation& r, int D, F go) {
    if (D % 16 || (!r.neighbours && r.half % 8)) return go(std::integral_constant<int, kAny>{}, std::integral_constant<int, 1>{});
    if (r.neighbours) return go(std::integral_constant<int, kNeighbours>{}, std::integral_constant<int, ITERS>{});
    return go(std::integral_constant<int, kHalves>{}, std::integral_constant<int, ITERS>{});
}

}  // namespace

hipError_t launch_rotate(const Rotate& a, hipStream_t stream) {
    const int bits = lane_bits_of(a.D), per = 64 >> bits, groups = (a.x.n + per - 1) / per, waves = kThreads / 64;
    return by_layout<kRotateIters>(a.r, a.D, [&](auto layout_, auto iters_) {
        constexpr int LAYOUT = decltype(layout_)::value, ITERS = decltype(iters_)::value;
        const int chunks = (groups + ITERS - 1) / ITERS, lds = waves * turns_of(a.r.half) * (int)sizeof(f32x2);
        hipLaunchKernelGGL((rotate_kernel<LAYOUT, ITERS>), grid_of((a.T + waves - 1) / waves * chunks), dim3(kThreads), lds, stream, a, bits, chunks);
        return hipGetLastError();
    });
}

hipError_t launch_rotate_append(const RotateAppend& a, hipStream_t stream) {
    const int mode = a.k_pow ? kBlocks : a.fp8 ? kHeads : kBf16, waves = kThreads / 64;
    const int bits = lane_bits_of(a.D), per = 64 >> bits, rows = a.q.n + (mode == kBlocks ? 0 : 2 * a.k.n);
    const int groups = (rows + per - 1) / per, units = mode == kBlocks ? 2 * a.k.n : 0;
    // few tokens each, so that the runs of a decode step spread over the chip, but no
    // fewer than waves, and no more than the lanes hold rows; where that makes many
    // workgroups, a block, as one that finds no run takes some us, too (a prompt of
    // 2000 tokens in blocks of 64, heads of 256: 17 us with 64 tokens, 22 with 16; 3913:
    // 18 and 38)
    int run_bits = 2;
    while (run_bits < std::min(8 - bits, 6) && (a.T * units >> run_bits) > kManyRuns) ++run_bits;
    if ((a.T * units >> run_bits) > kManyRuns) run_bits = std::max(run_bits, std::min(a.block_bits, 6));
    const int64_t run_groups = ((a.T + (1 << run_bits) - 1) >> run_bits) * units;
    const int lds = std::max(mode == kBlocks ? run_lds(a.r.half, a.block_bits, bits) : 0, waves * turns_of(a.r.half) * (int)sizeof(f32x2));
    auto of_mode = [&](auto mode_) {
        constexpr int M = decltype(mode_)::value;
        return by_layout<M == kBlocks ? kBesideRunsIters : kRowsIters>(a.r, a.D, [&](auto layout_, auto iters_) {
            constexpr int LAYOUT = decltype(layout_)::value, ITERS = decltype(iters_)::value;
            const int chunks = (groups + ITERS - 1) / ITERS;
            const int64_t all = run_groups + (a.T + waves - 1) / waves * chunks;
            if (!all) return hipSuccess;
            auto* kern = rotate_append_kernel<M, LAYOUT, ITERS>;
            static OncePerDevice once;
            const hipError_t attr = allow_lds(once, reinterpret_cast<const void*>(kern), kMaxLds);
            if (attr != hipSuccess) return attr;
            hipLaunchKernelGGL(kern, grid_of(all), dim3(kThreads), lds, stream, a, bits, std::max(chunks, 1), units, run_bits, run_groups);
            return hipGetLastError();
        });
    };
    if (mode == kBlocks) return of_mode(std::integral_constant<int, kBlocks>{});
    if (mode == kHeads) return of_mode(std::integral_constant<int, kHeads>{});
    return of_mode(std::integral_constant<int, kBf16>{});
}

}  // namespace fp8lin
