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
// position (0..3) stands in the step's two lowest bits, 2^-62 turns.
//
// A lane holds 8 pairs of a head, so D / 16 lanes hold a head, whatever the
// pairing: a head's sum of squares is a butterfly over them, its rotation stays
// in a lane, and both halves of the pairs are 16-byte accesses.  Everything
// between a value's load and its store is FP32, with one rounding at the end.
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
typedef uint64_t u64x2 __attribute__((ext_vector_type(2), aligned(8)));

// cos and sin of 2 pi phase / 2^64: the nearest quarter turn, then the series
// of the rest, |r| <= pi / 4, to r^8 and r^9 (next terms 2.5e-8 and 2e-9).
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
// turned.  VEC: a pair's 8 neighbours lie side by side (half and D in
// multiples of 8 and 16).
struct Lane {
    int j0, a, b;  // first dimensions of the pairs' sides (VEC)
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
    u32x4 a, b;  // VEC: 8 values each, as they lie in memory; else pair by pair
};
template <bool VEC>
__device__ __forceinline__ Packed load_pairs(const uint16_t* row, const Lane& l, int half, int D, bool neighbours) {
    Packed p{{0, 0, 0, 0}, {0, 0, 0, 0}};
    if constexpr (VEC) {
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
template <bool VEC>
__device__ __forceinline__ void unpack(const Packed& p, bool neighbours, float (&a)[kPairs], float (&b)[kPairs]) {
    auto value = [](const u32x4& w, int i) { return bf16_bits_to_f32((w[i / 2] >> (16 * (i & 1))) & 0xffffu); };
    if (VEC && neighbours) {
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

template <bool VEC>
__device__ __forceinline__ void store_bf16(uint16_t* row, const Lane& l, int half, int D, bool neighbours,
                                           const float (&a)[kPairs], const float (&b)[kPairs]) {
    if constexpr (VEC) {
        u32x4 x, y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = neighbours ? pack_bf16x2(f32x2{a[i], b[i]}) : pack_bf16x2(f32x2{a[2 * i], a[2 * i + 1]});
            y[i] = neighbours ? pack_bf16x2(f32x2{a[4 + i], b[4 + i]}) : pack_bf16x2(f32x2{b[2 * i], b[2 * i + 1]});
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

// E4M3FN of two values cut to +-448, to nearest even; NaN stays NaN.
__device__ __forceinline__ float cut(float v) { return v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f); }
__device__ __forceinline__ uint32_t codes4(float x, float y, float z, float w) {
    const int p = __builtin_amdgcn_cvt_pk_fp8_f32(cut(x), cut(y), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cut(z), cut(w), p, true);
}
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* row, const Lane& l, int half, int D, bool neighbours,
                                            const float (&a)[kPairs], const float (&b)[kPairs]) {
    if constexpr (VEC) {
        u32x2 x, y;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = neighbours ? codes4(a[2 * i], b[2 * i], a[2 * i + 1], b[2 * i + 1]) : codes4(a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]);
            y[i] = neighbours ? codes4(a[4 + 2 * i], b[4 + 2 * i], a[5 + 2 * i], b[5 + 2 * i])
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

// A token's cosines and sines of the lane's pairs, times the magnitude.
struct Turn {
    float c[kPairs], s[kPairs];
};
__device__ __forceinline__ void turn_of(const Rotation& r, int64_t t, int j0, Turn& turn) {
    uint64_t step[kPairs];
    // a step of 0 turns nothing
    const int n = r.steps ? min(max(r.half - j0, 0), kPairs) : 0;
    if (n == kPairs) {
#pragma unroll
        for (int i = 0; i < kPairs; i += 2) {
            const u64x2 w = *reinterpret_cast<const u64x2*>(r.steps + j0 + i);
            step[i] = w.x;
            step[i + 1] = w.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) step[i] = i < n ? r.steps[j0 + i] : 0;
    }
    if (n == 0) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            turn.c[i] = 1.0f;
            turn.s[i] = 0.0f;
        }
        return;
    }
    if (r.axes == 1 || r.axis == 0) {
        const uint64_t at = (uint64_t)r.positions[t];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) cos_sin(at * step[i], turn.c[i], turn.s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
            cos_sin((uint64_t)r.positions[(int64_t)min((int)step[i] & 3, r.axes - 1) * r.axis + t] * step[i], turn.c[i], turn.s[i]);
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        turn.c[i] = i < n ? turn.c[i] * r.magnitude : 1.0f;
        turn.s[i] = i < n ? turn.s[i] * r.magnitude * r.sign : 0.0f;
    }
}
__device__ __forceinline__ void rotate_pairs(const Turn& t, float (&a)[kPairs], float (&b)[kPairs]) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        const float x = a[i], y = b[i];
        a[i] = x * t.c[i] - y * t.s[i];
        b[i] = y * t.c[i] + x * t.s[i];
    }
}

// The lane's factors of the norm, center + weight.
template <bool VEC>
__device__ __forceinline__ void norm_weights(const uint16_t* w, float center, const Lane& l, int half, int D, bool neighbours,
                                             float (&a)[kPairs], float (&b)[kPairs]) {
    unpack<VEC>(load_pairs<VEC>(w, l, half, D, neighbours), neighbours, a, b);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        a[i] += center;
        b[i] += center;
    }
}
// x / sqrt(mean(x^2) + eps) times the factors, over the `lanes` lanes of a head.
__device__ __forceinline__ void norm_pairs(float (&a)[kPairs], float (&b)[kPairs], const float (&wa)[kPairs],
                                           const float (&wb)[kPairs], int lanes, int D, float eps) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) sum += a[i] * a[i] + b[i] * b[i];
    for (int d = 1; d < lanes; d <<= 1) sum += __shfl_xor(sum, d, 64);
    const float inv = __builtin_amdgcn_rsqf(sum / (float)D + eps);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        a[i] *= inv * wa[i];
        b[i] *= inv * wb[i];
    }
}

// ---- rotation alone -----------------------------------------------------------

// A wave takes a token and `iters` times 64 / lanes of its heads.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void rotate_kernel(Rotate a, int lane_bits, int chunks, int iters) {
    const int lane = threadIdx.x & 63, lanes = 1 << lane_bits, l = lane & (lanes - 1), g = lane >> lane_bits;
    const int64_t wave = group_index() * (kThreads / 64) + (threadIdx.x >> 6), t = wave / chunks;
    if (t >= a.T) return;
    const int first = (int)(wave - t * chunks) * iters * (64 >> lane_bits) + g;
    const Lane at = lane_of(kPairs * l, a.r.half, a.D, a.r.neighbours);
    if (at.j0 >= a.D / 2) return;
    Turn turn;
    turn_of(a.r, t, at.j0, turn);
    for (int i = 0; i < iters; ++i) {
        const int h = first + i * (64 >> lane_bits);
        if (h >= a.x.n) return;
        float x[kPairs], y[kPairs];
        unpack<VEC>(load_pairs<VEC>(a.x.x + t * a.x.tok + h * a.x.head, at, a.r.half, a.D, a.r.neighbours), a.r.neighbours, x, y);
        rotate_pairs(turn, x, y);
        store_bf16<VEC>(a.y + t * a.y_tok + h * a.y_head, at, a.r.half, a.D, a.r.neighbours, x, y);
    }
}

// ---- rotation on the way into the cache -----------------------------------------

enum Mode { kBf16, kHeads, kBlocks };

// A token's rows: its query heads, and (but in kBlocks) its keys and values.
template <int MODE, bool VEC>
__device__ void append_rows(const RotateAppend& a, int lane_bits, int chunks, int iters, int64_t wave) {
    const int lane = threadIdx.x & 63, lanes = 1 << lane_bits, l = lane & (lanes - 1), g = lane >> lane_bits;
    const int64_t t = wave / chunks;
    if (t >= a.T) return;
    const int first = (int)(wave - t * chunks) * iters * (64 >> lane_bits) + g;
    const bool nb = a.r.neighbours;
    const int half = a.r.half, D = a.D, rows = a.q.n + (MODE == kBlocks ? 0 : 2 * a.k.n);
    const Lane at = lane_of(kPairs * l, half, D, nb);
    const bool live = at.j0 < D / 2;
    Turn turn;
    if (live) turn_of(a.r, t, at.j0, turn);
    const int64_t slot = MODE == kBlocks ? -1 : a.slots[t];
    for (int i = 0; i < iters; ++i) {
        const int row = first + i * (64 >> lane_bits);
        const bool ok = live && row < rows, is_q = row < a.q.n, is_v = row >= a.q.n + a.k.n;
        const int h = is_q ? row : is_v ? row - a.q.n - a.k.n : row - a.q.n;
        float x[kPairs] = {}, y[kPairs] = {}, wx[kPairs] = {}, wy[kPairs] = {};
        const uint16_t* norm = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        if (ok) {
            const Heads& from = is_q ? a.q : is_v ? a.v : a.k;
            unpack<VEC>(load_pairs<VEC>(from.x + t * from.tok + h * from.head, at, half, D, nb), nb, x, y);
            if (norm) norm_weights<VEC>(norm, a.center, at, half, D, nb, wx, wy);
        }
        if (a.q_norm || a.k_norm) {
            // all lanes: a head's lanes agree on whether it is normed
            float u[kPairs], v[kPairs];
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                u[k] = x[k];
                v[k] = y[k];
            }
            norm_pairs(u, v, wx, wy, lanes, D, a.eps);
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                x[k] = norm ? u[k] : x[k];
                y[k] = norm ? v[k] : y[k];
            }
        }
        if (!ok) continue;
        if (!is_v) rotate_pairs(turn, x, y);
        if (is_q) {
            store_bf16<VEC>(a.y + t * a.y_tok + h * a.y_head, at, half, D, nb, x, y);
            continue;
        }
        if constexpr (MODE != kBlocks) {
            if (slot < 0 || slot >= a.limit) continue;
            const PagedCache& c = is_v ? a.vc : a.kc;
            const int64_t dst = (slot >> a.page_bits) * c.page + (slot & (((int64_t)1 << a.page_bits) - 1)) * c.slot + h * c.head;
            if constexpr (MODE == kHeads) {
                // an IEEE division, as paged_append's
                const float s = (is_v ? a.v_scale : a.k_scale)[h];
#pragma unroll
                for (int k = 0; k < kPairs; ++k) {
                    x[k] /= s;
                    y[k] /= s;
                }
                store_codes<VEC>(static_cast<uint8_t*>(const_cast<void*>(c.data)) + dst, at, half, D, nb, x, y);
            } else {
                store_bf16<VEC>(static_cast<uint16_t*>(const_cast<void*>(c.data)) + dst, at, half, D, nb, x, y);
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

constexpr int kKeep = 4;  // rows whose values a lane keeps between the two passes

// One head's rows t0 .. t0 + n, all of one block, by a workgroup: their largest
// value gives the block's power of two; where that grows, the block's other
// codes are multiplied; then the rows' codes.
template <bool VEC>
__device__ void append_run(const RotateAppend& a, int lane_bits, int64_t t0, int64_t n, int h, bool is_v) {
    __shared__ float tops[kThreads / 64];
    __shared__ uint32_t written[4];  // the block's slots that the rows write
    const int tid = threadIdx.x, lanes = 1 << lane_bits, l = tid & (lanes - 1), g = tid >> lane_bits, G = kThreads >> lane_bits;
    const bool nb = a.r.neighbours;
    const int half = a.r.half, D = a.D, block = 1 << a.block_bits;
    const Lane at = lane_of(kPairs * l, half, D, nb);
    const bool live = at.j0 < D / 2;
    const Heads& from = is_v ? a.v : a.k;
    const uint16_t* norm = is_v ? nullptr : a.k_norm;
    float wx[kPairs] = {}, wy[kPairs] = {};
    if (norm && live) norm_weights<VEC>(norm, a.center, at, half, D, nb, wx, wy);
    if (tid < 4) written[tid] = 0;
    __syncthreads();

    auto values = [&](int64_t i, float (&x)[kPairs], float (&y)[kPairs]) {
#pragma unroll
        for (int k = 0; k < kPairs; ++k) x[k] = y[k] = 0.0f;
        const bool ok = live && i < n;
        if (ok) unpack<VEC>(load_pairs<VEC>(from.x + (t0 + i) * from.tok + h * from.head, at, half, D, nb), nb, x, y);
        if (norm) norm_pairs(x, y, wx, wy, lanes, D, a.eps);
        if (ok && !is_v && a.r.steps) {
            Turn turn;
            turn_of(a.r, t0 + i, at.j0, turn);
            rotate_pairs(turn, x, y);
        }
    };
    auto largest = [](const float (&x)[kPairs], const float (&y)[kPairs], float top) {
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            const float u = fabsf(x[k]), v = fabsf(y[k]);
            top = fmaxf(top, u < __builtin_inff() ? u : 0.0f);
            top = fmaxf(top, v < __builtin_inff() ? v : 0.0f);
        }
        return top;
    };
    float x[kKeep][kPairs], y[kKeep][kPairs], top = 0.0f;
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
        if (k * G < n) {
            values(k * G + g, x[k], y[k]);
            top = largest(x[k], y[k], top);
        }
    }
    for (int64_t i = kKeep * G; i < n; i += G) {
        float u[kPairs], v[kPairs];
        values(i + g, u, v);
        top = largest(u, v, top);
    }
    for (int64_t i = tid; i < n; i += kThreads) {
        const int s = (int)(a.slots[t0 + i] & (block - 1));
        atomicOr(&written[s >> 5], 1u << (s & 31));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, tops[w]);

    const PagedCache& c = is_v ? a.vc : a.kc;
    const int64_t slot0 = a.slots[t0] >> a.block_bits << a.block_bits, page = slot0 >> a.page_bits;
    const int in_page = (int)(slot0 & (((int64_t)1 << a.page_bits) - 1));
    uint8_t* codes = static_cast<uint8_t*>(const_cast<void*>(c.data)) + page * c.page + in_page * c.slot + h * c.head;
    uint8_t* byte = (is_v ? a.v_pow : a.k_pow) + ((page << (a.page_bits - a.block_bits)) + (in_page >> a.block_bits)) * a.k.n + h;
    int power = block_power(top);
    if (!(written[0] & 1)) {
        const int old = min((int)*byte, kMaxPower);
        if (old < power) {
            const float f = power_of(127 + old - power);
            for (int e = tid; e < block * (D / 4); e += kThreads) {
                const int s = e / (D / 4), d = 4 * (e % (D / 4));
                if (written[s >> 5] >> (s & 31) & 1) continue;
                uint32_t* p = reinterpret_cast<uint32_t*>(codes + s * c.slot + d);
                const f32x2 lo = fp8x2_to_f32<false>(*p), hi = fp8x2_to_f32<true>(*p);
                *p = codes4(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
            }
        }
        power = max(power, old);
    }
    const float inv = power_of(254 - power);
    auto store = [&](int64_t i, float (&u)[kPairs], float (&v)[kPairs]) {
        if (!live || i >= n) return;
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            u[k] *= inv;
            v[k] *= inv;
        }
        store_codes<VEC>(codes + (a.slots[t0 + i] & (block - 1)) * c.slot, at, half, D, nb, u, v);
    };
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
        if (k * G < n) store(k * G + g, x[k], y[k]);
    for (int64_t i = kKeep * G; i < n; i += G) {
        float u[kPairs], v[kPairs];
        values(i + g, u, v);
        store(i + g, u, v);
    }
    __syncthreads();  // every thread has read the old byte
    if (tid == 0) *byte = (uint8_t)power;
}

// Workgroups below `row_groups` take the tokens' rows; the others, of one head
// of the keys or values each, the runs that begin in kChunk tokens.
template <int MODE, bool VEC>
__global__ __launch_bounds__(kThreads) void rotate_append_kernel(RotateAppend a, int lane_bits, int chunks, int iters,
                                                                 int64_t row_groups, int run_bits) {
    const int64_t group = group_index();
    if (MODE != kBlocks || group < row_groups) {
        append_rows<MODE, VEC>(a, lane_bits, chunks, iters, group * (kThreads / 64) + (threadIdx.x >> 6));
        return;
    }
    if constexpr (MODE == kBlocks) {
        const int64_t item = group - row_groups;
        const int unit = (int)(item % (2 * a.k.n));
        const int64_t first = item / (2 * a.k.n) << run_bits, last = min(first + (1 << run_bits), a.T);
        auto block_of = [&](int64_t t) {
            const int64_t s = t < 0 || t >= a.T ? -1 : a.slots[t];
            return s < 0 || s >= a.limit ? -1 : s >> a.block_bits;
        };
        int64_t before = block_of(first - 1);
        for (int64_t t = first; t < last; ++t) {
            const int64_t mine = block_of(t);
            if (mine >= 0 && mine != before) {
                int64_t n = 1;
                while (t + n < a.T && block_of(t + n) == mine) ++n;
                append_run<VEC>(a, lane_bits, t, n, unit >> 1, unit & 1);
                __syncthreads();
            }
            before = mine;
        }
    }
}

int lane_bits_of(int D) {
    int bits = 0;
    while ((16 << bits) < D) ++bits;
    return bits;
}
bool side_by_side(const Rotation& r, int D) { return D % 16 == 0 && (r.neighbours || r.half % 8 == 0); }

}  // namespace

hipError_t launch_rotate(const Rotate& a, hipStream_t stream) {
    const int bits = lane_bits_of(a.D), per = 64 >> bits, groups = (a.x.n + per - 1) / per;
    const int iters = 1, chunks = (groups + iters - 1) / iters;
    const dim3 grid = grid_of((a.T * chunks + 3) / 4), block(kThreads);
    if (side_by_side(a.r, a.D)) hipLaunchKernelGGL(rotate_kernel<true>, grid, block, 0, stream, a, bits, chunks, iters);
    else hipLaunchKernelGGL(rotate_kernel<false>, grid, block, 0, stream, a, bits, chunks, iters);
    return hipGetLastError();
}

hipError_t launch_rotate_append(const RotateAppend& a, hipStream_t stream) {
    const int mode = a.k_pow ? kBlocks : a.fp8 ? kHeads : kBf16;
    const int bits = lane_bits_of(a.D), per = 64 >> bits, rows = a.q.n + (mode == kBlocks ? 0 : 2 * a.k.n);
    const int groups = (rows + per - 1) / per, iters = 1, chunks = (groups + iters - 1) / iters;
    const int64_t row_groups = (a.T * chunks + 3) / 4;
    const int run_bits = a.T > 512 ? 2 : 0;
    const int64_t runs = mode == kBlocks ? ((a.T + (1 << run_bits) - 1) >> run_bits) * 2 * a.k.n : 0;
    const dim3 grid = grid_of(row_groups + runs), block(kThreads);
    const bool vec = side_by_side(a.r, a.D);
    auto go = [&](auto mode_) {
        constexpr int M = decltype(mode_)::value;
        if (vec) hipLaunchKernelGGL((rotate_append_kernel<M, true>), grid, block, 0, stream, a, bits, chunks, iters, row_groups, run_bits);
        else hipLaunchKernelGGL((rotate_append_kernel<M, false>), grid, block, 0, stream, a, bits, chunks, iters, row_groups, run_bits);
        return hipGetLastError();
    };
    if (mode == kBlocks) return go(std::integral_constant<int, kBlocks>{});
    if (mode == kHeads) return go(std::integral_constant<int, kHeads>{});
    return go(std::integral_constant<int, kBf16>{});
}

}  // namespace fp8lin
