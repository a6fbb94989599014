// Attention of new tokens over a paged cache: what the two kernels of
// attention_few.hip and attention_tile.hip share.
//
// For row i of a request (a new token at position p_i, one query head),
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(c q_i.k_j - m_i),
// over the keys j <= p_i (all keys when not causal), c = scale * log2(e).
// One pass over the keys keeps a running m_i, the sum of weights and the
// weighted sum of values in FP32; two parts (m, l, O) of a row are joined as
// (M, l 2^(m-M) + l' 2^(m'-M), O 2^(m-M) + O' 2^(m'-M)), M = max(m, m').
// The weights are rounded to BF16 for the product with V, as the matrix
// cores take it (half a step of 2^-8 each, averaged over the keys); the sum
// of weights adds them unrounded.
//
// m_i only moves when a score passes it by more than 2^8: any m_i gives the
// same o_i, and weights up to 2^8 lose nothing in FP32 or BF16, so most key
// tiles need no rescaling of O and no maximum across lanes.
#pragma once
#include "device.hpp"
#include "gemm_fp8.hpp"
#include "paged.hpp"

namespace fp8lin {
namespace attn {

using gemm_fp8::i32x4;
using gemm_fp8::make_desc;
using gemm_fp8::wait_lgkm;
using gemm_fp8::wait_vm;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr float kLazy = 8.0f;  // log2 of the largest weight before m moves
constexpr int kGroups = 256;   // workgroups of a launch at one per CU
constexpr int kFewRows = 64;   // rows of a request that the few-rows kernel takes
constexpr int kTileRows = 256;  // rows of a tile of the other

// 64 lanes x 16 B from global (voff, bounds-checked) into LDS [m0v, m0v + 1024).
// K and V rows that one workgroup reads take the non-temporal policy.
template <bool NT>
__device__ __forceinline__ void dma(uint32_t m0v, uint32_t voff, i32x4 desc) {
    if constexpr (NT)
        gemm_fp8::dma16_nt(m0v, voff, desc, 0);
    else
        gemm_fp8::dma16(m0v, voff, desc, 0);
}

// Four values of a 16-bit matrix in LDS, read across rows: the 16 lanes of a
// group give the addresses of 4 rows x 16 columns (lane i: row i / 4, columns
// 4 (i % 4) ..), and lane i receives column i of the 4 rows.
__device__ __forceinline__ s16x4 read_tr16(uint32_t addr) {
    typedef __attribute__((address_space(3))) s16x4 lds_t;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(uintptr_t)addr);
}
// The same of an 8-bit matrix: 8 rows x 16 columns (lane i: row i / 2, columns
// 8 (i % 2) ..), lane i receives column i of the 8 rows.
__device__ __forceinline__ i32x2 read_tr8(uint32_t addr) {
    typedef __attribute__((address_space(3))) i32x2 lds_t;
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_t*)(uintptr_t)addr);
}
__device__ __forceinline__ u32x4 read16(uint32_t addr) {
    typedef __attribute__((address_space(3))) u32x4 lds_t;
    return *(lds_t*)(uintptr_t)addr;
}

// Two E4M3FN codes times a power of two to BF16, exactly (every code has 4
// significant bits; the instruction takes the scale's exponent): the scales of
// a cache's blocks cost no instruction here.
template <bool HI>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
__device__ __forceinline__ bf16x8 codes8_bf16(uint32_t lo, uint32_t hi, float scale_lo = 1.0f, float scale_hi = 1.0f) {
    return __builtin_bit_cast(bf16x8, u32x4{codes_bf16<false>(lo, scale_lo), codes_bf16<true>(lo, scale_lo),
                                            codes_bf16<false>(hi, scale_hi), codes_bf16<true>(hi, scale_hi)});
}

// E8M0 powers of two of a cache's blocks, a byte each.  As long as a block is
// 16 tokens or more, the 16 keys of one page that a DMA brings have one.
__device__ __forceinline__ uint32_t power_index(const PagedAttention& a, int id, int64_t key, int hk) {
    const int in_page = (int)(key & ((1 << a.page_bits) - 1));
    return (((uint32_t)id << (a.page_bits - a.block_bits)) + (uint32_t)(in_page >> a.block_bits)) * (uint32_t)a.HK + (uint32_t)hk;
}
// The bytes of all blocks, below 2^32; other offsets read 0.
__device__ __forceinline__ i32x4 power_desc(const PagedAttention& a, const uint8_t* bytes) {
    return make_desc(bytes, ((uint32_t)a.pages << (a.page_bits - a.block_bits)) * (uint32_t)a.HK);
}
constexpr uint32_t kNoPower = 0xffffffffu;
// A byte a lane from global (voff, bounds-checked), as 32 bits into LDS [m0v, m0v + 256).
__device__ __forceinline__ void dma_byte(uint32_t m0v, uint32_t voff, i32x4 desc) {
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_ubyte %1, %2, 0 offen lds" ::"s"(m0v), "v"(voff), "s"(desc) : "memory", "m0");
}
__device__ __forceinline__ float power_at(uint32_t lds) {
    typedef __attribute__((address_space(3))) uint32_t lds_t;
    return __builtin_bit_cast(float, *(lds_t*)(uintptr_t)lds << 23);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 and 8 bytes at any BF16 element: gfx950 takes unaligned global accesses,
// so operands off the 16-byte grid need no other path.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef u32x2 __attribute__((aligned(2))) u32x2_any;

// N fragments of 8 values of a query row, from elements at(t).  A row past the
// tile gives those of some row: its scores and sums stay in its own lanes, and
// it is not written.
template <int N, class AT>
__device__ __forceinline__ void load_queries(const uint16_t* row, bf16x8 (&qf)[N], AT at) {
#pragma unroll
    for (int t = 0; t < N; ++t) qf[t] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4_any*>(row + at(t)));
}

__device__ __forceinline__ u32x2 load_gate4(const uint16_t* g) { return *reinterpret_cast<const u32x2_any*>(g); }
// o * sigmoid(gate) by the hardware's 2^x and reciprocal, a few units of FP32
// off; a gate of -inf gives 0, whatever o is short of NaN.
__device__ __forceinline__ void apply_gate(f32x4& o, u32x2 gv) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = bf16_bits_to_f32(((i < 2 ? gv.x : gv.y) >> (16 * (i & 1))) & 0xffffu);
        o[i] *= __builtin_amdgcn_rcpf(1.0f + exp2_fast(x * -1.44269504088896340736f));
    }
}
// The same of N groups of 4: a value's chain of six instructions waits on each,
// so all values take each step together.
template <int N>
__device__ __forceinline__ void apply_gates(f32x4 (&o)[N], const u32x2 (&gv)[N]) {
    float e[4 * N];
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
        const u32x2 w = gv[i / 4];
        e[i] = exp2_fast(-1.44269504088896340736f * bf16_bits_to_f32(((i % 4 < 2 ? w.x : w.y) >> (16 * (i & 1))) & 0xffffu));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) e[i] = __builtin_amdgcn_rcpf(1.0f + e[i]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) o[i / 4][i % 4] *= e[i];
}
__device__ __forceinline__ void store_bf16x4(uint16_t* y, f32x4 o) {
    *reinterpret_cast<u32x2_any*>(y) = u32x2{pack_bf16x2(f32x2{o.x, o.y}), pack_bf16x2(f32x2{o.z, o.w})};
}
// out[d .. d+3] = bf16(o * sigmoid(gate)): one rounding.
__device__ __forceinline__ void store4(const PagedAttention& a, int64_t tok, int head, int d, f32x4 o) {
    if (a.gate) apply_gate(o, load_gate4(a.gate + tok * a.g_tok + head * a.g_head + d));
    store_bf16x4(a.out + tok * a.o_tok + head * a.o_head + d, o);
}

// Whether the values of keys first, first + 1, .. < last hold an infinity or
// NaN (on the lane that sees one), by wave `wave` of `waves` that share them.
template <int D, bool F8>
__device__ __forceinline__ bool odd_values(const PagedAttention& a, const int32_t* table, int hk, int first, int last, int wave,
                                           int waves) {
    constexpr int ES = F8 ? 1 : 2, LANES = D * ES / 16, PER = 64 / LANES;  // 16 bytes a lane, keys at once
    // an exponent of all ones (E4M3FN: all bits but the sign) carries into the bit above it
    constexpr uint32_t BITS = F8 ? 0x7f7f7f7fu : 0x7f807f80u, ONE = F8 ? 0x01010101u : 0x00800080u;
    const int lane = threadIdx.x & 63;
    const char* base = static_cast<const char*>(a.v.data) + hk * a.v.head * ES + 16 * (lane % LANES);
    uint32_t odd = 0;
#pragma unroll 8
    for (int k = first + PER * wave; k < last; k += PER * waves) {
        const int key = min(k + lane / LANES, last - 1), id = table[key >> a.page_bits];
        const bool there = (unsigned)id < (unsigned)a.pages;
        const int64_t at = (int64_t)(there ? id : 0) * a.v.page + (int64_t)(key & ((1 << a.page_bits) - 1)) * a.v.slot;
        const u32x4 w = *reinterpret_cast<const u32x4*>(base + at * ES);
#pragma unroll
        for (int i = 0; i < 4; ++i) odd |= there ? (w[i] & BITS) + ONE : 0;
    }
    return (odd & (F8 ? 0x80808080u : 0x80008000u)) != 0;
}

// One row by plain FP32 sums, a key at a time, by a wave: for the rows near
// values that only some rows may see and that are infinities or NaN, which the
// matrix product would carry, as 0 * inf, into the other rows of its tile.
template <int D, int KIND>
__device__ void plain_row(const PagedAttention& a, const PagedSeq& s, int b, int hk, int flat) {
    constexpr bool F8 = KIND != kCacheBf16;
    constexpr int LANES = D / 4;  // 4 dimensions a lane
    const int lane = threadIdx.x & 63, d = 4 * (lane % LANES);
    const int32_t* table = a.table + (int64_t)b * a.ldt;
    const float c = a.scale2 * (KIND == kCacheHeads ? a.k_scale[hk] : 1.0f);
    auto value4 = [&](const PagedCache& cache, const uint8_t* powers, int id, int key) {
        f32x4 x = {0, 0, 0, 0};
        if ((unsigned)id >= (unsigned)a.pages) return x;
        const int64_t at = (int64_t)id * cache.page + (int64_t)(key & ((1 << a.page_bits) - 1)) * cache.slot + hk * cache.head + d;
        if constexpr (F8) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(cache.data) + at);
            const f32x2 lo = fp8x2_to_f32<false>(w), hi = fp8x2_to_f32<true>(w);
            x = f32x4{lo.x, lo.y, hi.x, hi.y};
            if constexpr (KIND == kCacheBlocks) {
                const float f = __builtin_bit_cast(float, (uint32_t)powers[power_index(a, id, key, hk)] << 23);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] *= f;
            }
        } else {
            const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(cache.data) + at);
            x = f32x4{bf16_bits_to_f32(w.x & 0xffffu), bf16_bits_to_f32(w.x >> 16), bf16_bits_to_f32(w.y & 0xffffu),
                      bf16_bits_to_f32(w.y >> 16)};
        }
        return x;
    };
    const int tok = flat / a.G, head = hk * a.G + flat % a.G;
    const int lim = a.causal ? min(max(s.len - s.n + tok + 1, 0), s.len) : s.len;
    const uint16_t* q = a.q + (int64_t)(s.off + tok) * a.q_tok + (int64_t)head * a.q_head + d;
    float m = -__builtin_inff(), l = 0.0f;
    f32x4 qv, o = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) qv[i] = bf16_bits_to_f32(q[i]);
    for (int key = 0; key < lim; ++key) {
        const int id = table[key >> a.page_bits];
        const f32x4 k = value4(a.k, a.k_pow, id, key), v = value4(a.v, a.v_pow, id, key);
        float x = lane < LANES ? qv.x * k.x + qv.y * k.y + qv.z * k.z + qv.w * k.w : 0.0f;
        x = wave_sum(x) * c;
        const float mn = fmaxf(m, x), ms = mn == -__builtin_inff() ? 0.0f : mn;
        const float f = m == -__builtin_inff() ? 0.0f : exp2_fast(m - ms), p = exp2_fast(x - ms);
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * f + p * v[i];
        m = mn;
    }
    const float inv = l == 0.0f ? 0.0f : (KIND == kCacheHeads ? a.v_scale[hk] : 1.0f) / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = l == 0.0f ? 0.0f : o[i] * inv;
    if (lane < LANES) store4(a, s.off + tok, head, d, o);
}

// The workspace: per workgroup where its piece begins (request, kv head, row
// tile, key tile; request -1: no piece), the request's first row and the tile's
// rows, and for each wave whether it met values that not all of its rows may
// see and that are no finite numbers; then the partial sums of split units: O
// (BM x D floats, the kernel's own order), m and l of the BM rows.  A workgroup
// leaves at most two: slot 0 for the piece that begins inside a unit (its
// first), slot 1 for the one that begins a unit (its last).
typedef int i32x4v __attribute__((ext_vector_type(4)));
constexpr int kBeginInts = 16, kBeginFloats = kGroups * kBeginInts;
__device__ __forceinline__ i32x4v* begin_of(float* ws, int group) { return reinterpret_cast<i32x4v*>(ws + group * kBeginInts); }
__device__ __forceinline__ int* bad_of(float* ws, int group, int wave) {
    return reinterpret_cast<int*>(ws + group * kBeginInts + 8) + wave;
}
template <int BM, int D>
struct Partial {
    static constexpr int64_t kFloats = (int64_t)BM * D + 2 * BM;
    static constexpr int64_t kBytes = 4 * (kBeginFloats + 2 * kGroups * kFloats);
    static __device__ __forceinline__ float* at(float* ws, int group, int slot) {
        return ws + kBeginFloats + (2 * group + slot) * kFloats;
    }
};

// `rows`: the most of a request.  Without `join` the units' partial sums are
// left to launch_tile's `few`, which joins both kernels' in one launch.
hipError_t launch_few(const PagedAttention& a, int D, CacheKind kind, int rows, bool join, hipStream_t stream);
hipError_t launch_tile(const PagedAttention& a, const PagedAttention* few, int D, CacheKind kind, hipStream_t stream);
constexpr int kMixedRows = 32;  // rows of a few-rows tile of a mixed batch

// Joins the pieces of the units that the boundaries between workgroups cut,
// and writes their rows.  Every workgroup lists the split units from the
// pieces' beginnings and takes every gridDim.x-th part of them: 64 (WAVES 4:
// its waves share the pieces of a unit, which are many and small in a decode
// step) or 1024 (WAVES 1) groups of 4 values.  ORDER::place(e, row, d): row and
// first dimension of the e-th 4 floats of a piece's O.  The units of workgroups
// with marked waves are computed again, row by row, instead.
template <int BM, int D, int KIND, int WAVES, class ORDER>
__device__ __forceinline__ void join(const PagedAttention& a, int block, int blocks) {
    constexpr int PER = 256 / WAVES, PARTS = BM * D / 4 / PER;
    __shared__ i32x4v begin[kGroups], rows[kGroups];
    __shared__ int unit[kGroups], unit_last[kGroups], wave_units[4];
    __shared__ f32x4 so[WAVES][PER];
    __shared__ float sm[WAVES][PER], sl[WAVES][PER];
    static_assert(kGroups == 256, "a thread per piece");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ uint8_t bad[kGroups];
    {
        const i32x4v* at = begin_of(a.ws, tid);
        begin[tid] = at[0];
        rows[tid] = at[1];
        const i32x4v x = at[2], y = at[3];
        bad[tid] = begin[tid].x >= 0 && (x.x | x.y | x.z | x.w | y.x | y.y | y.z | y.w);
    }
    const bool any_bad = __syncthreads_or(bad[tid]);
    auto same = [](const i32x4v& x, const i32x4v& y) { return x.x == y.x && x.y == y.y && x.z == y.z; };
    // the first boundary inside a unit
    const i32x4v mine = begin[tid];
    const bool first = tid > 0 && mine.x >= 0 && mine.w > 0 && !(same(begin[tid - 1], mine) && begin[tid - 1].w > 0);
    const uint64_t mask = __ballot(first);
    if (lane == 0) wave_units[wave] = __popcll(mask);
    __syncthreads();
    int at = __popcll(mask & ((1ull << lane) - 1)), units = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) at += wave_units[w];
        units += wave_units[w];
    }
    if (first) unit[at] = tid;
    if (tid > 0 && mine.x >= 0 && mine.w > 0 && (tid == kGroups - 1 || !same(begin[tid + 1], mine)))
        unit_last[at + (first ? 0 : -1)] = tid;
    __syncthreads();
    if constexpr (WAVES == 1) {
        // Bound by its vector instructions: what a row's values share (its place, its
        // factors, 2^x of the maxima) is computed once for the SHARE groups of 4 that
        // a thread takes of it, 64 apart in this order.  A prompt of 3913 tokens, heads
        // of 256, took 167 us with one group a thread and takes 159 (join and all).
        constexpr int SHARE = 4, ITEMS = PARTS / SHARE;
        for (int item = block; item < units * ITEMS; item += blocks) {
            const int w = unit[item / ITEMS], e = (item % ITEMS) * (PER * SHARE) + wave * (64 * SHARE) + lane;
            const i32x4v u = begin[w];
            const int r0 = u.z * BM, off = rows[w].x, nr = rows[w].y;
            int row, d;
            ORDER::place(e, row, d);
            if (row >= nr) continue;
            const int flat = r0 + row, tok = off + flat / a.G, head = u.y * a.G + flat % a.G;
            u32x2 gate[SHARE];
            if (a.gate) {
#pragma unroll
                for (int k = 0; k < SHARE; ++k) gate[k] = load_gate4(a.gate + tok * a.g_tok + head * a.g_head + d + ORDER::kNext * k);
            }
            // the unit's pieces: workgroups w - 1 (slot 1), w, .. last (slot 0)
            const int last = unit_last[item / ITEMS];
            if (any_bad) {
                bool skip = false;
                for (int g = w - 1; g <= last; ++g) skip |= bad[g] != 0;
                if (skip) continue;
            }
            float M = -__builtin_inff(), l = 0.0f;
            f32x4 o[SHARE];
#pragma unroll
            for (int k = 0; k < SHARE; ++k) o[k] = f32x4{0, 0, 0, 0};
            constexpr int UN = 2;  // pieces whose loads are in flight together
            for (int g0 = w - 1; g0 <= last; g0 += UN) {
                float m1[UN], l1[UN];
                f32x4 o1[UN][SHARE];
                bool there[UN];
#pragma unroll
                for (int i = 0; i < UN; ++i) {
                    const int g = g0 + i;
                    // an empty piece: the next one begins where it does
                    there[i] = g <= last && !(g < last && g >= w && begin[g + 1].w == begin[g].w);
                    // loaded without a condition (another piece's), so that all are in flight
                    const int from = there[i] ? g : w - 1;
                    const float* part = Partial<BM, D>::at(a.ws, from, from < w);
                    m1[i] = part[(int64_t)BM * D + row];
                    l1[i] = part[(int64_t)BM * D + BM + row];
#pragma unroll
                    for (int k = 0; k < SHARE; ++k) o1[i][k] = *reinterpret_cast<const f32x4*>(part + 4 * (int64_t)(e + 64 * k));
                }
#pragma unroll
                for (int i = 0; i < UN; ++i) {
                    if (!there[i]) continue;
                    // as below, the products' places in the fused operations said
                    const float mn = fmaxf(M, m1[i]);
                    const float f0 = M == -__builtin_inff() ? 0.0f : exp2_fast(M - mn);
                    const float f1 = m1[i] == -__builtin_inff() ? 0.0f : exp2_fast(m1[i] - mn);
                    l = __builtin_fmaf(l1[i], f1, l * f0);
#pragma unroll
                    for (int k = 0; k < SHARE; ++k)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[k][j] = __builtin_fmaf(o1[i][k][j], f1, o[k][j] * f0);
                    M = mn;
                }
            }
            const float inv = l == 0.0f ? 0.0f : (a.v_scale ? a.v_scale[u.y] : 1.0f) / l;
#pragma unroll
            for (int k = 0; k < SHARE; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[k][j] = l == 0.0f ? 0.0f : o[k][j] * inv;
            if (a.gate) apply_gates<SHARE>(o, gate);
            uint16_t* out = a.out + tok * a.o_tok + head * a.o_head + d;
#pragma unroll
            for (int k = 0; k < SHARE; ++k) store_bf16x4(out + ORDER::kNext * k, o[k]);
        }
    } else {
        const int q = wave, et = lane;
        // A tile's rows from its first to its last part, of all units before the next
        // part: a decode step has a few of a tile's 16 rows, and the parts of the others,
        // at the end, are passed over by all alike (61 requests, 12/2 heads of 256: 99 us a
        // call, 103 with each unit's parts side by side).
        for (int item = block; item < units * PARTS; item += blocks) {
            const int at_unit = item % units, e0 = item / units * PER, e = e0 + et;
            const int w = unit[at_unit];
            const i32x4v u = begin[w];
            const int r0 = u.z * BM, off = rows[w].x, nr = rows[w].y;
            int row, d;
            ORDER::place(e0, row, d);
            if (row >= nr) continue;  // of the whole workgroup
            ORDER::place(e, row, d);
            const bool ok = row < nr;
            const int flat = r0 + min(row, nr - 1), tok = off + flat / a.G, head = u.y * a.G + flat % a.G;
            u32x2 gate = {0, 0};
            if (a.gate) gate = load_gate4(a.gate + tok * a.g_tok + head * a.g_head + d);
            // the unit's pieces: workgroups w - 1 (slot 1), w, .. last (slot 0)
            const int last = unit_last[at_unit];
            if (any_bad) {
                bool skip = false;
                for (int g = w - 1; g <= last; ++g) skip |= bad[g] != 0;
                if (skip) continue;
            }
            float M = -__builtin_inff(), l = 0.0f;
            f32x4 o = {0, 0, 0, 0};
            // A factor of 0 is multiplied in like any other: a part whose scores are
            // all NaN has m = -inf and l = NaN, and a NaN stays one however little
            // its part weighs; a part of nothing adds l = 0, O = 0.
            auto add = [&](float m1, float l1, f32x4 o1) {
                const float mn = fmaxf(M, m1);
                const float f0 = M == -__builtin_inff() ? 0.0f : exp2_fast(M - mn);
                const float f1 = m1 == -__builtin_inff() ? 0.0f : exp2_fast(m1 - mn);
                l = l * f0 + l1 * f1;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = o[i] * f0 + o1[i] * f1;
                M = mn;
            };
            if (ok) {
                constexpr int UN = 8;  // pieces whose loads are in flight together
                for (int g0 = w - 1 + q; g0 <= last; g0 += WAVES * UN) {
                    float m1[UN], l1[UN];
                    f32x4 o1[UN];
#pragma unroll
                    for (int i = 0; i < UN; ++i) {
                        const int g = g0 + i * WAVES;
                        // an empty piece: the next one begins where it does
                        const bool there = g <= last && !(g < last && g >= w && begin[g + 1].w == begin[g].w);
                        // loaded without a condition (another piece's), so that all are in flight
                        const int from = there ? g : w - 1;
                        const float* part = Partial<BM, D>::at(a.ws, from, from < w);
                        m1[i] = part[(int64_t)BM * D + row];
                        l1[i] = part[(int64_t)BM * D + BM + row];
                        o1[i] = *reinterpret_cast<const f32x4*>(part + 4 * (int64_t)e);
                        if (!there) {
                            m1[i] = -__builtin_inff();
                            l1[i] = 0.0f;
                            o1[i] = f32x4{0, 0, 0, 0};
                        }
                    }
#pragma unroll
                    for (int i = 0; i < UN; ++i) add(m1[i], l1[i], o1[i]);
                }
            }
            __syncthreads();
            so[q][et] = o;
            sm[q][et] = M;
            sl[q][et] = l;
            __syncthreads();
            if (q == 0)
#pragma unroll
                for (int i = 1; i < WAVES; ++i) add(sm[i][et], sl[i][et], so[i][et]);
            if (q == 0 && ok) {
                const float inv = l == 0.0f ? 0.0f : (a.v_scale ? a.v_scale[u.y] : 1.0f) / l;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = l == 0.0f ? 0.0f : o[i] * inv;
                if (a.gate) apply_gate(o, gate);
                store_bf16x4(a.out + tok * a.o_tok + head * a.o_head + d, o);
            }
        }
    }
    if (any_bad) {
        using Split = PagedSplit<BM, 16, 0>;
        for (int g = 0; g < kGroups; ++g) {
            if (!bad[g]) continue;
            const i32x4v last = g + 1 < kGroups ? begin[g + 1] : i32x4v{-1, 0, 0, 0};
            for (i32x4v u = begin[g]; u.x < a.B;) {
                const bool end = last.x >= 0 && same(u, last);
                if (end && last.w == 0) break;
                const PagedSeq s = paged_seq(a, u.x);
                const int R = Split::tiles(a, s), r0 = u.z * BM;
                if (u.z < R)
                    for (int r = block * 4 + wave; r < (int)min((int64_t)BM, (int64_t)s.n * a.G - r0); r += 4 * blocks)
                        plain_row<D, KIND>(a, s, u.x, u.y, r0 + r);
                if (end) break;
                if (++u.z >= R) {
                    u.z = 0;
                    if (++u.y >= a.HK) {
                        u.y = 0;
                        ++u.x;
                    }
                }
            }
        }
    }
}
template <int BM, int D, int KIND, int WAVES, class ORDER>
__global__ __launch_bounds__(256) void join_kernel(PagedAttention a) {
    join<BM, D, KIND, WAVES, ORDER>(a, blockIdx.x, gridDim.x);
}

// The order of O in the partial sums of the few-rows kernel: by row.
template <int D>
struct FewOrder {
    static __device__ __forceinline__ void place(int e, int& row, int& d) {
        row = e / (D / 4);
        d = 4 * (e % (D / 4));
    }
};

// The order of O in the partial sums of the kernel with 32 rows per MFMA tile:
// as their registers hold it.
template <int D>
struct TileOrder {
    static constexpr int kNext = 8;  // dimensions between a lane's groups of one row, up to 4 of them
    static __device__ __forceinline__ void place(int e, int& row, int& d) {
        const int lane = e & 63, b = (e >> 6) & 3, dt = (e >> 8) % (D / 32), wave = (e >> 8) / (D / 32);
        row = 32 * wave + (lane & 31);
        d = 32 * dt + 8 * b + 4 * (lane >> 5);
    }
};

}  // namespace attn
}  // namespace fp8lin
