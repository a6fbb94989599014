// Attention of many rows per request and kv head: prompts and their chunks.
// Bound by the matrix cores, by what feeds them and by the vector units.  A
// workgroup of 4 waves, one per SIMD with up to 512 registers each, holds 256
// rows (consecutive tokens, the G query heads of a kv head side by side), a
// wave 64 of them, and walks the keys in tiles of 64 that all waves read from
// LDS.
//
// Per step of 32 keys, MFMA 32x32x16: S^T [keys, rows] = K Q^T leaves 4
// consecutive keys of one row in a lane's registers, which is what the second
// product O^T [D, rows] += V^T P^T takes as its B operand; V^T comes from the
// transposing LDS reads, its keys in the same order.  So a row's maximum and
// sum stay in one lane pair and nothing passes through LDS between the
// products.
//
// 64 rows a wave, not 32: every K or V fragment (1 KB from LDS) then feeds two
// MFMAs.  With one each, LDS delivers just what the MFMAs take and the loop ran
// at half the rate (8 waves of 32 rows, heads of 256: 404 us for a prompt of
// 3913 tokens).  Heads of 256 take the whole register file: 256 accumulation
// registers of O^T, 128 of queries, 32 of S^T, 32 of two steps' weights.
//
// The steps are skewed: the products of step s - 1 with V are issued while the
// weights of step s are computed.  The source spreads those a few vector
// instructions behind each pair of MFMAs, in groups that sched_barrier keeps in
// order, but nothing holds their results there: the compiler moves the 2^x, the
// sums and the packing of a step past its MFMAs, behind the branch that rescales
// O.  So softmax and MFMAs run one after the other in a wave (MFMAs busy in 42%
// of the cycles of a prompt of 3913 tokens, heads of 256), and where two waves
// share a SIMD (heads of 64 and 128) the counters show little of one's hidden
// behind the other's (a mixed batch: MFMAs 37%, vector work some 47%).  The MFMAs
// are one asm statement each, with O in accumulation and S in vector registers;
// the compiler counts the LDS waits.
//
// K and V of a tile arrive by direct-to-LDS DMA into two buffers each, as they
// are in the cache; the codes of an 8-bit cache are converted when a fragment
// is read.  One barrier per tile, between its last product with K and its first
// with V: there K of the next tile and V of this one have arrived, and K of
// this tile and V of the last one are no longer read, so the DMAs of the tiles
// after go out.
//
// Heads of 256, 12/2, BF16: a prompt of 3913 tokens (94 GFLOP) 137 us, and 33 us
// for the join, MFMAs busy in 42 % of the cycles; 512 tokens after 6919 (45
// GFLOP) 68 and 17 us: a launch's 256 pieces each write 256 KB of partial sums.
#include <algorithm>

#include "attention.hpp"

namespace fp8lin {
namespace attn {
namespace {

constexpr int kBM = kTileRows, kBN = 64, kKeys = 16;  // kKeys: keys of a tile that a wave brings
// A unit's start and end, in keys (heads of 256: up to 30 us at 64 keys in 4 us).
// With 192, 320, 448 and 640 at 256 a prompt of 3913 tokens takes 217, 173, 164
// and 167 us, a chunk of 512 77, 78, 78 and 79, a mixed batch (heads of 128)
// 170, 160, 153 and 150.
template <int D>
constexpr int kTileStart = 448 * D / 256;
constexpr int kTileMinTiles = 4;

template <int D, bool F8>
struct Tile {
    static constexpr int ROWB = D * (F8 ? 1 : 2);            // bytes of a key
    static constexpr int HALF = kBN * ROWB, LDS = 4 * HALF;  // K or V of a tile; two buffers of each
    static constexpr int RPI = 1024 / ROWB, LPR = 64 / RPI;  // keys of a DMA instruction, its lanes per key
    static constexpr int NI = kKeys / RPI;                   // instructions of a wave's part of K or V
    static constexpr int PICK = ROWB >= 256 ? 16 : ROWB / 16;  // chunks (16 bytes) that xk permutes
    // Chunk permutations: 16 keys at one chunk (K), or the 4 (8-bit: 8) keys of
    // a transposing read at its 64 (32) bytes, must hit distinct columns of the
    // 256 bytes that LDS serves at once.
    static __device__ __forceinline__ int xk(int r) {
        if constexpr (ROWB >= 256) return r & 15;
        if constexpr (ROWB == 128) return (r >> 1) & 7;
        return (r >> 2) & 3;
    }
    static __device__ __forceinline__ int xv(int r) {
        if constexpr (!F8) return ROWB >= 256 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
        if constexpr (ROWB == 256) return ((r & 3) | ((r >> 1) & 4)) << 1;
        if constexpr (ROWB == 128) return (((r >> 1) & 1) | ((r >> 2) & 2)) << 1;
        return ((r >> 3) & 1) << 1;
    }
};

// S = K Q^T, O += V^T P^T.  The two wait states in front cover a vector
// instruction that wrote an operand just before.
__device__ __forceinline__ void mfma_first(f32x16& s, const u32x4& k, const bf16x8& q) {
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(k), "v"(q));
}
__device__ __forceinline__ void mfma_s(f32x16& s, const u32x4& k, const bf16x8& q) {
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(k), "v"(q));
}
__device__ __forceinline__ void mfma_o(f32x16& o, const u32x4& v, const u32x4& p) {
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(o) : "v"(v), "v"(p));
}
// The accumulators are read by vector instructions after this.
template <int RB, int NT>
__device__ __forceinline__ void drain(f32x16 (&o)[RB][NT]) {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" : "+a"(o[0][0]));
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int dt = 0; dt < NT; ++dt)
            if (rb | dt) asm volatile("" : "+a"(o[rb][dt]));
}
__device__ __forceinline__ void clear(f32x16& o) {
    const u32x4 zero = {0, 0, 0, 0};
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "=a"(o) : "v"(zero));
}

// The lane's D / 8 groups of 4 values of a row, 64 f32x4 apart, times inv (0 for
// a row without weights), gated, to out: group i is dimensions 8 i ..
template <int D>
__device__ __forceinline__ void finish_row(const PagedAttention& a, const f32x4* o, float inv, const uint16_t* gate,
                                           uint16_t* out, bool ok) {
    constexpr int N = D / 16;
#pragma unroll
    for (int i0 = 0; i0 < 2 * N; i0 += N) {
        f32x4 x[N];
        u32x2 g[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = o[(i0 + i) * 64];
        if (a.gate) {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = load_gate4(gate + 8 * (i0 + i));
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = inv == 0.0f ? 0.0f : x[i][j] * inv;
        if (a.gate) apply_gates<N>(x, g);
        if (ok) {
#pragma unroll
            for (int i = 0; i < N; ++i) store_bf16x4(out + 8 * (i0 + i), x[i]);
        }
    }
}

template <int D, bool F8, int RB>
__global__ __launch_bounds__(64 * kBM / (32 * RB), 2 / RB) void tile_kernel(PagedAttention a) {
    constexpr int W = kBM / (32 * RB);  // waves
    using L = Tile<D, F8>;
    using Split = PagedSplit<kBM, kBN, kTileStart<D>>;
    extern __shared__ __align__(1024) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5, col = lane & 31;

    int64_t* pre = reinterpret_cast<int64_t*>(lds);
    Split::prefix(a, pre, 64 * W);
    const int64_t total = pre[a.B], chunk = Split::chunk(a, total, gridDim.x, kTileMinTiles);
    const int group = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int64_t p0 = group * chunk, p1 = min(p0 + chunk, total);
    i32x4v* begin = begin_of(a.ws, group);
    if (p0 >= total) {
        if (tid == 0) begin[0] = i32x4v{-1, 0, 0, 0};
        return;
    }
    typename Split::Loc cur, end;
    Split::piece(a, pre, p0, p1, cur, end);
    PagedSeq s = paged_seq(a, cur.b);
    if (lane < 8 / W) *bad_of(a.ws, group, wave + W * lane) = 0;
    if (tid == 0) {
        begin[0] = i32x4v{cur.b, cur.hk, cur.r, cur.kt};
        begin[1] = i32x4v{s.off, (int)min((int64_t)kBM, (int64_t)s.n * a.G - (int64_t)cur.r * kBM), 0, 0};
    }
    __syncthreads();
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
    // which keys of a tile this wave brings: of K and V, or with 8 waves of one
    const int part = wave & 3;
    const bool of_k = W == 4 || wave < 4, of_v = W == 4 || wave >= 4;
    // K of tile t at (t & 1) HALF, V behind both.  This lane's reads within a
    // tile: a chunk is picked by an exclusive or of the bits above, a key by an
    // offset.
    const uint32_t k_lane = lds0 + col * L::ROWB + ((half ^ L::xk(col)) << 4);
    // keys 4 half + 0..3 (8-bit: and 8 more, 4 half + 8..11), 16 dimensions by lane & 16
    const int vi = lane & 15, vr = F8 ? 4 * half + ((vi >> 1) & 3) + 8 * (vi >> 3) : 4 * half + (vi >> 2);
    const int vc = F8 ? (lane >> 4) & 1 : 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1);
    const uint32_t v_lane = lds0 + 2 * L::HALF + vr * L::ROWB + ((vc ^ L::xv(vr)) << 4) + 8 * (lane & 1);

    for (;;) {
        const int R = Split::tiles(a, s);
        const int nkt = R ? Split::key_tiles(a, s, cur.r) : 0;
        const bool last = cur.b == end.b && cur.hk == end.hk && cur.r == end.r;
        const int k0 = cur.kt, k1 = last ? end.kt : nkt;
        if (R && k1 > k0) {
            const int r0 = cur.r * kBM, nr = (int)min((int64_t)kBM, (int64_t)s.n * a.G - r0);
            const float c = a.scale2 * (F8 ? a.k_scale[cur.hk] : 1.0f);
            const int row0 = 32 * RB * wave, ctx = s.len - s.n;
            const int32_t* table = a.table + (int64_t)cur.b * a.ldt;
            // page id of the keys that this wave brings of tile t
            auto page_of = [&](int t) {
                const int64_t key = (int64_t)t * kBN + kKeys * part;
                const int id = table[min(key, (int64_t)max(s.len - 1, 0)) >> a.page_bits];
                return t < k1 && key < s.len ? id : -1;
            };
            // this wave's keys of tile t of a cache, and the i-th of the NI
            // instructions that bring them
            struct Part {
                i32x4 desc;
                uint32_t m0;
                int slot;
            };
            auto part_of = [&](const PagedCache& cache, int t, int id, bool is_v) {
                constexpr int ES = F8 ? 1 : 2;
                const int64_t key = (int64_t)t * kBN + kKeys * part;
                const int there = (unsigned)id < (unsigned)a.pages ? (int)min((int64_t)s.len - key, (int64_t)kKeys) : 0;
                const int64_t at = (int64_t)id * cache.page + (key & ((1 << a.page_bits) - 1)) * cache.slot + cur.hk * cache.head;
                const uint32_t bytes = there > 0 ? (uint32_t)(((there - 1) * cache.slot + D) * ES) : 0;
                return Part{make_desc(static_cast<const char*>(cache.data) + (bytes ? at * ES : 0), bytes),
                            (uint32_t)__builtin_amdgcn_readfirstlane(lds0 + (is_v ? 2 * L::HALF : 0) + (t & 1) * L::HALF + kKeys * part * L::ROWB),
                            (int)cache.slot * ES};
            };
            auto bring = [&](const Part& p, int i, bool is_v) {
                const int r = L::RPI * i + lane / L::LPR;  // kKeys * part is a multiple of 16: no part in xk, xv
                const int ch = (lane % L::LPR) ^ (is_v ? L::xv(r) : L::xk(r));
                dma<false>(p.m0 + i * 1024, (uint32_t)(r * p.slot + ch * 16), p.desc);
            };
            auto bring_all = [&](const PagedCache& cache, int t, int id, bool is_v) {
                const Part p = part_of(cache, t, id, is_v);
#pragma unroll
                for (int i = 0; i < L::NI; ++i) bring(p, i, is_v);
            };
            int id0 = page_of(k0), id1 = page_of(k0 + 1);

            // B operand: row 32 rb + col, dimensions 16 t + 8 half .. (8-bit: of 32 by
            // half, as 16 codes come at once)
            bf16x8 qf[RB][D / 16];
            int lim[RB];             // keys that the lane's row may see
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int row = row0 + 32 * rb + col, flat = r0 + row, tok = flat / a.G;
                const bool ok = row < nr;
                const uint16_t* q = a.q + (int64_t)(s.off + (ok ? tok : 0)) * a.q_tok + (int64_t)(cur.hk * a.G + flat % a.G) * a.q_head;
                load_queries<D / 16>(q, qf[rb], [&](int t) { return F8 ? 16 * (t & ~1) + 16 * half + 8 * (t & 1) : 16 * t + 8 * half; });
                lim[rb] = !ok ? 0 : a.causal ? min(max(ctx + tok + 1, 0), s.len) : s.len;
            }
            // keys that the wave's first row may see: below it no mask
            const int open = a.causal ? min(max(ctx + (r0 + row0) / a.G + 1, 0), s.len) : s.len;

            id0 = __builtin_amdgcn_readfirstlane(id0);
            id1 = __builtin_amdgcn_readfirstlane(id1);
            if (of_k) {
                bring_all(a.k, k0, id0, false);
                bring_all(a.k, k0 + 1, id1, false);
            }
            if (of_v) bring_all(a.v, k0, id0, true);
            int id2 = page_of(k0 + 2);

            f32x16 o[RB][D / 32], st[RB];
            u32x4 pw[RB][2];  // weights of the step before, the B operand
            float m[RB], l[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                m[rb] = -__builtin_inff();
                l[rb] = 0.0f;
            }

            // Fragments in flight: the first ones of a phase are read in the
            // last groups of the phase before.
            constexpr int PER = F8 ? 2 : 1, NK = D / 16 / PER, NV = 2 * D / 32;  // fragments of a K read; reads of a step
            constexpr int AHEAD = 4, AK = NK < AHEAD ? NK : AHEAD;
            static_assert(NV % AHEAD == 0 && (NK % AHEAD == 0 || NK < AHEAD));
            u32x4 f[AHEAD];
            auto load_k = [&](uint32_t kb, int sub, int i) {
                f[i % AK] = read16((kb ^ ((2 * i & (L::PICK - 1)) << 4)) + 32 * sub * L::ROWB + (2 * i & ~(L::PICK - 1)) * 16);
            };
            auto load_v = [&](uint32_t vb, int sub, int i) {
                const int ks = i / (D / 32), dt = i % (D / 32);
                if constexpr (F8) {
                    const u32x2 w = __builtin_bit_cast(u32x2, read_tr8((vb ^ (dt << 5)) + (32 * sub + 16 * ks) * L::ROWB));
                    f[i % AHEAD].x = w.x;
                    f[i % AHEAD].y = w.y;
                } else {
                    const uint32_t at = (vb ^ (dt << 6)) + (32 * sub + 16 * ks) * L::ROWB;
                    const u32x2 lo = __builtin_bit_cast(u32x2, read_tr16(at)), hi = __builtin_bit_cast(u32x2, read_tr16(at + 8 * L::ROWB));
                    f[i % AHEAD] = u32x4{lo.x, lo.y, hi.x, hi.y};
                }
            };
            // S^T of the 32 keys `sub` of the tile at kb; NEXT: the first
            // fragments of V's keys `vsub` follow
            auto qk = [&](uint32_t kb, auto sub_, auto next_, uint32_t vb, auto vsub_) {
                constexpr int sub = decltype(sub_)::value, vsub = decltype(vsub_)::value;
                constexpr bool NEXT = decltype(next_)::value;
#pragma unroll
                for (int i = 0; i < NK; ++i) {
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
                        const u32x4 w = f[i % AK];
                        const u32x4 k = F8 ? __builtin_bit_cast(u32x4, e ? codes8_bf16(w.z, w.w) : codes8_bf16(w.x, w.y)) : w;
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) {
                            if (i + e == 0) mfma_first(st[rb], k, qf[rb][0]);
                            else mfma_s(st[rb], k, qf[rb][PER * i + e]);
                        }
                    }
                    if (i + AK < NK) {
                        load_k(kb, sub, i + AK);
                    } else if constexpr (NEXT) {
                        load_v(vb, vsub, i + AK - NK);
                        if (i == NK - 1)
#pragma unroll
                            for (int j = AK; j < AHEAD; ++j) load_v(vb, vsub, j);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            // PV: O += P V of the last step (keys `sub` of the tile whose V is at
            // vb).  SM: the weights of this step (32 keys from key0), each stage
            // (scores less the maximum, 2^x, sums and packing) written a group
            // behind the one before, so that no instruction waits on the last
            // one's result; the compiler keeps the stages' order, not their
            // places between the MFMAs.  The first fragments of K's keys `ksub`
            // at kb follow.
            // each(i): what else goes out with group i.
            auto weigh = [&](auto pv_, auto sm_, uint32_t vb, auto sub_, int key0, uint32_t kb, auto ksub_, auto each) {
                constexpr bool PV = decltype(pv_)::value, SM = decltype(sm_)::value;
                constexpr int sub = decltype(sub_)::value, ksub = decltype(ksub_)::value;
                // groups: the row maxima, the test of them, the first weights and
                // over how many groups their first stage is spread
                constexpr int TOP = NV > 8 ? 2 : 1, TEST = TOP + 1, FIRST = TEST + (NV > 4 ? 1 : 0);
                constexpr int SPREAD = NV - FIRST > 2 ? NV - FIRST - 2 : 1;
                u32x4 pn[RB][2];
                float ms[RB], f_m[RB], top[RB];
                bool moved = false;
                auto stage = [&](int i, int which) {
#pragma unroll
                    for (int x = 0; x < 8 * RB; ++x)
                        if (x * SPREAD / (8 * RB) == i) {
                            const int rb = x % RB, j = 2 * (x / RB);
                            if (which == 0) {
                                st[rb][j] = __builtin_fmaf(st[rb][j], c, -ms[rb]);
                                st[rb][j + 1] = __builtin_fmaf(st[rb][j + 1], c, -ms[rb]);
                            } else if (which == 1) {
                                st[rb][j] = exp2_fast(st[rb][j]);
                                st[rb][j + 1] = exp2_fast(st[rb][j + 1]);
                            } else {
                                l[rb] += st[rb][j] + st[rb][j + 1];
                                pn[rb][j >> 3][(j & 7) >> 1] = pack_bf16x2(f32x2{st[rb][j], st[rb][j + 1]});
                            }
                        }
                };
                if constexpr (!PV) {
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(st[rb]));
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if constexpr (PV) {
                        const int ks = i / (D / 32), dt = i % (D / 32);
                        const u32x4 w = f[i % AHEAD];
                        const u32x4 v = F8 ? __builtin_bit_cast(u32x4, codes8_bf16(w.x, w.y)) : w;
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) mfma_o(o[rb][dt], v, pw[rb][ks]);
                        if (i + AHEAD < NV) load_v(vb, sub, i + AHEAD);
                    }
                    if (i + AHEAD >= NV && i + AHEAD - NV < AK) load_k(kb, ksub, i + AHEAD - NV);
                    each(i);
                    if constexpr (SM) {
                        if (i == 1) {
                            // four (RB 1: two, and the waits) MFMAs after the last one that wrote S
                            if constexpr (PV) {
                                if constexpr (RB == 1) asm volatile("s_nop 7" : "+v"(st[0]));
#pragma unroll
                                for (int rb = 0; rb < RB; ++rb) asm volatile("" : "+v"(st[rb]));
                            }
                            if (key0 + 32 > open) {
#pragma unroll
                                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                                    for (int j = 0; j < 16; ++j)
                                        if (key0 + 8 * (j >> 2) + 4 * half + (j & 3) >= lim[rb]) st[rb][j] = -__builtin_inff();
                            }
                        }
                        if (i == TOP) {
#pragma unroll
                            for (int rb = 0; rb < RB; ++rb) {
                                top[rb] = st[rb][0];
#pragma unroll
                                for (int j = 1; j < 16; ++j) top[rb] = fmaxf(top[rb], st[rb][j]);
                                f_m[rb] = 1.0f;
                            }
                        }
                        if (i == TEST) {
                            moved = __any(top[0] * c > m[0] + kLazy || top[RB - 1] * c > m[RB - 1] + kLazy);
                            if (moved) {
#pragma unroll
                                for (int rb = 0; rb < RB; ++rb) {
                                    const float t = fmaxf(top[rb], __shfl_xor(top[rb], 32, 64));
                                    const float mn = fmaxf(m[rb], t * c);
                                    f_m[rb] = m[rb] == -__builtin_inff() ? 0.0f : exp2_fast(m[rb] - mn);
                                    m[rb] = mn;
                                    l[rb] *= f_m[rb];
                                }
                            }
#pragma unroll
                            for (int rb = 0; rb < RB; ++rb) ms[rb] = m[rb] == -__builtin_inff() ? 0.0f : m[rb];
                        }
                        if (i >= FIRST) {
                            stage(i - FIRST, 0);
                            stage(i - FIRST - 1, 1);
                            stage(i - FIRST - 2, 2);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (SM) {
#pragma unroll
                    for (int i = NV; i < FIRST + SPREAD + 2; ++i) {
                        stage(i - FIRST, 0);
                        stage(i - FIRST - 1, 1);
                        stage(i - FIRST - 2, 2);
                    }
                    if (PV && moved) {
                        drain(o);
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                            for (int dt = 0; dt < D / 32; ++dt) {
                                // one tile at a time through the vector registers
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[rb][dt][j] *= f_m[rb];
                                asm volatile("s_nop 7" : "+a"(o[rb][dt]));
                                __builtin_amdgcn_sched_barrier(0);
                            }
                    }
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        pw[rb][0] = pn[rb][0];
                        pw[rb][1] = pn[rb][1];
                    }
                }
            };
            std::integral_constant<int, 0> sub0;
            std::integral_constant<int, 1> sub1;
            std::bool_constant<true> yes;
            std::bool_constant<false> no;
            auto nothing = [](int) {};

            wait_vm<W == 4 ? 2 * L::NI : 0>();  // K of the first tile
            __syncthreads();
            const uint32_t kb0 = k_lane + (k0 & 1) * L::HALF;
#pragma unroll
            for (int i = 0; i < AK; ++i) load_k(kb0, 0, i);
            qk(kb0, sub0, no, 0, sub0);
            weigh(no, yes, 0, sub0, k0 * kBN, kb0, sub1, nothing);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int dt = 0; dt < D / 32; ++dt) clear(o[rb][dt]);
            int t = k0;
#pragma unroll 1
            for (;;) {
                const uint32_t vb = v_lane + (t & 1) * L::HALF, kb = k_lane + (t & 1) * L::HALF;
                const uint32_t kn = k_lane + ((t + 1) & 1) * L::HALF;
                qk(kb, sub1, no, 0, sub0);
                wait_vm<0>();
                __syncthreads();
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) load_v(vb, 0, i);
                const int id = __builtin_amdgcn_readfirstlane(id2);
                const Part pk = part_of(a.k, t + 2, id, false), pv = part_of(a.v, t + 1, id1, true);
                id1 = id;
                weigh(yes, yes, vb, sub0, t * kBN + 32, kn, sub0, [&](int i) {
#pragma unroll
                    for (int x = 0; x < 2 * L::NI; ++x)
                        if (x * NV / (2 * L::NI) == i && (x < L::NI ? of_k : of_v)) bring(x < L::NI ? pk : pv, x % L::NI, x >= L::NI);
                });
                id2 = page_of(t + 3);  // read behind the next wait
                if (++t == k1) break;
                qk(kn, sub0, yes, vb, sub1);
                weigh(yes, yes, vb, sub1, t * kBN, kn, sub1, nothing);
            }
            const uint32_t vb_last = v_lane + ((k1 - 1) & 1) * L::HALF;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) load_v(vb_last, 1, i);
            weigh(yes, no, vb_last, sub1, 0, kb0, sub0, nothing);
            wait_vm<0>();
            drain(o);
            if (a.causal) {
                // keys of the piece that the tile's first row may not see, by all waves
                const int open0 = min(max(ctx + r0 / a.G + 1, 0), s.len);
                if (odd_values<D, F8>(a, table, cur.hk, max(open0, k0 * kBN), min(s.len, k1 * kBN), wave, W))
                    *bad_of(a.ws, group, wave) = 1;
            }

            // A whole unit goes through its slot as well (the last piece's, not
            // yet in use): with O out of the registers its rows' gates can all
            // be in flight, each thread reading back what it wrote.
            const bool whole = k0 == 0 && k1 == nkt;
            float* part = Partial<kBM, D>::at(a.ws, group, k0 == 0);
            f32x4* mine = reinterpret_cast<f32x4*>(part) + wave * RB * D / 8 * 64 + lane;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int row = row0 + 32 * rb + col;
                l[rb] += __shfl_xor(l[rb], 32, 64);
                if (row0 < nr) {
#pragma unroll
                    for (int dt = 0; dt < D / 32; ++dt) {
#pragma unroll
                        for (int b = 0; b < 4; ++b)
                            mine[((rb * D / 32 + dt) * 4 + b) * 64] =
                                f32x4{o[rb][dt][4 * b], o[rb][dt][4 * b + 1], o[rb][dt][4 * b + 2], o[rb][dt][4 * b + 3]};
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (half == 0 && !whole) {
                        part[(int64_t)kBM * D + row] = m[rb];
                        part[(int64_t)kBM * D + kBM + row] = l[rb];
                    }
                }
            }
            if (whole) {
                asm volatile("" ::: "memory");
#pragma unroll 1
                for (int rb = 0; rb < RB; ++rb) {
                    const int row = row0 + 32 * rb + col, flat = r0 + min(row, nr - 1), tok = s.off + flat / a.G;
                    const int64_t head = cur.hk * a.G + flat % a.G;
                    const float sum = rb ? l[RB - 1] : l[0], vs = F8 ? a.v_scale[cur.hk] : 1.0f;
                    finish_row<D>(a, mine + rb * D / 8 * 64, sum == 0.0f ? 0.0f : vs / sum, a.gate + tok * a.g_tok + head * a.g_head + 4 * half,
                               a.out + tok * a.o_tok + head * a.o_head + 4 * half, row < nr);
                }
            }
            __syncthreads();
        }
        if (last) return;
        cur.kt = 0;
        if (++cur.r >= R) {
            cur.r = 0;
            if (++cur.hk >= a.HK) {
                cur.hk = 0;
                do {
                    if (++cur.b >= a.B) return;
                    s = paged_seq(a, cur.b);
                } while (s.n == 0);
            }
        }
    }
}

}  // namespace

namespace {

constexpr int kFewJoin = 2 * kGroups, kTileJoin = 8 * kGroups;  // workgroups

// The joins of a mixed batch: the first workgroups the few-rows kernel's.
template <int D, bool F8>
__global__ __launch_bounds__(256) void join_mixed_kernel(PagedAttention few, PagedAttention a) {
    if (blockIdx.x < kFewJoin)
        join<kMixedRows, D, F8, 4, FewOrder<D>>(few, blockIdx.x, kFewJoin);
    else
        join<kBM, D, F8, 1, TileOrder<D>>(a, blockIdx.x - kFewJoin, kTileJoin);
}

template <int D, bool F8, int RB>
hipError_t run(const PagedAttention& a, const PagedAttention* few, hipStream_t stream) {
    constexpr int LDS = std::max<int>(Tile<D, F8>::LDS, PagedSplit<kBM, kBN, 0>::lds_bytes(kPagedMaxRequests));
    auto* kern = tile_kernel<D, F8, RB>;
    static OncePerDevice once;
    const hipError_t attr = allow_lds(once, reinterpret_cast<const void*>(kern), LDS);
    if (attr != hipSuccess) return attr;
    hipLaunchKernelGGL(kern, dim3(kGroups), dim3(64 * kBM / (32 * RB)), LDS, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (few)
        hipLaunchKernelGGL((join_mixed_kernel<D, F8>), dim3(kFewJoin + kTileJoin), dim3(256), 0, stream, *few, a);
    else
        hipLaunchKernelGGL((join_kernel<kBM, D, F8, 1, TileOrder<D>>), dim3(kTileJoin), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_tile(const PagedAttention& a, const PagedAttention* few, int D, bool fp8, hipStream_t stream) {
    if (D == 64) return fp8 ? run<64, true, 1>(a, few, stream) : run<64, false, 1>(a, few, stream);
    if (D == 128) return fp8 ? run<128, true, 1>(a, few, stream) : run<128, false, 1>(a, few, stream);
    return fp8 ? run<256, true, 2>(a, few, stream) : run<256, false, 2>(a, few, stream);
}

static int64_t ws_floats(int D, int64_t bm) { return kBeginFloats + 2 * kGroups * (bm * D + 2 * bm); }

}  // namespace attn

size_t paged_attention_ws_bytes(int D, int64_t max_rows) {
    using namespace attn;
    return (size_t)4 * (max_rows <= 16         ? ws_floats(D, 16)
                        : max_rows <= kFewRows ? ws_floats(D, 32)
                                               : ws_floats(D, kTileRows) + ws_floats(D, kMixedRows));
}

// Either kernel computes any number of rows; the rule is what each is fast at
// (heads of 256, 12/2, BF16 cache; few against tile, us: 60000 keys, 48 rows 57
// and 81, 96 rows 78 and 83, 192 rows 128 and 85; 16 requests of 4000 keys, 48
// rows 61 and 65, 66 rows 89 and 67).  Where some request may have more than
// kFewRows rows, a batch is computed in two: a request of a few rows in a
// 256-row tile streams its keys at the pace of one wave's steps (13 requests,
// three of them chunks of 400 to 700 tokens, 32/8 heads of 128: 153 us in two
// against 165).  One launch joins both kernels' partial sums: two cost 6 us more.
hipError_t launch_paged_attention(PagedAttention a, int D, bool fp8, int64_t max_rows, hipStream_t stream) {
    a.rows_from = 0;
    a.rows_to = INT64_MAX;
    if (max_rows <= attn::kFewRows) return attn::launch_few(a, D, fp8, (int)max_rows, true, stream);
    if (a.B == 1) return attn::launch_tile(a, nullptr, D, fp8, stream);
    PagedAttention few = a;
    few.rows_to = attn::kFewRows;
    few.ws = a.ws + attn::ws_floats(D, attn::kTileRows);
    const hipError_t e = attn::launch_few(few, D, fp8, attn::kFewRows, false, stream);
    if (e != hipSuccess) return e;
    a.rows_from = attn::kFewRows;
    return attn::launch_tile(a, &few, D, fp8, stream);
}

}  // namespace fp8lin
