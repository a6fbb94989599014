// Attention of many rows per request and kv head over a BF16 cache with heads
// of 256: what attention_tile.hip computes, for the shape whose accumulators
// fill the register file.
//
// A head of 256 makes 8 KB of K and V per key tile feed only 32 rows' products
// per wave in the general kernel: every MFMA needs its own 1 KB from LDS,
// which is all that LDS delivers.  Here a wave holds 64 rows (4 waves, one per
// SIMD, 512 registers each), so a K or V fragment serves two MFMAs:
//   256 accumulation registers: O^T, 2 x 8 tiles of 32 x 32
//   128 registers: the queries; 32: S^T of 32 keys; 32: two steps' weights
// With one wave per SIMD nothing else hides the softmax, so the steps of 32
// keys are skewed: the products of step s - 1 with V run while the weights of
// step s are computed, a few vector instructions after each pair of MFMAs.
// The MFMAs are one asm statement each, in that order, with O in accumulation
// and S in vector registers; the compiler keeps the order of the groups
// (sched_barrier) and counts the LDS waits.
//
// K and V of a tile of 64 keys arrive by direct-to-LDS DMA into two buffers
// each.  One barrier per tile, between its last product with K and its first
// with V: there K of the next tile and V of this one have arrived, and K of
// this tile and V of the last one are no longer read, so the DMAs of the tiles
// after go out.
#include <algorithm>

#include "attention.hpp"

namespace fp8lin {
namespace attn {
namespace {

constexpr int kD = 256, kW = 4, kRB = 2, kBM = 32 * kRB * kW, kBN = 64, kRow = 2 * kD;
constexpr int kHalf = kBN * kRow;  // K or V of a tile
constexpr int kWideLds = 4 * kHalf;
constexpr int kWideStart = 256;    // a unit's start and end (16 us) in keys (64 in 4 us)
constexpr int kWideMinTiles = 4;

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
__device__ __forceinline__ void drain(f32x16 (&o)[kRB][kD / 32]) {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" : "+a"(o[0][0]));
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
        for (int dt = 0; dt < kD / 32; ++dt)
            if (rb | dt) asm volatile("" : "+a"(o[rb][dt]));
}
__device__ __forceinline__ void clear(f32x16& o) {
    const u32x4 zero = {0, 0, 0, 0};
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "=a"(o) : "v"(zero));
}

// The lane's 8 D / 64 groups of 4 values of a row, 64 f32x4 apart, divided by
// the sum of weights, gated, to out: group i is dimensions 8 i ..
__device__ __forceinline__ void finish_row(const PagedAttention& a, const f32x4* o, float l, const uint16_t* gate, uint16_t* out,
                                           bool ok) {
    constexpr int N = kD / 16;
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
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = l == 0.0f ? 0.0f : x[i][j] * inv;
        if (a.gate) apply_gates<N>(x, g);
        if (ok) {
#pragma unroll
            for (int i = 0; i < N; ++i) store_bf16x4(out + 8 * (i0 + i), x[i]);
        }
    }
}

__device__ __forceinline__ int xk(int r) { return r & 15; }
__device__ __forceinline__ int xv(int r) { return (r & 3) << 2; }

__global__ __launch_bounds__(64 * kW, 1) void wide_kernel(PagedAttention a) {
    using Split = PagedSplit<kBM, kBN, kWideStart>;
    constexpr int KEYS = kBN / kW;  // keys that a wave brings of each tile
    extern __shared__ __align__(1024) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5, col = lane & 31;

    int64_t* pre = reinterpret_cast<int64_t*>(lds);
    Split::prefix(a, pre, 64 * kW);
    const int64_t total = pre[a.B], chunk = Split::chunk(a, total, gridDim.x, kWideMinTiles);
    const int group = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int64_t p0 = group * chunk, p1 = min(p0 + chunk, total);
    i32x4v* begin = reinterpret_cast<i32x4v*>(a.ws) + 2 * group;
    if (p0 >= total) {
        if (tid == 0) begin[0] = i32x4v{-1, 0, 0, 0};
        return;
    }
    typename Split::Loc cur, end;
    Split::piece(a, pre, p0, p1, cur, end);
    PagedSeq s = paged_seq(a, cur.b);
    if (tid == 0) {
        begin[0] = i32x4v{cur.b, cur.hk, cur.r, cur.kt};
        begin[1] = i32x4v{s.off, (int)min((int64_t)kBM, (int64_t)s.n * a.G - (int64_t)cur.r * kBM), 0, 0};
    }
    __syncthreads();
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
    // K of tile t at (t & 1) kHalf, V behind both
    // LDS addresses of this lane's reads within a tile: a chunk is picked by an
    // exclusive or of the bits above, a key by an offset
    const uint32_t k_lane = lds0 + col * kRow + ((half ^ xk(col)) << 4);
    const int vr = 4 * half + ((lane & 15) >> 2);
    const uint32_t v_lane = lds0 + 2 * kHalf + vr * kRow + (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ xv(vr)) << 4) +
                            8 * (lane & 1);

    for (;;) {
        const int R = Split::tiles(a, s);
        const int nkt = R ? Split::key_tiles(a, s, cur.r) : 0;
        const bool last = cur.b == end.b && cur.hk == end.hk && cur.r == end.r;
        const int k0 = cur.kt, k1 = last ? end.kt : nkt;
        if (R && k1 > k0) {
            const int r0 = cur.r * kBM, nr = (int)min((int64_t)kBM, (int64_t)s.n * a.G - r0);
            const float c = a.scale2;
            const int row0 = 32 * kRB * wave, ctx = s.len - s.n;
            const int32_t* table = a.table + (int64_t)cur.b * a.ldt;
            // page id of the keys that this wave brings of tile t
            auto page_of = [&](int t) {
                const int64_t key = (int64_t)t * kBN + KEYS * wave;
                const int id = table[min(key, (int64_t)max(s.len - 1, 0)) >> a.page_bits];
                return t < k1 && key < s.len ? id : -1;
            };
            auto bring = [&](const PagedCache& cache, int t, int id, bool is_v) {
                const int64_t key = (int64_t)t * kBN + KEYS * wave;
                const int there = (unsigned)id < (unsigned)a.pages ? (int)min((int64_t)s.len - key, (int64_t)KEYS) : 0;
                const int64_t at = (int64_t)id * cache.page + (key & ((1 << a.page_bits) - 1)) * cache.slot + cur.hk * cache.head;
                const uint32_t bytes = there > 0 ? (uint32_t)(((there - 1) * cache.slot + kD) * 2) : 0;
                const i32x4 desc = make_desc(static_cast<const char*>(cache.data) + (bytes ? at * 2 : 0), bytes);
                const uint32_t m0 = lds0 + (is_v ? 2 * kHalf : 0) + (t & 1) * kHalf + KEYS * wave * kRow;
#pragma unroll
                for (int i = 0; i < KEYS / 2; ++i) {
                    const int r = 2 * i + half;  // KEYS * wave is a multiple of 16: no part in xk, xv
                    const int ch = col ^ (is_v ? xv(r) : xk(r));
                    dma<false>(__builtin_amdgcn_readfirstlane(m0 + i * 1024), (uint32_t)(r * (int)cache.slot * 2 + ch * 16), desc);
                }
            };
            int id0 = page_of(k0), id1 = page_of(k0 + 1);

            bf16x8 qf[kRB][kD / 16];  // B operand: row 32 rb + col, dimensions 16 t + 8 half ..
            int lim[kRB];             // keys that the lane's row may see
#pragma unroll
            for (int rb = 0; rb < kRB; ++rb) {
                const int row = row0 + 32 * rb + col, flat = r0 + row, tok = flat / a.G;
                const bool ok = row < nr;
                const uint16_t* q = a.q + (int64_t)(s.off + (ok ? tok : 0)) * a.q_tok + (int64_t)(cur.hk * a.G + flat % a.G) * a.q_head;
                load_queries<kD / 16>(q, qf[rb], [&](int t) { return 16 * t + 8 * half; });
                lim[rb] = !ok ? 0 : a.causal ? min(max(ctx + tok + 1, 0), s.len) : s.len;
            }
            // keys that the wave's first row may see: below it no mask
            const int open = a.causal ? min(max(ctx + (r0 + row0) / a.G + 1, 0), s.len) : s.len;

            id0 = __builtin_amdgcn_readfirstlane(id0);
            id1 = __builtin_amdgcn_readfirstlane(id1);
            bring(a.k, k0, id0, false);
            bring(a.k, k0 + 1, id1, false);
            bring(a.v, k0, id0, true);
            int id2 = page_of(k0 + 2);

            f32x16 o[kRB][kD / 32], st[kRB];
            u32x4 pw[kRB][2];  // weights of the step before, the B operand
            float m[kRB], l[kRB];
#pragma unroll
            for (int rb = 0; rb < kRB; ++rb) {
                m[rb] = -__builtin_inff();
                l[rb] = 0.0f;
            }

            // S^T of the 32 keys `sub` of the tile at kb
            auto qk = [&](uint32_t kb, auto sub_) {
                constexpr int sub = decltype(sub_)::value, AHEAD = 4;
                u32x4 f[AHEAD];
                auto load = [&](int d) {
                    return read16((kb ^ ((2 * d & 15) << 4)) + 32 * sub * kRow + (2 * d & ~15) * 16);
                };
#pragma unroll
                for (int d = 0; d < AHEAD; ++d) f[d] = load(d);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < kD / 16; ++d) {
                    if (d == 0) {
                        mfma_first(st[0], f[0], qf[0][0]);
                        mfma_first(st[1], f[0], qf[1][0]);
                    } else {
                        mfma_s(st[0], f[d % AHEAD], qf[0][d]);
                        mfma_s(st[1], f[d % AHEAD], qf[1][d]);
                    }
                    if (d + AHEAD < kD / 16) f[d % AHEAD] = load(d + AHEAD);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            // O += P V of the last step (keys `sub` of the tile whose V is at
            // vb) with PV, the weights of this step (32 keys from key0) with SM
            auto weigh = [&](auto pv_, auto sm_, uint32_t vb, auto sub_, int key0) {
                constexpr bool PV = decltype(pv_)::value, SM = decltype(sm_)::value;
                constexpr int sub = decltype(sub_)::value, AHEAD = 4, N = 2 * kD / 32;
                u32x4 f[AHEAD], pn[kRB][2];
                auto load = [&](int i) {
                    const int ks = i / (kD / 32), dt = i % (kD / 32);
                    const uint32_t at = (vb ^ (dt << 6)) + (32 * sub + 16 * ks) * kRow;
                    const s16x4 lo = read_tr16(at), hi = read_tr16(at + 8 * kRow);
                    return u32x4{__builtin_bit_cast(u32x2, lo).x, __builtin_bit_cast(u32x2, lo).y,
                                 __builtin_bit_cast(u32x2, hi).x, __builtin_bit_cast(u32x2, hi).y};
                };
                float ms[kRB], f_m[kRB];
                bool moved = false;
                if constexpr (PV) {
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i) f[i] = load(i);
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(st[0]), "+v"(st[1]));
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if constexpr (PV) {
                        const int ks = i / (kD / 32), dt = i % (kD / 32);
                        mfma_o(o[0][dt], f[i % AHEAD], pw[0][ks]);
                        mfma_o(o[1][dt], f[i % AHEAD], pw[1][ks]);
                        if (i + AHEAD < N) f[i % AHEAD] = load(i + AHEAD);
                    }
                    if constexpr (SM) {
                        if (i == 1) {
                            // four MFMAs after the last one that wrote S
                            if constexpr (PV) asm volatile("" : "+v"(st[0]), "+v"(st[1]));
                            if (key0 + 32 > open) {
#pragma unroll
                                for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
                                    for (int j = 0; j < 16; ++j)
                                        if (key0 + 8 * (j >> 2) + 4 * half + (j & 3) >= lim[rb]) st[rb][j] = -__builtin_inff();
                            }
                        }
                        if (i == 2) {
                            float top[kRB];
#pragma unroll
                            for (int rb = 0; rb < kRB; ++rb) {
                                top[rb] = st[rb][0];
#pragma unroll
                                for (int j = 1; j < 16; ++j) top[rb] = fmaxf(top[rb], st[rb][j]);
                                f_m[rb] = 1.0f;
                            }
                            moved = __any(top[0] * c > m[0] + kLazy || top[1] * c > m[1] + kLazy);
                            if (moved) {
#pragma unroll
                                for (int rb = 0; rb < kRB; ++rb) {
                                    const float t = fmaxf(top[rb], __shfl_xor(top[rb], 32, 64));
                                    const float mn = fmaxf(m[rb], t * c);
                                    f_m[rb] = m[rb] == -__builtin_inff() ? 0.0f : exp2_fast(m[rb] - mn);
                                    m[rb] = mn;
                                    l[rb] *= f_m[rb];
                                }
                            }
#pragma unroll
                            for (int rb = 0; rb < kRB; ++rb) ms[rb] = m[rb] == -__builtin_inff() ? 0.0f : m[rb];
                        }
                        if (i >= 3 && i < 15) {
                            // 16 pairs of weights over 12 groups: 1 or 2 each
#pragma unroll
                            for (int x = 0; x < 16; ++x)
                                if (x * 12 / 16 == i - 3) {
                                    const int rb = x >> 3, j = 2 * (x & 7);
                                    const float p = exp2_fast(__builtin_fmaf(st[rb][j], c, -ms[rb]));
                                    const float q = exp2_fast(__builtin_fmaf(st[rb][j + 1], c, -ms[rb]));
                                    l[rb] += p + q;
                                    pn[rb][j >> 3][(j & 7) >> 1] = pack_bf16x2(f32x2{p, q});
                                }
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (SM) {
                    if (PV && moved) {
                        drain(o);
#pragma unroll
                        for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
                            for (int dt = 0; dt < kD / 32; ++dt) {
                                // one tile at a time through the vector registers
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[rb][dt][j] *= f_m[rb];
                                asm volatile("s_nop 7" : "+a"(o[rb][dt]));
                                __builtin_amdgcn_sched_barrier(0);
                            }
                    }
#pragma unroll
                    for (int rb = 0; rb < kRB; ++rb) {
                        pw[rb][0] = pn[rb][0];
                        pw[rb][1] = pn[rb][1];
                    }
                }
            };
            std::integral_constant<int, 0> sub0;
            std::integral_constant<int, 1> sub1;
            std::bool_constant<true> yes;
            std::bool_constant<false> no;

            wait_vm<KEYS>();  // K of the first tile; KEYS / 2 DMAs per K or V
            __syncthreads();
            qk(k_lane + (k0 & 1) * kHalf, sub0);
            weigh(no, yes, 0, sub0, k0 * kBN);
#pragma unroll
            for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
                for (int dt = 0; dt < kD / 32; ++dt) clear(o[rb][dt]);
            int t = k0;
#pragma unroll 1
            for (;;) {
                const uint32_t vb = v_lane + (t & 1) * kHalf;
                qk(k_lane + (t & 1) * kHalf, sub1);
                wait_vm<0>();
                __syncthreads();
                const int id = __builtin_amdgcn_readfirstlane(id2);
                bring(a.k, t + 2, id, false);
                bring(a.v, t + 1, id1, true);
                id1 = id;
                id2 = page_of(t + 3);  // read behind the next wait
                weigh(yes, yes, vb, sub0, t * kBN + 32);
                if (++t == k1) break;
                qk(k_lane + (t & 1) * kHalf, sub0);
                weigh(yes, yes, vb, sub1, t * kBN);
            }
            weigh(yes, no, v_lane + ((k1 - 1) & 1) * kHalf, sub1, 0);
            wait_vm<0>();
            drain(o);

            // A whole unit goes through its slot as well (the last piece's, not
            // yet in use): with O out of the registers its rows' gates can all
            // be in flight, each thread reading back what it wrote.
            const bool whole = k0 == 0 && k1 == nkt;
            float* part = Partial<kBM, kD>::at(a.ws, group, k0 == 0);
            f32x4* mine = reinterpret_cast<f32x4*>(part) + wave * kRB * kD / 8 * 64 + lane;
#pragma unroll
            for (int rb = 0; rb < kRB; ++rb) {
                const int row = row0 + 32 * rb + col;
                l[rb] += __shfl_xor(l[rb], 32, 64);
                if (row0 < nr) {
#pragma unroll
                    for (int dt = 0; dt < kD / 32; ++dt) {
#pragma unroll
                        for (int b = 0; b < 4; ++b)
                            mine[((rb * kD / 32 + dt) * 4 + b) * 64] =
                                f32x4{o[rb][dt][4 * b], o[rb][dt][4 * b + 1], o[rb][dt][4 * b + 2], o[rb][dt][4 * b + 3]};
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (half == 0 && !whole) {
                        part[(int64_t)kBM * kD + row] = m[rb];
                        part[(int64_t)kBM * kD + kBM + row] = l[rb];
                    }
                }
            }
            if (whole) {
                asm volatile("" ::: "memory");
#pragma unroll 1
                for (int rb = 0; rb < kRB; ++rb) {
                    const int row = row0 + 32 * rb + col, flat = r0 + min(row, nr - 1), tok = s.off + flat / a.G;
                    const int64_t head = cur.hk * a.G + flat % a.G;
                    finish_row(a, mine + rb * kD / 8 * 64, rb ? l[1] : l[0], a.gate + tok * a.g_tok + head * a.g_head + 4 * half,
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

hipError_t launch_wide(const PagedAttention& a, hipStream_t stream) {
    constexpr int LDS = std::max<int>(kWideLds, PagedSplit<kBM, kBN, 0>::lds_bytes(kPagedMaxRequests));
    static const hipError_t attr =
        hipFuncSetAttribute(reinterpret_cast<const void*>(wide_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (attr != hipSuccess) return attr;
    hipLaunchKernelGGL(wide_kernel, dim3(kGroups), dim3(64 * kW), LDS, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((join_kernel<kBM, kD, 1, TileOrder<kD>>), dim3(8 * kGroups), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace attn
}  // namespace fp8lin
