// Attention of many rows per request and kv head: prompts and their chunks.
// Bound by the matrix cores and by what feeds them.  A workgroup of W waves
// holds 32 W rows (consecutive tokens, the G query heads of a kv head side by
// side), each wave 32 of them with its queries and its part of O in registers,
// and walks the keys in tiles of 64 that all waves read from LDS (two buffers:
// the next tile arrives while one is computed, one barrier per tile).
//
// Per 32 keys, MFMA 32x32x16: S^T [keys, rows] = K Q^T leaves 4 consecutive
// keys of one row in a lane's registers, which is what the second product
// O^T [D, rows] += V^T P^T takes as its B operand; V^T comes from the
// transposing LDS reads, its keys in the same order.  So a row's maximum and
// sum stay in one lane pair and nothing passes through LDS between the
// products.
//
// BF16 caches go to LDS by direct DMA; the codes of an 8-bit cache through
// registers, converted once per workgroup on the way, so that the products see
// the same layout.
#include <algorithm>

#include "attention.hpp"

namespace fp8lin {
namespace attn {
namespace {

constexpr int kTileKeys = 64;
constexpr int kTileMinTiles = 4;
constexpr int kTileStart = 128;  // a unit's start and end, in keys
constexpr int kTileWaves = 8;

template <int D>
struct Tile {
    static constexpr int ROWB = 2 * D;               // bytes of a key in LDS
    static constexpr int HALF = kTileKeys * ROWB;    // K or V of a tile
    static constexpr int BUF = 2 * HALF;
    static constexpr int LDS = 2 * BUF;
    // chunk (16 bytes) permutations, as in attention_few.hip: 16 keys at one
    // chunk (K), 4 keys of 64 bytes (V)
    static __device__ __forceinline__ int xk(int r) { return ROWB >= 256 ? r & 15 : (r >> 1) & 7; }
    static __device__ __forceinline__ int xv(int r) { return ROWB >= 256 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }
};

template <int D, bool F8, int W>
__global__ __launch_bounds__(64 * W, 1) void tile_kernel(PagedAttention a) {
    using L = Tile<D>;
    constexpr int BM = 32 * W, KEYS = kTileKeys / W;  // keys that a wave brings of each tile
    using Split = PagedSplit<BM, kTileKeys, kTileStart>;
    extern __shared__ __align__(1024) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5, col = lane & 31;

    int64_t* pre = reinterpret_cast<int64_t*>(lds);
    Split::prefix(a, pre, 64 * W);
    const int64_t total = pre[a.B], chunk = Split::chunk(a, total, gridDim.x, kTileMinTiles);
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
        begin[1] = i32x4v{s.off, (int)min((int64_t)BM, (int64_t)s.n * a.G - (int64_t)cur.r * BM), 0, 0};
    }
    __syncthreads();
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;

    for (;;) {
        const int R = Split::tiles(a, s);
        const int nkt = R ? Split::key_tiles(a, s, cur.r) : 0;
        const bool last = cur.b == end.b && cur.hk == end.hk && cur.r == end.r;
        const int k0 = cur.kt, k1 = last ? end.kt : nkt;
        if (R && k1 > k0) {
            const int r0 = cur.r * BM, nr = (int)min((int64_t)BM, (int64_t)s.n * a.G - r0);
            const float c = a.scale2 * (F8 ? a.k_scale[cur.hk] : 1.0f);
            const int row = 32 * wave + col, flat = r0 + row, tok = flat / a.G;
            const bool ok = row < nr;
            const bool busy = 32 * wave < nr;
            bf16x8 qf[D / 16];  // B operand: row col, dimensions 16 t + 8 half ..
            {
                const uint16_t* q = a.q + (int64_t)(s.off + (ok ? tok : 0)) * a.q_tok + (int64_t)(cur.hk * a.G + flat % a.G) * a.q_head;
                load_queries<D / 16>(q, qf, [&](int t) { return 16 * t + 8 * half; });
            }
            const int ctx = s.len - s.n;
            const int lim = !ok ? 0 : a.causal ? min(max(ctx + tok + 1, 0), s.len) : s.len;
            // keys that the wave's first and last row may see
            const int wave_last = min(r0 + 32 * wave + 32, r0 + nr) - 1;
            const int open = a.causal ? min(max(ctx + (r0 + 32 * wave) / a.G + 1, 0), s.len) : s.len;
            const int close = !busy ? 0 : a.causal ? min(max(ctx + wave_last / a.G + 1, 0), s.len) : s.len;
            f32x16 o[D / 32];
            float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;

            const int32_t* table = a.table + (int64_t)cur.b * a.ldt;
            // page id of the keys that this wave brings of tile t
            auto page_of = [&](int t) {
                const int64_t key = (int64_t)t * kTileKeys + KEYS * wave;
                return t < k1 && key < s.len ? table[key >> a.page_bits] : -1;
            };
            struct Src {
                const char* base;
                uint32_t bytes;
            };
            auto source = [&](const PagedCache& cache, int t, int id) {
                constexpr int ES = F8 ? 1 : 2;
                const int64_t key = (int64_t)t * kTileKeys + KEYS * wave;
                const int there = t < k1 && (unsigned)id < (unsigned)a.pages ? (int)min((int64_t)s.len - key, (int64_t)KEYS) : 0;
                const int64_t at = (int64_t)id * cache.page + (key & ((1 << a.page_bits) - 1)) * cache.slot + cur.hk * cache.head;
                Src r;
                r.bytes = there > 0 ? (uint32_t)(((there - 1) * cache.slot + D) * ES) : 0;
                r.base = static_cast<const char*>(cache.data) + (r.bytes ? at * ES : 0);
                return r;
            };
            // BF16: both halves of tile t into buffer t & 1 by DMA
            auto bring = [&](int t, int id) {
                constexpr int RPI = 1024 / L::ROWB, LPR = 64 / RPI;
#pragma unroll
                for (int is_v = 0; is_v < 2; ++is_v) {
                    const PagedCache& cache = is_v ? a.v : a.k;
                    const Src src = source(cache, t, id);
                    const i32x4 desc = make_desc(src.base, src.bytes);
#pragma unroll
                    for (int i = 0; i < KEYS / RPI; ++i) {
                        const int r = i * RPI + lane / LPR, rt = KEYS * wave + r;
                        const int ch = (lane % LPR) ^ (is_v ? L::xv(rt) : L::xk(rt));
                        const uint32_t m0 = lds0 + (t & 1) * L::BUF + is_v * L::HALF + (KEYS * wave + i * RPI) * L::ROWB;
                        dma<false>(__builtin_amdgcn_readfirstlane(m0), (uint32_t)(r * (int)cache.slot * 2 + ch * 16), desc);
                    }
                }
            };
            // 8-bit: 16 codes per lane and load, KEYS rows of D codes
            constexpr int NL = F8 ? (KEYS * D + 1023) / 1024 : 1, LPR8 = D / 16;
            u32x4 code[2][NL];
            auto fetch = [&](int t, int id) {
#pragma unroll
                for (int is_v = 0; is_v < 2; ++is_v) {
                    const PagedCache& cache = is_v ? a.v : a.k;
                    const Src src = source(cache, t, id);
                    const rsrc_t rsrc = make_rsrc(src.base, src.bytes);
#pragma unroll
                    for (int i = 0; i < NL; ++i) {
                        const int r = (i * 64 + lane) / LPR8, ch = lane % LPR8;
                        code[is_v][i] = buf_load16<0>(rsrc, r < KEYS ? (uint32_t)(r * (int)cache.slot + ch * 16) : kBufferOob);
                    }
                }
            };
            auto put = [&](int t) {
#pragma unroll
                for (int is_v = 0; is_v < 2; ++is_v)
#pragma unroll
                    for (int i = 0; i < NL; ++i) {
                        const int r = (i * 64 + lane) / LPR8, ch = 2 * (lane % LPR8), rt = KEYS * wave + r;
                        const int x = is_v ? L::xv(rt) : L::xk(rt);
                        uint8_t* at = lds + (t & 1) * L::BUF + is_v * L::HALF + rt * L::ROWB;
                        if (KEYS * D >= 1024 || r < KEYS) {
                            const u32x4 w = code[is_v][i];
                            *reinterpret_cast<bf16x8*>(at + ((ch ^ x) << 4)) = codes8_bf16(w.x, w.y);
                            *reinterpret_cast<bf16x8*>(at + (((ch + 1) ^ x) << 4)) = codes8_bf16(w.z, w.w);
                        }
                    }
            };

            int id = __builtin_amdgcn_readfirstlane(page_of(k0));
            if constexpr (F8) {
                fetch(k0, id);
                put(k0);
            } else {
                bring(k0, id);
            }
            id = page_of(k0 + 1);
#pragma unroll 1
            for (int t = k0; t < k1; ++t) {
                if constexpr (F8) {
                    __syncthreads();
                    fetch(t + 1, __builtin_amdgcn_readfirstlane(id));
                } else {
                    wait_vm<0>();
                    __syncthreads();
                    bring(t + 1, __builtin_amdgcn_readfirstlane(id));
                }
                id = page_of(t + 2);
                const uint32_t kb = lds0 + (t & 1) * L::BUF, vb = kb + L::HALF;
#pragma unroll
                for (int sub = 0; sub < kTileKeys / 32; ++sub) {
                    const int key0 = t * kTileKeys + 32 * sub;
                    if (key0 >= close) continue;
                    f32x16 st;
#pragma unroll
                    for (int i = 0; i < 16; ++i) st[i] = 0.0f;
                    const int kr = 32 * sub + col;
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        const bf16x8 kf = __builtin_bit_cast(
                            bf16x8, read16(kb + kr * L::ROWB + (((2 * d + half) ^ L::xk(kr)) << 4)));
                        st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[d], st, 0, 0, 0);
                    }
                    if (key0 + 32 > open) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (key0 + 8 * (i >> 2) + 4 * half + (i & 3) >= lim) st[i] = -__builtin_inff();
                    }
                    float top = st[0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) top = fmaxf(top, st[i]);
                    if (__any(top * c > m + kLazy)) {
                        top = fmaxf(top, __shfl_xor(top, 32, 64));
                        const float mn = fmaxf(m, top * c);
                        const float f = m == -__builtin_inff() ? 0.0f : exp2_fast(m - mn);
                        m = mn;
                        l *= f;
#pragma unroll
                        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[dt][i] *= f;
                    }
                    const float ms = m == -__builtin_inff() ? 0.0f : m;
                    u32x4 pw[2];
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float x = exp2_fast(__builtin_fmaf(st[i], c, -ms));
                        const float y = exp2_fast(__builtin_fmaf(st[i + 1], c, -ms));
                        l += x + y;
                        pw[i >> 3][(i & 7) >> 1] = pack_bf16x2(f32x2{x, y});
                    }
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        // keys 16 ks + 4 half + 0..3 and the same + 8, of dimension 32 dt + col
                        const int vr = 32 * sub + 16 * ks + 4 * half + ((lane & 15) >> 2);
                        const int ch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), by = 8 * (lane & 1);
#pragma unroll
                        for (int dt = 0; dt < D / 32; ++dt) {
                            const s16x4 lo = read_tr16(vb + vr * L::ROWB + (((4 * dt + ch) ^ L::xv(vr)) << 4) + by);
                            const s16x4 hi = read_tr16(vb + (vr + 8) * L::ROWB + (((4 * dt + ch) ^ L::xv(vr + 8)) << 4) + by);
                            typedef short s16x8 __attribute__((ext_vector_type(8)));
                            const s16x8 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vf),
                                                                            __builtin_bit_cast(bf16x8, pw[ks]), o[dt], 0, 0, 0);
                        }
                    }
                }
                if constexpr (F8) put(t + 1);
            }
            if constexpr (!F8) wait_vm<0>();
            l += __shfl_xor(l, 32, 64);

            if (k0 == 0 && k1 == nkt) {
                __syncthreads();
                store_tile<D>(a, reinterpret_cast<float*>(lds + wave * store_bytes<D>()), o,
                              l == 0.0f ? 0.0f : (F8 ? a.v_scale[cur.hk] : 1.0f) / l, s.off, cur.hk, r0 + 32 * wave, nr - 32 * wave);
            } else if (busy) {
                float* part = Partial<BM, D>::at(a.ws, group, k0 == 0);
#pragma unroll
                for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        *reinterpret_cast<f32x4*>(part + 4 * (((wave * (D / 32) + dt) * 4 + b) * 64 + lane)) =
                            f32x4{o[dt][4 * b], o[dt][4 * b + 1], o[dt][4 * b + 2], o[dt][4 * b + 3]};
                if (half == 0) {
                    part[(int64_t)BM * D + row] = m;
                    part[(int64_t)BM * D + BM + row] = l;
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

template <int D, bool F8, int W>
hipError_t run(const PagedAttention& a, hipStream_t stream) {
    constexpr int BM = 32 * W, LDS = std::max<int>({Tile<D>::LDS, PagedSplit<BM, kTileKeys, 0>::lds_bytes(kPagedMaxRequests), W * store_bytes<D>()});
    auto* kern = tile_kernel<D, F8, W>;
    static const hipError_t attr =
        hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (attr != hipSuccess) return attr;
    hipLaunchKernelGGL(kern, dim3(kGroups), dim3(64 * W), LDS, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    auto* join = join_kernel<BM, D, 1, TileOrder<D>>;
    hipLaunchKernelGGL(join, dim3(8 * kGroups), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_tile(const PagedAttention& a, int D, bool fp8, hipStream_t stream) {
    if (D == 64) return fp8 ? run<64, true, kTileWaves>(a, stream) : run<64, false, kTileWaves>(a, stream);
    if (D == 128) return fp8 ? run<128, true, kTileWaves>(a, stream) : run<128, false, kTileWaves>(a, stream);
    return fp8 ? run<256, true, kTileWaves>(a, stream) : launch_wide(a, stream);
}

}  // namespace attn

namespace {
constexpr int kFewRows = 64;  // rows that the few-rows kernel takes; see launch_paged_attention
}

size_t paged_attention_ws_bytes(int D, int64_t max_rows) {
    const int64_t bm = max_rows <= 16 ? 16 : max_rows <= 32 ? 32 : max_rows <= kFewRows ? 64 : 32 * attn::kTileWaves;
    return (size_t)(4 * (attn::kBeginFloats + 2 * attn::kGroups * (bm * D + 2 * bm)));
}

// Either kernel computes any number of rows; the rule is what each is fast at.
hipError_t launch_paged_attention(const PagedAttention& a, int D, bool fp8, int64_t max_rows, hipStream_t stream) {
    if (max_rows <= kFewRows) return attn::launch_few(a, D, fp8, (int)max_rows, stream);
    return attn::launch_tile(a, D, fp8, stream);
}

}  // namespace fp8lin
