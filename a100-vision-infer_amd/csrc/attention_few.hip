// Attention of a few rows per request and kv head: the decode step (G rows)
// and drafted tokens (up to kFewRows = 64 rows, in tiles of 16 or 32).  Bound by reading K and V
// once.  One workgroup of 4 waves per CU; every wave holds all the tile's rows
// and its own key tiles, which it brings into its own part of LDS by
// direct-to-LDS DMA, so that the stream needs no barrier between waves and no
// registers for loads in flight; the waves' sums are joined in LDS when a unit
// ends.  61 requests, 465 MB of 8-bit keys and values, 12/2 heads of 256: 86 us,
// 5.4 TB/s; 7 requests with drafts, 205 MB of BF16: 47 us, 4.4 TB/s.
//
// Per key tile (KT keys: 16, or 32 of an 8-bit cache), MFMA 16x16x32:
//   S^T [keys, rows] = K Q^T, so that a lane holds 4 consecutive keys of one
//   row, which is what the second product takes as its B operand without a
//   move across lanes:
//   O^T [D, rows] += V^T P^T, V^T read from LDS by the transposing reads.
// K and V rows lie in LDS as they are in the cache, their 16-byte chunks
// permuted by row so that the reads hit distinct banks; each DMA lane fetches
// the chunk that its LDS place holds.  Rows past the request's keys, and pages
// whose id is out of range, are read as zeros by the buffer's bounds check.
#include "attention.hpp"

namespace fp8lin {
namespace attn {
namespace {

constexpr int kFewWaves = 4;
constexpr int kFewMinTiles = 4;  // key tiles of the shortest piece, one per wave

template <int D, bool F8>
struct Few {
    static constexpr int KT = F8 ? 32 : 16;           // keys of a tile
    static constexpr int ROWB = D * (F8 ? 1 : 2);     // bytes of a key
    static constexpr int SLOT = KT * ROWB;            // K or V of a tile: 32 D bytes
    static constexpr int NI = SLOT / 1024;            // DMA instructions of a slot
    static constexpr int RPI = 1024 / ROWB;           // keys of an instruction
    static constexpr int LPR = 64 / RPI;              // its lanes per key
    static constexpr int DEPTH = 16384 / SLOT;        // tiles of a wave's ring
    static constexpr int WAVE = 2 * DEPTH * SLOT;     // 32 KB per wave
    static constexpr int LDS = kFewWaves * WAVE;      // 128 KB
    // What a unit's start and end cost, as keys that stream in that time: 5 us
    // (its queries and first tiles, the join) at a CU's 30 KB per us.
    static constexpr int START = 160 * 1024 / (2 * ROWB);
    static constexpr int IN_FLIGHT = (2 * DEPTH - 1) * NI;

    // Chunk permutations: 16 keys (K) at one chunk, or the keys of a
    // transposing read (V), must hit distinct 16- or 32-byte columns of the
    // 256 bytes that LDS serves at once.
    static __device__ __forceinline__ int xk(int r) {
        if constexpr (ROWB >= 256) return r & 15;
        if constexpr (ROWB == 128) return (r >> 1) & 7;
        return (r >> 2) & 3;
    }
    static __device__ __forceinline__ int xv(int r) {
        if constexpr (!F8) {
            if constexpr (ROWB >= 256) return (r & 7) << 1;
            return ((r >> 1) & 3) << 1;
        } else {
            if constexpr (ROWB >= 256) return (r & 7) | ((r >> 1) & 8);
            if constexpr (ROWB == 128) return ((r >> 1) & 3) | ((r >> 2) & 4);
            return ((r >> 2) & 1) | ((r >> 3) & 2);
        }
    }
};

template <int D, bool F8, int NT>
__global__ __launch_bounds__(64 * kFewWaves, 1) void few_kernel(PagedAttention a) {
    using F = Few<D, F8>;
    constexpr int BM = 16 * NT, KT = F::KT, SUB = KT / 16, ES = F8 ? 1 : 2;
    using Split = PagedSplit<BM, KT, F::START>;
    extern __shared__ __align__(1024) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int quad = lane >> 4, col = lane & 15;

    int64_t* pre = reinterpret_cast<int64_t*>(lds);
    Split::prefix(a, pre, 64 * kFewWaves);
    const int64_t total = pre[a.B], chunk = Split::chunk(a, total, gridDim.x, kFewMinTiles);
    // consecutive pieces on one XCD
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
    if (lane < 2) *bad_of(a.ws, group, wave + 4 * lane) = 0;
    if (tid == 0) {
        begin[0] = i32x4v{cur.b, cur.hk, cur.r, cur.kt};
        begin[1] = i32x4v{s.off, (int)min((int64_t)BM, (int64_t)s.n * a.G - (int64_t)cur.r * BM), 0, 0};
    }
    __syncthreads();

    const uint32_t ring = (uint32_t)(uintptr_t)lds + wave * F::WAVE;
    // this lane's place in a DMA instruction: key lr of RPI, chunk lc
    const int lr = lane / F::LPR, lc = lane % F::LPR;

    for (;;) {
        const int R = Split::tiles(a, s);
        const int nkt = R ? Split::key_tiles(a, s, cur.r) : 0;
        const bool last = cur.b == end.b && cur.hk == end.hk && cur.r == end.r;
        const int k0 = cur.kt, k1 = last ? end.kt : nkt;
        if (R && k1 > k0) {
            const int r0 = cur.r * BM, nr = (int)min((int64_t)BM, (int64_t)s.n * a.G - r0);
            const int nt_used = (nr + 15) >> 4;
            // page ids of this wave's next key tiles, a lane each; the first ones
            // come with the queries
            const int32_t* table = a.table + (int64_t)cur.b * a.ldt;
            constexpr int BATCH = 64 / SUB;  // tiles whose page ids one load brings
            int ids;
            auto load_ids = [&](int j0) {
                const int64_t key = ((int64_t)k0 + wave + (int64_t)kFewWaves * (j0 + lane / SUB)) * KT + 16 * (lane % SUB);
                const int id = table[min(key, (int64_t)s.len - 1 + (s.len == 0)) >> a.page_bits];
                ids = key < s.len ? id : -1;
            };
            load_ids(0);
            const float c = a.scale2 * (F8 ? a.k_scale[cur.hk] : 1.0f);
            // queries (B operand: row col, dimensions 64 t + 16 quad + 8 e ..)
            bf16x8 qf[NT][D / 32];
            int lim[NT];  // keys that the lane's row may see
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int row = 16 * nt + col, flat = r0 + row, tok = flat / a.G;
                const bool ok = row < nr;
                const uint16_t* q = a.q + (int64_t)(s.off + (ok ? tok : 0)) * a.q_tok + (int64_t)(cur.hk * a.G + flat % a.G) * a.q_head;
                load_queries<D / 32>(q, qf[nt], [&](int t) { return 32 * (t & ~1) + 16 * quad + 8 * (t & 1); });
                lim[nt] = !ok ? 0 : a.causal ? min(max(s.len - s.n + tok + 1, 0), s.len) : s.len;
            }
            // the fewest keys that a row of the tile may see: tiles below need no mask
            const int open = a.causal ? min(max(s.len - s.n + r0 / a.G + 1, 0), s.len) : s.len;
            f32x4 o[NT][D / 16];
            float m[NT], l[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                m[nt] = -__builtin_inff();
                l[nt] = 0.0f;
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt) o[nt][dt] = f32x4{0, 0, 0, 0};
            }

            // ---- this wave's key tiles k0 + wave, + 4, ... ----
            const int n = k0 + wave < k1 ? (k1 - k0 - wave + kFewWaves - 1) / kFewWaves : 0;
            const char* kbase = static_cast<const char*>(a.k.data) + cur.hk * a.k.head * ES;
            const char* vbase = static_cast<const char*>(a.v.data) + cur.hk * a.v.head * ES;
            // K (V) of the wave's tile j into its ring place
            auto issue = [&](int j, bool is_v) {
                const PagedCache& cache = is_v ? a.v : a.k;
                const uint32_t m0 = ring + (2 * (j % F::DEPTH) + is_v) * F::SLOT;
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    const int64_t key = ((int64_t)k0 + wave + (int64_t)kFewWaves * j) * KT + 16 * sub;
                    const int id = __builtin_amdgcn_readlane(ids, (j % BATCH) * SUB + sub);
                    const int there = j < n && (unsigned)id < (unsigned)a.pages ? (int)min((int64_t)s.len - key, (int64_t)16) : 0;
                    const int64_t at = (int64_t)id * cache.page + (key & ((1 << a.page_bits) - 1)) * cache.slot;
                    const uint32_t bytes = there > 0 ? (uint32_t)(((there - 1) * cache.slot + D) * ES) : 0;
                    const i32x4 desc = make_desc((is_v ? vbase : kbase) + (bytes ? at * ES : 0), bytes);
#pragma unroll
                    for (int i = 0; i < F::NI / SUB; ++i) {
                        const int r = i * F::RPI + lr, rt = 16 * sub + r;
                        const int ch = lc ^ (is_v ? F::xv(rt) : F::xk(rt));
                        const uint32_t voff = (uint32_t)(r * (int)cache.slot * ES + ch * 16);
                        dma<true>(__builtin_amdgcn_readfirstlane(m0 + (sub * (F::NI / SUB) + i) * 1024), voff, desc);
                    }
                }
            };
#pragma unroll 1
            for (int j = 0; j < F::DEPTH; ++j) {
                issue(j, false);
                issue(j, true);
            }
#pragma unroll 1
            for (int j = 0; j < n; ++j) {
                const uint32_t ks = ring + 2 * (j % F::DEPTH) * F::SLOT, vs = ks + F::SLOT;
                const int key0 = (k0 + wave + kFewWaves * j) * KT;
                if ((j + F::DEPTH) % BATCH == 0) load_ids(j + F::DEPTH);
                wait_vm<F::IN_FLIGHT>();
                f32x4 st[NT][SUB];
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    const int row = 16 * sub + col;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) st[nt][sub] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int t = 0; t < D / 64; ++t) {
                        bf16x8 kf[2];
                        if constexpr (F8) {
                            const u32x4 w = read16(ks + row * F::ROWB + (((4 * t + quad) ^ F::xk(row)) << 4));
                            kf[0] = codes8_bf16(w.x, w.y);
                            kf[1] = codes8_bf16(w.z, w.w);
                        } else {
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                kf[e] = __builtin_bit_cast(
                                    bf16x8, read16(ks + row * F::ROWB + (((8 * t + 2 * quad + e) ^ F::xk(row)) << 4)));
                        }
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                st[nt][sub] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[e], qf[nt][2 * t + e], st[nt][sub],
                                                                                      0, 0, 0);
                    }
                }
                wait_lgkm<0>();
                issue(j + F::DEPTH, false);
                if (key0 + KT > open) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (key0 + 16 * sub + 4 * quad + i >= lim[nt]) st[nt][sub][i] = -__builtin_inff();
                }
                // weights, packed as the B operand of the second product
                u32x2 pw[NT][SUB];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float top = st[nt][0][0];
#pragma unroll
                    for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = fmaxf(top, st[nt][sub][i]);
                    if (__any(top * c > m[nt] + kLazy)) {
                        top = fmaxf(top, __shfl_xor(top, 16, 64));
                        top = fmaxf(top, __shfl_xor(top, 32, 64));
                        const float mn = fmaxf(m[nt], top * c);
                        const float f = m[nt] == -__builtin_inff() ? 0.0f : exp2_fast(m[nt] - mn);
                        m[nt] = mn;
                        l[nt] *= f;
#pragma unroll
                        for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[nt][dt][i] *= f;
                    }
                    const float ms = m[nt] == -__builtin_inff() ? 0.0f : m[nt];
#pragma unroll
                    for (int sub = 0; sub < SUB; ++sub) {
                        f32x4 p;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[i] = exp2_fast(__builtin_fmaf(st[nt][sub][i], c, -ms));
                            l[nt] += p[i];
                        }
                        pw[nt][sub] = u32x2{pack_bf16x2(f32x2{p.x, p.y}), pack_bf16x2(f32x2{p.z, p.w})};
                    }
                }
                wait_vm<F::IN_FLIGHT>();
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt) {
                    if constexpr (F8) {
                        // 8 keys of dimension 16 dt + col: 4 quad + 0..3 and 16 + 4 quad + 0..3
                        const int rr = col >> 1, row = (rr & 3) + 4 * quad + 16 * (rr >> 2);
                        const i32x2 w = read_tr8(vs + row * F::ROWB + ((dt ^ F::xv(row)) << 4) + 8 * (col & 1));
                        const bf16x8 vf = codes8_bf16((uint32_t)w.x, (uint32_t)w.y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const u32x4 pb = {pw[nt][0].x, pw[nt][0].y, pw[nt][SUB - 1].x, pw[nt][SUB - 1].y};
                            o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8, pb), o[nt][dt],
                                                                                0, 0, 0);
                        }
                    } else {
                        // 4 keys 4 quad + 0..3 of dimension 16 dt + col
                        const int row = 4 * quad + (col >> 2), ch = 2 * dt + ((col & 3) >> 1);
                        const s16x4 vf = read_tr16(vs + row * F::ROWB + ((ch ^ F::xv(row)) << 4) + 8 * (col & 1));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
                                vf, __builtin_bit_cast(s16x4, pw[nt][0]), o[nt][dt], 0, 0, 0);
                    }
                }
                wait_lgkm<0>();
                issue(j + F::DEPTH, true);
            }
            wait_vm<0>();
            if (a.causal) {
                // keys of the piece that the first row may not see, by all waves
                if (odd_values<D, F8>(a, table, cur.hk, max(open, k0 * KT), min(s.len, k1 * KT), wave, kFewWaves))
                    *bad_of(a.ws, group, wave) = 1;
            }

            // ---- join the four waves, 16 rows at a time ----
            constexpr int LD = D + 4;
            float* so = reinterpret_cast<float*>(lds);       // [waves][16][LD]
            float* sm = so + kFewWaves * 16 * LD;            // [waves][16]
            float* sl = sm + kFewWaves * 16;
            const bool whole = k0 == 0 && k1 == nkt;
            float* part = Partial<BM, D>::at(a.ws, group, k0 == 0);
            const float vscale = F8 ? a.v_scale[cur.hk] : 1.0f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                __syncthreads();
                if (nt < nt_used) {
                    float lt = l[nt];
                    lt += __shfl_xor(lt, 16, 64);
                    lt += __shfl_xor(lt, 32, 64);
                    if (quad == 0) {
                        sm[wave * 16 + col] = m[nt];
                        sl[wave * 16 + col] = lt;
                    }
#pragma unroll
                    for (int dt = 0; dt < D / 16; ++dt)
                        *reinterpret_cast<f32x4*>(so + (wave * 16 + col) * LD + 16 * dt + 4 * quad) = o[nt][dt];
                }
                __syncthreads();
                const int row = tid >> 4, flat = r0 + 16 * nt + row;
                if (16 * nt + row < nr) {
                    float M = sm[row];
#pragma unroll
                    for (int w = 1; w < kFewWaves; ++w) M = fmaxf(M, sm[w * 16 + row]);
                    float f[kFewWaves], lt = 0.0f;
#pragma unroll
                    for (int w = 0; w < kFewWaves; ++w) {
                        const float mw = sm[w * 16 + row];
                        f[w] = mw == -__builtin_inff() ? 0.0f : exp2_fast(mw - M);
                        lt += sl[w * 16 + row] * f[w];
                    }
                    const float inv = lt == 0.0f ? 0.0f : vscale / lt;
#pragma unroll
                    for (int k = 0; k < D / 64; ++k) {
                        const int d = 64 * k + 4 * (tid & 15);
                        f32x4 t = {0, 0, 0, 0};
#pragma unroll
                        for (int w = 0; w < kFewWaves; ++w) {
                            const f32x4 x = *reinterpret_cast<const f32x4*>(so + (w * 16 + row) * LD + d);
#pragma unroll
                            for (int i = 0; i < 4; ++i) t[i] += x[i] * f[w];
                        }
                        if (whole) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) t[i] = lt == 0.0f ? 0.0f : t[i] * inv;
                            store4(a, s.off + flat / a.G, cur.hk * a.G + flat % a.G, d, t);
                        } else {
                            *reinterpret_cast<f32x4*>(part + (16 * nt + row) * D + d) = t;
                        }
                    }
                    if (!whole && (tid & 15) == 0) {
                        part[(int64_t)BM * D + 16 * nt + row] = M;
                        part[(int64_t)BM * D + BM + 16 * nt + row] = lt;
                    }
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

template <int D, bool F8, int NT>
hipError_t run(const PagedAttention& a, bool with_join, hipStream_t stream) {
    constexpr int BM = 16 * NT, LDS = Few<D, F8>::LDS;
    static_assert(LDS >= PagedSplit<BM, 16, 0>::lds_bytes(kPagedMaxRequests), "the prefix of the requests' costs fits");
    static_assert(LDS >= kFewWaves * 16 * (D + 6) * 4, "the waves' sums fit");
    auto* kern = few_kernel<D, F8, NT>;
    static OncePerDevice once;
    const hipError_t attr = allow_lds(once, reinterpret_cast<const void*>(kern), LDS);
    if (attr != hipSuccess) return attr;
    hipLaunchKernelGGL(kern, dim3(kGroups), dim3(64 * kFewWaves), LDS, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !with_join) return e;
    auto* kern_join = join_kernel<BM, D, F8, 4, FewOrder<D>>;
    hipLaunchKernelGGL(kern_join, dim3(2 * kGroups), dim3(256), 0, stream, a);
    return hipGetLastError();
}

// Tiles of 32 rows at the most: requests of 33 to 64 rows read their keys twice.
// Tiles of 64 rows keep 256 registers of O for heads of 256 and spilled the rest
// (48 rows, 8000 keys, 12/2 heads: 60 us against 26); for smaller heads they
// gained 15 % on one long request (64 rows, 60000 8-bit keys, 32/8 heads of 128:
// 57 us against 66) and lost 27 % on a batch (16 x 4000 keys: 85 against 67).
template <int D, bool F8>
hipError_t run_rows(const PagedAttention& a, int rows, bool join, hipStream_t stream) {
    static_assert(kMixedRows == 32);
    return rows <= 16 ? run<D, F8, 1>(a, join, stream) : run<D, F8, 2>(a, join, stream);
}

}  // namespace

hipError_t launch_few(const PagedAttention& a, int D, bool fp8, int rows, bool join, hipStream_t stream) {
    if (D == 64) return fp8 ? run_rows<64, true>(a, rows, join, stream) : run_rows<64, false>(a, rows, join, stream);
    if (D == 128) return fp8 ? run_rows<128, true>(a, rows, join, stream) : run_rows<128, false>(a, rows, join, stream);
    return fp8 ? run_rows<256, true>(a, rows, join, stream) : run_rows<256, false>(a, rows, join, stream);
}

}  // namespace attn
}  // namespace fp8lin
