// Host-side arguments of the paged-cache kernels (paged.hip, attention_*.hip)
// and the device-side arithmetic that the attention kernels share: which part
// of which request a workgroup computes.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace fp8lin {

// A K or V cache [pages, page_size, kv_heads, D] with strides in elements
// (the last dimension contiguous); fp8: E4M3FN codes, else BF16.
struct PagedCache {
    const void* data;
    int64_t page, slot, head;
};

struct PagedAttention {
    const uint16_t *q, *gate;  // [T, H, D]; gate may be null
    uint16_t* out;
    int64_t q_tok, q_head, g_tok, g_head, o_tok, o_head;
    PagedCache k, v;
    const float *k_scale, *v_scale;  // [HK] or null
    const int32_t *table, *offsets, *lengths;
    int64_t ldt;
    int width, page_bits, pages;
    int B, T, H, HK, G;
    int64_t rows_from, rows_to;  // requests of rows_from < new tokens * G <= rows_to are computed, others left
    bool causal;
    float scale2;  // softmax scale * log2(e)
    float* ws;
};

constexpr int kPagedMaxRequests = 4096;
constexpr int kPagedMinPage = 16;

// Workgroups of the attention launch for D and the row tile that max_rows
// (the most rows, tokens times heads per kv head, that a request should
// bring) selects; the workspace that goes with them.
size_t paged_attention_ws_bytes(int D, int64_t max_rows);
hipError_t launch_paged_attention(PagedAttention a, int D, bool fp8, int64_t max_rows, hipStream_t stream);

hipError_t launch_paged_append(const uint16_t* k, const uint16_t* v, int64_t k_tok, int64_t k_head, int64_t v_tok,
                               int64_t v_head, const int64_t* slots, const PagedCache& kc, const PagedCache& vc, bool fp8,
                               const float* k_scale, const float* v_scale, int64_t T, int HK, int D, int page_bits,
                               int64_t pages, hipStream_t stream);
hipError_t launch_paged_layout(const int32_t* lengths, const int32_t* counts, const int32_t* table, int64_t ldt,
                               const int32_t* free_pages, int64_t free_count, const int32_t* cursor, int B, int width,
                               int page_bits, int64_t T, int32_t* offsets, int32_t* new_lengths, int64_t* slots,
                               int64_t* positions, int32_t* new_table, int64_t ldn, int32_t* new_cursor, int32_t* ws,
                               hipStream_t stream);
size_t paged_layout_ws_bytes(int64_t B, bool in_place);

// ---- the split of an attention launch over its workgroups -------------------
//
// A unit is one row tile (BM rows: consecutive tokens of a request, the G
// query heads of one kv head side by side) against the keys that its last row
// may see.  The units in the order (request, kv head, row tile) are laid on a
// line, each as long as it costs (START and its keys, times G), and workgroup w
// computes the piece [w, w + 1) * chunk of that line: every workgroup has the same
// amount of work, whatever the lengths.  A unit that falls into several
// pieces is joined afterwards from their partial sums.  The split depends on
// the lengths alone, so a call's result does not depend on timing.
struct PagedSeq {
    int off, n, len;
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedAttention& a, int b) {
    int lo = a.offsets[b], hi = a.offsets[b + 1];
    lo = min(max(lo, 0), a.T);
    hi = min(max(hi, lo), a.T);
    const int64_t rows = (int64_t)(hi - lo) * a.G;
    if (rows <= a.rows_from || rows > a.rows_to) hi = lo;
    const int64_t cap = (int64_t)a.width << a.page_bits;
    const int64_t len = min((int64_t)max(a.lengths[b], 0), cap);
    return PagedSeq{lo, hi - lo, (int)len};
}

template <int BM, int BN, int START>
struct PagedSplit {
    struct Loc {
        int b, hk, r, kt;
    };

    // Cost of the first x row tiles, x < R; ctx: keys before the new tokens.
    static __device__ __forceinline__ int64_t first(const PagedAttention& a, const PagedSeq& s, int64_t x) {
        if (!a.causal) return x * a.G * (START + max(s.len, 1));
        return x * a.G * (START + max(s.len - s.n, 0)) + BM * (x * (x + 1) / 2);
    }
    static __device__ __forceinline__ int tiles(const PagedAttention& a, const PagedSeq& s) {
        return (int)(((int64_t)s.n * a.G + BM - 1) / BM);
    }
    // Cost of row tile r of R.
    static __device__ __forceinline__ int64_t tile(const PagedAttention& a, const PagedSeq& s, int r) {
        if (!a.causal) return (int64_t)a.G * (START + max(s.len, 1));
        return (int64_t)a.G * (START + max(s.len - s.n, 0)) + min((int64_t)(r + 1) * BM, (int64_t)s.n * a.G);
    }
    // All row tiles of one kv head.
    static __device__ __forceinline__ int64_t head(const PagedAttention& a, const PagedSeq& s) {
        const int R = tiles(a, s);
        return R ? first(a, s, R - 1) + tile(a, s, R - 1) : 0;
    }
    // Key tiles of row tile r: at least one, so that a row without keys is
    // written too.
    static __device__ __forceinline__ int key_tiles(const PagedAttention& a, const PagedSeq& s, int r) {
        int limit = s.len;
        if (a.causal) {
            const int64_t rows = min((int64_t)(r + 1) * BM, (int64_t)s.n * a.G);
            limit = min(max(s.len - s.n + (int)((rows - 1) / a.G) + 1, 0), s.len);
        }
        return max((limit + BN - 1) / BN, 1);
    }

    // floor(x / y) for 0 <= x < 2^62, 0 < y, x / y below 2^31: by the FP64
    // quotient, whose error of under half a unit the two checks take back.
    static __device__ __forceinline__ int64_t div(int64_t x, int64_t y) {
        int64_t q = (int64_t)((double)x / (double)y);
        if (q * y > x) --q;
        if ((q + 1) * y <= x) ++q;
        return q;
    }

    // What a workgroup knows of the batch while it finds its piece, in LDS:
    // prefix[b] = cost of the requests before b, b <= B, then each request's
    // (new tokens, keys).
    static constexpr int lds_bytes(int B) { return 16 * B + 16; }
    static __device__ __forceinline__ int* held(const PagedAttention& a, int64_t* pre) {
        return reinterpret_cast<int*>(pre + a.B + 1);
    }
    // All threads of the workgroup, which synchronise here.
    static __device__ void prefix(const PagedAttention& a, int64_t* pre, int threads) {
        __shared__ int64_t wave_total[16];
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
        int* h = held(a, pre);
        int64_t base = 0;
        for (int b0 = 0; b0 < a.B; b0 += threads) {
            const int b = b0 + tid;
            int64_t cost = 0;
            if (b < a.B) {
                const PagedSeq s = paged_seq(a, b);
                cost = (int64_t)a.HK * head(a, s);
                h[2 * b] = s.n;
                h[2 * b + 1] = s.len;
            }
            int64_t run = cost;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int64_t o = __shfl_up(run, d, 64);
                if (lane >= d) run += o;
            }
            if (lane == 63) wave_total[wave] = run;
            __syncthreads();
            int64_t before = base + run - cost;
            for (int w = 0; w < waves; ++w) {
                if (w < wave) before += wave_total[w];
                base += wave_total[w];
            }
            if (b < a.B) pre[b] = before;
            __syncthreads();
        }
        if (tid == 0) pre[a.B] = base;
        __syncthreads();
    }

    // The place p of the line, 0 <= p < prefix[B]: within its unit, behind the
    // START, key tile kt = floor(part of the unit's cost before p * its key
    // tiles).
    static __device__ Loc locate(const PagedAttention& a, int64_t* pre, int64_t p) {
        int lo = 0, hi = a.B;  // pre[lo] <= p < pre[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] <= p) lo = mid; else hi = mid;
        }
        const int* h = held(a, pre) + 2 * lo;
        const PagedSeq s{0, h[0], h[1]};
        const int64_t per_head = head(a, s);
        int64_t q = p - pre[lo];
        Loc l;
        l.b = lo;
        l.hk = (int)min(max(div(q, per_head), (int64_t)0), (int64_t)a.HK - 1);
        q -= l.hk * per_head;
        int rl = 0, rh = tiles(a, s);
        while (rh - rl > 1) {
            const int mid = (rl + rh) >> 1;
            if (first(a, s, mid) <= q) rl = mid; else rh = mid;
        }
        l.r = rl;
        const int64_t start = (int64_t)START * a.G;
        q = max(q - first(a, s, rl) - start, (int64_t)0);
        // in FP64, as the product may pass 64 bits: a piece's end and the next
        // one's begin are the same computation, which grows with q
        const int kts = key_tiles(a, s, rl);
        l.kt = min(max((int)((double)q * kts / (double)(tile(a, s, rl) - start)), 0), kts - 1);
        return l;
    }
    // The pieces [p0, p1) of every wave's workgroup: even lanes find where it
    // begins, odd lanes where it ends (request B if it ends the line).
    static __device__ void piece(const PagedAttention& a, int64_t* pre, int64_t p0, int64_t p1, Loc& begin, Loc& end) {
        const int64_t p = (threadIdx.x & 1) ? p1 : p0;
        Loc l{a.B, 0, 0, 0};
        if (p < pre[a.B]) l = locate(a, pre, p);
        begin = Loc{__builtin_amdgcn_readlane(l.b, 0), __builtin_amdgcn_readlane(l.hk, 0), __builtin_amdgcn_readlane(l.r, 0),
                    __builtin_amdgcn_readlane(l.kt, 0)};
        end = Loc{__builtin_amdgcn_readlane(l.b, 1), __builtin_amdgcn_readlane(l.hk, 1), __builtin_amdgcn_readlane(l.r, 1),
                  __builtin_amdgcn_readlane(l.kt, 1)};
    }
    // Length of a piece: an even share, but no shorter than min_tiles key
    // tiles of a unit.  groups: a power of two.
    static __device__ __forceinline__ int64_t chunk(const PagedAttention& a, int64_t total, int groups, int min_tiles) {
        return max((total + groups - 1) >> (31 - __builtin_clz(groups)), (int64_t)min_tiles * BN * a.G);
    }
};

}  // namespace fp8lin
