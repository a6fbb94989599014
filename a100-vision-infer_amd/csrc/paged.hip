// The paged cache's bookkeeping and its writes:
//   - paged layout of a step: from the requests' lengths and their numbers of
//     new tokens to row offsets, pages taken from the free list, cache slots
//     and positions of the new tokens;
//   - append: the new tokens' keys and values into their slots, as BF16 or as
//     E4M3FN codes of value / scale.
#include <algorithm>

#include "device.hpp"
#include "paged.hpp"

namespace fp8lin {
namespace {

// ---- layout -----------------------------------------------------------------
//
// Request b holds len_b tokens and gets n_b more.  The entries of its block
// table row from page len_b / P to the page of its last new token that hold no
// page yet (< 0) take the next pages of the free list, in the order of the
// requests and their entries:
//   id(b, j) = free[cursor + fresh entries before (b, j)].
// Bound by launch and load latency: one launch for up to kScanRequests
// requests, in which every workgroup counts the fresh entries of the requests
// before its own by itself; beyond that (each of B workgroups would read B
// requests: 17.3 us a call against 16.9 in two launches at 1500), or where the
// new table is written over the old one (the counts would change under the
// other workgroups), a first launch of one workgroup leaves the sums in a
// workspace.  At 1024 requests a call takes 13 us in one launch and 17 in two,
// the host's share included; the kernel takes 4 us for one request and 8 for
// 509.
constexpr int kScanRequests = 1024;
constexpr int kLayoutThreads = 256;

struct Layout {
    const int32_t *lengths, *counts, *table, *free_pages, *cursor;
    int64_t ldt, ldn, free_count, T;
    int B, width, page_bits;
    int32_t *offsets, *new_lengths, *new_table, *new_cursor;
    int64_t *slots, *positions;
    int32_t* sums;  // [B][2] first row, first fresh entry; null: counted here
};

struct Span {
    int64_t len, n;
    int lo, hi;  // entries that may be fresh
};
__device__ __forceinline__ Span span_of(const Layout& a, int b) {
    Span s;
    s.len = max(a.lengths[b], 0);
    s.n = max(a.counts[b], 0);
    const int64_t P = (int64_t)1 << a.page_bits;
    s.lo = (int)min(s.len >> a.page_bits, (int64_t)a.width);
    s.hi = s.n ? (int)min((s.len + s.n + P - 1) >> a.page_bits, (int64_t)a.width) : s.lo;
    return s;
}

// Sums of n and of fresh entries over the requests [0, end), by all threads of
// the workgroup: a thread per request, the entries of a long prompt by all.
__device__ void count_before(const Layout& a, int end, int64_t& rows, int64_t& fresh) {
    constexpr int kLong = 4;
    __shared__ int64_t wave_rows[kLayoutThreads / 64], wave_fresh[kLayoutThreads / 64];
    __shared__ int long_list[kLayoutThreads], long_count;
    const int tid = threadIdx.x;
    int64_t r = 0, f = 0;
    for (int b0 = 0; b0 < end; b0 += kLayoutThreads) {
        if (tid == 0) long_count = 0;
        __syncthreads();
        const int b = b0 + tid;
        if (b < end) {
            const Span s = span_of(a, b);
            r += s.n;
            if (s.hi - s.lo <= kLong) {
#pragma unroll
                for (int i = 0; i < kLong; ++i)
                    if (s.lo + i < s.hi) f += a.table[(int64_t)b * a.ldt + s.lo + i] < 0;
            } else {
                long_list[atomicAdd(&long_count, 1)] = b;
            }
        }
        __syncthreads();
        for (int i = 0; i < long_count; ++i) {
            const Span s = span_of(a, long_list[i]);
            for (int j = s.lo + tid; j < s.hi; j += kLayoutThreads) f += a.table[(int64_t)long_list[i] * a.ldt + j] < 0;
        }
        __syncthreads();
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        r += __shfl_xor(r, d, 64);
        f += __shfl_xor(f, d, 64);
    }
    if ((tid & 63) == 0) {
        wave_rows[tid >> 6] = r;
        wave_fresh[tid >> 6] = f;
    }
    __syncthreads();
    rows = fresh = 0;
#pragma unroll
    for (int w = 0; w < kLayoutThreads / 64; ++w) {
        rows += wave_rows[w];
        fresh += wave_fresh[w];
    }
}

// One workgroup: the sums before every request, for layout_kernel.
__global__ __launch_bounds__(kLayoutThreads) void layout_sums_kernel(Layout a) {
    __shared__ int64_t wave_rows[kLayoutThreads / 64], wave_fresh[kLayoutThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int64_t rows = 0, fresh = 0;
    for (int b0 = 0; b0 < a.B; b0 += kLayoutThreads) {
        const int b = b0 + tid;
        int64_t r = 0, f = 0;
        if (b < a.B) {
            const Span s = span_of(a, b);
            r = s.n;
            for (int j = s.lo; j < s.hi; ++j) f += a.table[(int64_t)b * a.ldt + j] < 0;
        }
        int64_t ri = r, fi = f;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t ro = __shfl_up(ri, d, 64), fo = __shfl_up(fi, d, 64);
            if (lane >= d) {
                ri += ro;
                fi += fo;
            }
        }
        if (lane == 63) {
            wave_rows[wave] = ri;
            wave_fresh[wave] = fi;
        }
        __syncthreads();
        int64_t rb = rows + ri - r, fb = fresh + fi - f;
        for (int w = 0; w < kLayoutThreads / 64; ++w) {
            if (w < wave) {
                rb += wave_rows[w];
                fb += wave_fresh[w];
            }
            rows += wave_rows[w];
            fresh += wave_fresh[w];
        }
        if (b < a.B) {
            a.sums[2 * b] = (int32_t)min(rb, (int64_t)INT32_MAX);
            a.sums[2 * b + 1] = (int32_t)min(fb, (int64_t)INT32_MAX);
        }
        __syncthreads();
    }
}

// Workgroup (b, y): part y of request b's table row and new tokens.
__global__ __launch_bounds__(kLayoutThreads) void layout_kernel(Layout a) {
    __shared__ int32_t ids[kLayoutThreads];
    __shared__ int wave_fresh[kLayoutThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = blockIdx.x, y = blockIdx.y, Y = gridDim.y;
    int64_t row0, taken;
    if (a.sums) {
        row0 = a.sums[2 * b];
        taken = a.sums[2 * b + 1];
    } else {
        count_before(a, b, row0, taken);
    }
    const Span s = span_of(a, b);
    const int64_t first = a.cursor ? max(a.cursor[0], 0) : 0;
    const int32_t* table = a.table + (int64_t)b * a.ldt;
    int32_t* out = a.new_table + (int64_t)b * a.ldn;
    const int P = 1 << a.page_bits;
    // entries that no new token needs; the table may be its own output
    if (out != table) {
        for (int j = y * kLayoutThreads + tid; j < a.width; j += Y * kLayoutThreads)
            if (j < s.lo || j >= s.hi) out[j] = table[j];
    }
    for (int j0 = s.lo, part = 0; j0 < s.hi; j0 += kLayoutThreads, ++part) {
        const int j = j0 + tid;
        int32_t id = j < s.hi ? table[j] : 0;
        const bool fresh = id < 0;
        const uint64_t mask = __ballot(fresh);
        if (lane == 0) wave_fresh[wave] = __popcll(mask);
        __syncthreads();
        int64_t rank = taken + __popcll(mask & ((1ull << lane) - 1));
        for (int w = 0; w < kLayoutThreads / 64; ++w) {
            if (w < wave) rank += wave_fresh[w];
            taken += wave_fresh[w];
        }
        if (part % Y == y) {
            if (fresh) {
                const int64_t at = first + rank;
                id = at < a.free_count ? a.free_pages[at] : -1;
            }
            ids[tid] = id;
            if (j < s.hi) out[j] = id;
            __syncthreads();
            const int64_t lo = max(s.len, (int64_t)j0 << a.page_bits);
            const int64_t hi = min(s.len + s.n, (int64_t)min(j0 + kLayoutThreads, s.hi) << a.page_bits);
            for (int64_t pos = lo + tid; pos < hi; pos += kLayoutThreads) {
                const int64_t t = row0 + pos - s.len;
                if (t >= a.T) break;
                const int32_t page = ids[(pos >> a.page_bits) - j0];
                a.slots[t] = page < 0 ? -1 : ((int64_t)page << a.page_bits) + (pos & (P - 1));
                a.positions[t] = pos;
            }
        }
        __syncthreads();
    }
    // tokens past the table's last entry
    const int64_t cap = (int64_t)a.width << a.page_bits;
    for (int64_t pos = max(s.len, cap) + y * kLayoutThreads + tid; pos < s.len + s.n; pos += (int64_t)Y * kLayoutThreads) {
        const int64_t t = row0 + pos - s.len;
        if (t >= a.T) break;
        a.slots[t] = -1;
        a.positions[t] = pos;
    }
    if (y == 0 && tid == 0) {
        a.offsets[b] = (int32_t)min(row0, (int64_t)INT32_MAX);
        a.new_lengths[b] = (int32_t)min(s.len + s.n, (int64_t)INT32_MAX);
    }
    if (b == a.B - 1) {
        const int64_t end = row0 + s.n;
        for (int64_t t = end + y * kLayoutThreads + tid; t < a.T; t += (int64_t)Y * kLayoutThreads) {
            a.slots[t] = -1;
            a.positions[t] = 0;
        }
        if (y == 0 && tid == 0) {
            a.offsets[a.B] = (int32_t)min(end, (int64_t)INT32_MAX);
            a.new_cursor[0] = (int32_t)min(first + taken, (int64_t)INT32_MAX);
        }
    }
}

// ---- append -----------------------------------------------------------------

struct Append {
    const uint16_t* x[2];
    int64_t tok[2], head[2];
    PagedCache cache[2];
    const float* scale[2];
    const int64_t* slots;
    int64_t T, limit;
    int HK, D, page_bits;
};

// E4M3FN of clamp(x / s, +-448), to nearest even; NaN stays NaN.  An IEEE
// division: the code is that of the exact quotient's FP32 value.
__device__ __forceinline__ float to_code_range(float x, float s) {
    const float v = x / s;
    return v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f);
}

// A thread moves 8 values of a token's key (blockIdx.y 0) or value (1); 3913
// tokens, 2 heads of 256 into an 8-bit cache (12 MB): 6 us, launch included.  VEC:
// the inputs' rows start on 16 bytes.
template <bool F8, bool VEC>
__global__ __launch_bounds__(256) void append_kernel(Append a) {
    const int kv = blockIdx.y, vecs = a.HK * a.D / 8;
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t t = e / vecs;
    if (t >= a.T) return;
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.limit) return;
    const int at = (int)(e - t * vecs) * 8, h = at / a.D, d = at - h * a.D;
    const uint16_t* src = a.x[kv] + t * a.tok[kv] + h * a.head[kv] + d;
    u32x4 w;
    if constexpr (VEC) {
        w = load_u32x4(src);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)src[2 * i] | (uint32_t)src[2 * i + 1] << 16;
    }
    const PagedCache& c = a.cache[kv];
    const int64_t dst = (slot >> a.page_bits) * c.page + (slot & ((1 << a.page_bits) - 1)) * c.slot + h * c.head + d;
    if constexpr (F8) {
        const float s = a.scale[kv][h];
        uint32_t code[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                v[k] = to_code_range(bf16_bits_to_f32((w[2 * i + (k >> 1)] >> (16 * (k & 1))) & 0xffffu), s);
            int p = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
            code[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], p, true);
        }
        *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(const_cast<void*>(c.data)) + dst) = u32x2{code[0], code[1]};
    } else {
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(const_cast<void*>(c.data)) + dst) = w;
    }
}

}  // namespace

size_t paged_layout_ws_bytes(int64_t B, bool in_place) { return in_place || B > kScanRequests ? (size_t)(8 * B) : 0; }

hipError_t launch_paged_layout(const int32_t* lengths, const int32_t* counts, const int32_t* table, int64_t ldt,
                               const int32_t* free_pages, int64_t free_count, const int32_t* cursor, int B, int width,
                               int page_bits, int64_t T, int32_t* offsets, int32_t* new_lengths, int64_t* slots,
                               int64_t* positions, int32_t* new_table, int64_t ldn, int32_t* new_cursor, int32_t* ws,
                               hipStream_t stream) {
    Layout a{lengths, counts, table, free_pages, cursor, ldt, ldn, free_count, T, B, width, page_bits, offsets, new_lengths,
             new_table, new_cursor, slots, positions, nullptr};
    const bool in_place = new_table == table;
    int parts = 1;
    if (in_place || B > kScanRequests) {
        a.sums = ws;
        hipLaunchKernelGGL(layout_sums_kernel, dim3(1), dim3(kLayoutThreads), 0, stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (!in_place) {
        // enough workgroups for a few long rows, one per row in a large batch
        const int64_t most = (T >> page_bits) + width;
        parts = (int)std::min<int64_t>(std::max<int64_t>(512 / B, 1), (most + kLayoutThreads - 1) / kLayoutThreads);
        parts = std::max(parts, 1);
    }
    hipLaunchKernelGGL(layout_kernel, dim3(B, parts), dim3(kLayoutThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_paged_append(const uint16_t* k, const uint16_t* v, int64_t k_tok, int64_t k_head, int64_t v_tok,
                               int64_t v_head, const int64_t* slots, const PagedCache& kc, const PagedCache& vc, bool fp8,
                               const float* k_scale, const float* v_scale, int64_t T, int HK, int D, int page_bits,
                               int64_t pages, hipStream_t stream) {
    const Append a{{k, v}, {k_tok, v_tok}, {k_head, v_head}, {kc, vc}, {k_scale, v_scale}, slots, T, pages << page_bits, HK, D,
                   page_bits};
    auto on16 = [](const void* p, int64_t tok, int64_t head) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && tok % 8 == 0 && head % 8 == 0;
    };
    const bool vec = on16(k, k_tok, k_head) && on16(v, v_tok, v_head);
    const int64_t blocks = (T * (HK * (int64_t)D / 8) + 255) / 256;
    const dim3 grid((unsigned)blocks, 2), block(256);
    if (fp8) {
        if (vec) hipLaunchKernelGGL((append_kernel<true, true>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((append_kernel<true, false>), grid, block, 0, stream, a);
    } else {
        if (vec) hipLaunchKernelGGL((append_kernel<false, true>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((append_kernel<false, false>), grid, block, 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace fp8lin
