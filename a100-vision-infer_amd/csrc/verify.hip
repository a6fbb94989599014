// Verification of drafted tokens against the target's probabilities.
//
// Rows a .. a + n of a request are the target's logits after its last token
// and after each of its n drafts x_1 .. x_n.  With p = softmax(logits / T) of
// a row and q the draft's distribution there, x_i is kept while
// u_i q(x_i) < p(x_i); the token after the kept ones is drawn from
// max(p - q, 0) of the first row that refused its draft, or from p of the last
// row: the first j whose running sum of weights passes u * (sum of weights).
//
// Bound by reading the logits (and the draft's probabilities of one row per
// request).  All sums and exponentials are in 64 bits: the drawn token is an
// integer next to up to V borders of the running sum, and an FP32 sum of
// 248320 weights would move it past one in about a draw of a thousand.
//
//   1. verify_rows_kernel: slices of every row -> maximum, sum of exponentials;
//   2. verify_weigh_kernel: kept drafts per request; the sums of the weights of
//      its deciding row by slices;
//   3. verify_draw_kernel: the slice, then the token, that the number falls on.
#include <algorithm>

#include "device.hpp"
#include "verify.hpp"

namespace fp8lin {
namespace {

constexpr int kThreads = 256;

struct Args {
    const void* logits;
    int64_t ld;
    const float* probs;  // the draft's, or null: drafts without probabilities
    int64_t ldp, prob_rows;
    const int64_t* tokens;
    const float* u;
    const int32_t* offsets;
    const float* temperature;
    int B, slices, V, per;  // per: columns of a slice, a multiple of 8
    int64_t T;
    int32_t* accepted;
    int64_t* out;
    double* row_sum;    // [T][slices]
    float* row_max;     // [T][slices]
    int32_t* row_at;    // [T][slices] first column of the maximum
    double* weight;     // [B][slices][2] sums of max(p - q, 0) and of p
};

struct Request {
    int64_t a, n;  // first row, rows
};
__device__ __forceinline__ Request request(const Args& g, int b) {
    const int64_t lo = min(max((int64_t)g.offsets[b], (int64_t)0), g.T);
    const int64_t hi = min(max((int64_t)g.offsets[b + 1], lo), g.T);
    return Request{lo, hi - lo};
}

template <bool BF16>
__device__ __forceinline__ float logit(const Args& g, int64_t row, int64_t j) {
    if constexpr (BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(g.logits)[row * g.ld + j]);
    return static_cast<const float*>(g.logits)[row * g.ld + j];
}

// A temperature of zero (or below) stands for the most likely token.
__device__ __forceinline__ float temperature(const Args& g, int b) { return g.temperature ? g.temperature[b] : 1.0f; }
__device__ __forceinline__ bool greedy(float t) { return t <= 0.0f; }
__device__ __forceinline__ double slope(float t) { return greedy(t) ? 1.0 : 1.0 / (double)t; }

// e^((x - m) s), nothing for a logit of -inf; NaN for a NaN or a row of +inf.
__device__ __forceinline__ double weigh(float x, float m, double s) {
    return x == -__builtin_inff() ? 0.0 : exp(((double)x - (double)m) * s);
}

// Maximum, its first column and the sum of exponentials, joined.
struct Stat {
    float m;
    int at;
    double sum;
};
__device__ __forceinline__ void join(Stat& a, const Stat& b, double s) {
    const float m = fmaxf(a.m, b.m);
    const double fa = a.m == m ? 1.0 : a.m == -__builtin_inff() ? 0.0 : exp(((double)a.m - (double)m) * s);
    const double fb = b.m == m ? 1.0 : b.m == -__builtin_inff() ? 0.0 : exp(((double)b.m - (double)m) * s);
    // a part without finite logits has sum 0, or NaN that must stay
    a.sum = (a.sum == 0.0 ? 0.0 : a.sum * (a.sum != a.sum ? 1.0 : fa)) + (b.sum == 0.0 ? 0.0 : b.sum * (b.sum != b.sum ? 1.0 : fb));
    if (b.m > a.m || (b.m == a.m && b.at < a.at)) a.at = b.at;
    a.m = m;
}
__device__ __forceinline__ Stat lane_xor(const Stat& v, int d) {
    return Stat{__shfl_xor(v.m, d, 64), __shfl_xor(v.at, d, 64), __shfl_xor(v.sum, d, 64)};
}

__device__ __forceinline__ int owner_of(const Args& g, int64_t row) {
    int lo = 0, hi = g.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (g.offsets[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
}

// Workgroup (row, slice).  VEC: rows start on 16 bytes.
template <bool BF16, bool VEC>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(Args g) {
    __shared__ Stat part[kThreads / 64];
    const int64_t row = blockIdx.x;
    const int slice = blockIdx.y, tid = threadIdx.x;
    if (row >= g.offsets[g.B]) return;  // behind the last request
    const double s = slope(temperature(g, owner_of(g, row)));
    const int lo = slice * g.per, hi = min(lo + g.per, g.V);
    Stat v{-__builtin_inff(), INT32_MAX, 0.0};
    auto take = [&](const float (&x)[8], int j) {
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
        if (top > v.m) {
            if (v.m != -__builtin_inff()) v.sum *= exp(((double)v.m - (double)top) * s);
            v.m = top;
#pragma unroll
            for (int i = 7; i >= 0; --i)
                if (x[i] == top) v.at = j + i;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v.sum += weigh(x[i], v.m, s);
    };
    for (int j = lo + 8 * tid; j < hi; j += 8 * kThreads) {
        float x[8];
        if (VEC && j + 8 <= hi) {
            if constexpr (BF16) {
                const u32x4 w = load_u32x4(static_cast<const uint16_t*>(g.logits) + row * g.ld + j);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = bf16_bits_to_f32((w[i >> 1] >> (16 * (i & 1))) & 0xffffu);
            } else {
                const float* p = static_cast<const float*>(g.logits) + row * g.ld + j;
                const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = a[i];
                    x[4 + i] = b[i];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = j + i < hi ? logit<BF16>(g, row, j + i) : -__builtin_inff();
        }
        take(x, j);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) join(v, lane_xor(v, d), s);
    if ((tid & 63) == 0) part[tid >> 6] = v;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 64; ++w) join(v, part[w], s);
        const int64_t at = row * g.slices + slice;
        g.row_max[at] = v.m;
        g.row_at[at] = v.at;
        g.row_sum[at] = v.sum;
    }
}

// A row's statistics from its slices, by one wave; every lane gets them.
__device__ __forceinline__ Stat row_stat(const Args& g, int64_t row, double s) {
    const int lane = threadIdx.x & 63;
    Stat v{-__builtin_inff(), INT32_MAX, 0.0};
    for (int i = lane; i < g.slices; i += 64) {
        const int64_t at = row * g.slices + i;
        join(v, Stat{g.row_max[at], g.row_at[at], g.row_sum[at]}, s);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) join(v, lane_xor(v, d), s);
    return v;
}

// Whether the row is a distribution: some finite logit, no NaN, no +inf.
__device__ __forceinline__ bool valid(const Stat& v) { return v.sum > 0.0 && v.sum < __builtin_inf(); }

struct Decision {
    int64_t kept;   // accepted drafts; row a + kept decides the next token
    Stat stat;      // that row's
    int64_t probs;  // row of the draft's probabilities for the request's first draft
};

// The draft model's rows are those of all requests but their last ones: the
// request's first is a less the requests before it that have rows.
__device__ int64_t probs_row(const Args& g, int b, const Request& r) {
    int64_t before = 0;
    for (int i0 = 0; i0 < b; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        before += __syncthreads_count(i < b && request(g, i).n > 0);
    }
    return r.a - before;
}
__device__ __forceinline__ double draft_prob(const Args& g, int64_t row, int64_t j) {
    return row >= 0 && row < g.prob_rows ? (double)g.probs[row * g.ldp + j] : 0.0;
}

// By all threads of a workgroup: wave w tests drafts w, w + 4, ...
template <bool BF16>
__device__ Decision decide(const Args& g, int b, const Request& r) {
    __shared__ int first;
    __shared__ Stat stat;
    const int tid = threadIdx.x, wave = tid >> 6;
    const float t = temperature(g, b);
    const double s = slope(t);
    const int64_t probs = g.probs ? probs_row(g, b, r) : 0;
    if (tid == 0) first = (int)(r.n - 1);
    __syncthreads();
    for (int64_t i0 = 0; i0 < r.n - 1 && i0 <= first; i0 += kThreads / 64) {
        const int64_t i = i0 + wave;
        if (i < r.n - 1) {
            const Stat v = row_stat(g, r.a + i, s);
            const int64_t x = g.tokens[r.a + i + 1];
            bool keep = false;
            if (x >= 0 && x < g.V && valid(v)) {
                const double p = greedy(t) ? (v.at == x ? 1.0 : 0.0) : weigh(logit<BF16>(g, r.a + i, x), v.m, s) / v.sum;
                const double q = g.probs ? draft_prob(g, probs + i, x) : 1.0;
                keep = (double)g.u[r.a + i] * q < p;
            }
            if (!keep && (tid & 63) == 0) atomicMin(&first, (int)i);
        }
        __syncthreads();
    }
    const int64_t kept = first;
    if (wave == 0) {
        const Stat v = row_stat(g, r.a + kept, s);
        if (tid == 0) stat = v;
    }
    __syncthreads();
    return Decision{kept, stat, probs};
}

// The weight of column j in the deciding row, and its p.
template <bool BF16>
__device__ __forceinline__ double weight_at(const Args& g, const Request& r, const Decision& c, float t, double s,
                                            int64_t x, int j, double& p) {
    p = greedy(t) ? (j == c.stat.at ? 1.0 : 0.0) : weigh(logit<BF16>(g, r.a + c.kept, j), c.stat.m, s) / c.stat.sum;
    if (c.kept == r.n - 1) return p;
    if (!g.probs) return j == x ? 0.0 : p;
    return fmax(p - draft_prob(g, c.probs + c.kept, j), 0.0);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// Workgroup (request, slice).
template <bool BF16>
__global__ __launch_bounds__(kThreads) void verify_weigh_kernel(Args g) {
    __shared__ double ws[kThreads / 64], ps[kThreads / 64];
    const int b = blockIdx.x, slice = blockIdx.y, tid = threadIdx.x;
    const Request r = request(g, b);
    if (r.n == 0) return;
    const Decision c = decide<BF16>(g, b, r);
    const float t = temperature(g, b);
    const double s = slope(t);
    const int64_t x = c.kept < r.n - 1 ? g.tokens[r.a + c.kept + 1] : -1;
    const int lo = slice * g.per, hi = min(lo + g.per, g.V);
    double w = 0.0, p = 0.0;
    for (int j = lo + tid; j < hi; j += kThreads) {
        double pj;
        w += weight_at<BF16>(g, r, c, t, s, x, j, pj);
        p += pj;
    }
    w = wave_sum64(w);
    p = wave_sum64(p);
    if ((tid & 63) == 0) {
        ws[tid >> 6] = w;
        ps[tid >> 6] = p;
    }
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kThreads / 64; ++i) {
            w += ws[i];
            p += ps[i];
        }
        g.weight[((int64_t)b * g.slices + slice) * 2] = w;
        g.weight[((int64_t)b * g.slices + slice) * 2 + 1] = p;
    }
}

// One workgroup per request; the last one also clears the rows behind them.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(Args g) {
    __shared__ double run[kThreads], before_s;
    __shared__ int slice_s, pick_s, last_s;
    const int b = blockIdx.x, tid = threadIdx.x;
    const Request r = request(g, b);
    if (b == g.B - 1)
        for (int64_t i = r.a + r.n + tid; i < g.T; i += kThreads) g.out[i] = -1;
    if (r.n == 0) {
        if (tid == 0) g.accepted[b] = 0;
        return;
    }
    const Decision c = decide<BF16>(g, b, r);
    const float t = temperature(g, b);
    const double s = slope(t);
    const int64_t x = c.kept < r.n - 1 ? g.tokens[r.a + c.kept + 1] : -1;
    const bool ok = valid(c.stat);
    const double* weight = g.weight + (int64_t)b * g.slices * 2;
    if (tid == 0) {
        // nothing left where the target is not above the draft: p itself
        double total = 0.0;
        for (int i = 0; i < g.slices; ++i) total += weight[2 * i];
        const int of = total > 0.0 ? 0 : 1;
        if (of) {
            total = 0.0;
            for (int i = 0; i < g.slices; ++i) total += weight[2 * i + 1];
        }
        const double target = (double)g.u[r.a + r.n - 1] * total;
        double sum = 0.0, before = 0.0;
        int slice = 0;
        for (int i = 0; i < g.slices; ++i) {
            const double w = weight[2 * i + of];
            if (w > 0.0) {
                slice = i;
                before = sum;
            }
            sum += w;
            if (w > 0.0 && sum > target) break;
        }
        slice_s = 2 * slice + of;
        before_s = target - before;
        pick_s = INT32_MAX;
        last_s = -1;
    }
    __syncthreads();
    const int slice = slice_s >> 1, of = slice_s & 1;
    const double target = before_s;
    const int lo = slice * g.per, hi = min(lo + g.per, g.V), mine = g.per / kThreads + 1;
    const int j0 = min(lo + tid * mine, hi), j1 = min(j0 + mine, hi);
    double sum = 0.0;
    for (int j = j0; j < j1; ++j) {
        double p;
        const double w = weight_at<BF16>(g, r, c, t, s, x, j, p);
        sum += of ? p : w;
    }
    run[tid] = sum;
    __syncthreads();
    double before = 0.0;
    for (int i = 0; i < tid; ++i) before += run[i];
    int pick = INT32_MAX, last = -1;
    for (int j = j0; j < j1; ++j) {
        double p;
        const double w = weight_at<BF16>(g, r, c, t, s, x, j, p), v = of ? p : w;
        before += v;
        if (v > 0.0) {
            last = j;
            if (before > target && pick == INT32_MAX) pick = j;
        }
    }
    if (pick != INT32_MAX) atomicMin(&pick_s, pick);
    if (last >= 0) atomicMax(&last_s, last);
    __syncthreads();
    const int64_t token = !ok ? -1 : pick_s != INT32_MAX ? pick_s : last_s;
    for (int64_t i = tid; i < r.n; i += kThreads)
        g.out[r.a + i] = i < c.kept ? g.tokens[r.a + i + 1] : i == c.kept ? token : -1;
    if (tid == 0) g.accepted[b] = (int32_t)c.kept;
}

// Columns of a slice: enough slices to fill the chip, few enough to be joined
// by one wave in one go.
int slice_columns(int64_t T, int64_t V) {
    const int64_t want = std::min<int64_t>(64, std::max<int64_t>(1, 2048 / std::max<int64_t>(T, 1)));
    const int64_t per = std::max<int64_t>((V + want - 1) / want, 2048);
    return (int)((per + 7) / 8 * 8);
}

}  // namespace

size_t verify_ws_bytes(int64_t T, int64_t B, int64_t V) {
    const int64_t per = slice_columns(T, V), slices = (V + per - 1) / per;
    return (size_t)(T * slices * 16 + B * slices * 16);
}

hipError_t launch_verify(const void* logits, bool bf16, int64_t ld, const float* probs, int64_t ldp, int64_t prob_rows,
                         const int64_t* tokens, const float* u, const int32_t* offsets, const float* temperature, int64_t T,
                         int B, int V, int32_t* accepted, int64_t* out, void* ws, hipStream_t stream) {
    const int per = slice_columns(T, V), slices = (V + per - 1) / per;
    double* sums = static_cast<double*>(ws);
    double* weight = sums + T * slices;
    float* row_max = reinterpret_cast<float*>(weight + (int64_t)B * slices * 2);
    const Args g{logits, ld, probs, ldp, prob_rows, tokens, u, offsets, temperature, B, slices, V, per, T, accepted, out,
                 sums, row_max, reinterpret_cast<int32_t*>(row_max + T * slices), weight};
    const bool vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld % (bf16 ? 8 : 4) == 0;
    const dim3 rows((unsigned)T, slices), requests(B, slices), block(kThreads);
    if (T) {
        if (bf16) {
            if (vec) hipLaunchKernelGGL((verify_rows_kernel<true, true>), rows, block, 0, stream, g);
            else hipLaunchKernelGGL((verify_rows_kernel<true, false>), rows, block, 0, stream, g);
            hipLaunchKernelGGL(verify_weigh_kernel<true>, requests, block, 0, stream, g);
        } else {
            if (vec) hipLaunchKernelGGL((verify_rows_kernel<false, true>), rows, block, 0, stream, g);
            else hipLaunchKernelGGL((verify_rows_kernel<false, false>), rows, block, 0, stream, g);
            hipLaunchKernelGGL(verify_weigh_kernel<false>, requests, block, 0, stream, g);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (bf16) hipLaunchKernelGGL(verify_draw_kernel<true>, dim3(B), block, 0, stream, g);
    else hipLaunchKernelGGL(verify_draw_kernel<false>, dim3(B), block, 0, stream, g);
    return hipGetLastError();
}

}  // namespace fp8lin
