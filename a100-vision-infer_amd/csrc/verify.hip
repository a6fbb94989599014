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
//      its deciding row by slices.  Without draft probabilities (q = 1 at the
//      draft) those are the first kernel's, which leaves the row's draft out of
//      its sums then, and this one is not run;
//   3. verify_draw_kernel: the slice, then the token, that the number falls on.
// 48 requests, 170 rows of 248320, with probabilities: 48 us (FP64 exponentials;
// 84 MB), 28 us and 12 us.  Without: 192 rows 71 us a call (83 with the second
// kernel), one row of each of 256 requests 82 (162), 4 rows of one request 6 and
// 11 us (latency; 17 us a call, 22).
#include <algorithm>

#include "device.hpp"
#include "verify.hpp"

namespace fp8lin {
namespace {

constexpr int kThreads = 256;

struct Decision;

struct Args {
    const void* logits;
    int64_t ld;
    const float* probs;  // the draft's, or null: drafts without probabilities
    int64_t ldp, prob_rows;
    const int64_t* tokens;
    const float* u;
    const int32_t* offsets;
    const float* temperature;
    int B, V;
    int slices, per;    // of a row; per: columns of a slice, a multiple of 8
    int cuts, cut_per;  // of a request's deciding row
    int64_t T;
    int32_t* accepted;
    int64_t* out;
    double* row_sum;    // [T][slices]; without draft probabilities: without the row's draft
    float* row_max;     // [T][slices]
    int32_t* row_at;    // [T][slices] first column of the maximum
    double* weight;     // [B][cuts][2] sums of max(p - q, 0) and of p
    Decision* decision;  // [B], by verify_weigh_kernel
};

struct Request {
    int64_t a, n;  // first row, rows
};
__device__ __forceinline__ Request request(const Args& g, int b) {
    const int64_t lo = min(max((int64_t)g.offsets[b], (int64_t)0), g.T);
    const int64_t hi = min(max((int64_t)g.offsets[b + 1], lo), g.T);
    return Request{lo, hi - lo};
}

// A temperature of zero (or below) stands for the most likely token.
__device__ __forceinline__ float temperature(const Args& g, int b) { return g.temperature ? g.temperature[b] : 1.0f; }
__device__ __forceinline__ bool greedy(float t) { return t <= 0.0f; }
__device__ __forceinline__ double slope(float t) { return 1.4426950408889634074 / (greedy(t) ? 1.0 : (double)t); }

// 2^t for t <= 0 in 64 bits, nothing below 2^-1100 (and for NaN): 2^n 2^f,
// |f| <= 1/2, 2^f = sum (f ln 2)^k / k! to k = 11: the next term is up to
// 6.3e-15 of a value near 0.7, a relative error of at most 9e-15 with the
// roundings (8.6e-15, at f = -1/2), which moves a draw among 250 000 tokens with
// a probability below 3e-9.  20 instructions without a branch, where the
// library's exp takes 65: the rows of a batch of 48 requests (170 x 248320)
// 78 -> 48 us.
// The coefficients stay in scalar registers (laundered, or the compiler would
// load each into a vector register before every use).
struct Exp2 {
    double c[12];
    __device__ Exp2() {
        constexpr double ln2 = 0.693147180559945309417;
        double v = 1.0;
#pragma unroll
        for (int k = 0; k < 12; ++k) {
            c[k] = v;
            v *= ln2 / (k + 1);
        }
#pragma unroll
        for (int k = 0; k < 12; ++k) asm("" : "+s"(c[k]));
    }
    __device__ __forceinline__ double operator()(double t) const {
        t = fmax(t, -1100.0);
        const double n = __builtin_rint(t), f = t - n;
        double p = c[11];
#pragma unroll
        for (int k = 10; k >= 0; --k) p = __builtin_fma(p, f, c[k]);
        return __builtin_ldexp(p, (int)n);
    }
};
// e^((x - m) / T) with s = log2(e) / T; nothing for x of -inf (m finite) or
// NaN.  The difference first: logits may be far larger than their differences.
__device__ __forceinline__ double weigh(const Exp2& e, float x, float m, double s) { return e(((double)x - (double)m) * s); }

// Maximum, its first column and the sum of exponentials of a part of a row:
// maximum -inf and sum 0 for a part of nothing but -inf, sum NaN for one that
// holds a NaN or +inf.
struct Stat {
    float m;
    int at;
    double sum;
};
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}
// The statistics of a wave's 64 parts; every lane gets them.
__device__ __forceinline__ Stat wave_join(const Exp2& e, const Stat& v, double s) {
    Stat r = v;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const float m = __shfl_xor(r.m, d, 64);
        const int at = __shfl_xor(r.at, d, 64);
        if (m > r.m || (m == r.m && at < r.at)) {
            r.m = m;
            r.at = at;
        }
    }
    r.sum = wave_sum64(v.sum == 0.0 || v.sum != v.sum ? v.sum : v.sum * weigh(e, v.m, r.m, s));
    return r;
}

__device__ __forceinline__ int owner_of(const Args& g, int64_t row) {
    int lo = 0, hi = g.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (g.offsets[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
}

// 8 values of a row from column j, `fill` behind `end`.  VEC: rows start on 16
// bytes (and j is a multiple of 8).
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int j, int end, float fill, float (&x)[8]) {
    if (VEC && j + 8 <= end) {
        if constexpr (sizeof(T) == 2) {
            const u32x4 w = load_u32x4(row + j);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = bf16_bits_to_f32((w[i >> 1] >> (16 * (i & 1))) & 0xffffu);
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4*>(row + j), b = *reinterpret_cast<const f32x4*>(row + j + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = a[i];
                x[4 + i] = b[i];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // a column past the end loads the last one instead, so that all loads are in flight
            const T v = row[min(j + i, end - 1)];
            float f;
            if constexpr (sizeof(T) == 2) f = bf16_bits_to_f32(v);
            else f = v;
            x[i] = j + i < end ? f : fill;
        }
    }
}

// Workgroup (row, slice).  DIRECT: without draft probabilities.
template <class T, bool VEC, bool DIRECT>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(Args g) {
    __shared__ Stat part[kThreads / 64];
    const int64_t row = blockIdx.x;
    const int slice = blockIdx.y, tid = threadIdx.x;
    if (row < g.offsets[0] || row >= g.offsets[g.B]) return;  // of no request
    const int b = owner_of(g, row);
    const double s = slope(temperature(g, b));
    const Request r = request(g, b);
    const int64_t draft = DIRECT && row + 1 < r.a + r.n ? g.tokens[row + 1] : -1;
    const int x_col = draft >= 0 && draft < g.V ? (int)draft : -1;
    const int lo = slice * g.per, hi = min(lo + g.per, g.V);
    const T* logits = static_cast<const T*>(g.logits) + row * g.ld;
    const Exp2 e;
    Stat v{-__builtin_inff(), INT32_MAX, 0.0};
    bool bad = false;
    for (int j = lo + 8 * tid; j < hi; j += 8 * kThreads) {
        float x[8];
        load8<T, VEC>(logits, j, hi, -__builtin_inff(), x);
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
        if (top > v.m) {
            v.sum *= v.sum == 0.0 ? 0.0 : weigh(e, v.m, top, s);
            v.m = top;
#pragma unroll
            for (int i = 7; i >= 0; --i)
                if (x[i] == top) v.at = j + i;
        }
        const float m = v.m == -__builtin_inff() ? 0.0f : v.m;
#pragma unroll
        for (int i = 0; i < 8; ++i) bad |= x[i] != x[i];
        if (DIRECT && (unsigned)(x_col - j) < 8u)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i == x_col) x[i] = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 8; ++i) v.sum += weigh(e, x[i], m, s);
    }
    if (bad || v.m == __builtin_inff()) v.sum = __builtin_nan("");
    v = wave_join(e, v, s);
    if ((tid & 63) == 0) part[tid >> 6] = v;
    __syncthreads();
    if (tid < 64) {
        v = wave_join(e, tid < kThreads / 64 ? part[tid] : Stat{-__builtin_inff(), INT32_MAX, 0.0}, s);
        if (tid == 0) {
            const int64_t at = row * g.slices + slice;
            g.row_max[at] = v.m;
            g.row_at[at] = v.at;
            g.row_sum[at] = v.sum;
        }
    }
}

// A row's statistics from its slices (at most 64), by one wave.
__device__ __forceinline__ Stat row_stat(const Args& g, const Exp2& e, int64_t row, double s) {
    const int lane = threadIdx.x & 63;
    const int64_t at = row * g.slices + min(lane, g.slices - 1);
    Stat v{g.row_max[at], g.row_at[at], g.row_sum[at]};
    if (lane >= g.slices) v = Stat{-__builtin_inff(), INT32_MAX, 0.0};
    return wave_join(e, v, s);
}

// Whether the row is a distribution: some finite logit, no NaN, no +inf.
__device__ __forceinline__ bool valid(const Stat& v) { return v.sum > 0.0 && v.sum < __builtin_inf(); }

struct Decision {
    int64_t kept;   // accepted drafts; row a + kept decides the next token
    Stat stat;      // that row's, the sum of all columns
    double draft;   // the exponential of its draft
    int64_t probs;  // row of the draft's probabilities for the request's first draft
};

// The draft model's rows are those of all requests but their last ones: the
// request's first is a, less the rows before the first request and the requests
// before it that have rows.
__device__ int64_t probs_row(const Args& g, int b, const Request& r) {
    int64_t before = 0;
    for (int i0 = 0; i0 < b; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        before += __syncthreads_count(i < b && request(g, i).n > 0);
    }
    return r.a - request(g, 0).a - before;
}

// By all threads of a workgroup: wave w tests drafts w, w + 4, ...
template <class T>
__device__ Decision decide(const Args& g, int b, const Request& r) {
    constexpr int kWaves = kThreads / 64;
    __shared__ int first;
    __shared__ Stat stats[kWaves];
    __shared__ double drafts[kWaves];
    const int tid = threadIdx.x, wave = tid >> 6;
    const float t = temperature(g, b);
    const double s = slope(t);
    const Exp2 e;
    const int64_t probs = g.probs ? probs_row(g, b, r) : 0;
    if (tid == 0) first = (int)(r.n - 1);
    __syncthreads();
    // the row behind the last draft refuses nothing: it ends the loop
    for (int64_t i0 = 0;; i0 += kWaves) {
        const int64_t i = i0 + wave;
        if (i < r.n) {
            const int64_t row = r.a + i, x = i < r.n - 1 ? g.tokens[row + 1] : -1;
            const bool in = x >= 0 && x < g.V;
            const T* logits = static_cast<const T*>(g.logits) + row * g.ld;
            float at;
            if constexpr (sizeof(T) == 2) at = bf16_bits_to_f32(logits[in ? x : 0]);
            else at = logits[in ? x : 0];
            const int64_t qr = probs + i;
            const bool given = !g.probs || (qr >= 0 && qr < g.prob_rows);
            const double q = g.probs && in && given ? (double)g.probs[qr * g.ldp + x] : 1.0;
            const double u = (double)g.u[row];
            Stat v = row_stat(g, e, row, s);
            const double at_x = in ? weigh(e, at, v.m == -__builtin_inff() ? 0.0f : v.m, s) : 0.0;
            if (!g.probs) v.sum += at_x;
            const double p = greedy(t) ? (v.at == x ? 1.0 : 0.0) : at_x / v.sum;
            const bool keep = in && given && valid(v) && u * q < p;
            if ((tid & 63) == 0) {
                stats[wave] = v;
                drafts[wave] = at_x;
                if (!keep) atomicMin(&first, (int)i);
            }
        }
        __syncthreads();
        if (first < i0 + kWaves) break;
    }
    return Decision{first, stats[first % kWaves], drafts[first % kWaves], probs};
}

// The weights of 8 columns in the deciding row: max(p - q, 0) in w, and p.
template <class T, bool VEC>
struct Weights {
    Exp2 e;
    const T* logits;
    const float* q;
    float m;
    double s, scale;
    int at;      // the column of all weight, or -1
    int64_t x;   // the refused draft without probabilities, or -1
    bool q_vec;

    __device__ Weights(const Args& g, int b, const Request& r, const Decision& c) {
        const float t = temperature(g, b);
        const bool refused = c.kept < r.n - 1;
        const int64_t qr = c.probs + c.kept;
        logits = static_cast<const T*>(g.logits) + (r.a + c.kept) * g.ld;
        q = refused && g.probs && qr >= 0 && qr < g.prob_rows ? g.probs + qr * g.ldp : nullptr;
        q_vec = reinterpret_cast<uintptr_t>(q) % 16 == 0;
        x = refused && !g.probs ? g.tokens[r.a + c.kept + 1] : -1;
        m = c.stat.m;
        s = slope(t);
        scale = 1.0 / c.stat.sum;
        at = greedy(t) ? c.stat.at : -1;
    }
    __device__ __forceinline__ void get(int j, int end, double (&w)[8], double (&p)[8]) const {
        float lx[8], qx[8];
        load8<T, VEC>(logits, j, end, -__builtin_inff(), lx);
        if (q) {
            if (q_vec) load8<float, true>(q, j, end, 0.0f, qx);
            else load8<float, false>(q, j, end, 0.0f, qx);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = at >= 0 ? (j + i == at ? 1.0 : 0.0) : weigh(e, lx[i], m, s) * scale;
            w[i] = q ? fmax(p[i] - (double)qx[i], 0.0) : j + i == x ? 0.0 : p[i];
        }
    }
};

// Workgroup (request, slice).
template <class T, bool VEC>
__global__ __launch_bounds__(kThreads) void verify_weigh_kernel(Args g) {
    __shared__ double ws[kThreads / 64], ps[kThreads / 64];
    const int b = blockIdx.x, slice = blockIdx.y, tid = threadIdx.x;
    const Request r = request(g, b);
    if (r.n == 0) return;
    const Decision c = decide<T>(g, b, r);
    if (slice == 0 && tid == 0) g.decision[b] = c;
    const Weights<T, VEC> weights(g, b, r, c);
    const int lo = min(slice * g.cut_per, g.V), hi = min(lo + g.cut_per, g.V);
    double w = 0.0, p = 0.0;
    for (int j = lo + 8 * tid; j < hi; j += 8 * kThreads) {
        double w8[8], p8[8];
        weights.get(j, hi, w8, p8);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w += w8[i];
            p += p8[i];
        }
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
        g.weight[((int64_t)b * g.cuts + slice) * 2] = w;
        g.weight[((int64_t)b * g.cuts + slice) * 2 + 1] = p;
    }
}

// Running sums over the lanes of a wave.
__device__ __forceinline__ double wave_scan64(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(v, d, 64);
        if ((threadIdx.x & 63) >= d) v += o;
    }
    return v;
}

// One workgroup per request; the first and last ones also clear the rows before
// and behind them.
// DIRECT: without draft probabilities; the slices are the rows'.
template <class T, bool VEC, bool DIRECT>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(Args g) {
    __shared__ double wave_total[kThreads / 64], target_s;
    __shared__ int slice_s, pick_s, last_s;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Request r = request(g, b);
    if (b == 0)
        for (int64_t i = tid; i < r.a; i += kThreads) g.out[i] = -1;
    if (b == g.B - 1)
        for (int64_t i = r.a + r.n + tid; i < g.T; i += kThreads) g.out[i] = -1;
    if (r.n == 0) {
        if (tid == 0) g.accepted[b] = 0;
        return;
    }
    Decision c;
    if constexpr (DIRECT) c = decide<T>(g, b, r);
    else c = g.decision[b];
    const Weights<T, VEC> weights(g, b, r, c);
    const int cuts = DIRECT ? g.slices : g.cuts, per = DIRECT ? g.per : g.cut_per;
    if (wave == 0) {
        // a lane per slice; p itself where the target is nowhere above the draft
        double w = 0.0, p = 0.0;
        if constexpr (DIRECT) {
            const int64_t at = (r.a + c.kept) * cuts + min(lane, cuts - 1);
            const double sum = g.row_sum[at];
            const float top = g.row_max[at];
            const int64_t lo = (int64_t)lane * per;
            auto holds = [&](int64_t j) { return j >= lo && j < lo + per; };
            if (weights.at >= 0) {
                p = holds(weights.at) ? 1.0 : 0.0;
                w = weights.at == weights.x ? 0.0 : p;
            } else if (lane < cuts) {
                w = sum == 0.0 ? 0.0 : sum * weigh(weights.e, top, weights.m, weights.s) * weights.scale;
                p = weights.x >= 0 && holds(weights.x) ? w + c.draft * weights.scale : w;
            }
        } else if (lane < cuts) {
            const double* weight = g.weight + ((int64_t)b * cuts + lane) * 2;
            w = weight[0];
            p = weight[1];
        }
        const int of = __ballot(w > 0.0) ? 0 : 1;
        if (of) w = p;
        const double run = wave_scan64(w), target = (double)g.u[r.a + r.n - 1] * __shfl(run, 63, 64);
        const uint64_t some = __ballot(w > 0.0), past = __ballot(w > 0.0 && run > target);
        const int slice = past ? __ffsll((unsigned long long)past) - 1 : some ? 63 - __clzll((long long)some) : 0;
        const double before = __shfl(run - w, slice, 64);
        if (lane == 0) {
            slice_s = 2 * slice + of;
            target_s = target - before;
            pick_s = INT32_MAX;
            last_s = -1;
        }
    }
    __syncthreads();
    const int slice = slice_s >> 1, of = slice_s & 1;
    const double target = target_s;
    const int lo = min(slice * per, g.V), hi = min(lo + per, g.V);
    double base = 0.0;
    int pick = INT32_MAX, last = -1;
    for (int j0 = lo; j0 < hi; j0 += 8 * kThreads) {
        const int j = j0 + 8 * tid;
        double w8[8], p8[8], sum = 0.0;
        if (j < hi) {
            weights.get(j, hi, w8, p8);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += of ? p8[i] : w8[i];
        }
        const double run = wave_scan64(sum);
        if (lane == 63) wave_total[wave] = run;
        __syncthreads();
        double before = base + run - sum;
        for (int w = 0; w < kThreads / 64; ++w) {
            if (w < wave) before += wave_total[w];
            base += wave_total[w];
        }
        if (j < hi) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double v = of ? p8[i] : w8[i];
                before += v;
                if (v > 0.0) {
                    last = j + i;
                    if (before > target && pick == INT32_MAX) pick = j + i;
                }
            }
        }
        __syncthreads();
        if (base > target) break;  // by all threads: what follows is behind the token
    }
    if (pick != INT32_MAX) atomicMin(&pick_s, pick);
    if (last >= 0) atomicMax(&last_s, last);
    __syncthreads();
    const int64_t token = !valid(c.stat) ? -1 : pick_s != INT32_MAX ? pick_s : last_s;
    for (int64_t i = tid; i < r.n; i += kThreads)
        g.out[r.a + i] = i < c.kept ? g.tokens[r.a + i + 1] : i == c.kept ? token : -1;
    if (tid == 0) g.accepted[b] = (int32_t)c.kept;
}

// Columns of a slice of one of `rows` rows: enough slices to fill the chip, few
// enough to be joined by one wave in one go (64).
int slice_columns(int64_t rows, int64_t V, int64_t least = 1) {
    const int64_t want = std::min<int64_t>(64, std::max<int64_t>(least, 2048 / std::max<int64_t>(rows, 1)));
    const int64_t per = std::max<int64_t>((V + want - 1) / want, 2048);
    return (int)((per + 7) / 8 * 8);
}
// Without draft probabilities one workgroup goes through a slice of a row in
// the draw: 24 at the least (192 rows of 248320: 84 us a call with 11, 71 with
// 24, 72 with 48; with probabilities more than the chip holds only cost).
constexpr int64_t kDirectSlices = 24;
int64_t slices_of(int64_t V, int per) { return (V + per - 1) / per; }

template <class T, bool VEC>
hipError_t run(const Args& g, hipStream_t stream) {
    const dim3 block(kThreads);
    if (g.T) {
        if (g.probs) hipLaunchKernelGGL((verify_rows_kernel<T, VEC, false>), dim3((unsigned)g.T, g.slices), block, 0, stream, g);
        else hipLaunchKernelGGL((verify_rows_kernel<T, VEC, true>), dim3((unsigned)g.T, g.slices), block, 0, stream, g);
        if (g.probs) hipLaunchKernelGGL((verify_weigh_kernel<T, VEC>), dim3(g.B, g.cuts), block, 0, stream, g);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (g.probs) hipLaunchKernelGGL((verify_draw_kernel<T, VEC, false>), dim3(g.B), block, 0, stream, g);
    else hipLaunchKernelGGL((verify_draw_kernel<T, VEC, true>), dim3(g.B), block, 0, stream, g);
    return hipGetLastError();
}

}  // namespace

size_t verify_ws_bytes(int64_t T, int64_t B, int64_t V) {
    return (size_t)(T * slices_of(V, slice_columns(T, V, kDirectSlices)) * 16 + B * slices_of(V, slice_columns(B, V)) * 16 +
                    B * (int64_t)sizeof(Decision));
}

hipError_t launch_verify(const void* logits, bool bf16, int64_t ld, const float* probs, int64_t ldp, int64_t prob_rows,
                         const int64_t* tokens, const float* u, const int32_t* offsets, const float* temperature, int64_t T,
                         int B, int V, int32_t* accepted, int64_t* out, void* ws, hipStream_t stream) {
    Args g{};
    g.logits = logits, g.ld = ld, g.probs = probs, g.ldp = ldp, g.prob_rows = prob_rows;
    g.tokens = tokens, g.u = u, g.offsets = offsets, g.temperature = temperature;
    g.B = B, g.V = V, g.T = T, g.accepted = accepted, g.out = out;
    g.per = slice_columns(T, V, probs ? 1 : kDirectSlices), g.slices = (int)slices_of(V, g.per);
    g.cut_per = slice_columns(B, V), g.cuts = (int)slices_of(V, g.cut_per);
    g.row_sum = static_cast<double*>(ws);
    g.weight = g.row_sum + T * g.slices;
    g.decision = reinterpret_cast<Decision*>(g.weight + (int64_t)B * g.cuts * 2);
    g.row_max = reinterpret_cast<float*>(g.decision + B);
    g.row_at = reinterpret_cast<int32_t*>(g.row_max + T * g.slices);
    const bool vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld % (bf16 ? 8 : 4) == 0;
    return bf16 ? (vec ? run<uint16_t, true>(g, stream) : run<uint16_t, false>(g, stream))
                : (vec ? run<float, true>(g, stream) : run<float, false>(g, stream));
}

}  // namespace fp8lin
