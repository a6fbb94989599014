// Host-side arguments of the rotation kernels (rotate.hip).
#pragma once
#include "paged.hpp"

namespace fp8lin {

// Heads [T, heads, D] (BF16, strides in elements, the last dimension
// contiguous).
struct Heads {
    const uint16_t* x;
    int64_t tok, head;
    int n;
};

struct Rotation {
    const uint64_t* steps;  // [half]; null: nothing is rotated
    const int64_t* positions;
    int64_t axis;  // elements between the positions of two axes
    int axes;      // a pair whose axis is not there takes the last one
    int half;
    bool neighbours;
    float magnitude, sign;  // sign -1: the transposed rotation
};

// x's heads rotated into y.
struct Rotate {
    Heads x;
    uint16_t* y;
    int64_t y_tok, y_head;
    Rotation r;
    int64_t T;
    int D;
};
hipError_t launch_rotate(const Rotate& a, hipStream_t stream);

// q, normed and rotated, into y; k, normed and rotated, and v into their slots.
struct RotateAppend {
    Heads q, k, v;
    uint16_t* y;
    int64_t y_tok, y_head;
    const uint16_t *q_norm, *k_norm;  // [D] or null
    float eps, center;                // center: 1 if weights are offsets from 1
    Rotation r;
    PagedCache kc, vc;
    const float *k_scale, *v_scale;  // [HK] of an 8-bit cache, or null
    uint8_t *k_pow, *v_pow;          // E8M0 [pages, page_size / block, HK], or null
    const int64_t* slots;
    int64_t T, limit;  // tokens; slots of the cache
    int D, page_bits, block_bits;
    bool fp8;
};
hipError_t launch_rotate_append(const RotateAppend& a, hipStream_t stream);

}  // namespace fp8lin
