// Rotary positions: the host's frequency table, which travels in the kernel's parameter space, and the device code that rotates
// one head, shared by the operator of its own (rope.cu) and the writer of paged rows (pool.cu).
#pragma once
#include "internal.cuh"

struct mkv_rope {
    mkv_rope_desc desc;
    double freq[MKV_ROPE_MAX_DIMS / 2];  // radians per position
    double turns[MKV_ROPE_MAX_DIMS / 2]; // whole turns per position
    double m;                           // factor on cosine and sine
};

namespace mkv {

// What a launch carries: frequencies in turns per position, so that the whole turns of an angle can be taken off exactly before
// it is rounded to f32 (at position 1,000,000 an f32 angle is off by up to 0.03 radians).
struct RopeTab {
    double turns[MKV_ROPE_MAX_DIMS / 2];
    float m;
    uint32_t pairs; // rotated pairs, 0 = no rotation
    uint32_t interleaved;
    float sign; // -1: the transposed map
};
RopeTab rope_tab(const mkv_rope *r, bool backward);

// m * (cos, sin) of pair i at position p
__device__ __forceinline__ float2 rope_cs(const RopeTab &tab, uint32_t i, int32_t p) {
    const double t = (double)p * tab.turns[i];
    const float half_turns = 2.0f * (float)(t - rint(t)); // in [-1, 1]
    float s, c;
    sincospif(half_turns, &s, &c);
    return make_float2(tab.m * c, tab.m * tab.sign * s);
}

// Eight consecutive values as f32. VEC: 16-byte accesses.
template <bool VEC> __device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
    if constexpr (VEC) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = p[i];
    }
}
template <bool VEC> __device__ __forceinline__ void load8(const __half *p, float (&x)[8]) {
    if constexpr (VEC) {
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __half2float(p[i]);
    }
}
__device__ __forceinline__ void store1(float *p, float x) { *p = x; }
__device__ __forceinline__ void store1(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ float load1(const float *p) { return *p; }
__device__ __forceinline__ float load1(const __half *p) { return __half2float(*p); }
template <bool VEC> __device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
    if constexpr (VEC) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = x[i];
    }
}
template <bool VEC> __device__ __forceinline__ void store8(__half *p, const float (&x)[8]) {
    if constexpr (VEC) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = __float2half_rn(x[i]);
    }
}

// How the work of a head is cut into units of a thread; a unit holds both dims of its pairs, so that x and y may be the same memory.
//   ROPE_COPY: eight dims, none rotated; ROPE_HALF8: eight pairs (dims i.. and dims / 2 + i..), then eight dims a unit;
//   ROPE_INTER8: eight dims (four pairs or none); ROPE_ANY: one pair or one dim (odd sizes, strides or addresses).
enum { ROPE_COPY = 0, ROPE_HALF8 = 1, ROPE_INTER8 = 2, ROPE_ANY = 3 };
inline int rope_mode(uint32_t pairs, bool interleaved, uint32_t head_dim, bool aligned) {
    if (!aligned || head_dim % 8u != 0u) return ROPE_ANY;
    if (pairs == 0u) return ROPE_COPY;
    if (interleaved) return (2u * pairs) % 8u == 0u ? ROPE_INTER8 : ROPE_ANY;
    return pairs % 8u == 0u ? ROPE_HALF8 : ROPE_ANY;
}
__host__ __device__ inline uint32_t rope_units(int mode, uint32_t pairs, uint32_t head_dim) {
    return mode == ROPE_ANY ? head_dim - pairs : mode == ROPE_HALF8 ? head_dim / 8u - pairs / 8u : head_dim / 8u;
}
// One unit in two halves, so that the loads may be in flight while the cosines and sines are computed.
template <int MODE, class TI> __device__ __forceinline__ void rope_load(const TI *src, uint32_t u, uint32_t pairs, bool interleaved, float (&a)[8], float (&b)[8]) {
    if constexpr (MODE == ROPE_ANY) {
        if (u < pairs) {
            a[0] = load1(src + (interleaved ? 2u * u : u));
            b[0] = load1(src + (interleaved ? 2u * u + 1u : pairs + u));
        } else {
            a[0] = load1(src + pairs + u);
        }
    } else if constexpr (MODE == ROPE_HALF8) {
        const uint32_t nu = pairs / 8u;
        load8<true>(src + (u < nu ? 8u * u : 8u * (u + nu)), a);
        if (u < nu) load8<true>(src + pairs + 8u * u, b);
    } else {
        load8<true>(src + 8u * u, a);
    }
}
template <int MODE, class TO> __device__ __forceinline__ void rope_store(TO *dst, uint32_t u, uint32_t pairs, bool interleaved, const float2 *cs, float (&a)[8], float (&b)[8]) {
    if constexpr (MODE == ROPE_ANY) {
        if (u < pairs) {
            const float2 c = cs[u];
            store1(dst + (interleaved ? 2u * u : u), a[0] * c.x - b[0] * c.y);
            store1(dst + (interleaved ? 2u * u + 1u : pairs + u), a[0] * c.y + b[0] * c.x);
        } else {
            store1(dst + pairs + u, a[0]);
        }
    } else if constexpr (MODE == ROPE_HALF8) {
        const uint32_t nu = pairs / 8u;
        if (u < nu) {
            float y[8], z[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 c = cs[8u * u + i];
                y[i] = a[i] * c.x - b[i] * c.y;
                z[i] = a[i] * c.y + b[i] * c.x;
            }
            store8<true>(dst + 8u * u, y);
            store8<true>(dst + pairs + 8u * u, z);
        } else {
            store8<true>(dst + 8u * (u + nu), a);
        }
    } else {
        if (MODE == ROPE_INTER8 && 4u * u < pairs) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 c = cs[4u * u + i];
                const float y = a[2 * i] * c.x - a[2 * i + 1] * c.y, z = a[2 * i] * c.y + a[2 * i + 1] * c.x;
                a[2 * i] = y;
                a[2 * i + 1] = z;
            }
        }
        store8<true>(dst + 8u * u, a);
    }
}

} // namespace mkv
