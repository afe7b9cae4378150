/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_rows_io.h - loads and stores of f32 and bf16 rows as floats, and the
 * division of work items by launch constants, for the kernels that handle
 * many tokens' rows (dsv4_rope.hip, dsv4_kvrows.hip, dsv4_tree.hip).
 * Included inside an anonymous namespace. */
#pragma once

typedef __bf16 io_v2bf __attribute__((ext_vector_type(2)));
typedef float io_v2f __attribute__((ext_vector_type(2)));

/* Two f32 -> two bf16, to nearest even (v_cvt_pk_bf16_f32). */
__device__ __forceinline__ uint32_t io_bf2(float a, float b)
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(io_v2f{a, b}, io_v2bf));
}

/* N consecutive elements as floats; 16 bytes or 8 at a time where N elements
 * are that many, at any address of an element (the target's loads and stores of
 * global memory need no more). */
template <class T, int N>
__device__ __forceinline__ void io_load(const T *p, float *v)
{
    constexpr bool BF = sizeof(T) == 2;
    if constexpr (!BF && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            f32x4 t;
            __builtin_memcpy(&t, p + i, 16);
            v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
        }
    } else if constexpr (BF && N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            u32x4 t;
            __builtin_memcpy(&t, p + i, 16);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[i + 2 * k] = __uint_as_float(t[k] << 16);
                v[i + 2 * k + 1] = __uint_as_float(t[k] & 0xFFFF0000u);
            }
        }
    } else if constexpr (BF && N == 4) {
        uint2 t;
        __builtin_memcpy(&t, p, 8);
        v[0] = __uint_as_float(t.x << 16); v[1] = __uint_as_float(t.x & 0xFFFF0000u);
        v[2] = __uint_as_float(t.y << 16); v[3] = __uint_as_float(t.y & 0xFFFF0000u);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (BF) v[i] = __uint_as_float((uint32_t)p[i] << 16);
            else v[i] = p[i];
        }
    }
}

template <class T, int N>
__device__ __forceinline__ void io_store(T *p, const float *v)
{
    constexpr bool BF = sizeof(T) == 2;
    if constexpr (!BF && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const f32x4 t{v[i], v[i + 1], v[i + 2], v[i + 3]};
            __builtin_memcpy(p + i, &t, 16);
        }
    } else if constexpr (BF && N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const u32x4 t{io_bf2(v[i], v[i + 1]), io_bf2(v[i + 2], v[i + 3]),
                          io_bf2(v[i + 4], v[i + 5]), io_bf2(v[i + 6], v[i + 7])};
            __builtin_memcpy(p + i, &t, 16);
        }
    } else if constexpr (BF && N == 4) {
        const uint2 t = make_uint2(io_bf2(v[0], v[1]), io_bf2(v[2], v[3]));
        __builtin_memcpy(p, &t, 8);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (BF) p[i] = (uint16_t)io_bf2(v[i], 0.0f);
            else p[i] = v[i];
        }
    }
}

/* n / d for 0 <= n < 2^31 and a launch constant 1 <= d < 2^31, without a
 * division: the high word of n times ceil(2^32 (2^s - d) / d) and a shift
 * (Granlund and Montgomery's method). */
struct IoDiv {
    uint32_t d, m, s;
    explicit IoDiv(uint32_t v) : d(v), m(0), s(0)
    {
        while ((1ull << s) < v) s++;
        m = (uint32_t)((((1ull << s) - v) << 32) / v + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const
    {
        return (__umulhi(m, n) + n) >> s;
    }
};
