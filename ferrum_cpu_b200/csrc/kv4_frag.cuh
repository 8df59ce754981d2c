// What the attention kernels on the 4-bit cache share: levels as matrix fragments, planes of f32 values, rows into the cache.
#pragma once
#include "kv4_ops.cuh"
#include "pdl.cuh"

namespace fc {

// Eight levels of a word as four registers of exact f16 pairs (nibbles i and i + 4), 0 <= i < 4. 1024 + n has n in its low bits,
// 1024 + 16 n four bits up.
__device__ __forceinline__ uint32_t sub8(uint32_t x) {
    const __half2 r = __hsub2(*(const __half2*)&x, __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408)));
    return *(const uint32_t*)&r;
}
__device__ __forceinline__ uint32_t sub8_16(uint32_t x) {
    const __half2 r = __hfma2(*(const __half2*)&x, __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00)),
                              __halves2half2(__ushort_as_half(0xd480), __ushort_as_half(0xd480)));   // x / 16 - 72
    return *(const uint32_t*)&r;
}
__device__ __forceinline__ void levels_of(uint32_t w, uint32_t (&f)[4]) {
    f[0] = sub8((w & 0x000f000fu) | 0x64006400u);
    f[1] = sub8_16((w & 0x00f000f0u) | 0x64006400u);
    w >>= 8;
    f[2] = sub8((w & 0x000f000fu) | 0x64006400u);
    f[3] = sub8_16((w & 0x00f000f0u) | 0x64006400u);
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Pairs of f16.
__device__ __forceinline__ uint32_t hmul2u(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*(const __half2*)&a, *(const __half2*)&b);
    return *(const uint32_t*)&r;
}
__device__ __forceinline__ uint32_t hfma2u(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*(const __half2*)&a, *(const __half2*)&b, *(const __half2*)&c);
    return *(const uint32_t*)&r;
}
// a b - c
__device__ __forceinline__ uint32_t hfms2u(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*(const __half2*)&a, *(const __half2*)&b, __hneg2(*(const __half2*)&c));
    return *(const uint32_t*)&r;
}
// x, y (below 2^14 in size) as two f16 planes: hi + lo holds 22 bits of each, or 2^-25 where that is more.
__device__ __forceinline__ void planes_of(float x, float y, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    *hi = *(const uint32_t*)&h;
    *lo = *(const uint32_t*)&l;
}
// Weights are kept times 2^6 and the scales they meet are brought to [2^7, 2^8): the product stays below 2^14, and what f16 cannot hold is
// 2^-31 of the largest weight and 2^-32 of the largest scale.
constexpr float kLift = 6.0f;
constexpr int kScaleLift = 7;
// 2^e, -126 <= e <= 127
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }
// The power of two that brings values of at most `top` (finite, >= 0) into [2^13, 2^14); 2^126 at most.
__device__ __forceinline__ int plane_shift(float top) {
    const int e = (__float_as_int(top) >> 23) & 255;
    return min(140 - e, 126);
}

__device__ __forceinline__ void cp16(void* smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// NB words that lie one after the other, in the widest loads their place allows.
template <int NB>
__device__ __forceinline__ void load_words(const uint32_t* p, uint32_t (&w)[NB]) {
    if (NB % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 4; ++i) {
            const uint4 v = ((const uint4*)p)[i];
            w[4 * i] = v.x; w[(4 * i + 1) % NB] = v.y; w[(4 * i + 2) % NB] = v.z; w[(4 * i + 3) % NB] = v.w;
        }
    } else if (NB % 2 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
            const uint2 v = ((const uint2*)p)[i];
            w[2 * i] = v.x; w[(2 * i + 1) % NB] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NB; ++i) w[i] = p[i];
    }
}
// The scales of one row.
template <int NB>
__device__ __forceinline__ void load_scales(const __half* p, float (&d)[NB]) {
    if (NB % 2 == 0) {
        uint32_t w[NB / 2 ? NB / 2 : 1];
        load_words(((const uint32_t*)p), w);
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
            const float2 f = __half22float2(*(const __half2*)&w[i]);
            d[2 * i] = f.x; d[(2 * i + 1) % NB] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NB; ++i) d[i] = __half2float(p[i]);
    }
}

// Four consecutive values a lane, eight lanes a block: the block's scale and the lane's levels plus 8. The quotient of two f32 never
// rounds onto a tie that it does not have (x has 24 bits, (k + 1/2) d at most 16: they differ by more than half a unit of the
// quotient), so rint of it is the nearest level of the exact quotient. NaN counts as 0 and infinities saturate the scale: whatever a
// row holds, the cache stays finite, and no masked position can hurt another.
__device__ __forceinline__ void quantize4(const float4& v, __half* d, int (&level)[4]) {
    float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = x[i] == x[i] ? x[i] : 0.0f;
    float hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    const float m = hi >= -lo ? hi : lo;
    *d = __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f));
    const float f = __half2float(*d);
#pragma unroll
    for (int i = 0; i < 4; ++i) level[i] = f == 0.0f ? 8 : 8 + (int)fminf(fmaxf(rintf(__fdiv_rn(x[i], f)), -8.0f), 7.0f);
}
// A row's words of keys: lane 8 q + c of a warp holds channels 4 c .. + 3 of block b = b0 + q. The even lanes of a block return
// word c / 2 of it.
__device__ __forceinline__ uint32_t key_word(const int (&level)[4], int lane) {
    uint32_t w = (uint32_t)(level[0] | level[1] << 4 | level[2] << 8 | level[3] << 12) << (16 * (lane & 1));
    return w | __shfl_xor_sync(0xffffffffu, w, 1);
}
// A row's half words of values: lanes c = 0 and 1 of a block return those of g = 4 c .. 4 c + 3 (two in a register).
__device__ __forceinline__ uint2 value_halves(const int (&level)[4], int lane) {
    const int at = 4 * ((lane & 7) >> 1);            // nibble j = c / 2
    uint2 w = make_uint2((uint32_t)level[0] << at | (uint32_t)level[1] << (16 + at), (uint32_t)level[2] << at | (uint32_t)level[3] << (16 + at));
#pragma unroll
    for (int o = 4; o > 1; o >>= 1) {
        w.x |= __shfl_xor_sync(0xffffffffu, w.x, o);
        w.y |= __shfl_xor_sync(0xffffffffu, w.y, o);
    }
    return w;
}

}  // namespace fc
