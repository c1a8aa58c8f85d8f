// Shared device code of the kernels on dense matrices (8-bit rows, norms, 8-bit product, distillation, AdamW): element types,
// chunks of eight elements, reductions over a wave and over the threads of a row.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "geo_sc.h"

namespace geo_sc {

using f32 = float;
using bf16 = __bf16;
using f16 = _Float16;

inline int dtype_bytes(int dtype) { return dtype == GEO_SC_F32 ? 4 : 2; }
inline bool dtype_known(int dtype) { return dtype == GEO_SC_F32 || dtype == GEO_SC_BF16 || dtype == GEO_SC_F16; }

// Eight consecutive elements, at any alignment that the element has: gfx950 reads and writes 16 bytes at any byte address,
// so odd row lengths and strides keep the wide accesses.
constexpr int kChunk = 8;

// ONCE: see reads_once().  (A choice at run time breaks the row of loads: 8191 x 4096 bf16 normed, both passes, 133 us, so 121.)
template <bool ONCE, typename T>
__device__ __forceinline__ void fetch_whole(const T* p, T (&raw)[kChunk])
{
    typedef int Piece __attribute__((ext_vector_type(4), aligned(2)));
    if constexpr (ONCE) {
#pragma unroll
        for (int i = 0; i < (int)sizeof raw / 16; ++i) {
            const Piece u = __builtin_nontemporal_load((const Piece*)p + i);
            __builtin_memcpy((char*)raw + 16 * i, &u, 16);
        }
    } else {
        __builtin_memcpy(raw, p, sizeof raw);
    }
}
template <bool ONCE = false, typename T>
__device__ __forceinline__ void load_chunk(const T* p, float (&v)[kChunk])
{
    T raw[kChunk];
    fetch_whole<ONCE>(p, raw);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) v[j] = (float)raw[j];
}
// the chunk at column c of a row of `cols` columns; `fill` behind the row's end
template <bool ONCE = false, typename T>
__device__ __forceinline__ void load_chunk(const T* row, int64_t c, int64_t cols, float fill, float (&v)[kChunk])
{
    if (c + kChunk <= cols) {
        load_chunk<ONCE>(row + c, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < kChunk; ++j) v[j] = c + j < cols ? (float)row[c + j] : fill;
}
// the same as it lies in memory, zeros behind the row's end: what is converted later need not be waited for at the load
template <bool ONCE, typename T>
__device__ __forceinline__ void fetch_chunk(const T* row, int64_t c, int64_t cols, T (&raw)[kChunk])
{
    if (c + kChunk <= cols) {
        fetch_whole<ONCE>(row + c, raw);
        return;
    }
#pragma unroll
    for (int j = 0; j < kChunk; ++j) raw[j] = c + j < cols ? row[c + j] : (T)0.f;
}
// `streamed`: past the caches, see streams()
template <typename T>
__device__ __forceinline__ void store_chunk(T* row, int64_t c, int64_t cols, const float (&v)[kChunk], bool streamed = false)
{
    typedef int Piece __attribute__((ext_vector_type(4), aligned(2)));
    T raw[kChunk];
#pragma unroll
    for (int j = 0; j < kChunk; ++j) raw[j] = (T)v[j];
    if (c + kChunk <= cols) {
        if (streamed) {
#pragma unroll
            for (int p = 0; p < (int)sizeof raw / 16; ++p) {
                Piece u;
                __builtin_memcpy(&u, (const char*)raw + 16 * p, 16);
                __builtin_nontemporal_store(u, (Piece*)(row + c) + p);
            }
        } else {
            __builtin_memcpy(row + c, raw, sizeof raw);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < kChunk; ++j)
        if (c + j < cols) row[c + j] = raw[j];
}
// Whether rows that a kernel reads once are read past what the caches hold for others.  8191 x 4096 bf16 normed, both passes, 161 us
// -> 121, 16384 x 4096 fp32 rows in 8 bits 82 -> 74.  Not where lines are shared by loads that straddle words (8192 x 2047 bf16,
// 136 -> 145), or by the two loads of a chunk of fp32 at odd places (8192 x 4095, 226 -> 237).
inline bool reads_once(int dtype, const void* p, int64_t stride)
{
    return !(((uintptr_t)p | (uint64_t)(stride * dtype_bytes(dtype))) % (dtype == GEO_SC_F32 ? 16 : 4));
}
// Whether a kernel's output goes past the caches.  What passes half of the 256 MB that the memory side caches is not found there by
// the next kernel anyway, and in them it drives out what is read: 8191 x 4096 bf16 rows normed (134 MB of sum and
// values) 88 us -> 74 (59 with what reads_once() says), the gradient of 4096 x 32768 logits (268 MB) 126 -> 117.  Smaller outputs stay for their reader.
inline bool streams(int64_t bytes) { return bytes >= (int64_t)128 << 20; }
// the same with the type known at run time only (one branch for all lanes)
__device__ __forceinline__ void store_chunk(void* base, int dtype, int64_t offset, int64_t c, int64_t cols, const float (&v)[kChunk],
                                            bool streamed)
{
    if (dtype == GEO_SC_F32) store_chunk((f32*)base + offset, c, cols, v, streamed);
    else if (dtype == GEO_SC_BF16) store_chunk((bf16*)base + offset, c, cols, v, streamed);
    else store_chunk((f16*)base + offset, c, cols, v, streamed);
}
__device__ __forceinline__ void load_chunk(const void* base, int dtype, int64_t offset, int64_t c, int64_t cols, float fill,
                                           float (&v)[kChunk])
{
    if (dtype == GEO_SC_F32) load_chunk((const f32*)base + offset, c, cols, fill, v);
    else if (dtype == GEO_SC_BF16) load_chunk((const bf16*)base + offset, c, cols, fill, v);
    else load_chunk((const f16*)base + offset, c, cols, fill, v);
}

// Calls launch(first, count) for consecutive shares of `groups` workgroups of `threads`: a launch counts its threads in 32 bits, and
// one of more starts what the count leaves of them, without an error.
template <typename F>
void in_launches(int64_t groups, int threads, F launch)
{
    const int64_t most = 0xffffffffll / threads;
    for (int64_t first = 0; first < groups; first += most) launch(first, (uint32_t)(groups - first < most ? groups - first : most));
}

// Bits of |v|: as unsigned integers they order like the magnitudes, with infinity above every number and NaN above infinity,
// so their maximum is the largest magnitude where all are numbers and says where one is not.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
constexpr uint32_t kInfinityBits = 0x7f800000u;

// Every lane receives the wave's result; the order of the additions is the same on every run.
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    return v;
}

// Sum and maximum over the `waves` waves that share a row, in one exchange through LDS.  `turn` alternates between two
// sets of slots, so that one barrier per call is enough where calls follow each other.
struct RowSlots {
    float sum[2][16];
    uint32_t most[2][16];
};
__device__ __forceinline__ void row_reduce(float& sum, uint32_t& most, int waves, RowSlots& slots, int turn)
{
    sum = wave_sum(sum);
    most = wave_max(most);
    if (waves == 1) return;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        slots.sum[turn & 1][wave] = sum;
        slots.most[turn & 1][wave] = most;
    }
    __syncthreads();
    float s = 0.f;
    uint32_t m = 0;
    for (int k = 0; k < waves; ++k) {
        s += slots.sum[turn & 1][k];
        m = max(m, slots.most[turn & 1][k]);
    }
    sum = s;
    most = m;
}

// Reciprocal and scale of a row from the bits of its largest magnitude.  `unit` multiplies the scale (r of a norm, else 1).
// A row that holds an infinity or NaN becomes q = 0 with scale NaN: its values are NaN.  Magnitudes below 2^-100 are
// brought up by 2^100 first, where 127 / a would pass the largest float.
struct RowScale {
    float lift, inverse, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t bits, float unit, bool sound)
{
    RowScale r;
    const float a = __uint_as_float(bits);
    r.lift = a < 0x1p-100f ? 0x1p100f : 1.f;
    r.inverse = a > 0.f ? 127.f / (a * r.lift) : 0.f;
    r.scale = a * unit * (1.f / 127.f);
    if (bits >= kInfinityBits || !sound) {
        r.inverse = 0.f;
        r.scale = __uint_as_float(0x7fc00000u);
    }
    return r;
}

// The chunk at column c of a row in 8 bits, and the values v that it then stands for.
__device__ __forceinline__ void store_eight(int8_t* row, int64_t c, int64_t cols, const RowScale& rs, const float (&n)[kChunk], float (&v)[kChunk])
{
    int8_t q[kChunk];
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
        // (a NaN's conversion to an integer is whatever the hardware makes of it: such rows write zeros)
        const float k = rs.inverse == 0.f ? 0.f : rintf(n[j] * rs.lift * rs.inverse);
        q[j] = (int8_t)(int)k;
        v[j] = k * rs.scale;
    }
    if (c + kChunk <= cols) {
        __builtin_memcpy(row + c, q, sizeof q);
    } else {
#pragma unroll
        for (int j = 0; j < kChunk; ++j)
            if (c + j < cols) row[c + j] = q[j];
    }
}

// The power of two that brings the largest magnitude, which is a number and not zero, to 1 .. 4 (denormals less far).
__device__ __forceinline__ float power_up(uint32_t peak)
{
    const int field = 254 - (int)(peak >> 23);
    return __uint_as_float((uint32_t)(field < 1 ? 1 : field > 253 ? 253 : field) << 23);
}
// Threads of a row with `chunks` chunks: whole waves, at most 1024, of which each has `held` chunks.
inline int threads_of_row(int64_t chunks, int held)
{
    const int64_t threads = ((chunks + held - 1) / held + 63) / 64 * 64;
    return threads < 1024 ? (int)threads : 1024;
}

}  // namespace geo_sc
