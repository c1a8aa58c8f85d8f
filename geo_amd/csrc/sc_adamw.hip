// One AdamW step on many tensors.
//
//   g = grad s,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  r = sqrt(v)
//   p = p (1 - lr wd) - (m lr / (1 - b1^t)) / (r / sqrt(1 - b2^t) + eps)
//
// Everything in fp32, each operation rounded by itself (no fused multiply-add), so that a program of elementary operations has the
// same bits.  Bound by memory, each element is read and written once: 139.6M fp32 masters with bf16 gradients and copies, 3.9 GB, in 764 us
// (5.1 TB/s), 120M of them with 8-bit states, 1.9 GB, in 370 (5.2 TB/s; decoding, root, quotient and rounding are some 110 instructions an element
// there, 0.9 of that time by themselves).  15 tensors of 2.1M elements in all with 8-bit states 11.4 us, 12 small ones 5.9.
//
// States of 8 bits: m and r as floats of 4 exponent and 3 mantissa bits, times a power of two per block of 256 elements.  The root and
// not v, which would need twice the exponents.  A power of two, because codes then stay what they are when a
// block's largest number moves within its octave; any other scale would round all of them anew in every step.  Three bits of
// mantissa alone would freeze the states: with b2 = 0.999 a step moves r by 1 / 2000 of itself, a code is 1 / 16 to 1 / 8, and to
// the nearest it would stay where it is until a gradient of eleven times r comes.  So a number goes up with the probability of its place
// between two codes, by a sequence that is even over the places of a block and over the steps (multiples of two irrational
// numbers, modulo one): the mean is right, the same inputs give the same bits, and no random numbers have to be kept.
#include "sc_dense.h"

#include <math.h>

#include <type_traits>

#pragma clang fp contract(off)

namespace geo_sc {
namespace {

constexpr int kTensors = 48;                   // of a launch: their descriptions fill the 4 KB of a launch's arguments
constexpr int kBlock = 256;                    // elements that share a scale: half a wave's chunks
constexpr int kThreads = 256, kTile = kThreads * kChunk;   // elements of a workgroup
static_assert(kBlock == 32 * kChunk, "a block is half a wave");

struct Steps {   // what depends on the number of the step
    float size, inverse_root;   // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    uint32_t number;            // t
};
struct Constants {
    float scale, b1, c1, b2, c2, keep, eps, lo, hi;
    int copy_dtype;
    Steps steps;
    const Steps* device_steps;   // or NULL
    bool streamed;               // what is written
};
struct Tensor {
    void* param;
    const void* grad;
    void *avg, *sq;
    uint8_t *avg_scale, *sq_scale;
    void* copy;
    float* clamped;
    int64_t elements;
};
struct Share {
    Constants c;
    int count;
    uint32_t first[kTensors];   // workgroup
    Tensor tensors[kTensors];
};
static_assert(sizeof(Share) <= 4096, "the arguments of a launch");
static_assert(kTensors <= 64, "a lane for each tensor");

__host__ __device__ inline Steps steps_at(double lr, double b1, double b2, int64_t t)
{
    return {(float)(lr / (1.0 - pow(b1, (double)t))), (float)(1.0 / sqrt(1.0 - pow(b2, (double)t))), (uint32_t)t};
}
static_assert(sizeof(Steps) <= 16, "the workspace");

__global__ void k_adamw_count(int64_t* step, double lr, double b1, double b2, Steps* to)
{
    *to = steps_at(lr, b1, b2, ++*step);
}

// the largest over the 32 lanes of a block
__device__ __forceinline__ uint32_t block_max(uint32_t v)
{
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    return v;
}
// A scale's byte is the exponent field of a float; 0 is half of the smallest normal one, 255 no number.
__device__ __forceinline__ float scale_of(uint8_t byte) { return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : (uint32_t)byte << 23); }
__device__ __forceinline__ void decode(const uint8_t (&codes)[kChunk], float (&v)[kChunk])
{
#ifdef __HIP_DEVICE_COMPILE__
    uint32_t words[2];
    __builtin_memcpy(words, codes, sizeof words);
#pragma unroll
    for (int j = 0; j < kChunk; j += 2) {
        const auto two = j & 2 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)words[j / 4], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)words[j / 4], false);
        v[j] = two[0];
        v[j + 1] = two[1];
    }
#endif
}
// The code of v >= 0, up to 256; `dither` of 2^32 is the fraction of a step from which on it goes up.
__device__ __forceinline__ uint32_t encode(float v, uint32_t dither)
{
    const bool tiny = v < 0x1p-6f;   // steps of 2^-9: those that 2^-6 .. 2^-5 has
    const uint32_t up = __float_as_uint(tiny ? v + 0x1p-6f : v) + (dither >> 12);
    return (up >> 20) - (tiny ? 121 * 8 : 120 * 8);
}

// The states of a chunk.  `block`: the tensor's block that the lane's chunk is in; `place`: the chunk's first element in it.
template <int BITS>
struct States;
template <>
struct States<32> {
    float m[kChunk], v[kChunk];
    template <bool ONCE>
    __device__ __forceinline__ void load(const Tensor& t, int64_t c)
    {
        load_chunk<ONCE>((const float*)t.avg, c, t.elements, 0.f, m);
        load_chunk<ONCE>((const float*)t.sq, c, t.elements, 0.f, v);
    }
    __device__ __forceinline__ void store(const Tensor& t, int64_t c, const float (&)[kChunk], uint32_t, bool streamed)
    {
        if (c >= t.elements) return;
        store_chunk((float*)t.avg, c, t.elements, m, streamed);
        store_chunk((float*)t.sq, c, t.elements, v, streamed);
    }
};
template <>
struct States<8> {
    float m[kChunk], v[kChunk];
    static __device__ __forceinline__ void codes(const void* from, int64_t c, int64_t n, uint8_t (&raw)[kChunk])
    {
        const uint8_t* p = (const uint8_t*)from;
        if (c + kChunk <= n) {
            __builtin_memcpy(raw, p + c, kChunk);
            return;
        }
#pragma unroll
        for (int j = 0; j < kChunk; ++j) raw[j] = c + j < n ? p[c + j] : 0;
    }
    template <bool ONCE>
    __device__ __forceinline__ void load(const Tensor& t, int64_t c)
    {
        uint8_t a[kChunk], s[kChunk];
        codes(t.avg, c, t.elements, a);
        codes(t.sq, c, t.elements, s);
        const bool there = c < t.elements;
        const float up = there ? scale_of(t.avg_scale[c / kBlock]) : 0.f, root_up = there ? scale_of(t.sq_scale[c / kBlock]) : 0.f;
        decode(a, m);
        decode(s, v);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            m[j] *= up;
            v[j] *= root_up;
            v[j] *= v[j];
        }
    }
    template <bool ROOT>
    static __device__ __forceinline__ void put(void* to, uint8_t* scale, int64_t c, int64_t n, const float (&x)[kChunk], uint32_t first)
    {
        // (behind the tensor's end x is zero)
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) most = max(most, magnitude_bits(x[j]));
        const bool numbers = !__any(most >= kInfinityBits);   // of the wave's chunks: nearly always
        if (!numbers) {
            most = 0;
#pragma unroll
            for (int j = 0; j < kChunk; ++j) most = max(most, magnitude_bits(x[j]) < kInfinityBits ? magnitude_bits(x[j]) : 0);
        }
        most = block_max(most) >> 23;
        const uint32_t field = most > 8 ? most - 7 : 1;
        const float down = __uint_as_float((254 - field) << 23);
        uint8_t raw[kChunk];
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            uint32_t code = encode(fabsf(x[j]) * down, first + (uint32_t)j * 0x9E3779B1u);
            if (!numbers && magnitude_bits(x[j]) >= kInfinityBits) code = 0x7f;
            if (ROOT) code = x[j] > 0.f ? max(code, 1u) : code;
            else code |= __float_as_uint(x[j]) >> 31 << 7;
            raw[j] = (uint8_t)code;
        }
        if (c >= n) return;
        if (c % kBlock == 0) scale[c / kBlock] = (uint8_t)field;
        uint8_t* p = (uint8_t*)to;
        if (c + kChunk <= n) {
            __builtin_memcpy(p + c, raw, kChunk);
            return;
        }
#pragma unroll
        for (int j = 0; j < kChunk; ++j)
            if (c + j < n) p[c + j] = raw[j];
    }
    __device__ __forceinline__ void store(const Tensor& t, int64_t c, const float (&root)[kChunk], uint32_t number, bool)
    {
        const uint32_t first = (uint32_t)(c % kBlock) * 0x9E3779B1u + number * 0x6A09E667u;
        put<false>(t.avg, t.avg_scale, c, t.elements, m, first);
        put<true>(t.sq, t.sq_scale, c, t.elements, root, first + 0x80000000u);
    }
};

// A workgroup takes 2048 elements of one tensor, a thread eight side by side.  ONCE: past the caches, see reads_once().
template <typename P, typename G, int BITS, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_adamw(Share s)
{
    // the tensor: each lane looks at the first workgroup of one
    const int lane = threadIdx.x & 63;
    const bool begun = lane < s.count && s.first[lane < kTensors ? lane : 0] <= blockIdx.x;
    const int i = __popcll(__ballot(begun)) - 1;
    const Tensor& t = s.tensors[i];
    const Constants& k = s.c;
    const Steps steps = k.device_steps ? *k.device_steps : k.steps;
    const int64_t c = (int64_t)(blockIdx.x - s.first[i]) * kTile + threadIdx.x * kChunk, n = t.elements;
    float p[kChunk], g[kChunk], root[kChunk];
    States<BITS> states;
    // (lanes behind the tensor's end go on: their block's largest number is asked of all)
    load_chunk<ONCE>((const P*)t.param, c, n, 0.f, p);
    load_chunk<ONCE>((const G*)t.grad, c, n, 0.f, g);
    states.template load<ONCE>(t, c);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
        const float grad = g[j] * k.scale;
        states.m[j] = states.m[j] * k.b1 + grad * k.c1;
        states.v[j] = states.v[j] * k.b2 + (grad * grad) * k.c2;
        root[j] = sqrtf(states.v[j]);
        p[j] = p[j] * k.keep - (states.m[j] * steps.size) / (root[j] * steps.inverse_root + k.eps);
    }
    states.store(t, c, root, steps.number, k.streamed);
    if (c >= n) return;
    store_chunk((P*)t.param, c, n, p, k.streamed);
    if (t.copy) store_chunk(t.copy, k.copy_dtype, 0, c, n, p, k.streamed);
    if (t.clamped) {
        float v[kChunk];
#pragma unroll
        for (int j = 0; j < kChunk; ++j) v[j] = p[j] < k.lo ? k.lo : p[j] > k.hi ? k.hi : p[j];
        store_chunk(t.clamped, c, n, v, k.streamed);
    }
}

template <typename P, typename G>
void run(const Share& s, uint32_t groups, int bits, hipStream_t stream)
{
    const auto go = [&](auto width) {
        if (s.c.streamed) k_adamw<P, G, width(), true><<<dim3(groups), dim3(kThreads), 0, stream>>>(s);
        else k_adamw<P, G, width(), false><<<dim3(groups), dim3(kThreads), 0, stream>>>(s);
    };
    if (bits == 8) go(std::integral_constant<int, 8>());
    else go(std::integral_constant<int, 32>());
}
template <typename P>
void run(const Share& s, uint32_t groups, int grad_dtype, int bits, hipStream_t stream)
{
    if (grad_dtype == GEO_SC_F32) run<P, f32>(s, groups, bits, stream);
    else if (grad_dtype == GEO_SC_BF16) run<P, bf16>(s, groups, bits, stream);
    else run<P, f16>(s, groups, bits, stream);
}

// what a call must have, but for the workspace
int check(int count, const geo_sc_adamw_tensor* tensors, const geo_sc_adamw_options* o)
{
    if (count < 0 || (count && !tensors) || !o || o->struct_bytes != sizeof *o) return GEO_SC_ERR_INVALID_ARGUMENT;
    if (!dtype_known(o->param_dtype) || !dtype_known(o->grad_dtype) || (o->state_bits != 8 && o->state_bits != 32) || !(o->lr >= 0) ||
        !(o->beta1 >= 0 && o->beta1 < 1) || !(o->beta2 >= 0 && o->beta2 < 1) || !(o->eps >= 0) || !(o->weight_decay >= 0) ||
        !(o->lo <= o->hi) || (!o->device_step && o->step < 1))
        return GEO_SC_ERR_INVALID_ARGUMENT;
    const bool eight = o->state_bits == 8;
    for (int i = 0; i < count; ++i) {
        const geo_sc_adamw_tensor& t = tensors[i];
        if (t.elements < 0) return GEO_SC_ERR_INVALID_ARGUMENT;
        if (t.elements == 0) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (eight && (!t.avg_scale || !t.sq_scale)) ||
            (t.copy && !dtype_known(o->copy_dtype)))
            return GEO_SC_ERR_INVALID_ARGUMENT;
        if (t.elements > (int64_t)kTile * (0xffffffffll / kThreads)) return GEO_SC_ERR_UNSUPPORTED;   // (one launch's threads)
    }
    return GEO_SC_OK;
}

// Past the caches where what is written fills them, and everything that is loaded lies at whole lines' parts.
bool past_caches(int count, const geo_sc_adamw_tensor* tensors, const geo_sc_adamw_options* o)
{
    const bool eight = o->state_bits == 8;
    int64_t written = 0;
    uint64_t places = 0;
    for (int i = 0; i < count; ++i) {
        const geo_sc_adamw_tensor& t = tensors[i];
        written += t.elements * (dtype_bytes(o->param_dtype) + (eight ? 2 : 8) + (t.copy ? dtype_bytes(o->copy_dtype) : 0) + (t.clamped ? 4 : 0));
        if (t.elements) places |= (uintptr_t)t.param | (uintptr_t)t.grad | (eight ? 0 : (uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq);
    }
    return streams(written) && places % 16 == 0;
}

// Calls launch(share, groups) with the tensors of one launch after the other: c's constants, `groups` workgroups.
template <typename F>
void in_shares(const Constants& c, int count, const geo_sc_adamw_tensor* tensors, F launch)
{
    Share s = {};
    s.c = c;
    uint32_t groups = 0;
    const auto flush = [&]() {
        if (groups) launch(s, groups);
        s.count = 0;
        groups = 0;
    };
    for (int i = 0; i < count; ++i) {
        const geo_sc_adamw_tensor& t = tensors[i];
        if (!t.elements) continue;
        const uint32_t more = (uint32_t)((t.elements + kTile - 1) / kTile);
        if (s.count == kTensors || (uint64_t)groups + more > 0xffffffffll / kThreads) flush();
        s.first[s.count] = groups;
        s.tensors[s.count++] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.avg_scale, t.sq_scale, t.copy, t.clamped, t.elements};
        groups += more;
    }
    flush();
}

}  // namespace
}  // namespace geo_sc

using namespace geo_sc;

extern "C" int geo_sc_adamw_plan(int count, const geo_sc_adamw_tensor* tensors, const geo_sc_adamw_options* o, int* launches, int* uncached)
{
    if (!launches || !uncached) return GEO_SC_ERR_INVALID_ARGUMENT;
    if (const int rc = check(count, tensors, o)) return rc;
    *launches = 0;
    in_shares({}, count, tensors, [&](const Share&, uint32_t) { ++*launches; });
    *uncached = past_caches(count, tensors, o);
    return GEO_SC_OK;
}

extern "C" int geo_sc_adamw(int count, const geo_sc_adamw_tensor* tensors, const geo_sc_adamw_options* o, void* workspace,
                            size_t workspace_bytes, geo_sc_stream_t stream)
{
    if (const int rc = check(count, tensors, o)) return rc;
    if (o->device_step && (!workspace || workspace_bytes < sizeof(Steps) || (uintptr_t)workspace % 8)) return GEO_SC_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    Constants c = {};
    c.scale = (float)o->grad_scale;
    c.b1 = (float)o->beta1;
    c.c1 = (float)(1 - o->beta1);
    c.b2 = (float)o->beta2;
    c.c2 = (float)(1 - o->beta2);
    c.keep = (float)(1 - o->lr * o->weight_decay);
    c.eps = (float)o->eps;
    c.lo = o->lo;
    c.hi = o->hi;
    c.copy_dtype = o->copy_dtype;
    if (o->device_step) {
        k_adamw_count<<<dim3(1), dim3(1), 0, st>>>(o->device_step, o->lr, o->beta1, o->beta2, (Steps*)workspace);
        c.device_steps = (const Steps*)workspace;
    } else {
        c.steps = steps_at(o->lr, o->beta1, o->beta2, o->step);
    }
    c.streamed = past_caches(count, tensors, o);
    bool launched = o->device_step;
    in_shares(c, count, tensors, [&](const Share& s, uint32_t groups) {
        launched = true;
        if (o->param_dtype == GEO_SC_F32) run<f32>(s, groups, o->grad_dtype, o->state_bits, st);
        else if (o->param_dtype == GEO_SC_BF16) run<bf16>(s, groups, o->grad_dtype, o->state_bits, st);
        else run<f16>(s, groups, o->grad_dtype, o->state_bits, st);
    });
    if (!launched) return GEO_SC_OK;
    return hipGetLastError() == hipSuccess ? GEO_SC_OK : GEO_SC_ERR_LAUNCH;
}
