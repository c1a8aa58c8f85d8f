// Matrix product in 8-bit integers with a scale for each row of either operand, and its gradients.
//
//   y[m][n] = x_scale[m] w_scale[n] sum_k x[m][k] w[n][k]
//
// The sum is an exact 32-bit integer (|x w| <= 2^14, so up to 131071 terms); the two scales come in once, at the end.  Integer
// sums do not depend on their order, so cutting the inner dimension between waves or workgroups changes no result.
//
// Gradients, straight through the rounding of the operands (g: gradient of y):
//   dx[m][k] = sum_n (g[m][n] w_scale[n]) w[n][k],   dw[n][k] = sum_m (g[m][n] x_scale[m]) x[m][k]
// The 8-bit operand is exact in fp16; a row of the scaled gradient is brought by a power of two to where its largest magnitude
// fills fp16's range, and held as a sum of fp16 terms: one where g is bf16 (11 bits for products of 8-bit numbers), two where it is
// fp16 or fp32 (23 bits; nothing of a term is lost above 2^-39 of the row's largest), which makes the inner dimension twice as
// long.  Sums in fp32; the power of two comes out at the end, exactly.  (Terms of bf16 need no powers of two, but one rounds the
// scaled gradient as coarsely as the result is rounded, and fp32 takes three.)
//
// Both products run on one kernel: the 16x16 matrix instructions of int8 (64 deep) and fp16 (32 deep) take the same 16 bytes per
// lane of either operand, so tiles are counted in bytes of the inner dimension.
#include "sc_dense.h"

namespace geo_sc {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* LdsPtr;

constexpr int kStage = 64;    // bytes of the inner dimension per stage: one matrix instruction deep
template <int N>
using Int = std::integral_constant<int, N>;
constexpr int kUnits = 256;   // compute units
constexpr int64_t kMostGroups = 0xfffffe;   // workgroups of 256 threads in a launch, which counts threads in 32 bits

struct TileArgs {
    const uint8_t *x, *w;              // rows of `inner` bytes each
    int64_t x_stride, w_stride;        // bytes
    int64_t rows, cols, inner;
    int w_stages;                      // w's inner dimension repeats after this many stages (terms of the gradient)
    const float *x_scale, *w_scale;    // NULL: 1
    void* y;
    int64_t y_stride;                  // elements
    int dtype;
    int stages_per_split;
    int splits;
    uint32_t* partial;                 // [splits][rows][cols] 32-bit sums, or NULL: one split that writes y
    int tiles_m, tiles_n;
};
// One launch computes up to two products: workgroups from second_at on the second.
struct TwoProducts {
    TileArgs first, second;
    uint32_t second_at;
};

// One load of 16 bytes per lane straight into LDS, lane after lane from `to` on.  (The host's pass over this file knows no
// such load, and a kernel that it cannot check gets no stub.)
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, uint8_t* to, int offset, int uniform_offset)
{
#ifdef __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (LdsPtr)to, 16, offset, uniform_offset, 0, 0);
#endif
}

// 16 bytes of a row from byte k on; zeros behind its end.  A piece that passes the end is the row's last 16 bytes, shifted.
__device__ __forceinline__ v4i load_piece(const uint8_t* row, int64_t k, int64_t inner)
{
    unsigned __int128 v = 0;
    if (inner < 16) {
#pragma unroll 1
        for (int64_t j = inner; j-- > k;) v = v << 8 | row[j];
        return __builtin_bit_cast(v4i, v);
    }
    const int64_t at = k + 16 <= inner ? k : inner - 16, shift = k - at;
    __builtin_memcpy(&v, row + at, 16);
    return __builtin_bit_cast(v4i, shift < 16 ? v >> (8 * (int)shift) : (unsigned __int128)0);
}

// 16 N bytes from any address.  Loads at odd addresses take the memory pipeline twice and more (4096 x 16384 bytes of w at odd
// strides, 16 rows of x: 39 us, at multiples of four 18): whole words are loaded, those that hold the first byte to the last,
// and shifted.
template <int N>
struct Shifted {
    typedef int Four __attribute__((ext_vector_type(4), aligned(4)));
    const uint8_t* from;
    int shift, last;
    Shifted() = default;
    __device__ __forceinline__ explicit Shifted(const uint8_t* p)
        : from((const uint8_t*)((uintptr_t)p & ~(uintptr_t)3)), shift((int)((uintptr_t)p & 3)), last(shift ? 16 * N : 16 * N - 4)
    {
    }
    struct Words {
        Four four[N];
        uint32_t last;
    };
    __device__ __forceinline__ Words load(int64_t offset) const   // a multiple of four
    {
        Words t;
#pragma unroll
        for (int i = 0; i < N; ++i) t.four[i] = *(const Four*)(from + offset + 16 * i);
        t.last = *(const uint32_t*)(from + offset + last);
        return t;
    }
    __device__ __forceinline__ v4i piece(const Words& t, int i) const
    {
        uint32_t u[5];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = (uint32_t)t.four[i][k];
        u[4] = i + 1 < N ? (uint32_t)t.four[i + 1 < N ? i + 1 : i][0] : t.last;
        v4i v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (int)__builtin_amdgcn_alignbyte(u[k + 1], u[k], (uint32_t)shift);
        return v;
    }
};

template <bool INT8>
struct Matrix;
template <>
struct Matrix<true> {
    typedef v4i Sum;
    static __device__ __forceinline__ void add(const v4i& a, const v4i& b, Sum& s) { s = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, s, 0, 0, 0); }
    // The same on sums that stay in their accumulation registers: of the builtin's, with as many registers as the tiles need, the
    // compiler copied three for every product (8192 x 16384 x 4096: 750 us, so 565).  It keeps no distance from these products: what
    // else reads the sums comes behind settle(), and a test follows the built code for what comes between.
    static __device__ __forceinline__ void add_in_place(const v4i& a, const v4i& b, Sum& s)
    {
        asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(s) : "v"(a), "v"(b));
    }
};
template <>
struct Matrix<false> {
    typedef v4f Sum;
    static __device__ __forceinline__ void add(const v4i& a, const v4i& b, Sum& s)
    {
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), s, 0, 0, 0);
    }
    static __device__ __forceinline__ void add_in_place(const v4i& a, const v4i& b, Sum& s)
    {
        asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(s) : "v"(a), "v"(b));
    }
};

// four consecutive columns of a row of y
__device__ __forceinline__ void store_four(void* y, int dtype, int64_t at, int64_t left, const float (&v)[4])
{
    const auto put = [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        T raw[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        if (left >= 4) {
            __builtin_memcpy(p + at, raw, sizeof raw);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (r < left) p[at + r] = raw[r];
        }
    };
    if (dtype == GEO_SC_F32) put((f32*)y);
    else if (dtype == GEO_SC_BF16) put((bf16*)y);
    else put((f16*)y);
}

// Scales and stores four sums of consecutive columns, or hands them to the join as they are.
template <typename Sum>
__device__ __forceinline__ void finish_four(const TileArgs& a, int split, int64_t m, int64_t n, const Sum& s, float xs, const float (&ws)[4])
{
    const int64_t left = a.cols - n;
    if (m >= a.rows || left <= 0) return;
    if (a.partial) {
        uint32_t* out = a.partial + ((int64_t)split * a.rows + m) * a.cols + n;
        if (left >= 4) {
            __builtin_memcpy(out, &s, 16);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const auto one = s[r];   // (a bit cast of the element itself takes the vector's first)
                if (r < left) out[r] = __builtin_bit_cast(uint32_t, one);
            }
        }
        return;
    }
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (float)s[r] * xs * ws[r];
    store_four(a.y, a.dtype, m * a.y_stride + n, left, v);
}

__device__ __forceinline__ float scale_at(const float* scale, int64_t i, int64_t count) { return scale && i < count ? scale[i] : 1.f; }

// ---------------------------------------------------------------- epilogue
//
//   z = x_scale w_scale sum + bias,   y = act(z) + residual;   for the backward slope = act'(z)
// In fp32, y rounded once.  The slope and not z is kept: z in 16 bits would be off by up to a 2048th of itself, the slope in fp16 is off by
// as much of a number that is 1.13 at most, whatever z is.

struct Epilogue {
    const void *bias, *residual;   // or NULL; the residual's type is y's
    void* slope;                   // [rows][cols]; or NULL
    int64_t residual_stride;
    int bias_dtype, slope_dtype, activation;
};
bool slope_type_known(int dtype) { return dtype == GEO_SC_F32 || dtype == GEO_SC_F16 || dtype == GEO_SC_U8; }

// z becomes act(z), d its slope.  NaN stays NaN.
// gelu: z P(z) with P(z) = 1 - Q(z) the normal distribution's share below z, its slope P + z p.  With x = |z| / sqrt 2 and u = 1 / (1 + 0.3275911 x),
// 2 Q(|z|) = (a1 u + .. + a5 u^5) exp(-x^2) to 1.5e-7 (Abramowitz and Stegun 7.1.26), from the exponential that the density p takes anyway.
// The hardware's exponential and reciprocal are within a unit each.  A wave of a large tile is alone on its SIMD and does 256
// numbers a lane, four cycles an instruction (the transcendental ones sixteen).
template <int N>
__device__ __forceinline__ void activate(int kind, float (&z)[N], float (&d)[N])
{
    if (kind == GEO_SC_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            d[j] = z[j] <= 0.f ? 0.f : 1.f;   // (what comes back to a NaN goes on, as behind torch's relu)
            z[j] = z[j] < 0.f ? 0.f : z[j];
        }
    } else if (kind == GEO_SC_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float u = __builtin_amdgcn_rcpf(1.f + 0.3275911f * 0.70710678f * fabsf(z[j]));
            const float e = __builtin_amdgcn_exp2f(z[j] * z[j] * (-0.5f * 1.44269504f));
            const float series = u * (0.254829592f + u * (-0.284496736f + u * (1.421413741f + u * (-1.453152027f + u * 1.061405429f))));
            const float tail = 0.5f * series * e, below = z[j] < 0.f ? tail : 1.f - tail;
            d[j] = below + z[j] * e * 0.39894228f;
            z[j] *= below;
        }
    } else if (kind == GEO_SC_ACT_SILU) {   // z times s = 1 / (1 + exp(-z)); slope s + z s (1 - s)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z[j] * -1.44269504f));
            z[j] *= s;
            d[j] = s + z[j] * (1.f - s);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) d[j] = 1.f;
    }
}

// N consecutive columns of a row, of which `left` are there
template <int N, typename T>
__device__ __forceinline__ void load_columns(const T* p, int64_t left, float (&v)[N])
{
    if (left >= N) {
        T raw[N];
        __builtin_memcpy(raw, p, sizeof raw);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (float)raw[j];
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < left ? (float)p[j] : 0.f;
    }
}
template <int N>
__device__ __forceinline__ void load_columns(const void* p, int dtype, int64_t at, int64_t left, float (&v)[N])
{
    if (dtype == GEO_SC_F32) load_columns((const f32*)p + at, left, v);
    else if (dtype == GEO_SC_BF16) load_columns((const bf16*)p + at, left, v);
    else load_columns((const f16*)p + at, left, v);
}
template <int N, typename T>
__device__ __forceinline__ void store_columns(T* p, int64_t left, const float (&v)[N])
{
    T raw[N];
#pragma unroll
    for (int j = 0; j < N; ++j) raw[j] = (T)v[j];
    if (left >= N) {
        __builtin_memcpy(p, raw, sizeof raw);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < left) p[j] = raw[j];
    }
}
template <int N>
__device__ __forceinline__ void store_columns(void* p, int dtype, int64_t at, int64_t left, const float (&v)[N])
{
    if (dtype == GEO_SC_F32) store_columns((f32*)p + at, left, v);
    else if (dtype == GEO_SC_BF16) store_columns((bf16*)p + at, left, v);
    else store_columns((f16*)p + at, left, v);
}
template <int N>
__device__ __forceinline__ void load_bias(const Epilogue& e, int64_t n, int64_t cols, float (&v)[N])
{
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = 0.f;
    if (e.bias && n < cols) load_columns(e.bias, e.bias_dtype, n, cols - n, v);
}
template <int N>
__device__ __forceinline__ void store_slope(const Epilogue& e, int64_t at, int64_t left, const float (&d)[N])
{
    if (e.slope_dtype == GEO_SC_F32) store_columns((f32*)e.slope + at, left, d);
    else if (e.slope_dtype == GEO_SC_F16) store_columns((f16*)e.slope + at, left, d);
    else store_columns((uint8_t*)e.slope + at, left, d);
}
// N columns from n on of row m: their sums scaled and the bias added come in as z
template <int N>
__device__ __forceinline__ void finish_columns(const TileArgs& a, const Epilogue& e, int64_t m, int64_t n, float (&z)[N])
{
    const int64_t left = a.cols - n;
    if (m >= a.rows || left <= 0) return;
    float d[N];
    activate(e.activation, z, d);
    if (e.slope) store_slope(e, m * a.y_stride + n, left, d);
    if (e.residual) {
        load_columns(e.residual, a.dtype, m * e.residual_stride + n, left, d);
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] += d[j];
    }
    store_columns(a.y, a.dtype, m * a.y_stride + n, left, z);
}
// the same from four sums and their scales
__device__ __forceinline__ void finish_four(const TileArgs& a, const Epilogue& e, int64_t m, int64_t n, const v4i& s, float xs, const float (&ws)[4])
{
    float z[4], bias[4];
    load_bias(e, n, a.cols, bias);
#pragma unroll
    for (int r = 0; r < 4; ++r) z[r] = (float)s[r] * xs * ws[r] + bias[r];
    finish_columns(a, e, m, n, z);
}

// ---------------------------------------------------------------- tiles
//
// Tiles of B rows of x by B rows of w; four waves, each with a quarter of the outputs in 16x16 squares.  w is the matrix
// instruction's first operand, so a lane's four sums are consecutive columns of y.
//
// A stage is 64 bytes of every row, one matrix instruction deep, in LDS as four 16-byte pieces per row at positions
// piece ^ (row / 4 & 2): then no two of the lanes that the LDS serves at once (of its read of 16 bytes, measured: 0 - 3, 12 - 15 and 20 - 27, and so
// on) meet in a bank.
constexpr int kRing = 4, kWaves = 4;

template <int B, bool INT8>
struct Tiling {
    typedef typename Matrix<INT8>::Sum Sum;
    static constexpr int T = B / 32;               // squares of a wave in either direction
    static constexpr int L = B / 16 / kWaves;      // a wave's loads of either operand for a stage, 16 rows each
    static constexpr int kBytes = 2 * B * kStage;  // of a stage
    static constexpr int kArea = 16 * T * 64;      // bytes of 16 rows of a wave's sums
};

// Quotients are computed in vector registers; of the whole wave's they say so here, or descriptors that are formed from them are taken for
// the lanes' own, and every load goes through a loop over them.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// Where a workgroup works: its product's tile and split.
struct Spot {
    TileArgs a;
    int64_t m0, n0;
    uint32_t split, die;
    int begin, stop, end;   // stages: whole ones up to stop, one more where the inner dimension ends inside it
};

// Workgroups go to the eight dies in turn: each die takes a contiguous share of the tiles, so that neighbours share its L2, in
// strips of four tiles of rows.
template <int B>
__device__ __forceinline__ Spot spot_of(const TwoProducts& both, uint32_t work)
{
    Spot p;
    const bool is_second = work >= both.second_at;
    p.a = is_second ? both.second : both.first;
    const uint32_t group = work - (is_second ? both.second_at : 0), all = (uint32_t)p.a.tiles_m * p.a.tiles_n;
    p.split = uniform(group / all);
    p.die = uniform(group % all & 7);
    const uint32_t tile = p.die * (all / 8) + (p.die < all % 8 ? p.die : all % 8) + (group % all >> 3);
    constexpr uint32_t kStrip = 4;
    const uint32_t strip = uniform(tile / (kStrip * p.a.tiles_n)), inside = tile - strip * kStrip * p.a.tiles_n;
    const uint32_t height = p.a.tiles_m - strip * kStrip < kStrip ? p.a.tiles_m - strip * kStrip : kStrip;
    p.m0 = (int64_t)(strip * kStrip + uniform(inside % height)) * B;
    p.n0 = (int64_t)uniform(inside / height) * B;
    const int stages = (int)((p.a.inner + kStage - 1) / kStage), whole = (int)(p.a.inner / kStage);
    p.begin = p.split * p.a.stages_per_split;
    p.end = p.begin + p.a.stages_per_split < stages ? p.begin + p.a.stages_per_split : stages;
    p.stop = p.end < whole ? p.end : whole;
    return p;
}

__device__ __forceinline__ int w_stage(const TileArgs& a, int k) { return k >= a.w_stages ? k - a.w_stages : k; }   // (at most two terms)
// row that a lane loads for the i-th time, from the tile's first; rows behind the operand's last are its last again, their
// outputs are not stored
__device__ __forceinline__ int64_t load_row(int64_t first, int64_t rows, int i, int wave, int lane)
{
    const int64_t r = (int64_t)(i * kWaves + wave) * 16 + (lane >> 2);
    return first + r < rows ? r : rows - 1 - first;
}
__device__ __forceinline__ int load_piece_of(int lane) { return (lane & 3) ^ (lane >> 4 & 2); }

// A stage through registers: any alignment, zeros behind the end of a row.
template <int L>
__device__ __forceinline__ void fetch_stage(const Spot& p, int k, int wave, int lane, v4i (&v)[2 * L])
{
    const int64_t xk = (int64_t)k * kStage + load_piece_of(lane) * 16, wk = (int64_t)w_stage(p.a, k) * kStage + load_piece_of(lane) * 16;
#pragma unroll
    for (int i = 0; i < L; ++i) v[i] = load_piece(p.a.x + (p.m0 + load_row(p.m0, p.a.rows, i, wave, lane)) * p.a.x_stride, xk, p.a.inner);
#pragma unroll
    for (int i = 0; i < L; ++i) v[L + i] = load_piece(p.a.w + (p.n0 + load_row(p.n0, p.a.cols, i, wave, lane)) * p.a.w_stride, wk, p.a.inner);
}
template <int L>
__device__ __forceinline__ void put_stage(uint8_t* to, int wave, int lane, const v4i (&v)[2 * L])
{
#pragma unroll
    for (int i = 0; i < 2 * L; ++i) *(v4i*)(to + (i * kWaves + wave) * 1024 + lane * 16) = v[i];
}

// A wave's fragments of a stage: T of w, then T of x.
template <int B>
struct Fragments {
    static constexpr int T = B / 32;
    int x, w;   // bytes from the stage's begin
    __device__ Fragments(int wave, int lane)
    {
        const int mine = (lane & 15) * kStage + (((lane >> 4) ^ (lane >> 2 & 2)) << 4);
        x = wave % 2 * T * 16 * kStage + mine;
        w = (B + wave / 2 * T * 16) * kStage + mine;
    }
    __device__ __forceinline__ void read_one(v4i (&f)[2 * T], const uint8_t* from, int t) const
    {
        f[t] = *(const v4i*)(from + (t < T ? w + t * 16 * kStage : x + (t - T) * 16 * kStage));
    }
    __device__ __forceinline__ void read(v4i (&f)[2 * T], const uint8_t* from) const
    {
#pragma unroll
        for (int t = 0; t < 2 * T; ++t) read_one(f, from, t);
    }
};
// kInPlace: see Matrix::add_in_place
template <bool INT8, bool kInPlace, int T>
__device__ __forceinline__ void multiply_one(const v4i (&f)[2 * T], typename Matrix<INT8>::Sum (&sum)[T][T], int t)
{
    if constexpr (kInPlace) Matrix<INT8>::add_in_place(f[t / T], f[T + t % T], sum[t / T][t % T]);
    else Matrix<INT8>::add(f[t / T], f[T + t % T], sum[t / T][t % T]);
}
template <bool INT8, bool kInPlace, int T>
__device__ __forceinline__ void multiply(const v4i (&f)[2 * T], typename Matrix<INT8>::Sum (&sum)[T][T])
{
#pragma unroll
    for (int t = 0; t < T * T; ++t) multiply_one<INT8, kInPlace, T>(f, sum, t);
}

// The last products' sums are in their registers.  The compiler does not know the products for what they are and keeps no
// distance; every sum passes through a statement behind the wait, so that no read of one can come before it.
template <int T, typename Sum>
__device__ __forceinline__ void settle(Sum (&sum)[T][T])
{
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
        for (int i = 0; i < T; i += 2) asm volatile("" : "+a"(sum[j][i]), "+a"(sum[j][i + 1]));
}

// The scales of a wave's rows and columns, all asked for at once: each by itself would be waited for by itself.
template <int T>
struct TileScales {
    float x[T], w[T][4];
    __device__ __forceinline__ void load(const Spot& p, int wave, int lane)
    {
#pragma unroll
        for (int j = 0; j < T; ++j) {
            x[j] = 1.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) w[j][r] = 1.f;
        }
        if (p.a.w_scale) {
#pragma unroll
            for (int j = 0; j < T; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t n = p.n0 + (wave / 2 * T + j) * 16 + (lane >> 4) * 4 + r;
                    w[j][r] = p.a.w_scale[n < p.a.cols ? n : p.a.cols - 1];
                }
        }
        if (p.a.x_scale) {
#pragma unroll
            for (int i = 0; i < T; ++i) {
                const int64_t m = p.m0 + (wave % 2 * T + i) * 16 + (lane & 15);
                x[i] = p.a.x_scale[m < p.a.rows ? m : p.a.rows - 1];
            }
        }
    }
};

template <int B>
__device__ __forceinline__ bool inside(const Spot& p) { return p.m0 + B <= p.a.rows && p.n0 + B <= p.a.cols; }

// A tile's sums scaled, rounded and stored, or handed to the join as they are.  Out through LDS, each wave in an area of its own: a
// lane holds four columns of one row, the lanes that share a row store 16 bytes each and fill its lines.  Positions of the
// 16-byte pieces ^ row: no two lanes of a quarter wave meet in a bank.
template <int B, bool INT8>
__device__ __forceinline__ void finish_tile(const Spot& p, typename Matrix<INT8>::Sum (&sum)[B / 32][B / 32], const TileScales<B / 32>& scales,
                                            uint8_t* area, int wave, int lane)
{
    constexpr int T = B / 32;
    const bool fits = inside<B>(p);
    const auto finish = [&](auto* y, int64_t stride, auto value) {
        using Y = std::remove_pointer_t<decltype(y)>;
        constexpr int kEach = 16 / (int)sizeof(Y), kPieces = T * 16 / kEach, kAtOnce = 64 / kPieces;   // elements, pieces of a row, rows of a store
        constexpr int kMix = (kPieces < 16 ? kPieces : 16) - 1, kBatch = 4 / (int)sizeof(Y);           // squares of rows that the area holds
        const int row = lane & 15, column = (lane >> 4) * 4;
#pragma unroll
        for (int first = 0; first < T; first += kBatch) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
                for (int j = 0; j < T; ++j) {
                    typename Matrix<INT8>::Sum s = sum[j][first + i];
                    asm volatile("" : "+v"(s));   // (here, and not for all types at once before the choice of one)
                    Y four[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) four[r] = value(s[r], first + i, j, r);
                    const int at = j * 16 + column, where = (i * 16 + row) * kPieces + ((at / kEach) ^ (row & kMix));
                    __builtin_memcpy(area + where * 16 + at % kEach * sizeof(Y), four, sizeof four);
                }
            __builtin_amdgcn_wave_barrier();
            const int64_t m1 = p.m0 + (wave % 2 * T + first) * 16, n = p.n0 + wave / 2 * T * 16 + lane % kPieces * kEach;
            v4i u[16 * kBatch / kAtOnce];
#pragma unroll
            for (int h = 0; h < 16 * kBatch / kAtOnce; ++h) {
                const int r = h * kAtOnce + lane / kPieces;
                u[h] = *(const v4i*)(area + (r * kPieces + (lane % kPieces ^ (r & kMix))) * 16);
            }
            if (fits) {
#pragma unroll
                for (int h = 0; h < 16 * kBatch / kAtOnce; ++h)
                    __builtin_memcpy(y + (m1 + h * kAtOnce + lane / kPieces) * stride + n, &u[h], 16);
            } else {
#pragma unroll
                for (int h = 0; h < 16 * kBatch / kAtOnce; ++h) {
                    const int64_t m = m1 + h * kAtOnce + lane / kPieces;
                    Y raw[kEach];
                    __builtin_memcpy(raw, &u[h], 16);
                    if (m < p.a.rows && n + kEach <= p.a.cols) {
                        __builtin_memcpy(y + m * stride + n, raw, 16);
                    } else if (m < p.a.rows) {
#pragma unroll
                        for (int t = 0; t < kEach; ++t)
                            if (n + t < p.a.cols) y[m * stride + n + t] = raw[t];
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    };
    const auto scaled = [&](auto one, int i, int j, int r) { return (float)one * scales.x[i] * scales.w[j][r]; };
    if (p.a.partial)
        finish(p.a.partial + (int64_t)p.split * p.a.rows * p.a.cols, p.a.cols, [&](auto one, int, int, int) { return __builtin_bit_cast(uint32_t, one); });
    else if (p.a.dtype == GEO_SC_F32) finish((f32*)p.a.y, p.a.y_stride, scaled);
    else if (p.a.dtype == GEO_SC_BF16) finish((bf16*)p.a.y, p.a.y_stride, [&](auto one, int i, int j, int r) { return (bf16)scaled(one, i, j, r); });
    else finish((f16*)p.a.y, p.a.y_stride, [&](auto one, int i, int j, int r) { return (f16)scaled(one, i, j, r); });
}

// The same through the epilogue: the sums times their rows' scales into LDS, ROWS of a wave's rows at a time, and out of it a lane eight
// columns of a row.  A wave of a large tile is alone on its SIMD, so nothing is waited for where it is used: the sums out of LDS and the
// residual's rows are asked for kBatch rows at a time, a batch ahead.  4096 x 4096 x 2048 bf16 with silu, bias and residual 46 us where the
// product alone takes 37; asked for row by row 62.
template <int B, int ROWS>
struct EpilogueTile {
    static constexpr int T = B / 32, kCols = T * 16, kPieces = kCols / 4, kMix = (kPieces < 16 ? kPieces : 16) - 1;
    static constexpr int kLanes = kCols / kChunk, kAtOnce = 64 / kLanes;   // lanes of a row, rows at once
    static constexpr int kPasses = ROWS / kAtOnce;
    static_assert(ROWS % 16 == 0 && kCols % ROWS == 0 && kPasses % (B == 256 ? 4 : 2) == 0, "");
    const Epilogue& e;
    float ws[kChunk], bias[kChunk], xs[T];

    // A wave whose columns end inside a chunk has that chunk begin earlier: its lane, and those behind it, form the last eight columns
    // once more, the same numbers as the lane before, and nothing depends on a lane.  (Masked loads cannot be asked for ahead: the tiles
    // of the last rows of 4095 x 4099 with a residual took 25 us more.)  One that has fewer than eight columns is masked.
    static __device__ __forceinline__ int64_t begin(const Spot& p, int wave) { return p.n0 + wave / 2 * kCols; }
    static __device__ __forceinline__ int64_t column(const Spot& p, int wave, int lane)
    {
        const int64_t n = begin(p, wave) + lane % kLanes * kChunk, last = p.a.cols - kChunk;
        return n > last && last >= begin(p, wave) ? last : n;
    }
    // asks for the scales and the bias
    __device__ __forceinline__ void ask(const Spot& p, int wave, int lane)
    {
        const int64_t n = column(p, wave, lane);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) ws[j] = 0.f;
        if (n < p.a.cols) load_columns(p.a.w_scale + n, p.a.cols - n, ws);
        load_bias(e, n, p.a.cols, bias);
#pragma unroll
        for (int i = 0; i < T; ++i) {
            const int64_t m = p.m0 + wave % 2 * kCols + i * 16 + (lane & 15);
            xs[i] = p.a.x_scale[m < p.a.rows ? m : p.a.rows - 1];
        }
    }
    enum Way { kWhole, kOverlap, kMasked };
    template <typename Y, Way WAY>
    struct Batch {   // of rows: what the registers hold, and in the rarer ways less code
        static constexpr int kRows = B == 256 && sizeof(Y) == 2 && WAY == kWhole ? 4 : 2, kStep = kRows * kAtOnce, kWords = kChunk * (int)sizeof(Y) / 4;
        static __device__ __forceinline__ float element(const uint32_t (&words)[kWords], int j)
        {
            if constexpr (sizeof(Y) == 4) return __uint_as_float(words[j]);
            else return (float)__builtin_bit_cast(Y, (uint16_t)(words[j / 2] >> (16 * (j & 1))));
        }
        // the residual from row m on, as it lies in memory
        static __device__ __forceinline__ void ask(const Spot& p, const Epilogue& e, int64_t m, int64_t n, uint32_t (&words)[16])
        {
            if (!e.residual) return;
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int64_t mine = m + i * kAtOnce;
                const Y* row = (const Y*)e.residual + (mine < p.a.rows ? mine : p.a.rows - 1) * e.residual_stride;   // (behind the last row that row once more)
                if constexpr (WAY == kMasked) {   // (and behind the last column that one)
                    Y one[kChunk];
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) one[j] = row[n + j < p.a.cols ? n + j : p.a.cols - 1];
                    __builtin_memcpy(words + i * kWords, one, sizeof one);
                } else {
                    __builtin_memcpy(words + i * kWords, row + n, kWords * 4);
                }
            }
        }
    };
    // What is written out of `area`: ROWS rows from `first` of the wave's on.  `ahead`: the residual of the first batch.
    template <typename Y, Way WAY>
    __device__ __forceinline__ void rows(const Spot& p, const uint8_t* area, int wave, int lane, int first, uint32_t (&ahead)[16]) const
    {
        typedef Batch<Y, WAY> Of;
        constexpr int kBatch = Of::kRows, kStep = Of::kStep;
        const int64_t stride = p.a.y_stride, n = column(p, wave, lane), left = p.a.cols - n, m0 = p.m0 + wave % 2 * kCols + first + lane / kLanes;
        const int mine = lane / kLanes, piece = lane % kLanes * 2, from = (int)(n - begin(p, wave));
        const auto ask_sums = [&](float (&v)[kBatch][kChunk], int r) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int row = (r + i * kAtOnce + mine) % ROWS;
                if constexpr (WAY == kOverlap) {
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) {
                        const int c = from + j;
                        v[i][j] = *(const float*)(area + (row * kPieces + ((c >> 2) ^ (row & kMix))) * 16 + (c & 3) * 4);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) __builtin_memcpy(v[i] + 4 * h, area + (row * kPieces + ((piece + h) ^ (row & kMix))) * 16, 16);
                }
            }
        };
        float sums_ahead[kBatch][kChunk];
        ask_sums(sums_ahead, 0);
        int64_t at = m0 * stride + n;
#pragma unroll 1
        for (int r = 0; r < ROWS; r += kStep) {
            uint32_t residual[kBatch][Of::kWords];
            float z[kBatch][kChunk];
            __builtin_memcpy(residual, ahead, sizeof residual);
            __builtin_memcpy(z, sums_ahead, sizeof z);
            ask_sums(sums_ahead, r + kStep);   // (behind the last ones the first once more)
            if (r + kStep < ROWS) Of::ask(p, e, m0 + r + kStep, n, ahead);
#pragma unroll
            for (int i = 0; i < kBatch; ++i, at += kAtOnce * stride) {
                float d[kChunk];
#pragma unroll
                for (int j = 0; j < kChunk; ++j) z[i][j] = z[i][j] * ws[j] + bias[j];
                activate(e.activation, z[i], d);
                if (m0 + r + i * kAtOnce >= p.a.rows || (WAY == kMasked && left <= 0)) continue;
                const int64_t there = WAY == kMasked ? left : kChunk;
                if (e.slope) store_slope(e, at, there, d);
                if (e.residual) {
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) z[i][j] += Of::element(residual[i], j);
                }
                store_columns((Y*)p.a.y + at, there, z[i]);
            }
        }
    }
    // ROWS of the wave's rows, from FIRST on, into `area`
    template <int FIRST>
    __device__ __forceinline__ void put(v4i (&sum)[T][T], uint8_t* area, int lane) const
    {
#pragma unroll
        for (int i = 0; i < ROWS / 16; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j) {
                const int row = i * 16 + (lane & 15), to = j * 4 + (lane >> 4);
                v4i s = sum[j][FIRST / 16 + i];
                asm volatile("" : "+v"(s));   // (out of its accumulation registers here)
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = (float)s[r] * xs[FIRST / 16 + i];
                __builtin_memcpy(area + (row * kPieces + (to ^ (row & kMix))) * 16, v, 16);
            }
    }
    // A loop over the shares of ROWS rows, with the types and ways inside it: each of them has its code once, and no branch of a kernel has to
    // go further than an instruction can say (128 KB).
    __device__ __forceinline__ void finish(const Spot& p, v4i (&sum)[T][T], uint8_t* area, int wave, int lane) const
    {
        const int64_t there = p.a.cols - begin(p, wave), n = column(p, wave, lane), m0 = p.m0 + wave % 2 * kCols + lane / kLanes;
        if (there <= 0) return;
        const auto of_kind = [&](auto work) {
            const auto of_way = [&](auto y) {
                if (there >= kCols) work(y, std::integral_constant<Way, kWhole>());
                else if (there >= kChunk) work(y, std::integral_constant<Way, kOverlap>());
                else work(y, std::integral_constant<Way, kMasked>());
            };
            if (p.a.dtype == GEO_SC_F32) of_way(f32());
            else if (p.a.dtype == GEO_SC_BF16) of_way(bf16());
            else of_way(f16());
        };
        uint32_t ahead[16] = {};
        const auto ask_first = [&](int first) {
            of_kind([&](auto y, auto way) { Batch<decltype(y), way()>::ask(p, e, m0 + first, n, ahead); });
        };
        ask_first(0);
        put<0>(sum, area, lane);   // (in front of the loop: their registers are free from here on)
#pragma unroll 1
        for (int first = 0;;) {
            __builtin_amdgcn_wave_barrier();
            of_kind([&](auto y, auto way) { rows<decltype(y), way()>(p, area, wave, lane, first, ahead); });
            __builtin_amdgcn_wave_barrier();
            first += ROWS;
            if (first >= kCols) break;
            ask_first(first);
            static_assert(kCols <= 2 * ROWS || kCols == 4 * ROWS, "");
            if constexpr (kCols > ROWS)
                if (first == ROWS) put<ROWS>(sum, area, lane);
            if constexpr (kCols > 2 * ROWS) {
                if (first == 2 * ROWS) put<2 * ROWS>(sum, area, lane);
                if (first == 3 * ROWS) put<3 * ROWS>(sum, area, lane);
            }
        }
    }
};

// Rows that start at multiples of 16 bytes, and four whole stages of every split.  The loads write LDS themselves, into a ring of
// kRing stages: while a wave multiplies stage s out of registers, stage s + 1 moves from LDS to its other registers and the stages
// up to s + kRing are on their way.  One barrier per stage: it says that every wave's share of stage s + 1 has come and
// that all have read stage s, whose place stage s + kRing takes.
// Bound by power: 8192 x 16384 x 4096 in 446 - 452 us (2.43 - 2.46 POP/s) at 1.95 GHz, where the products alone run at 2.17; both gradients of
// 4096 x 4096 x 4096 bf16 in 200 us (1.37 PFLOP/s).
// finish(p, sum, ring, wave, lane) stores the sums of a tile; `ring` gives the place of a stage, kBytes each, which is free then.
template <int B, bool INT8, typename Finish>
__device__ __forceinline__ void tiles_body(const TwoProducts& both, Finish finish)
{
    typedef Tiling<B, INT8> G;
    constexpr int T = G::T, L = G::L;
    // (arrays of their own, not one: the compiler keeps reads of one apart from loads into another)
    __shared__ __align__(16) uint8_t ring0[G::kBytes], ring1[G::kBytes], ring2[G::kBytes], ring3[G::kBytes];
    const auto place = [&](auto which) -> uint8_t* {
        constexpr int r = decltype(which)::value % kRing;
        if constexpr (r == 0) return ring0;
        else if constexpr (r == 1) return ring1;
        else if constexpr (r == 2) return ring2;
        else return ring3;
    };
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const Fragments<B> fragments(wave, lane);

    Spot p;
    int x_off[L], w_off[L];
    __amdgpu_buffer_rsrc_t xr, wr;
    int xk, wk, x_begin, x_end, w_begin, w_end;   // bytes of the inner dimension: next to load; where its turn ends and goes on
    const auto load_one = [&](uint8_t* to, int i) {
        if (i < L) load_to_lds(xr, to + (i * kWaves + wave) * 1024, x_off[i], xk);
        else load_to_lds(wr, to + (i * kWaves + wave) * 1024, w_off[i - L], wk);
    };
    const auto advance = [&]() {
        xk += kStage;
        wk += kStage;
        wk = xk == x_end ? w_begin : wk == w_end ? 0 : wk;
        xk = xk == x_end ? x_begin : xk;
    };
    const auto load = [&](uint8_t* to) {
#pragma unroll
        for (int i = 0; i < 2 * L; ++i) load_one(to, i);
        advance();
    };
    const auto start = [&](uint32_t work) {
        p = spot_of<B>(both, work);
#pragma unroll
        for (int i = 0; i < L; ++i) {
            x_off[i] = (int)(load_row(p.m0, p.a.rows, i, wave, lane) * p.a.x_stride) + load_piece_of(lane) * 16;
            w_off[i] = (int)(load_row(p.n0, p.a.cols, i, wave, lane) * p.a.w_stride) + load_piece_of(lane) * 16;
        }
        xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.a.x + p.m0 * p.a.x_stride), 0, 0x7fffffff, 0x00020000);
        wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.a.w + p.n0 * p.a.w_stride), 0, 0x7fffffff, 0x00020000);
        // Each die starts at a place of its own in the inner dimension: all at once at the same columns of power-of-two strides
        // meet in the same channels of the memory (the loads alone of 8192 x 16384 x 4096: 340 us, so 282).
        const int first = p.begin + (int)((int64_t)(p.stop - p.begin) * p.die / 8);
        x_begin = p.begin * kStage;
        x_end = p.stop * kStage;
        w_begin = w_stage(p.a, p.begin) * kStage;
        w_end = p.a.w_stages < 0x7fffffff / kStage ? p.a.w_stages * kStage : -1;
        xk = first * kStage;
        wk = w_stage(p.a, first) * kStage;
        load(ring0);
        load(ring1);
        load(ring2);
        load(ring3);
    };
    // All but the newest `flying` loads of a wave have come, for all waves, and all have what they read before.
    const auto arrive = [&](auto flying) { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(flying)::value) : "memory"); };

    typename G::Sum sum[T][T];
    v4i f[2][2 * T];
    // Multiplies stage k, which is in f[which & 1]; `steady`: at least kRing stages follow.  Everything else stands between the
    // products, little at a time: a wave issues in order, one instruction in four cycles, and a product takes sixteen.  The
    // next stage's reads in the first half, the loads over all of it, their next place in the second.
    constexpr int kLoads = 2 * L, kProducts = T * T, kPer = kProducts / kLoads;
    const auto stage = [&](auto which, int k, auto steady) {
        constexpr int r = decltype(which)::value;
        constexpr bool kSteady = decltype(steady)::value;
        if (kSteady || k + kRing <= p.stop) arrive(Int<(kRing - 2) * kLoads>());
        else if (k + kRing - 1 <= p.stop) arrive(Int<(kRing - 3) * kLoads>());
        else arrive(Int<0>());
        if (!kSteady && k + kRing < p.stop) load(place(which));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < kProducts; ++u) {
            multiply_one<INT8, true, T>(f[r & 1], sum, u);
            __builtin_amdgcn_sched_barrier(0);
            // (behind the last stage the reads bring what nobody uses)
#pragma unroll
            for (int t = 0; t < 2 * T; ++t)
                if (t * kProducts / (4 * T) == u) fragments.read_one(f[(r + 1) & 1], place(Int<r + 1>()), t);
            if constexpr (kSteady) {
                if (u % kPer == kPer / 2) load_one(place(which), u / kPer);
                if (u == kProducts - 1) advance();
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    start(blockIdx.x);
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
        for (int i = 0; i < T; ++i) sum[j][i] = typename G::Sum{0, 0, 0, 0};
    arrive(Int<(kRing - 1) * kLoads>());
    fragments.read(f[0], ring0);
    int k = p.begin;
    for (; k + 2 * kRing <= p.stop; k += kRing) {
        stage(Int<0>(), k, std::true_type());
        stage(Int<1>(), k + 1, std::true_type());
        stage(Int<2>(), k + 2, std::true_type());
        stage(Int<3>(), k + 3, std::true_type());
    }
    for (; k < p.stop; k += kRing) {
        stage(Int<0>(), k, std::false_type());
        if (k + 1 < p.stop) stage(Int<1>(), k + 1, std::false_type());
        if (k + 2 < p.stop) stage(Int<2>(), k + 2, std::false_type());
        if (k + 3 < p.stop) stage(Int<3>(), k + 3, std::false_type());
    }
    finish.ask(p, wave, lane);
    if (p.stop < p.end) {   // a last stage that is not whole
        v4i v[2 * L];
        fetch_stage<L>(p, p.stop, wave, lane, v);
        __syncthreads();
        put_stage<L>(ring0, wave, lane, v);
        __syncthreads();
        fragments.read(f[0], ring0);
        multiply<INT8, true, T>(f[0], sum);
    }
    settle(sum);
    finish(p, sum, wave == 0 ? ring0 : wave == 1 ? ring1 : wave == 2 ? ring2 : ring3, wave, lane);
}
template <int B, bool INT8>
__global__ __launch_bounds__(kWaves * 64) void k_tiles(TwoProducts both)
{
    __shared__ __align__(16) uint8_t areas[kWaves][Tiling<B, INT8>::kArea];
    struct Finish {
        uint8_t (*areas)[Tiling<B, INT8>::kArea];
        TileScales<B / 32> scales;
        __device__ __forceinline__ void ask(const Spot& p, int wave, int lane) { scales.load(p, wave, lane); }
        __device__ __forceinline__ void operator()(const Spot& p, typename Matrix<INT8>::Sum (&sum)[B / 32][B / 32], uint8_t*, int wave, int lane)
        {
            finish_tile<B, INT8>(p, sum, scales, areas[wave], wave, lane);
        }
    };
    tiles_body<B, INT8>(both, Finish{areas, {}});
}
// (the ring takes the sums on their way out: 128 KB of LDS for the largest tile)
template <int B>
__global__ __launch_bounds__(kWaves * 64, 256 / B) void k_tiles_epilogue(TwoProducts both, Epilogue e)
{
    struct Finish {
        EpilogueTile<B, B / 2 < 64 ? B / 2 : 64> tile;
        __device__ __forceinline__ void ask(const Spot& p, int wave, int lane) { tile.ask(p, wave, lane); }
        __device__ __forceinline__ void operator()(const Spot& p, v4i (&sum)[B / 32][B / 32], uint8_t* place, int wave, int lane)
        {
            __syncthreads();   // all have read the last stage
            tile.finish(p, sum, place, wave, lane);
        }
    };
    tiles_body<B, true>(both, Finish{{e}});
}

// Fewer stages than the ring of k_tiles holds, at any alignment: stages through registers, the next one on its way while one is
// multiplied.  1000 x 1000 x 239: 6.6 us, its launch and one way to memory and back.
template <int B, bool INT8, bool EPILOGUE>
__global__ __launch_bounds__(kWaves * 64) void k_tiles_any(TwoProducts both, Epilogue e)
{
    typedef Tiling<B, INT8> G;
    constexpr int T = G::T, L = G::L;
    constexpr int kArea = EPILOGUE ? 32 * T * 64 : G::kArea;   // (32 rows of sums)
    __shared__ __align__(16) uint8_t buffers[2][G::kBytes];
    __shared__ __align__(16) uint8_t areas[kWaves][kArea];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const Fragments<B> fragments(wave, lane);
    const Spot p = spot_of<B>(both, blockIdx.x);
    typename G::Sum sum[T][T];
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
        for (int i = 0; i < T; ++i) sum[j][i] = typename G::Sum{0, 0, 0, 0};
    v4i v[2 * L], f[2 * T];
    fetch_stage<L>(p, p.begin, wave, lane, v);
    put_stage<L>(buffers[0], wave, lane, v);
    __syncthreads();
    for (int k = p.begin; k < p.end; ++k) {
        if (k + 1 < p.end) fetch_stage<L>(p, k + 1, wave, lane, v);
        fragments.read(f, buffers[(k - p.begin) & 1]);
        multiply<INT8, false, T>(f, sum);
        if (k + 1 < p.end) put_stage<L>(buffers[(k - p.begin + 1) & 1], wave, lane, v);
        __syncthreads();
    }
    if constexpr (EPILOGUE) {
        EpilogueTile<B, 32> tile = {e};
        tile.ask(p, wave, lane);
        tile.finish(p, sum, areas[wave], wave, lane);
    } else {
        TileScales<T> scales;
        scales.load(p, wave, lane);
        finish_tile<B, INT8>(p, sum, scales, areas[wave], wave, lane);
    }
}

// Rows that start anywhere, laid out anew at multiples of 16 bytes for k_tiles: a piece of a row per thread.  What lies behind a
// row's end up to such a multiple is zero.  (4096 x 4096 x 4095, odd strides: 76 us, of which the copies 10; k_tiles_any on them as
// they lie 231.  1009 x 1003 x 1111: 10.6 and 16.7.)
struct AlignArgs {
    const uint8_t* from[2];   // x, w; NULL: is aligned
    uint8_t* to[2];
    int64_t stride[2];
    uint32_t works[2], pieces;
    int64_t inner;
};
__global__ __launch_bounds__(256) void k_align_rows(AlignArgs a)
{
    const uint32_t groups = (a.works[0] + 255) / 256, which = blockIdx.x >= groups;
    const uint32_t work = (blockIdx.x - (which ? groups : 0)) * 256 + threadIdx.x;
    if (work >= a.works[which]) return;
    const int64_t row = work / a.pieces, c = (int64_t)(work % a.pieces) * 16;
    const uint8_t* from = a.from[which] + row * a.stride[which];
    v4i v;
    if (c + 16 <= a.inner) {
        const Shifted<1> any(from + c);
        v = any.piece(any.load(0), 0);
    } else {
        v = load_piece(from, c, a.inner);
    }
    *(v4i*)(a.to[which] + (int64_t)work * 16) = v;
}

// Few rows of x (at most 16 MT): y is bound by the one read of w.  A wave reads 128 bytes of 16 rows of w per step, 32 per lane,
// straight into the registers that the matrix instruction takes, and the same bytes of x; a workgroup's waves, and the
// grid's second dimension, cut the inner dimension, and the sums meet in LDS.  SHIFTED: rows that start anywhere.
constexpr int kFewWaves = 8, kStep = 2 * kStage;
template <int MT, bool SHIFTED, bool EPILOGUE>
__global__ __launch_bounds__(kFewWaves * 64) void k_few_rows(TileArgs a, uint32_t first_tile, Epilogue e)
{
    __shared__ __align__(16) v4i sums[kFewWaves][MT][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t n0 = ((int64_t)first_tile + blockIdx.x) * 16;
    const int row = lane & 15, at = (lane >> 4) * 32;
    typedef Shifted<2> Any;
    using Place = std::conditional_t<SHIFTED, Any, const uint8_t*>;
    Place xp[MT], wp;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = i * 16 + row;
        xp[i] = Place(a.x + (m < a.rows ? m : a.rows - 1) * a.x_stride + at);
    }
    const uint8_t* w_row = a.w + (n0 + row < a.cols ? n0 + row : a.cols - 1) * a.w_stride;
    wp = Place(w_row + at);
    v4i sum[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) sum[i] = v4i{0, 0, 0, 0};
    const int steps = (int)((a.inner + kStep - 1) / kStep), whole = (int)(a.inner / kStep);
    const int begin = blockIdx.y * (a.stages_per_split / 2);
    const int end = begin + a.stages_per_split / 2 < steps ? begin + a.stages_per_split / 2 : steps;
    const int end_whole = end < whole ? end : whole;
    struct Plain {
        v4i two[2];
    };
    using Bytes = std::conditional_t<SHIFTED, Any::Words, Plain>;   // 32 of a row, as they are loaded
    struct Step {
        Bytes w, x[MT];
    };
    const auto load_one = [&](const Place& from, int64_t o) {
        if constexpr (SHIFTED) {
            return from.load(o);
        } else {
            Plain t;
            __builtin_memcpy(t.two, from + o, 32);
            return t;
        }
    };
    const auto half_of = [&](const Place& from, const Bytes& t, int h) {
        if constexpr (SHIFTED) return from.piece(t, h);
        else return t.two[h];
    };
    const auto multiply = [&](const Step& t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const v4i w = half_of(wp, t.w, h);
#pragma unroll
            for (int i = 0; i < MT; ++i) Matrix<true>::add(w, half_of(xp[i], t.x[i], h), sum[i]);
        }
    };
    const auto load = [&](Step& t, int k) {
        const int64_t o = (int64_t)k * kStep;
        t.w = load_one(wp, o);
#pragma unroll
        for (int i = 0; i < MT; ++i) t.x[i] = load_one(xp[i], o);
    };
    // kAhead steps on their way at once, x at the distance of w: loads come back in order.  (The steady part by itself, with
    // no condition around its loads: behind one, the compiler waits for all of them.)
    constexpr int kAhead = 16 / (MT + 1);
    Step ahead[kAhead];
    int k = begin + wave;
    if (k + (2 * kAhead - 1) * kFewWaves < end_whole) {
#pragma unroll
        for (int d = 0; d < kAhead; ++d) load(ahead[d], k + d * kFewWaves);
        for (; k + (2 * kAhead - 1) * kFewWaves < end_whole; k += kAhead * kFewWaves) {
#pragma unroll
            for (int d = 0; d < kAhead; ++d) {
                multiply(ahead[d]);
                load(ahead[d], k + (d + kAhead) * kFewWaves);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int d = 0; d < kAhead; ++d) multiply(ahead[d]);
        k += kAhead * kFewWaves;
    }
    const int left = k < end_whole ? (end_whole - k + kFewWaves - 1) / kFewWaves : 0;   // fewer than 2 kAhead
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int d = 0; d < kAhead; ++d)
            if (half * kAhead + d < left) load(ahead[d], k + (half * kAhead + d) * kFewWaves);
#pragma unroll
        for (int d = 0; d < kAhead; ++d)
            if (half * kAhead + d < left) multiply(ahead[d]);
    }
    if (end > end_whole && (end_whole - begin) % kFewWaves == wave) {   // the last step, where it is not whole
        const int64_t o = (int64_t)end_whole * kStep + at;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const v4i w = load_piece(w_row, o + h * 16, a.inner);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int64_t m = i * 16 + row;
                Matrix<true>::add(w, load_piece(a.x + (m < a.rows ? m : a.rows - 1) * a.x_stride, o + h * 16, a.inner), sum[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[wave][i][lane] = sum[i];
    __syncthreads();
    for (int t = wave; t < MT; t += kFewWaves) {
        v4i s = sums[0][t][lane];
#pragma unroll
        for (int k = 1; k < kFewWaves; ++k) s += sums[k][t][lane];
        const int64_t m = t * 16 + (lane & 15), n = n0 + (lane >> 4) * 4;
        float ws[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) ws[r] = scale_at(a.w_scale, n + r, a.cols);
        if constexpr (EPILOGUE) finish_four(a, e, m, n, s, scale_at(a.x_scale, m, a.rows), ws);
        else finish_four(a, blockIdx.y, m, n, s, scale_at(a.x_scale, m, a.rows), ws);
    }
}

// The same for rows that start at multiples of 16 bytes: loads in the
// order of the matrix instruction's operands give neighbouring lanes different rows, and the memory pipeline takes such a load's
// lanes one by one (4096 x 16384 bytes of w: 16 us for 16 rows of x, 31 for 48).  Here each wave has a ring of its own in LDS, which
// the loads fill in lines, and no barrier but where the waves' sums meet.  Workgroups stay: a wave's stages run on from one
// 16 columns of y to its next, so that w streams.  48 rows by 4096 x 16384 in 21.5 us: 3.1 TB/s of w, and x three times as much out of L2.
template <int MT, bool EPILOGUE>
__global__ __launch_bounds__(kFewWaves * 64) void k_few_streamed(TileArgs a, Epilogue e)
{
    constexpr int kStageBytes = (1 + MT) * 1024, kPlaces = 16384 / kStageBytes;
    static_assert(kPlaces >= 3 && kPlaces <= 8, "");
    __shared__ __align__(16) uint8_t p0[kFewWaves][kStageBytes], p1[kFewWaves][kStageBytes], p2[kFewWaves][kStageBytes],
        p3[kFewWaves][kStageBytes], p4[kFewWaves][kStageBytes], p5[kFewWaves][kStageBytes], p6[kFewWaves][kStageBytes], p7[kFewWaves][kStageBytes];
    __shared__ __align__(16) v4i sums[kFewWaves][MT][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const auto place = [&](auto which) -> uint8_t* {
        constexpr int r = decltype(which)::value % kPlaces;
        if constexpr (r == 0) return p0[wave];
        else if constexpr (r == 1) return p1[wave];
        else if constexpr (r == 2) return p2[wave];
        else if constexpr (r == 3) return p3[wave];
        else if constexpr (r == 4) return p4[wave];
        else if constexpr (r == 5) return p5[wave];
        else if constexpr (r == 6) return p6[wave];
        else return p7[wave];
    };
    const int whole = (int)(a.inner / kStage), each = (whole - wave + kFewWaves - 1) / kFewWaves;   // a wave's stages of a tile: at least 1
    const int tiles = (int)((a.cols + 15) / 16), my_tiles = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    const int total = each * my_tiles;

    // loads: 16 rows of 64 bytes, a lane a piece; the pieces of rows r lie at positions piece ^ (r / 4 & 2)
    const int piece = ((lane & 3) ^ (lane >> 4 & 2)) * 16, load_row = lane >> 2;
    int x_off[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = i * 16 + load_row;
        x_off[i] = (int)((m < a.rows ? m : a.rows - 1) * a.x_stride) + piece;
    }
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.x), 0, 0x7fffffff, 0x00020000);
    int load_tile = blockIdx.x, load_stage = wave;
    const auto load = [&](uint8_t* to) {   // the wave's next stage
        const int64_t n0 = (int64_t)load_tile * 16, last = a.cols - 1 - n0;
        const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.w + n0 * a.w_stride), 0, 0x7fffffff, 0x00020000);
        const int w_off = (int)((load_row < last ? load_row : last) * a.w_stride) + piece, at = load_stage * kStage;
        load_to_lds(wr, to, w_off, at);
#pragma unroll
        for (int i = 0; i < MT; ++i) load_to_lds(xr, to + (1 + i) * 1024, x_off[i], at);
        load_stage += kFewWaves;
        if (load_stage >= whole) {
            load_stage = wave;
            load_tile += gridDim.x;
        }
    };
    v4i sum[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) sum[i] = v4i{0, 0, 0, 0};
    const int mine = (lane & 15) * kStage + (((lane >> 4) ^ (lane >> 2 & 2)) << 4);
    const auto multiply = [&](const uint8_t* from) {
        const v4i w = *(const v4i*)(from + mine);
#pragma unroll
        for (int i = 0; i < MT; ++i) Matrix<true>::add(w, *(const v4i*)(from + (1 + i) * 1024 + mine), sum[i]);
    };
    // (of a wave that finishes: its rows of y are the same in every tile)
    const int64_t m = wave * 16 + (lane & 15);
    const float xs = wave < MT ? a.x_scale[m < a.rows ? m : a.rows - 1] : 0.f;
    typedef float Scales __attribute__((ext_vector_type(16), aligned(4)));
    typedef const Scales __attribute__((address_space(4)))* ConstScales;
    typedef const float __attribute__((address_space(4)))* ConstFloat;
    int tile = blockIdx.x, left = each;
    // An epilogue comes later, at one place for all stages: in every one of them its code would be there as often as there are places.
    // (A tile has as many stages at least as there are places: no two are held at once.)
    float held[4];
    int64_t held_n = 0;
    bool holds = false;
    const auto finish_held = [&]() {
        if (!EPILOGUE || !holds) return;
        holds = false;
        if (wave >= MT) return;
        float bias[4];
        load_bias(e, held_n, a.cols, bias);
#pragma unroll
        for (int r = 0; r < 4; ++r) held[r] += bias[r];
        finish_columns(a, e, m, held_n, held);
    };
    const auto finish = [&]() {   // the waves' sums of a tile
        const int64_t n0 = (int64_t)tile * 16;
        if (whole * kStage < a.inner && wave == kFewWaves - 1) {   // the last stage, where it is not whole
            const int64_t n = n0 + (lane & 15), k = (int64_t)whole * kStage + (lane >> 4) * 16;
            const v4i w = load_piece(a.w + (n < a.cols ? n : a.cols - 1) * a.w_stride, k, a.inner);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int64_t r = i * 16 + (lane & 15);
                Matrix<true>::add(w, load_piece(a.x + (r < a.rows ? r : a.rows - 1) * a.x_stride, k, a.inner), sum[i]);
            }
        }
        // (barriers that leave the loads on their way)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the last tile's sums have been read
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            sums[wave][i][lane] = sum[i];
            sum[i] = v4i{0, 0, 0, 0};
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (wave < MT) {
            v4i s = sums[0][wave][lane];
#pragma unroll
            for (int k = 1; k < kFewWaves; ++k) s += sums[k][wave][lane];
            // (sixteen scales by a scalar load: a vector load would be waited for behind all that are on their way)
            Scales w16;
            if (n0 + 16 <= a.cols) {
                w16 = *(ConstScales)(a.w_scale + n0);
            } else {
                for (int t = 0; t < 16; ++t) w16[t] = n0 + t < a.cols ? *(ConstFloat)(a.w_scale + n0 + t) : 0.f;
            }
            float ws[4], v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) ws[r] = lane < 16 ? w16[r] : lane < 32 ? w16[4 + r] : lane < 48 ? w16[8 + r] : w16[12 + r];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (float)s[r] * xs * ws[r];
            const int64_t n = n0 + (lane >> 4) * 4;
            if constexpr (EPILOGUE) {
#pragma unroll
                for (int r = 0; r < 4; ++r) held[r] = v[r];
                held_n = n;
            } else {
                if (m < a.rows && n < a.cols) store_four(a.y, a.dtype, m * a.y_stride + n, a.cols - n, v);
            }
        }
        holds = EPILOGUE;
        tile += gridDim.x;
        left = each;
    };
    const auto stage = [&](auto which, int at, auto steady) {
        if (decltype(steady)::value || at + kPlaces <= total) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kPlaces - 1) * (1 + MT)) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        multiply(place(which));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // what was read may be overwritten
        if (decltype(steady)::value || at + kPlaces < total) load(place(which));
        if (--left == 0) finish();
    };
    const auto for_places = [&](auto f) {
        [&]<int... R>(std::integer_sequence<int, R...>) { (f(Int<R>()), ...); }
        (std::make_integer_sequence<int, kPlaces>());
    };
    int at = 0;
    if (total >= 2 * kPlaces) {   // (the steady part by itself, with no condition around its loads: behind one, the compiler waits for all)
        for_places([&](auto which) { load(place(which)); });
        for (; at + 2 * kPlaces <= total; at += kPlaces) {
            finish_held();
            for_places([&](auto which) { stage(which, at + decltype(which)::value, std::true_type()); });
        }
    } else {
        for_places([&](auto which) {
            if (decltype(which)::value < total) load(place(which));
        });
    }
    for (; at < total; at += kPlaces) {
        finish_held();
        for_places([&](auto which) {
            if (at + decltype(which)::value < total) stage(which, at + decltype(which)::value, std::false_type());
        });
    }
    finish_held();
}

// y from the sums of the splits, of both products of a launch: memory, and 3 us at the least
template <bool INT8, bool EPILOGUE>
__global__ __launch_bounds__(256) void k_join_splits(TwoProducts both, Epilogue e)
{
    const bool is_second = blockIdx.x >= both.second_at;
    const TileArgs a = is_second ? both.second : both.first;
    // (products that are cut have fewer than 2^32 outputs: less than a tile for each compute unit)
    const uint32_t at = (blockIdx.x - (is_second ? both.second_at : 0)) * 256 + threadIdx.x, fours = (uint32_t)((a.cols + 3) / 4);
    const int64_t m = at / fours, n = (int64_t)(at % fours) * 4, left = a.cols - n;
    if (m >= a.rows) return;
    typename Matrix<INT8>::Sum s = {0, 0, 0, 0};
    for (int k = 0; k < a.splits; ++k) {
        const uint32_t* p = a.partial + ((int64_t)k * a.rows + m) * a.cols + n;
        uint32_t one[4] = {0, 0, 0, 0};
        if (left >= 4) {
            __builtin_memcpy(one, p, 16);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (r < left) one[r] = p[r];
        }
        s += __builtin_bit_cast(typename Matrix<INT8>::Sum, one);
    }
    const float xs = scale_at(a.x_scale, m, a.rows);
    if constexpr (EPILOGUE) {
        float ws[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) ws[r] = scale_at(a.w_scale, n + r, a.cols);
        finish_four(a, e, m, n, s, xs, ws);
        return;
    }
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (float)s[r] * xs * scale_at(a.w_scale, n + r, a.cols);
    store_four(a.y, a.dtype, m * a.y_stride + n, left, v);
}

// ---------------------------------------------------------------- which kernel, and how the inner dimension is cut

struct Shape {
    int64_t rows, cols, inner;   // bytes of the inner dimension; rows 0: no such product
    int64_t tiles(int64_t t) const { return ((rows + t - 1) / t) * ((cols + t - 1) / t); }
    int64_t steps() const { return (inner + 2 * kStage - 1) / (2 * kStage); }   // a split has whole steps of two stages
};
struct Plan {
    int few;        // squares of 16 rows of k_few_rows; 0: k_tiles
    int tile;       // rows and columns of k_tiles' tile
    int splits[2], stages_per_split[2];
};

// Cuts a product's inner dimension into about `splits`, none of fewer than `least` steps, the last of three at least.
void cut(Plan* p, int which, const Shape& s, int64_t splits, int64_t least)
{
    const int64_t steps = s.steps();
    if (splits > steps / least) splits = steps / least;
    if (splits > 64) splits = 64;
    if (splits < 1 || s.rows * ((s.cols + 3) / 4) > 0x7fffffff) splits = 1;   // (the join counts in 32 bits)
    int64_t per_split = (steps + splits - 1) / splits;
    while (per_split < steps && steps - (steps - 1) / per_split * per_split < 3) ++per_split;
    p->stages_per_split[which] = (int)(2 * per_split);
    p->splits[which] = (int)((steps + per_split - 1) / per_split);
}

// What a tile costs, us, measured: `stage` of a stage where a compute unit has as many workgroups as it holds (and each of them
// alone no less than `alone`), `rest` of everything else.  int8 and fp16 are within a tenth of each other.
struct TileCost {
    int tile, held;
    double stage, alone, rest;
};
constexpr TileCost kTileCosts[] = {{256, 1, .60, .56, 10}, {128, 2, .26, .24, 4}, {64, 4, .115, .08, 3}};
constexpr int64_t kLeastSteps = 8;

// The tile, and the splits of either product, of the least time by that table: what all compute units do together or what the
// longest workgroup does, whichever is more, and the join of the splits.  Of 4096 x 4096 x 4096 tiles of 256 take 57 us, of 128 75, of
// 64 122; of 1009 x 1003 x 1111 29, 11 and 6; both fp32 gradients of 1024 x 4096 x 1024 by 128 take 98 us, cut 78.
Plan plan_of(const Shape& s, const Shape& t, bool int8)
{
    Plan best = {};
    if (int8 && s.rows <= 64) {
        best.few = (int)((s.rows + 15) / 16);
        // (a split and its join cost 3 us, in which a workgroup goes through 16 KB of its rows)
        const int64_t groups = (s.cols + 15) / 16;
        cut(&best, 0, s, groups < kUnits ? kUnits / groups : 1, 128);
        return best;
    }
    const Shape shapes[2] = {s, t};
    const int count = t.rows ? 2 : 1;
    double least = 0;
    for (const TileCost& c : kTileCosts) {
        double work = 0;
        for (int i = 0; i < count; ++i) work += (double)shapes[i].tiles(c.tile) * 2 * shapes[i].steps();
        const double together = c.stage * work / kUnits;
        for (int is_cut = 0; is_cut < 2; ++is_cut) {
            Plan p = {};
            p.tile = c.tile;
            double groups = 0, longest = 0, join = 0;
            for (int i = 0; i < count; ++i) {
                cut(&p, i, shapes[i], is_cut ? (int64_t)(2 * shapes[i].steps() * c.alone / together) + 1 : 1, kLeastSteps);
                groups += (double)shapes[i].tiles(c.tile) * p.splits[i];
                if (p.stages_per_split[i] * c.alone > longest) longest = p.stages_per_split[i] * c.alone;
                if (p.splits[i] > 1) join += 8e-6 / 4 * p.splits[i] * shapes[i].rows * shapes[i].cols;
            }
            const double rounds = (double)((int64_t)groups / (kUnits * c.held) + 1);
            const double time = (together > longest ? together : longest) + c.rest * rounds + (join > 0 ? 4 + join : 0);
            if (!best.tile || time < least) {
                best = p;
                least = time;
            }
        }
    }
    return best;
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
size_t partial_bytes(const Plan& p, int which, const Shape& s) { return p.splits[which] > 1 ? align256((size_t)p.splits[which] * s.rows * s.cols * 4) : 0; }

// loads that write LDS take 16-byte addresses, and offsets of 31 bits from a tile's first row
bool loads_fit(const uint8_t* p, int64_t stride, int64_t rows, int64_t inner)
{
    return (uintptr_t)p % 16 == 0 && stride % 16 == 0 && stride * rows + inner < 0x7fffffff;
}

bool is_direct(const TileArgs& a, int tile)
{
    const int64_t last = a.inner / kStage - (int64_t)(a.splits - 1) * a.stages_per_split;   // whole stages of the last split
    return last >= kRing && loads_fit(a.x, a.x_stride, tile, a.inner) && loads_fit(a.w, a.w_stride, tile, a.inner);
}

// The aligned copies that a product in tiles takes (none where it has fewer stages than k_tiles needs).
struct Copies {
    size_t x, w;   // bytes, 0: none
};
Copies copies_of(TileArgs a, const Plan& p, int64_t rows, int64_t cols)
{
    const int64_t stride = (a.inner + 15) / 16 * 16;
    a.splits = p.splits[0];
    a.stages_per_split = p.stages_per_split[0];
    if (p.few || is_direct(a, p.tile) || (rows + cols) * (stride / 16) > kMostGroups * 256) return {};   // (one launch)
    const bool x = !loads_fit(a.x, a.x_stride, p.tile, a.inner), w = !loads_fit(a.w, a.w_stride, p.tile, a.inner);
    if (x) a.x = nullptr, a.x_stride = stride;   // (a place of any alignment)
    if (w) a.w = nullptr, a.w_stride = stride;
    if (!is_direct(a, p.tile)) return {};
    return {x ? align256((size_t)rows * stride) : 0, w ? align256((size_t)cols * stride) : 0};
}

// Measured, us: 4096 x 4096, k_few_rows / streamed: 1 row 5.0 / 5.2, 4 rows 5.4 / 5.2, 16 rows 6.4 / 5.5; 4096 x 1024: 3.2 / 3.8 for
// any; 4096 x 16384: 16 rows 19.1 / 17.1, 48 rows 31 / 22, 64 rows 39 / 25.  Rows at odd addresses, 4096 x 16384: 1 row 18, 16 rows 24,
// 48 rows 41 (loaded as they lie 34, 39, 112).
bool is_streamed(const TileArgs& a)
{
    return a.splits == 1 && a.rows > 2 && a.inner >= 4 * kFewWaves * kStage && loads_fit(a.x, a.x_stride, 64, a.inner) &&
           loads_fit(a.w, a.w_stride, 16, a.inner);
}

// `e`: the epilogue, or NULL
template <int MT>
void run_few(const TileArgs& a, const Epilogue* e, hipStream_t s)
{
    constexpr int kPlaces = 16384 / ((1 + MT) * 1024);   // (an epilogue: as many stages of a tile for each wave)
    if (is_streamed(a) && (!e || a.inner / kStage / kFewWaves >= kPlaces)) {
        const int64_t tiles = (a.cols + 15) / 16;
        const dim3 grid((uint32_t)(tiles < kUnits ? tiles : kUnits)), block(kFewWaves * 64);
        if (e) k_few_streamed<MT, true><<<grid, block, 0, s>>>(a, *e);
        else k_few_streamed<MT, false><<<grid, block, 0, s>>>(a, {});
        return;
    }
    const bool words = ((uintptr_t)a.x | (uintptr_t)a.w | (uint64_t)a.x_stride | (uint64_t)a.w_stride) % 4 == 0;
    in_launches((a.cols + 15) / 16, kFewWaves * 64, [&](int64_t first, uint32_t tiles) {
        const dim3 grid(tiles, (uint32_t)a.splits), block(kFewWaves * 64);
        const auto run = [&](auto shifted) {
            if (e) k_few_rows<MT, shifted(), true><<<grid, block, 0, s>>>(a, (uint32_t)first, *e);
            else k_few_rows<MT, shifted(), false><<<grid, block, 0, s>>>(a, (uint32_t)first, {});
        };
        if (words) run(std::false_type());
        else run(std::true_type());
    });
}

template <int B, bool INT8>
bool run_tiles(TwoProducts both, const Epilogue* e, bool direct, hipStream_t s)
{
    const auto groups = [](TileArgs& a) {
        a.tiles_m = (int)((a.rows + B - 1) / B);
        a.tiles_n = (int)((a.cols + B - 1) / B);
        return (int64_t)a.tiles_m * a.tiles_n * a.splits;
    };
    const int64_t first = groups(both.first), works = first + (both.second.rows ? groups(both.second) : 0);
    if (works > kMostGroups) return false;   // (more outputs than the memory holds, but for products of less than a tile's height)
    both.second_at = (uint32_t)first;
    const dim3 grid((uint32_t)works), block(kWaves * 64);
    if constexpr (INT8) {
        if (e) {
            if (direct) k_tiles_epilogue<B><<<grid, block, 0, s>>>(both, *e);
            else k_tiles_any<B, true, true><<<grid, block, 0, s>>>(both, *e);
            return true;
        }
    }
    if (direct) k_tiles<B, INT8><<<grid, block, 0, s>>>(both);
    else k_tiles_any<B, INT8, false><<<grid, block, 0, s>>>(both, {});
    return true;
}

// The rows and columns of a product that its last tiles are for, if they are no more than 64 in a direction, as products of their own
// in tiles of 64: 4096 x 4099 takes 272 tiles of 256, a second round of the compute units for 3 rows of w's.
constexpr int64_t kMostStrip = 64;
struct Strips {
    TileArgs main, down, right;   // all but the last rows and columns; the last rows; the last columns of the others (rows 0: none)
    Epilogue down_epilogue, right_epilogue;
};
Strips cut_strips(const TileArgs& a, int tile, const Epilogue* e)
{
    Strips s = {};
    s.main = a;
    const int64_t last_rows = a.rows % tile, last_cols = a.cols % tile;
    const bool down = last_rows && last_rows <= kMostStrip && a.rows > tile, right = last_cols && last_cols <= kMostStrip && a.cols > tile;
    const int y_bytes = dtype_bytes(a.dtype);
    const auto shift = [&](TileArgs& t, Epilogue& f, int64_t row, int64_t col) {
        const int64_t at = row * a.y_stride + col;
        t.x += row * a.x_stride;
        t.w += col * a.w_stride;
        if (t.x_scale) t.x_scale += row;
        if (t.w_scale) t.w_scale += col;
        t.y = (char*)t.y + at * y_bytes;
        if (!e) return;
        f = *e;
        if (f.bias) f.bias = (const char*)f.bias + col * dtype_bytes(f.bias_dtype);
        if (f.residual) f.residual = (const char*)f.residual + (row * f.residual_stride + col) * y_bytes;
        if (f.slope) f.slope = (char*)f.slope + at * (f.slope_dtype == GEO_SC_F32 ? 4 : f.slope_dtype == GEO_SC_F16 ? 2 : 1);
    };
    if (down) {
        s.main.rows -= last_rows;
        s.down = a;
        s.down.rows = last_rows;
        shift(s.down, s.down_epilogue, s.main.rows, 0);
    }
    if (right) {
        s.main.cols -= last_cols;
        s.right = s.main;
        s.right.cols = last_cols;
        shift(s.right, s.right_epilogue, 0, s.main.cols);
    }
    return s;
}
int64_t rounds_of(const TileArgs& a, const TileArgs& b, const TileCost& cost)
{
    const auto tiles = [&](const TileArgs& t) { return ((t.rows + cost.tile - 1) / cost.tile) * ((t.cols + cost.tile - 1) / cost.tile); };
    const int64_t at_once = kUnits * cost.held;
    return (tiles(a) + (b.rows ? tiles(b) : 0) + at_once - 1) / at_once;
}
// Whether strips cost less than the rounds that they save: those last as long as the shorter product's tiles (a compute unit that ends
// them early goes on with the longer one's), a strip is a launch by itself whose few workgroups walk its whole inner dimension.
// Of 158 products and pairs of gradients whose strips save a round, on average within half a per cent of the better way by this rule; 11 off it
// always with strips (1071 x 2974 x 1955, both gradients bf16, four of them: 102 us, 59 without), 5 never (4095 x 4099 x 2047, one: 67 us, 107
// without).
constexpr double kStripRest = 4.5, kStripStage = .16;   // us of a strip, and of each of its stages
bool strips_pay(const TileArgs& a, const TileArgs& b, const Strips& of_a, const Strips& of_b, int tile)
{
    const TileCost& cost = tile == 256 ? kTileCosts[0] : kTileCosts[1];
    const auto stages = [](const TileArgs& t) { return (double)((t.inner + kStage - 1) / kStage); };
    const double shorter = b.rows && stages(b) < stages(a) ? stages(b) : stages(a);
    const double saved = (double)(rounds_of(a, b, cost) - rounds_of(of_a.main, of_b.main, cost)) * (cost.alone * shorter + cost.rest);
    double spent = 0;
    for (const TileArgs* t : {&of_a.down, &of_a.right, &of_b.down, &of_b.right})
        if (t->rows) spent += kStripRest + kStripStage * stages(*t);
    return saved > spent;
}

void set_splits(TwoProducts* both, const Plan& p)
{
    both->first.splits = p.splits[0];
    both->first.stages_per_split = p.stages_per_split[0];
    both->second.splits = p.splits[1];
    both->second.stages_per_split = p.stages_per_split[1];
}
uint8_t* const kAligned = (uint8_t*)256;   // of a workspace, for a query
// How k_tiles goes over its products: whether their rows are taken as they lie, and whether strips are cut off them.
struct Tiles {
    bool direct, cut;
    Strips first, second;
};
Tiles tiles_of(const TwoProducts& both, const Plan& p, const Epilogue* e)
{
    Tiles t = {};
    t.direct = is_direct(both.first, p.tile) && (!both.second.rows || is_direct(both.second, p.tile));
    if (!t.direct || p.tile <= 64 || p.splits[0] != 1 || (both.second.rows && p.splits[1] != 1)) return t;
    t.first = cut_strips(both.first, p.tile, e);
    t.second = cut_strips(both.second, p.tile, nullptr);
    t.cut = strips_pay(both.first, both.second, t.first, t.second, p.tile);
    return t;
}

// Runs one product, or two in one launch (second.rows 0: one).  The caller has made the plan and the partial sums' memory.
// `e`: the epilogue of the one product, or NULL; where the inner dimension is cut, the join has it.
template <bool INT8>
int run_products(TwoProducts both, const Epilogue* e, const Plan& p, hipStream_t s)
{
    const Epilogue* const now = both.first.partial ? nullptr : e;
    set_splits(&both, p);
    if (p.few) {
        if (p.few == 1) run_few<1>(both.first, now, s);
        else if (p.few == 2) run_few<2>(both.first, now, s);
        else if (p.few == 3) run_few<3>(both.first, now, s);
        else run_few<4>(both.first, now, s);
    } else {
        const Tiles t = tiles_of(both, p, now);
        if (t.cut) {
            const auto strip = [&](const TileArgs& a, const Epilogue& e) {
                TwoProducts one = {};
                one.first = a;
                return !a.rows || run_tiles<64, INT8>(one, now ? &e : nullptr, true, s);
            };
            if (!strip(t.first.down, t.first.down_epilogue) || !strip(t.first.right, t.first.right_epilogue) || !strip(t.second.down, {}) ||
                !strip(t.second.right, {}))
                return GEO_SC_ERR_UNSUPPORTED;
            both.first = t.first.main;
            both.second = t.second.main;
        }
        const bool fits = p.tile == 256   ? run_tiles<256, INT8>(both, now, t.direct, s)
                          : p.tile == 128 ? run_tiles<128, INT8>(both, now, t.direct, s)
                                          : run_tiles<64, INT8>(both, now, t.direct, s);
        if (!fits) return GEO_SC_ERR_UNSUPPORTED;
    }
    const auto joins = [](const TileArgs& a) { return a.partial ? (uint32_t)((a.rows * ((a.cols + 3) / 4) + 255) / 256) : 0u; };
    both.second_at = joins(both.first);
    const uint32_t all = both.second_at + joins(both.second);
    if (all) {
        if constexpr (INT8) {
            if (e) k_join_splits<true, true><<<dim3(all), dim3(256), 0, s>>>(both, *e);
            else k_join_splits<true, false><<<dim3(all), dim3(256), 0, s>>>(both, {});
        } else {
            k_join_splits<false, false><<<dim3(all), dim3(256), 0, s>>>(both, {});
        }
    }
    return hipGetLastError() == hipSuccess ? GEO_SC_OK : GEO_SC_ERR_LAUNCH;
}

// ---------------------------------------------------------------- operands of the gradients
//
// Two launches.  k_grad_peaks, in blocks of peak_rows x peak_cols of g: the largest |g[m][n] w_scale[n]| of each row in the block,
// the largest |g[m][n] x_scale[m]| of each column.  k_grad_operands, its workgroups in three ranges:
//   g in tiles of 64 x 64: the blocks' maxima joined to powers of two dx_back[m], dw_back[n];
//     dx_left[m][term][n] = terms of g[m][n] w_scale[n] / dx_back[m],  dw_left[n][term][m] = terms of g[m][n] x_scale[m] / dw_back[n]
//   w in tiles of 64 x 128: dx_right[k][n] = w[n][k] in fp16
//   x in tiles of 64 x 128: dw_right[k][m] = x[m][k] in fp16
// Rows of an output are padded to whole stages of 64 elements per term, with zeros.  Bound by memory: 4096 x 4096 x 4096 bf16 reads 67
// MB, writes 134 MB in 45 us (4.5 TB/s).
constexpr int kSide = 64, kWide = 128;
constexpr int kPeakWide = 64 * kChunk;     // columns that a wave looks at
constexpr int kPeakBatch = 8;              // rows that it asks for at once
constexpr int kPeakWaves = 16;             // of a workgroup, at most
constexpr int64_t kMostPeakRows = 2048;    // rows of a block, whose maxima are kept in LDS

struct OperandArgs {
    const void* g;
    int dtype;
    int64_t g_stride, x_stride, w_stride, rows, cols, inner;
    const int8_t *x, *w;
    const float *x_scale, *w_scale;
    int64_t rows_padded, cols_padded, peak_rows, peak_cols;
    uint32_t row_blocks, col_blocks, g_tiles, w_tiles;   // tiles: workgroups of the first two ranges
    uint32_t *row_peaks, *col_peaks;                 // [col_blocks][rows], [row_blocks][cols]: bits of the maxima
    const void* slope;                               // [rows][cols] that g is multiplied by on its way in, or NULL
    int slope_dtype;
    float* col_sums;                                 // [row_blocks][cols] of g slope, or NULL
    void* dbias;
    int dbias_dtype;
    float *dx_back, *dw_back;
    f16 *dx_left, *dx_right, *dw_left, *dw_right;    // NULL, with its peaks: that gradient is not wanted
};

// The power of two that brings magnitudes up to `peak` to 2^14 .. 2^15, and its inverse.  Of a row with an infinity or NaN, whose
// every result is one, it leaves the others finite.  The inverse is no denormal, for peaks below 2^-112 either.
__device__ __forceinline__ float power_for(uint32_t peak, float* back)
{
    const uint32_t e = peak >> 23 & 255, field = e > 15 ? 268 - e : 253;
    *back = __uint_as_float((254 - field) << 23);
    return __uint_as_float(field << 23);
}

// (where the slope is zero nothing comes through, no infinity either)
__device__ __forceinline__ float through_slope(float g, float slope) { return slope == 0.f ? 0.f : g * slope; }

// the terms of v: each the fp16 nearest to what the earlier ones leave
template <int TERMS>
__device__ __forceinline__ void store_terms(const float (&v)[kChunk], f16* out, int64_t padded)
{
    f16 t[TERMS][kChunk];
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
        t[0][j] = (f16)v[j];
        if constexpr (TERMS == 2) {
            const float left = v[j] - (float)t[0][j];
            t[1][j] = fabsf(left) < __uint_as_float(kInfinityBits) ? (f16)left : (f16)0.f;   // of an infinity nothing is left
        }
    }
#pragma unroll
    for (int i = 0; i < TERMS; ++i) __builtin_memcpy(out + i * padded, t[i], sizeof t[i]);
}

// A wave takes eight rows of 512 columns at once, a lane eight columns of them; a workgroup's waves pass over its block's rows, then
// over further columns.  What lies outside is the last row and the last columns once more: a maximum stays what it is.
// Bound by memory, the block's rows all asked for at once: 4096 x 4096 bf16 in 16 us.
// NARROW: g has fewer columns than a lane takes.  SLOPE: g is multiplied by a slope of type S on its way in.  SUMS: the columns' sums too, where
// they are asked for.  Either takes four rows at once: the registers for eight are more than a wave of such workgroups has.
template <typename T, bool NARROW, bool SUMS, bool SLOPE, typename S>
__global__ __launch_bounds__(kPeakWaves * 64) void k_grad_peaks(OperandArgs a)
{
    constexpr int kBatch = SLOPE || SUMS ? 4 : kPeakBatch;
    __shared__ uint32_t row_most[kMostPeakRows], col_most[kPeakWaves * kPeakWide];   // (a wave writes its own rows')
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const uint32_t across = blockIdx.x / a.row_blocks, down = blockIdx.x % a.row_blocks;
    const int64_t r0 = down * a.peak_rows, r1 = r0 + a.peak_rows < a.rows ? r0 + a.peak_rows : a.rows;
    const int64_t c0 = across * a.peak_cols, c1 = c0 + a.peak_cols < a.cols ? c0 + a.peak_cols : a.cols;
    for (int64_t from = c0; from < c1; from += kPeakWide) {
        const int64_t own = from + lane * kChunk, c = NARROW || own + kChunk <= a.cols ? own : a.cols - kChunk;
        float ws[kChunk] = {};
        uint32_t most[kChunk] = {};
        float sums[kChunk] = {};
        if (a.row_peaks) load_chunk(a.w_scale, c, a.cols, 0.f, ws);
        for (int64_t r = r0 + wave * kBatch; r < r1; r += waves * kBatch) {
            T raw[kBatch][kChunk];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const T* row = (const T*)a.g + (r + i < r1 ? r + i : r1 - 1) * a.g_stride;
                if constexpr (NARROW) {
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) raw[i][j] = c + j < a.cols ? row[c + j] : (T)0.f;
                } else {
                    __builtin_memcpy(raw[i], row + c, sizeof raw[i]);
                }
            }
            S slope[SLOPE ? kBatch : 1][kChunk];
            if constexpr (SLOPE) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const S* row = (const S*)a.slope + (r + i < r1 ? r + i : r1 - 1) * a.cols;
                    if constexpr (NARROW) {
#pragma unroll
                        for (int j = 0; j < kChunk; ++j) slope[i][j] = c + j < a.cols ? row[c + j] : (S)0;
                    } else {
                        __builtin_memcpy(slope[i], row + c, sizeof slope[i]);
                    }
                }
            }
            uint32_t m[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const float xs = a.col_peaks ? fabsf(a.x_scale[r + i < r1 ? r + i : r1 - 1]) : 0.f;
                m[i] = 0;
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    float v = (float)raw[i][j];
                    if constexpr (SLOPE) v = through_slope(v, (float)slope[i][j]);
                    if constexpr (SUMS) sums[j] += r + i < r1 ? v : 0.f;
                    v = fabsf(v);
                    most[j] = max(most[j], __float_as_uint(v * xs));
                    m[i] = max(m[i], __float_as_uint(v * fabsf(ws[j])));
                }
            }
            if (a.row_peaks) {
                // lanes trade halves of their rows until each holds one, row lane % kBatch
#pragma unroll
                for (int half = kBatch / 2; half >= 1; half /= 2)
#pragma unroll
                    for (int i = 0; i < half; ++i) {
                        const bool upper = lane & half;
                        const uint32_t keep = upper ? m[i + half] : m[i], give = upper ? m[i] : m[i + half];
                        m[i] = max(keep, (uint32_t)__shfl_xor((int)give, half));
                    }
#pragma unroll
                for (int d = kBatch; d < 64; d *= 2) m[0] = max(m[0], (uint32_t)__shfl_xor((int)m[0], d));
                const int64_t at = r - r0 + lane;
                if (lane < kBatch && r + lane < r1) row_most[at] = from > c0 ? max(row_most[at], m[0]) : m[0];
            }
        }
        if (a.col_peaks) {
#pragma unroll
            for (int j = 0; j < kChunk; ++j) col_most[(wave * kChunk + j) * 64 + lane] = most[j];
            __syncthreads();
            for (int k = threadIdx.x; k < kPeakWide; k += blockDim.x) {
                uint32_t one = 0;
                for (int v = 0; v < waves; ++v) one = max(one, col_most[v * kPeakWide + k]);
                const int64_t mine = from + k % 64 * kChunk, n = (NARROW || mine + kChunk <= a.cols ? mine : a.cols - kChunk) + k / 64;
                if (n < a.cols) a.col_peaks[down * a.cols + n] = one;
            }
            __syncthreads();
        }
        if (SUMS && a.col_sums) {
#pragma unroll
            for (int j = 0; j < kChunk; ++j) col_most[(wave * kChunk + j) * 64 + lane] = __float_as_uint(sums[j]);
            __syncthreads();
            for (int k = threadIdx.x; k < kPeakWide; k += blockDim.x) {
                float one = 0.f;
                for (int v = 0; v < waves; ++v) one += __uint_as_float(col_most[v * kPeakWide + k]);
                const int64_t mine = from + k % 64 * kChunk, n = (NARROW || mine + kChunk <= a.cols ? mine : a.cols - kChunk) + k / 64;
                if (n < a.cols) a.col_sums[down * a.cols + n] = one;
            }
            __syncthreads();
        }
    }
    if (!a.row_peaks) return;
    __syncthreads();
    for (int64_t r = threadIdx.x; r < r1 - r0; r += blockDim.x) a.row_peaks[across * a.rows + r0 + r] = row_most[r];
}

// The maxima and sums of more than kMostJoined blocks of rows, into the first block's place: every tile of k_grad_operands would
// read the maxima, of kJoinedElements elements or more in as much time as this takes at the least, and its first tiles add up the sums, one after
// the other.  k_grad_operands alone / both, us: 5579 x 2138 30 / 28 + 5, 16384 x 256 16.4 / 15.7 + 3.8, 16384 x 1024 31.3 / 26.4 + 3.8, 65536 x 1024
// 134 / 113 + 4.8; with sums 16384 x 1024 52 / 32 + 4.6, 2000 x 2000 30 / 16 + 10, 65536 x 64 44 / 16 + 4.8.
constexpr uint32_t kMostJoined = 32;
constexpr int64_t kJoinedElements = (int64_t)1 << 24;
__global__ __launch_bounds__(256) void k_join_peaks(OperandArgs a)
{
    const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const uint32_t share = threadIdx.x >> 6;
    __shared__ uint32_t most[4][64];
    __shared__ float sums[4][64];
    uint32_t m = 0;
    float s = 0.f;
    if (c < a.cols) {
        if (a.col_peaks) {
#pragma unroll 16
            for (uint32_t k = share; k < a.row_blocks; k += 4) m = max(m, a.col_peaks[k * a.cols + c]);
        }
        if (a.col_sums) {
#pragma unroll 16
            for (uint32_t k = share; k < a.row_blocks; k += 4) s += a.col_sums[k * a.cols + c];
        }
    }
    most[share][threadIdx.x & 63] = m;
    sums[share][threadIdx.x & 63] = s;
    __syncthreads();   // (all have read: a column is one workgroup's)
    if (share || c >= a.cols) return;
    const int i = threadIdx.x;
    if (a.col_peaks) a.col_peaks[c] = max(max(most[0][i], most[1][i]), max(most[2][i], most[3][i]));
    if (a.col_sums) a.col_sums[c] = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
}

// out[c][r] = q[r][c] in fp16 for a tile of 64 rows and 128 columns.  A thread turns four columns of eight rows: it reads a
// word of each row (a row of 33 words: no two lanes meet in a bank) and writes eight rows' values of each column.
constexpr int kWideWords = kWide / 4 + 1;
__device__ __forceinline__ void widen_tile(const int8_t* q, int64_t stride, int64_t rows, int64_t cols, int64_t padded, uint32_t tile, f16* out,
                                           uint32_t* lds)
{
    const uint32_t across = (uint32_t)((cols + kWide - 1) / kWide);
    const int64_t r0 = (int64_t)(tile / across) * kSide, c0 = (int64_t)(tile % across) * kWide;
#pragma unroll
    for (int i = 0; i < kSide * kWide / 16 / 256; ++i) {
        const int piece = i * 256 + threadIdx.x, r = piece / (kWide / 16), c = piece % (kWide / 16) * 16;
        v4i v = {0, 0, 0, 0};
        if (r0 + r < rows && c0 + c < cols) v = load_piece((const uint8_t*)(q + (r0 + r) * stride), c0 + c, cols);
#pragma unroll
        for (int j = 0; j < 4; ++j) lds[r * kWideWords + c / 4 + j] = v[j];
    }
    __syncthreads();
    const int r = threadIdx.x % 8 * 8, c = threadIdx.x / 8 * 4;
    uint32_t words[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) words[j] = lds[(r + j) * kWideWords + c / 4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (c0 + c + j >= cols) break;
        f16 t[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = (f16)(float)(int8_t)(words[k] >> (8 * j));
        __builtin_memcpy(out + (c0 + c + j) * padded + r0 + r, t, sizeof t);
    }
}

// (SLOPE by itself, and no more loads of maxima at once than eight waves on a SIMD have registers for: bf16 7266 x 13203 without a slope 194 us, 243
// with the slope's code in it and eight loads, 205 before there was either; 4096 x 4096 43, 44 and 46.)
template <int TERMS, bool SLOPE>
__global__ __launch_bounds__(256) void k_grad_operands(OperandArgs a)
{
    __shared__ float tile[kSide][kSide + 1];
    __shared__ uint32_t most[2][4][kSide];
    static_assert(sizeof tile >= kSide * kWideWords * 4, "a tile of 8-bit numbers fits");
    if (blockIdx.x >= a.g_tiles) {
        const uint32_t at = blockIdx.x - a.g_tiles;
        if (at < a.w_tiles) widen_tile(a.w, a.w_stride, a.cols, a.inner, a.cols_padded, at, a.dx_right, (uint32_t*)tile);
        else widen_tile(a.x, a.x_stride, a.rows, a.inner, a.rows_padded, at - a.w_tiles, a.dw_right, (uint32_t*)tile);
        return;
    }
    const uint32_t across = (uint32_t)(a.cols_padded / kSide);
    const int64_t r0 = (int64_t)(blockIdx.x / across) * kSide, c0 = (int64_t)(blockIdx.x % across) * kSide;
    constexpr int kPasses = kSide * kSide / kChunk / 256;
    float v[kPasses][kChunk];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int at = i * 256 + threadIdx.x, r = at / (kSide / kChunk), c = at % (kSide / kChunk) * kChunk;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) v[i][j] = 0.f;
        if (r0 + r < a.rows && c0 + c < a.cols) {
            load_chunk(a.g, a.dtype, (r0 + r) * a.g_stride, c0 + c, a.cols, 0.f, v[i]);
            if constexpr (SLOPE) {
                float slope[kChunk];
                if (a.slope_dtype == GEO_SC_U8) load_columns((const uint8_t*)a.slope + (r0 + r) * a.cols + c0 + c, a.cols - c0 - c, slope);
                else load_chunk(a.slope, a.slope_dtype, (r0 + r) * a.cols, c0 + c, a.cols, 0.f, slope);
#pragma unroll
                for (int j = 0; j < kChunk; ++j) v[i][j] = through_slope(v[i][j], slope[j]);
            }
        }
    }
    if (a.dbias && r0 == 0 && threadIdx.x < kSide && c0 + threadIdx.x < a.cols) {
        float sum = 0.f;
        for (uint32_t k = 0; k < a.row_blocks; ++k) sum += a.col_sums[k * a.cols + c0 + threadIdx.x];
        if (a.dbias_dtype == GEO_SC_F32) ((f32*)a.dbias)[c0 + threadIdx.x] = sum;
        else if (a.dbias_dtype == GEO_SC_BF16) ((bf16*)a.dbias)[c0 + threadIdx.x] = (bf16)sum;
        else ((f16*)a.dbias)[c0 + threadIdx.x] = (f16)sum;
    }
    // the blocks' maxima of the tile's rows and columns, a quarter of the blocks per wave
    const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    uint32_t row_most = 0, col_most = 0;
    if (a.dx_left && r0 + lane < a.rows)
        for (uint32_t k = wave; k < a.col_blocks; k += 4) row_most = max(row_most, a.row_peaks[k * a.rows + r0 + lane]);
    if (a.dw_left && c0 + lane < a.cols)
#pragma unroll 4
        for (uint32_t k = wave; k < a.row_blocks; k += 4) col_most = max(col_most, a.col_peaks[k * a.cols + c0 + lane]);
    most[0][wave][lane] = row_most;
    most[1][wave][lane] = col_most;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int at = i * 256 + threadIdx.x, r = at / (kSide / kChunk), c = at % (kSide / kChunk) * kChunk;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) tile[r][c + j] = v[i][j];
    }
    __syncthreads();
    const auto power = [&](int which, int i, float* back) {
        return power_for(max(max(most[which][0][i], most[which][1][i]), max(most[which][2][i], most[which][3][i])), back);
    };
    float back;
    if (a.dx_left) {
        if (c0 == 0 && threadIdx.x < kSide && r0 + threadIdx.x < a.rows) {
            power(0, threadIdx.x, &back);
            a.dx_back[r0 + threadIdx.x] = back;
        }
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int at = i * 256 + threadIdx.x, r = at / (kSide / kChunk), c = at % (kSide / kChunk) * kChunk;
            if (r0 + r >= a.rows) continue;
            float k[kChunk] = {};
            if (c0 + c < a.cols) load_chunk(a.w_scale, c0 + c, a.cols, 0.f, k);
            const float up = power(0, r, &back);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) v[i][j] = v[i][j] * k[j] * up;
            store_terms<TERMS>(v[i], a.dx_left + (r0 + r) * TERMS * a.cols_padded + c0 + c, a.cols_padded);
        }
    }
    if (!a.dw_left) return;
    if (r0 == 0 && threadIdx.x < kSide && c0 + threadIdx.x < a.cols) {
        power(1, threadIdx.x, &back);
        a.dw_back[c0 + threadIdx.x] = back;
    }
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int at = i * 256 + threadIdx.x, c = at / (kSide / kChunk), r = at % (kSide / kChunk) * kChunk;
        if (c0 + c >= a.cols) continue;
        float k[kChunk] = {}, t[kChunk];
        if (r0 + r < a.rows) load_chunk(a.x_scale, r0 + r, a.rows, 0.f, k);
        const float up = power(1, c, &back);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) t[j] = tile[r + j][c] * k[j] * up;
        store_terms<TERMS>(t, a.dw_left + (c0 + c) * TERMS * a.rows_padded + r0 + r, a.rows_padded);
    }
}

int terms_of(int grad_dtype) { return grad_dtype == GEO_SC_BF16 ? 1 : 2; }
int64_t padded_to_side(int64_t n) { return (n + kSide - 1) / kSide * kSide; }   // whole stages of fp16 elements
// rows or columns of a block of which one maximum is taken: some `count` blocks where that leaves each `least` at least
int64_t peak_block(int64_t n, int64_t count, int64_t least, int64_t most)
{
    const int64_t block = ((n + count - 1) / count + least - 1) / least * least;
    return block < most ? block : most;
}

// the workspace of the backward: both gradients' operands, then the splits' sums
struct GradLayout {
    Shape dx, dw;
    Plan plan;   // the first product is dx, or dw where dx is not wanted
    size_t dx_left, dx_right, dx_back, dw_left, dw_right, dw_back, row_peaks, col_peaks, col_sums, first_partial, second_partial, bytes;
    int64_t peak_rows, peak_cols;
};
GradLayout grad_layout(int64_t rows, int64_t cols, int64_t inner, int terms, bool need_dx, bool need_dw, bool need_dbias)
{
    GradLayout l = {};
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align256(bytes);
        return here;
    };
    l.peak_cols = peak_block(cols, 32, kPeakWide, (int64_t)1 << 40);
    // (a workgroup for each compute unit: 16384 x 1024 in 256 blocks 16 us, in 64 32)
    const int64_t across = (cols + l.peak_cols - 1) / l.peak_cols;
    l.peak_rows = peak_block(rows, across >= 8 ? 32 : across >= 2 ? 256 / across : 128, 32, kMostPeakRows);
    if (need_dx) {
        const int64_t p = padded_to_side(cols);
        l.row_peaks = take((size_t)((cols + l.peak_cols - 1) / l.peak_cols) * rows * 4);
        l.dx_back = take((size_t)rows * 4);
        l.dx = {rows, inner, terms * p * 2};
        l.dx_left = take((size_t)rows * terms * p * 2);
        l.dx_right = take((size_t)inner * p * 2);
    }
    if (need_dw) {
        const int64_t p = padded_to_side(rows);
        l.col_peaks = take((size_t)((rows + l.peak_rows - 1) / l.peak_rows) * cols * 4);
        l.dw_back = take((size_t)cols * 4);
        l.dw = {cols, inner, terms * p * 2};
        l.dw_left = take((size_t)cols * terms * p * 2);
        l.dw_right = take((size_t)inner * p * 2);
    }
    const Shape none = {};
    if (need_dx || need_dw) l.plan = plan_of(need_dx ? l.dx : l.dw, need_dx && need_dw ? l.dw : none, false);
    l.first_partial = take(partial_bytes(l.plan, 0, need_dx ? l.dx : l.dw));
    l.second_partial = take(need_dx && need_dw ? partial_bytes(l.plan, 1, l.dw) : 0);
    if (need_dbias) l.col_sums = take((size_t)((rows + l.peak_rows - 1) / l.peak_rows) * cols * 4);
    l.bytes = at;
    return l;
}

// The products of the gradients on a workspace that begins at `base`, without their outputs; the first is dx, or dw where dx is not wanted.
TwoProducts grad_products(const GradLayout& l, uint8_t* base, int terms, bool need_dx, bool need_dw)
{
    const auto product = [&](const Shape& shape, size_t left, size_t right, size_t back, bool cut, size_t partial) {
        TileArgs a = {};
        a.x = base + left;
        a.w = base + right;
        a.x_stride = shape.inner;
        a.w_stride = shape.inner / terms;
        a.rows = shape.rows;
        a.cols = shape.cols;
        a.inner = shape.inner;
        a.w_stages = (int)(a.w_stride / kStage);
        a.x_scale = (const float*)(base + back);
        a.y_stride = shape.cols;
        a.partial = cut ? (uint32_t*)(base + partial) : nullptr;
        return a;
    };
    TwoProducts both = {};
    if (need_dx) both.first = product(l.dx, l.dx_left, l.dx_right, l.dx_back, l.plan.splits[0] > 1, l.first_partial);
    if (need_dw)
        (need_dx ? both.second : both.first) = product(l.dw, l.dw_left, l.dw_right, l.dw_back, l.plan.splits[need_dx ? 1 : 0] > 1,
                                                       need_dx ? l.second_partial : l.first_partial);
    return both;
}

Plan forward_plan(const int8_t* x, int64_t x_stride, const int8_t* w, int64_t w_stride, int64_t rows, int64_t cols, int64_t inner, TileArgs* a)
{
    a->x = (const uint8_t*)x;
    a->w = (const uint8_t*)w;
    a->x_stride = x_stride;
    a->w_stride = w_stride;
    a->rows = rows;
    a->cols = cols;
    a->inner = inner;
    return plan_of({rows, cols, inner}, Shape{}, true);
}

bool sizes_fit(int64_t rows, int64_t cols, int64_t inner)
{
    return rows >= 1 && cols >= 1 && inner >= 1 && rows <= 0x3fffffff && cols <= 0x3fffffff && inner <= 131071;
}

int forward(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride, const float* w_scale, int64_t rows,
            int64_t cols, int64_t inner, void* y, int dtype, const Epilogue* e, void* workspace, size_t workspace_bytes, hipStream_t stream)
{
    if (!sizes_fit(rows, cols, inner) || !dtype_known(dtype) || x_stride < 0 || w_stride < 0 || !x || !w || !x_scale || !w_scale || !y)
        return GEO_SC_ERR_INVALID_ARGUMENT;
    TwoProducts both = {};
    TileArgs& a = both.first;
    const Plan plan = forward_plan(x, x_stride, w, w_stride, rows, cols, inner, &a);
    const size_t partial = partial_bytes(plan, 0, {rows, cols, inner});
    const Copies copies = copies_of(a, plan, rows, cols);
    const size_t need = partial + copies.x + copies.w;
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) return GEO_SC_ERR_WORKSPACE;
    if (copies.x || copies.w) {
        AlignArgs g = {};
        uint8_t* to = (uint8_t*)workspace + partial;
        g.inner = inner;
        g.pieces = (uint32_t)((inner + 15) / 16);
        const auto copy = [&](int which, const uint8_t*& from, int64_t& stride, int64_t count, uint8_t* at) {
            g.from[which] = from;
            g.stride[which] = stride;
            g.works[which] = (uint32_t)count * g.pieces;
            g.to[which] = at;
            from = at;
            stride = (int64_t)g.pieces * 16;
        };
        if (copies.x) copy(0, a.x, a.x_stride, rows, to);
        if (copies.w) copy(1, a.w, a.w_stride, cols, to + copies.x);
        k_align_rows<<<dim3((g.works[0] + 255) / 256 + (g.works[1] + 255) / 256), dim3(256), 0, stream>>>(g);
    }
    a.w_stages = 0x7fffffff;
    a.x_scale = x_scale;
    a.w_scale = w_scale;
    a.y = y;
    a.y_stride = cols;
    a.dtype = dtype;
    a.partial = partial ? (uint32_t*)workspace : nullptr;
    return run_products<true>(both, e, plan, stream);
}

int backward(const void* grad, int grad_dtype, int64_t grad_stride, const void* slope, int slope_type, const int8_t* x, int64_t x_stride,
             const float* x_scale, const int8_t* w, int64_t w_stride, const float* w_scale, int64_t rows, int64_t cols, int64_t inner, void* dx,
             int dx_dtype, void* dw, int dw_dtype, void* dbias, int dbias_dtype, void* workspace, size_t workspace_bytes, hipStream_t s)
{
    if (!sizes_fit(rows, cols, inner) || !dtype_known(grad_dtype) || (dx && !dtype_known(dx_dtype)) || (dw && !dtype_known(dw_dtype)) ||
        (dbias && !dtype_known(dbias_dtype)) || (slope && !slope_type_known(slope_type)) ||
        grad_stride < 0 || (grad_stride && rows > 1 && grad_stride < cols) || x_stride < 0 || w_stride < 0 || !grad || (dx && (!w || !w_scale)) ||
        (dw && (!x || !x_scale)))
        return GEO_SC_ERR_INVALID_ARGUMENT;
    if (!dx && !dw && !dbias) return GEO_SC_OK;
    const int terms = terms_of(grad_dtype);
    const GradLayout l = grad_layout(rows, cols, inner, terms, dx, dw, dbias);
    if (!workspace || workspace_bytes < l.bytes || (uintptr_t)workspace % 16) return GEO_SC_ERR_WORKSPACE;
    const auto tiles = [](int64_t r, int64_t rs, int64_t c, int64_t cs) { return ((r + rs - 1) / rs) * ((c + cs - 1) / cs); };
    const bool products = dx || dw;   // (for the bias alone: the first row of tiles)
    const int64_t g_tiles = tiles(products ? rows : 1, kSide, cols, kSide), w_tiles = dx ? tiles(cols, kSide, inner, kWide) : 0,
                  x_tiles = dw ? tiles(rows, kSide, inner, kWide) : 0;
    const int64_t blocks = tiles(rows, l.peak_rows, cols, l.peak_cols);
    if (g_tiles + w_tiles + x_tiles > kMostGroups || blocks > kMostGroups / (kPeakWaves * 64 / 256)) return GEO_SC_ERR_UNSUPPORTED;
    uint8_t* base = (uint8_t*)workspace;
    OperandArgs o = {};
    o.g = grad;
    o.dtype = grad_dtype;
    o.g_stride = grad_stride;
    o.x_stride = x_stride;
    o.w_stride = w_stride;
    o.rows = rows;
    o.cols = cols;
    o.inner = inner;
    o.x = x;
    o.w = w;
    o.x_scale = x_scale;
    o.w_scale = w_scale;
    o.rows_padded = padded_to_side(rows);
    o.cols_padded = padded_to_side(cols);
    if (dx) {
        o.dx_left = (f16*)(base + l.dx_left), o.dx_right = (f16*)(base + l.dx_right);
        o.dx_back = (float*)(base + l.dx_back), o.row_peaks = (uint32_t*)(base + l.row_peaks);
    }
    if (dw) {
        o.dw_left = (f16*)(base + l.dw_left), o.dw_right = (f16*)(base + l.dw_right);
        o.dw_back = (float*)(base + l.dw_back), o.col_peaks = (uint32_t*)(base + l.col_peaks);
    }
    o.slope = slope;
    o.slope_dtype = slope_type;
    if (dbias) {
        o.col_sums = (float*)(base + l.col_sums);
        o.dbias = dbias;
        o.dbias_dtype = dbias_dtype;
    }
    o.peak_rows = l.peak_rows;
    o.peak_cols = l.peak_cols;
    o.row_blocks = (uint32_t)((rows + l.peak_rows - 1) / l.peak_rows);
    o.col_blocks = (uint32_t)((cols + l.peak_cols - 1) / l.peak_cols);
    o.g_tiles = (uint32_t)g_tiles;
    o.w_tiles = (uint32_t)w_tiles;
    // (with a slope or sums, half as many waves: two workgroups on a compute unit, where one would leave the last few a round of their own)
    const int most_waves = slope || dbias ? kPeakWaves / 2 : kPeakWaves;
    const dim3 peak_threads((uint32_t)((l.peak_rows < most_waves * kPeakBatch ? l.peak_rows / kPeakBatch : most_waves) * 64));
    const auto peaks_of = [&](auto one, auto with_sums, auto with_slope, auto of_slope) {
        using T = decltype(one);
        using S = decltype(of_slope);
        if (cols < kChunk) k_grad_peaks<T, true, with_sums(), with_slope(), S><<<dim3((uint32_t)blocks), peak_threads, 0, s>>>(o);
        else k_grad_peaks<T, false, with_sums(), with_slope(), S><<<dim3((uint32_t)blocks), peak_threads, 0, s>>>(o);
    };
    const auto peaks = [&](auto one) {
        const std::true_type yes;
        const std::false_type no;
        if (!slope && !dbias) peaks_of(one, no, no, one);
        else if (!slope) peaks_of(one, yes, no, one);
        else if (slope_type == GEO_SC_F32) peaks_of(one, yes, yes, f32());
        else if (slope_type == GEO_SC_U8) peaks_of(one, yes, yes, uint8_t());
        else peaks_of(one, yes, yes, f16());
    };
    if (grad_dtype == GEO_SC_F32) peaks(f32());
    else if (grad_dtype == GEO_SC_BF16) peaks(bf16());
    else peaks(f16());
    if (o.row_blocks > kMostJoined && (o.col_sums || (o.col_peaks && rows * cols >= kJoinedElements))) {
        k_join_peaks<<<dim3((uint32_t)((cols + 63) / 64)), dim3(256), 0, s>>>(o);
        o.row_blocks = 1;
    }
    const dim3 grid((uint32_t)(g_tiles + w_tiles + x_tiles));
    if (terms == 1 && slope) k_grad_operands<1, true><<<grid, dim3(256), 0, s>>>(o);
    else if (terms == 1) k_grad_operands<1, false><<<grid, dim3(256), 0, s>>>(o);
    else if (slope) k_grad_operands<2, true><<<grid, dim3(256), 0, s>>>(o);
    else k_grad_operands<2, false><<<grid, dim3(256), 0, s>>>(o);
    if (!products) return hipGetLastError() == hipSuccess ? GEO_SC_OK : GEO_SC_ERR_LAUNCH;
    TwoProducts both = grad_products(l, base, terms, dx, dw);
    if (dx) both.first.y = dx, both.first.dtype = dx_dtype;
    TileArgs& of_w = dx ? both.second : both.first;
    if (dw) of_w.y = dw, of_w.dtype = dw_dtype;
    return run_products<false>(both, nullptr, l.plan, s);
}

}  // namespace
}  // namespace geo_sc

using namespace geo_sc;

extern "C" {

int geo_sc_matmul_q8_workspace_size(const int8_t* x, int64_t x_stride, const int8_t* w, int64_t w_stride, int64_t rows, int64_t cols,
                                    int64_t inner, size_t* bytes)
{
    if (!bytes || !sizes_fit(rows, cols, inner) || x_stride < 0 || w_stride < 0) return GEO_SC_ERR_INVALID_ARGUMENT;
    TileArgs a = {};
    const Plan plan = forward_plan(x, x_stride, w, w_stride, rows, cols, inner, &a);
    const Copies copies = copies_of(a, plan, rows, cols);
    *bytes = partial_bytes(plan, 0, {rows, cols, inner}) + copies.x + copies.w;
    return GEO_SC_OK;
}

int geo_sc_matmul_q8_plan(const int8_t* x, int64_t x_stride, const int8_t* w, int64_t w_stride, int64_t rows, int64_t cols, int64_t inner,
                          int* kernel, int* tile, int* splits)
{
    if (!kernel || !tile || !splits || !sizes_fit(rows, cols, inner) || x_stride < 0 || w_stride < 0) return GEO_SC_ERR_INVALID_ARGUMENT;
    TileArgs a = {};
    const Plan plan = forward_plan(x, x_stride, w, w_stride, rows, cols, inner, &a);
    const Copies copies = copies_of(a, plan, rows, cols);
    a.splits = plan.splits[0];
    a.stages_per_split = plan.stages_per_split[0];
    if (plan.few) *kernel = is_streamed(a) ? GEO_SC_Q8_FEW_STREAMED : GEO_SC_Q8_FEW_ROWS;
    else *kernel = is_direct(a, plan.tile) || copies.x || copies.w ? GEO_SC_Q8_TILES : GEO_SC_Q8_TILES_ANY;
    *tile = plan.few ? 16 * plan.few : plan.tile;
    *splits = plan.splits[0];
    return GEO_SC_OK;
}

int geo_sc_matmul_q8_strips(const int8_t* x, int64_t x_stride, const int8_t* w, int64_t w_stride, int64_t rows, int64_t cols, int64_t inner,
                            int64_t* last_rows, int64_t* last_cols)
{
    if (!last_rows || !last_cols || !sizes_fit(rows, cols, inner) || x_stride < 0 || w_stride < 0) return GEO_SC_ERR_INVALID_ARGUMENT;
    TwoProducts both = {};
    TileArgs& a = both.first;
    const Plan plan = forward_plan(x, x_stride, w, w_stride, rows, cols, inner, &a);
    const Copies copies = copies_of(a, plan, rows, cols);
    if (copies.x) a.x = kAligned, a.x_stride = (inner + 15) / 16 * 16;
    if (copies.w) a.w = kAligned, a.w_stride = (inner + 15) / 16 * 16;
    set_splits(&both, plan);
    *last_rows = *last_cols = 0;
    if (plan.few) return GEO_SC_OK;
    const Tiles t = tiles_of(both, plan, nullptr);
    if (t.cut) *last_rows = t.first.down.rows, *last_cols = t.first.right.cols;
    return GEO_SC_OK;
}

int geo_sc_matmul_q8_backward_strips(int64_t rows, int64_t cols, int64_t inner, int grad_dtype, int need_dx, int need_dw, int64_t* dx_rows,
                                     int64_t* dx_cols, int64_t* dw_rows, int64_t* dw_cols)
{
    if (!dx_rows || !dx_cols || !dw_rows || !dw_cols || !sizes_fit(rows, cols, inner) || !dtype_known(grad_dtype)) return GEO_SC_ERR_INVALID_ARGUMENT;
    *dx_rows = *dx_cols = *dw_rows = *dw_cols = 0;
    if (!need_dx && !need_dw) return GEO_SC_OK;
    const int terms = terms_of(grad_dtype);
    const GradLayout l = grad_layout(rows, cols, inner, terms, need_dx, need_dw, false);
    TwoProducts both = grad_products(l, kAligned, terms, need_dx, need_dw);
    set_splits(&both, l.plan);
    const Tiles t = tiles_of(both, l.plan, nullptr);
    if (!t.cut) return GEO_SC_OK;
    const Strips& of_w = need_dx ? t.second : t.first;
    if (need_dx) *dx_rows = t.first.down.rows, *dx_cols = t.first.right.cols;
    if (need_dw) *dw_rows = of_w.down.rows, *dw_cols = of_w.right.cols;
    return GEO_SC_OK;
}

int geo_sc_matmul_q8(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride, const float* w_scale,
                     int64_t rows, int64_t cols, int64_t inner, void* y, int dtype, void* workspace, size_t workspace_bytes,
                     geo_sc_stream_t stream)
{
    return forward(x, x_stride, x_scale, w, w_stride, w_scale, rows, cols, inner, y, dtype, nullptr, workspace, workspace_bytes, (hipStream_t)stream);
}

int geo_sc_matmul_q8_epilogue(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride, const float* w_scale,
                              int64_t rows, int64_t cols, int64_t inner, const geo_sc_q8_epilogue* epilogue, void* y, int dtype,
                              void* workspace, size_t workspace_bytes, geo_sc_stream_t stream)
{
    if (!epilogue || epilogue->struct_bytes != sizeof *epilogue || epilogue->activation < GEO_SC_ACT_NONE || epilogue->activation > GEO_SC_ACT_SILU ||
        (epilogue->bias && !dtype_known(epilogue->bias_dtype)) || epilogue->residual_stride < 0 ||
        (epilogue->slope && (!slope_type_known(epilogue->slope_dtype) ||
                             (epilogue->slope_dtype == GEO_SC_U8 && epilogue->activation > GEO_SC_ACT_RELU))))
        return GEO_SC_ERR_INVALID_ARGUMENT;
    const Epilogue e = {epilogue->bias,       epilogue->residual,    epilogue->slope,     epilogue->residual_stride,
                        epilogue->bias_dtype, epilogue->slope_dtype, epilogue->activation};
    return forward(x, x_stride, x_scale, w, w_stride, w_scale, rows, cols, inner, y, dtype, &e, workspace, workspace_bytes, (hipStream_t)stream);
}

int geo_sc_matmul_q8_backward_workspace_size(int64_t rows, int64_t cols, int64_t inner, int grad_dtype, int need_dx, int need_dw,
                                             size_t* bytes)
{
    if (!bytes || !sizes_fit(rows, cols, inner) || !dtype_known(grad_dtype)) return GEO_SC_ERR_INVALID_ARGUMENT;
    *bytes = need_dx || need_dw ? grad_layout(rows, cols, inner, terms_of(grad_dtype), need_dx, need_dw, false).bytes : 0;
    return GEO_SC_OK;
}

int geo_sc_matmul_q8_epilogue_backward_workspace_size(int64_t rows, int64_t cols, int64_t inner, int grad_dtype, int need_dx, int need_dw,
                                                      int need_dbias, size_t* bytes)
{
    if (!bytes || !sizes_fit(rows, cols, inner) || !dtype_known(grad_dtype)) return GEO_SC_ERR_INVALID_ARGUMENT;
    *bytes = grad_layout(rows, cols, inner, terms_of(grad_dtype), need_dx, need_dw, need_dbias).bytes;
    return GEO_SC_OK;
}

int geo_sc_matmul_q8_backward(const void* grad, int grad_dtype, int64_t grad_stride, const int8_t* x, int64_t x_stride,
                              const float* x_scale, const int8_t* w, int64_t w_stride, const float* w_scale, int64_t rows, int64_t cols,
                              int64_t inner, void* dx, int dx_dtype, void* dw, int dw_dtype, void* workspace, size_t workspace_bytes,
                              geo_sc_stream_t stream)
{
    return backward(grad, grad_dtype, grad_stride, nullptr, 0, x, x_stride, x_scale, w, w_stride, w_scale, rows, cols, inner, dx, dx_dtype, dw,
                    dw_dtype, nullptr, 0, workspace, workspace_bytes, (hipStream_t)stream);
}

int geo_sc_matmul_q8_epilogue_backward(const void* grad, int grad_dtype, int64_t grad_stride, const void* slope, int slope_dtype, const int8_t* x,
                                       int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride, const float* w_scale, int64_t rows,
                                       int64_t cols, int64_t inner, void* dx, int dx_dtype, void* dw, int dw_dtype, void* dbias, int dbias_dtype,
                                       void* workspace, size_t workspace_bytes, geo_sc_stream_t stream)
{
    return backward(grad, grad_dtype, grad_stride, slope, slope_dtype, x, x_stride, x_scale, w, w_stride, w_scale, rows, cols, inner, dx,
                    dx_dtype, dw, dw_dtype, dbias, dbias_dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
