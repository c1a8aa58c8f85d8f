// Rows in 8 bits with a scale each, and the root-mean-square norm that ends in them.
//
//   a = max_j |n_j|,  scale = a / 127,  q_j = round(n_j * 127 / a)   (half to even; a = 0: scale 0 and q 0)
//   norm: t = x + residual,  r = 1 / sqrt(mean_j t_j^2 + eps),  n_j = t_j r w_j
//
// r is common to a row, so it cancels in q: q_j = round(t_j w_j * 127 / max|t w|) and scale = max|t w| r / 127.  The sum of
// squares and the maximum then need one pass and one exchange between the row's waves, and the row stays in registers
// from its only read to its only write.  Where the squares or the products pass the range of fp32 the row is read again and taken
// times a power of two, which cancels in q alike (in_range, scaled_row).
//
// Backward of the norm, straight through the rounding, with g the gradient of the values and h that of the sum:
//   u = g w,   dt = r (u - t r mean(u t r)) + h,   dx = dresidual = dt,   dw = sum over the rows of g t r
// (t r is at most the root of the columns: no product with it passes the range that u has.)
// t is formed again from x and residual: the sum that the forward returns is rounded to their type, which would show in dw
// (bf16: 2.5e-3 of its size, where its own rounding is 1.7e-3).
#include <type_traits>

#include "sc_dense.h"

namespace geo_sc {
namespace {

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

struct RowsArgs {
    const void *x, *residual, *weight;
    int64_t rows, cols, x_stride, residual_stride, q_stride;
    float eps;
    int8_t* q;
    float *scale, *rstd;
    void *total, *values;
    int values_dtype;
    bool streamed;   // total and values
};

template <typename T, bool NORM, bool ONCE>
__device__ __forceinline__ void read_chunk(const RowsArgs& a, int64_t row, int64_t c, float (&t)[kChunk])
{
    load_chunk<ONCE>((const T*)a.x + row * a.x_stride, c, a.cols, 0.f, t);
    if constexpr (NORM) {
        if (a.residual) {
            float s[kChunk];
            load_chunk<ONCE>((const T*)a.residual + row * a.residual_stride, c, a.cols, 0.f, s);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) t[j] += s[j];
        }
    }
}

template <typename T, bool NORM>
__device__ __forceinline__ void write_chunk(const RowsArgs& a, int64_t row, int64_t c, const RowScale& rs, const float (&n)[kChunk])
{
    float v[kChunk];
    int8_t q[kChunk];
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
        // (a NaN's conversion to an integer is whatever the hardware makes of it: such rows write zeros)
        const float k = rs.inverse == 0.f ? 0.f : rintf(n[j] * rs.lift * rs.inverse);
        q[j] = (int8_t)(int)k;
        v[j] = k * rs.scale;
    }
    int8_t* out = a.q + row * a.q_stride;
    if (c + kChunk <= a.cols) {
        __builtin_memcpy(out + c, q, sizeof q);
    } else {
#pragma unroll
        for (int j = 0; j < kChunk; ++j)
            if (c + j < a.cols) out[c + j] = q[j];
    }
    if (a.values) store_chunk(a.values, a.values_dtype, row * a.cols, c, a.cols, v, a.streamed);
}

__device__ __forceinline__ float row_unit(const RowsArgs& a, float squares) { return 1.f / sqrtf(squares / (float)a.cols + a.eps); }

// Whether sums of squares and products with the weight, formed as they are, lost nothing to infinity or to zero.  (A row of zeros
// counts as outside: it looks like one whose squares and products vanished.)
__device__ __forceinline__ bool in_range(const RowsArgs& a, float squares, uint32_t most)
{
    return squares < __uint_as_float(kInfinityBits) && squares + a.eps * (float)a.cols > 0x1p-64f && most < kInfinityBits &&
           most >= __float_as_uint(0x1p-100f);
}
// The power of two that brings the largest magnitude, which is a number and not zero, to 1 .. 4 (denormals less far).
__device__ __forceinline__ float power_up(uint32_t peak)
{
    const int field = 254 - (int)(peak >> 23);
    return __uint_as_float((uint32_t)(field < 1 ? 1 : field > 253 ? 253 : field) << 23);
}
// r of a row, and r / up, the factor of t up, from the sum of the squares of t up.  Where eps up^2 is beyond all squares r is eps's alone.
__device__ __forceinline__ void scaled_units(const RowsArgs& a, float squares, float up, float& unit, float& factor)
{
    const float eps = a.eps * up * up;
    if (eps < 0x1p100f) {
        factor = 1.f / sqrtf(squares / (float)a.cols + eps);
        unit = factor * up;
    } else {
        unit = 1.f / sqrtf(a.eps);
        factor = unit * (1.f / up);
    }
}

// One row per threadIdx.y; the row's blockDim.x threads hold ITEMS chunks of eight columns each in registers from the only read to
// the write.  Bound by memory: 16384 x 4096 fp32 to q and bf16 values 403 MB in 73 us, 8191 x 4096 bf16 with residual to q, sum and
// values 302 MB in 59 (5.5 and 5.1 TB/s).  (Blocks that stay, go on to further rows and ask for the next one ahead: 91 us for
// the second, when these took 84; new blocks hide a row's reduction better.)
template <typename T, bool NORM, int ITEMS, bool ONCE>
__global__ __launch_bounds__(1024) void k_rows(RowsArgs a)
{
    __shared__ RowSlots slots;
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int threads = blockDim.x, t = threadIdx.x, waves = threads >> 6;   // (blocks of several rows have one wave per row: no barrier)
    if (row >= a.rows) return;
    const auto column = [&](int i) { return ((int64_t)i * threads + t) * kChunk; };
    float n[ITEMS][kChunk], squares = 0.f;
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (column(i) < a.cols) {
            read_chunk<T, NORM, ONCE>(a, row, column(i), n[i]);
            if constexpr (NORM) {
                if (a.total && a.residual) store_chunk((T*)a.total + row * a.cols, column(i), a.cols, n[i], a.streamed);
                float w[kChunk];
                load_chunk((const T*)a.weight, column(i), a.cols, 0.f, w);
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    squares += n[i][j] * n[i][j];
                    n[i][j] *= w[j];
                }
            }
#pragma unroll
            for (int j = 0; j < kChunk; ++j) most = max(most, magnitude_bits(n[i][j]));
        }
    row_reduce(squares, most, waves, slots, 0);
    float unit = NORM ? row_unit(a, squares) : 1.f, factor = unit;
    bool sound = true;
    if (NORM && __builtin_expect(!in_range(a, squares, most), false)) {   // (all threads of a row alike)
        uint32_t peak = 0;
        float none = 0.f;
#pragma unroll 1
        for (int i = 0; i < ITEMS; ++i)
            if (column(i) < a.cols) {
                read_chunk<T, NORM, false>(a, row, column(i), n[0]);
#pragma unroll
                for (int j = 0; j < kChunk; ++j) peak = max(peak, magnitude_bits(n[0][j]));
            }
        row_reduce(none, peak, waves, slots, 1);
        sound = peak < kInfinityBits;
        if (sound && peak) {
            const float up = power_up(peak);
            squares = 0.f;
            most = 0;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (column(i) < a.cols) {
                    read_chunk<T, NORM, false>(a, row, column(i), n[i]);
                    float w[kChunk];
                    load_chunk((const T*)a.weight, column(i), a.cols, 0.f, w);
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) {
                        n[i][j] *= up;
                        squares += n[i][j] * n[i][j];
                        n[i][j] *= w[j];
                        most = max(most, magnitude_bits(n[i][j]));
                    }
                }
            row_reduce(squares, most, waves, slots, 0);
            scaled_units(a, squares, up, unit, factor);
        }
    }
    const RowScale rs = row_scale(most, factor, sound);
    if (t == 0) {
        a.scale[row] = rs.scale;
        if (NORM && a.rstd) a.rstd[row] = unit;
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (column(i) < a.cols) write_chunk<T, NORM>(a, row, column(i), rs, n[i]);
}

// Rows that do not fit into a block's registers (more than 32768 columns): read a second time, out of L2, after the reduction.
// 512 x 100003 bf16 in 51 us.
template <typename T, bool NORM>
__global__ __launch_bounds__(1024) void k_rows_long(RowsArgs a)
{
    __shared__ RowSlots slots;
    const int64_t row = blockIdx.x, first = (int64_t)threadIdx.x * kChunk, step = (int64_t)blockDim.x * kChunk;
    float n[kChunk], squares = 0.f, up = 1.f;
    uint32_t most = 0;
    const auto take = [&](int64_t c, bool write_total) {
        read_chunk<T, NORM, false>(a, row, c, n);
        if constexpr (NORM) {
            if (write_total && a.total && a.residual) store_chunk((T*)a.total + row * a.cols, c, a.cols, n, a.streamed);
            float w[kChunk];
            load_chunk((const T*)a.weight, c, a.cols, 0.f, w);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
                n[j] *= up;
                squares += n[j] * n[j];
                n[j] *= w[j];
            }
        }
    };
    const auto scan = [&](bool write_total) {
        squares = 0.f;
        most = 0;
        for (int64_t c = first; c < a.cols; c += step) {
            take(c, write_total);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) most = max(most, magnitude_bits(n[j]));
        }
        row_reduce(squares, most, blockDim.x >> 6, slots, 0);
    };
    scan(true);
    float unit = NORM ? row_unit(a, squares) : 1.f, factor = unit;
    bool sound = true;
    if (NORM && __builtin_expect(!in_range(a, squares, most), false)) {
        uint32_t peak = 0;
        float none = 0.f;
        for (int64_t c = first; c < a.cols; c += step) {
            read_chunk<T, NORM, false>(a, row, c, n);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) peak = max(peak, magnitude_bits(n[j]));
        }
        row_reduce(none, peak, blockDim.x >> 6, slots, 1);
        sound = peak < kInfinityBits;
        if (sound && peak) {
            up = power_up(peak);
            scan(false);
            scaled_units(a, squares, up, unit, factor);
        }
    }
    const RowScale rs = row_scale(most, factor, sound);
    if (threadIdx.x == 0) {
        a.scale[row] = rs.scale;
        if (NORM && a.rstd) a.rstd[row] = unit;
    }
    for (int64_t c = first; c < a.cols; c += step) {
        take(c, false);
        write_chunk<T, NORM>(a, row, c, rs, n);
    }
}

// Threads of a row with `chunks` chunks: whole waves, at most 1024, of which each has `held` chunks.
int threads_of_row(int64_t chunks, int held)
{
    const int64_t threads = ((chunks + held - 1) / held + 63) / 64 * 64;
    return threads < 1024 ? (int)threads : 1024;
}

// the rows from `first` on
template <typename T>
RowsArgs rows_from(RowsArgs a, int64_t first)
{
    a.x = (const T*)a.x + first * a.x_stride;
    if (a.residual) a.residual = (const T*)a.residual + first * a.residual_stride;
    a.q += first * a.q_stride;
    a.scale += first;
    if (a.rstd) a.rstd += first;
    if (a.total) a.total = (T*)a.total + first * a.cols;
    if (a.values) a.values = (char*)a.values + first * a.cols * dtype_bytes(a.values_dtype);
    a.rows -= first;
    return a;
}

template <typename T, bool NORM>
int run_rows(RowsArgs a, hipStream_t s)
{
    constexpr int dtype = std::is_same_v<T, f32> ? GEO_SC_F32 : std::is_same_v<T, bf16> ? GEO_SC_BF16 : GEO_SC_F16;
    const bool once = reads_once(dtype, a.x, a.x_stride) && (!a.residual || reads_once(dtype, a.residual, a.residual_stride));
    a.streamed = streams(a.rows * a.cols * ((a.total && a.residual ? (int64_t)sizeof(T) : 0) + (a.values ? dtype_bytes(a.values_dtype) : 0)));
    const int64_t chunks = (a.cols + kChunk - 1) / kChunk;
    // Two chunks per thread where there are rows enough to fill the compute units: half as many waves reduce a row.  8191 x 4096
    // bf16 in 8 bits 23.5 us, with one 29.8.  Few rows are as fast as their longest thread.
    const int threads = threads_of_row(chunks, a.rows >= 2048 && chunks > 64 ? 2 : 1), per_block = threads == 64 ? 4 : 1;
    const int64_t items = (chunks + threads - 1) / threads;
    const dim3 block(threads, per_block);
    in_launches((a.rows + per_block - 1) / per_block, threads, [&](int64_t first, uint32_t grid) {
        const RowsArgs b = rows_from<T>(a, first * per_block);
        const auto held = [&](auto count) {
            if (once) k_rows<T, NORM, count(), true><<<grid, block, 0, s>>>(b);
            else k_rows<T, NORM, count(), false><<<grid, block, 0, s>>>(b);
        };
        if (items <= 1) held(std::integral_constant<int, 1>());
        else if (items <= 2) held(std::integral_constant<int, 2>());
        else if (items <= 4) held(std::integral_constant<int, 4>());
        else k_rows_long<T, NORM><<<grid, block, 0, s>>>(b);
    });
    return hipGetLastError() == hipSuccess ? GEO_SC_OK : GEO_SC_ERR_LAUNCH;
}

template <bool NORM>
int run_rows(const RowsArgs& a, int dtype, hipStream_t s)
{
    if (dtype == GEO_SC_F32) return run_rows<f32, NORM>(a, s);
    if (dtype == GEO_SC_BF16) return run_rows<bf16, NORM>(a, s);
    return run_rows<f16, NORM>(a, s);
}

// ---------------------------------------------------------------- backward of the norm

struct NormBackArgs {
    const void *grad_values, *grad_total, *x, *residual, *weight;   // grad_total, residual: or NULL
    int grad_dtype;
    int64_t rows, cols, grad_stride, grad_total_stride, x_stride, residual_stride;
    const float* rstd;
    void *dx;
    bool streamed;    // dx
    bool once;        // what is read
    float* partial;   // [blocks][cols]: sums of the weight's gradient, NULL: not wanted
    int64_t first_row;   // of a launch of k_norm_back_long
};

// A block takes every gridDim.x-th row; its threads keep the weight and their columns' sums of the weight's gradient in
// registers over all rows of the block.  Bound by memory: 8191 x 4096 bf16 with both gradients and residual 344 MB in 55 us (6.2
// TB/s; x and residual partly in the caches after the forward).  (Asking for the next row ahead of the exchange took 76 us where
// it took 71 without, before x and residual were read again: the registers that it needs cost a block per compute unit.)
template <typename T, typename G, int ITEMS, bool ONCE>
__global__ __launch_bounds__(1024) void k_norm_back(NormBackArgs a)
{
    __shared__ RowSlots slots;
    const int threads = blockDim.x, t = threadIdx.x, waves = threads >> 6;
    float w[ITEMS][kChunk], dw[ITEMS][kChunk];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int64_t c = ((int64_t)i * threads + t) * kChunk;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) w[i][j] = dw[i][j] = 0.f;
        if (c < a.cols) load_chunk((const T*)a.weight, c, a.cols, 0.f, w[i]);
    }
    const auto column = [&](int i) { return ((int64_t)i * threads + t) * kChunk; };
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, ++turn) {
        const float unit = a.rstd[row];
        float g[ITEMS][kChunk], v[ITEMS][kChunk], h[ITEMS][kChunk], along = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (column(i) < a.cols) {
                G grad[kChunk];
                T x[kChunk], residual[kChunk] = {}, also[kChunk] = {};
                fetch_chunk<ONCE>((const G*)a.grad_values + row * a.grad_stride, column(i), a.cols, grad);
                fetch_chunk<ONCE>((const T*)a.x + row * a.x_stride, column(i), a.cols, x);
                if (a.residual) fetch_chunk<ONCE>((const T*)a.residual + row * a.residual_stride, column(i), a.cols, residual);
                if (a.grad_total) fetch_chunk<ONCE>((const T*)a.grad_total + row * a.grad_total_stride, column(i), a.cols, also);
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    g[i][j] = (float)grad[j];
                    v[i][j] = ((float)x[j] + (float)residual[j]) * unit;
                    h[i][j] = (float)also[j];
                    dw[i][j] += g[i][j] * v[i][j];
                    g[i][j] *= w[i][j];
                    along += g[i][j] * v[i][j];
                }
            }
        uint32_t none = 0;
        row_reduce(along, none, waves, slots, turn);
        const float back = along / (float)a.cols;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (column(i) < a.cols) {
                float d[kChunk];
#pragma unroll
                for (int j = 0; j < kChunk; ++j) d[j] = unit * (g[i][j] - v[i][j] * back) + h[i][j];
                store_chunk((T*)a.dx + row * a.cols, column(i), a.cols, d, a.streamed);
            }
    }
    if (a.partial) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int64_t c = ((int64_t)i * threads + t) * kChunk;
            if (c < a.cols) store_chunk(a.partial + (int64_t)blockIdx.x * a.cols, c, a.cols, dw[i]);
        }
    }
}

// a chunk of t = x + residual
template <typename T>
__device__ __forceinline__ void load_sum(const NormBackArgs& a, int64_t row, int64_t c, float (&v)[kChunk])
{
    load_chunk((const T*)a.x + row * a.x_stride, c, a.cols, 0.f, v);
    if (!a.residual) return;
    float r[kChunk];
    load_chunk((const T*)a.residual + row * a.residual_stride, c, a.cols, 0.f, r);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) v[j] += r[j];
}

// Rows that do not fit into a block's registers (more than 16384 columns): dx row by row, read twice; the weight's gradient by
// columns, see k_weight_grad_columns.  512 x 100003 bf16, both, in 210 us.
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_back_long(NormBackArgs a)
{
    __shared__ RowSlots slots;
    const int threads = blockDim.x, waves = threads >> 6;
    const int64_t row = a.first_row + blockIdx.x, first = (int64_t)threadIdx.x * kChunk, step = (int64_t)threads * kChunk;
    const float r = a.rstd[row];
    float along = 0.f;
    float g[kChunk], v[kChunk], w[kChunk];
    const auto take = [&](int64_t c) {
        load_chunk(a.grad_values, a.grad_dtype, row * a.grad_stride, c, a.cols, 0.f, g);
        load_sum<T>(a, row, c, v);
        load_chunk((const T*)a.weight, c, a.cols, 0.f, w);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            v[j] *= r;
            g[j] *= w[j];
        }
    };
    for (int64_t c = first; c < a.cols; c += step) {
        take(c);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) along += g[j] * v[j];
    }
    uint32_t none = 0;
    row_reduce(along, none, waves, slots, 0);
    const float back = along / (float)a.cols;
    for (int64_t c = first; c < a.cols; c += step) {
        take(c);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) g[j] = r * (g[j] - v[j] * back);
        if (a.grad_total) {
            load_chunk((const T*)a.grad_total + row * a.grad_total_stride, c, a.cols, 0.f, w);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) g[j] += w[j];
        }
        store_chunk((T*)a.dx + row * a.cols, c, a.cols, g, a.streamed);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void k_weight_grad_columns(NormBackArgs a)
{
    const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * kChunk;
    if (c >= a.cols) return;
    float dw[kChunk] = {}, g[kChunk], v[kChunk];
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        load_chunk(a.grad_values, a.grad_dtype, row * a.grad_stride, c, a.cols, 0.f, g);
        load_sum<T>(a, row, c, v);
        const float r = a.rstd[row];
#pragma unroll
        for (int j = 0; j < kChunk; ++j) dw[j] += g[j] * (v[j] * r);
    }
    store_chunk(a.partial + (int64_t)blockIdx.y * a.cols, c, a.cols, dw);
}

// dweight[c] = the sum over the blocks' partial sums: 32 columns by 32 shares of the blocks in a workgroup, joined in a fixed
// order.  512 blocks of 4096 columns in 4.5 us.
constexpr int kJoinCols = 32, kJoinShares = 32;
template <typename T>
__global__ __launch_bounds__(kJoinCols * kJoinShares) void k_join_weight_grad(const float* partial, int64_t blocks, int64_t cols, T* dw)
{
    __shared__ float sums[kJoinShares][kJoinCols];
    const int64_t c = (int64_t)blockIdx.x * kJoinCols + threadIdx.x;
    float s = 0.f;
    if (c < cols) {
#pragma unroll 16
        for (int64_t b = threadIdx.y; b < blocks; b += kJoinShares) s += partial[b * cols + c];
    }
    sums[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < cols) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < kJoinShares; ++k) s += sums[k][threadIdx.x];
        dw[c] = (T)s;
    }
}

constexpr int64_t kHeldBackCols = 2 * 1024 * kChunk;   // columns that a block's registers hold in the backward

// blocks (= partial sums of the weight's gradient) of the backward.  8191 x 4096 bf16, both passes, us: 256 blocks 131, 384 124, 512
// 121, 768 128.
int64_t norm_back_blocks(int64_t rows, int64_t cols)
{
    const int64_t most = cols > kHeldBackCols ? 64 : 512;
    return rows < most ? rows : most;
}

template <typename T, typename G>
void run_norm_back_held(const NormBackArgs& a, int64_t blocks, hipStream_t s)
{
    const int64_t chunks = (a.cols + kChunk - 1) / kChunk;
    const int threads = threads_of_row(chunks, 1);
    const auto held = [&](auto count) {
        if (a.once) k_norm_back<T, G, count(), true><<<dim3((uint32_t)blocks), dim3(threads), 0, s>>>(a);
        else k_norm_back<T, G, count(), false><<<dim3((uint32_t)blocks), dim3(threads), 0, s>>>(a);
    };
    if (chunks <= threads) held(std::integral_constant<int, 1>());
    else held(std::integral_constant<int, 2>());
}

template <typename T>
int run_norm_back(const NormBackArgs& a, T* dw, hipStream_t s)
{
    const int64_t chunks = (a.cols + kChunk - 1) / kChunk, blocks = norm_back_blocks(a.rows, a.cols);
    if (a.cols > kHeldBackCols) {
        in_launches(a.rows, 1024, [&](int64_t first, uint32_t count) {
            NormBackArgs b = a;
            b.first_row = first;
            k_norm_back_long<T><<<dim3(count), dim3(1024), 0, s>>>(b);
        });
        if (a.partial)
            k_weight_grad_columns<T><<<dim3((uint32_t)((chunks + 255) / 256), (uint32_t)blocks), dim3(256), 0, s>>>(a);
    } else if (a.grad_dtype == GEO_SC_F32) {
        run_norm_back_held<T, f32>(a, blocks, s);
    } else if (a.grad_dtype == GEO_SC_BF16) {
        run_norm_back_held<T, bf16>(a, blocks, s);
    } else {
        run_norm_back_held<T, f16>(a, blocks, s);
    }
    if (a.partial)
        k_join_weight_grad<T><<<dim3((uint32_t)((a.cols + kJoinCols - 1) / kJoinCols)), dim3(kJoinCols, kJoinShares), 0, s>>>(
            a.partial, blocks, a.cols, dw);
    return hipGetLastError() == hipSuccess ? GEO_SC_OK : GEO_SC_ERR_LAUNCH;
}

bool sizes_fit(int64_t rows, int64_t cols) { return rows >= 0 && cols >= 1 && rows <= 0x7fffffff && cols <= 0x7fffffff; }

}  // namespace
}  // namespace geo_sc

using namespace geo_sc;

extern "C" {

int geo_sc_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_stride, int8_t* q, int64_t q_stride,
                         float* scale, void* values, int values_dtype, geo_sc_stream_t stream)
{
    if (!sizes_fit(rows, cols) || !dtype_known(dtype) || (values && !dtype_known(values_dtype)) || x_stride < 0 || q_stride < cols)
        return GEO_SC_ERR_INVALID_ARGUMENT;
    if (rows == 0) return GEO_SC_OK;
    if (!x || !q || !scale) return GEO_SC_ERR_INVALID_ARGUMENT;
    RowsArgs a = {};
    a.x = x;
    a.rows = rows;
    a.cols = cols;
    a.x_stride = x_stride;
    a.q_stride = q_stride;
    a.q = q;
    a.scale = scale;
    a.values = values;
    a.values_dtype = values_dtype;
    return run_rows<false>(a, dtype, (hipStream_t)stream);
}

int geo_sc_rms_norm_q8(const void* x, const void* residual, const void* weight, int dtype, int64_t rows, int64_t cols,
                       int64_t x_stride, int64_t residual_stride, float eps, int8_t* q, int64_t q_stride, float* scale,
                       void* total, void* values, int values_dtype, float* rstd, geo_sc_stream_t stream)
{
    if (!sizes_fit(rows, cols) || !dtype_known(dtype) || (values && !dtype_known(values_dtype)) || x_stride < 0 ||
        residual_stride < 0 || q_stride < cols || !(eps >= 0.f))
        return GEO_SC_ERR_INVALID_ARGUMENT;
    if (rows == 0) return GEO_SC_OK;
    if (!x || !weight || !q || !scale) return GEO_SC_ERR_INVALID_ARGUMENT;
    const RowsArgs a = {x, residual, weight, rows, cols, x_stride, residual_stride, q_stride, eps, q, scale, rstd, total, values,
                        values_dtype, false};
    return run_rows<true>(a, dtype, (hipStream_t)stream);
}

int geo_sc_rms_norm_q8_backward_workspace_size(int64_t rows, int64_t cols, size_t* bytes)
{
    if (!bytes || !sizes_fit(rows, cols)) return GEO_SC_ERR_INVALID_ARGUMENT;
    *bytes = (size_t)norm_back_blocks(rows, cols) * (size_t)cols * sizeof(float);
    return GEO_SC_OK;
}

int geo_sc_rms_norm_q8_backward(const void* grad_values, int grad_dtype, int64_t grad_stride, const void* grad_total,
                                int64_t grad_total_stride, const void* x, int64_t x_stride, const void* residual,
                                int64_t residual_stride, const void* weight, int dtype, int64_t rows, int64_t cols, const float* rstd,
                                void* dx, void* dweight, void* workspace, size_t workspace_bytes, geo_sc_stream_t stream)
{
    if (!sizes_fit(rows, cols) || rows < 1 || !dtype_known(dtype) || !dtype_known(grad_dtype) || grad_stride < 0 ||
        grad_total_stride < 0 || x_stride < 0 || residual_stride < 0 || !grad_values || !x || !weight || !rstd || !dx)
        return GEO_SC_ERR_INVALID_ARGUMENT;
    size_t need = 0;
    geo_sc_rms_norm_q8_backward_workspace_size(rows, cols, &need);
    if (dweight && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 4)) return GEO_SC_ERR_WORKSPACE;
    const bool once = reads_once(dtype, x, x_stride) && (!residual || reads_once(dtype, residual, residual_stride)) &&
                      reads_once(grad_dtype, grad_values, grad_stride) && (!grad_total || reads_once(dtype, grad_total, grad_total_stride));
    const NormBackArgs a = {grad_values, grad_total, x, residual, weight, grad_dtype, rows, cols, grad_stride, grad_total_stride,
                            x_stride, residual_stride, rstd, dx, streams(rows * cols * dtype_bytes(dtype)), once,
                            dweight ? (float*)workspace : nullptr, 0};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == GEO_SC_F32) return run_norm_back<f32>(a, (f32*)dweight, s);
    if (dtype == GEO_SC_BF16) return run_norm_back<bf16>(a, (bf16*)dweight, s);
    return run_norm_back<f16>(a, (f16*)dweight, s);
}

}  // extern "C"
