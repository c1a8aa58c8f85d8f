// The norm behind a block, its gate, the scaled residual and the norm in front of the next block, in one pass.
//
//   n1 = x r1,  r1 = 1 / sqrt(mean x^2 + eps);   m = post n1   (without a norm behind the block m = x)
//   t = scale residual + gate m;   n2 = t r2,  r2 = 1 / sqrt(mean t^2 + eps);   out = weight n2
//
// Per channel: weight, post, scale; gate per channel of a run of consecutive rows (a sample's).  A row's threads hold it in registers from
// its only read to its only write, with two exchanges between its waves.  8192 x 4096 bf16, a gate per sample: 268 MB in 73 us (3.7 TB/s; 49
// without post, gate and scale, whose loads stand behind the first exchange; asked for ahead of it, their registers cost more than the
// wait, 85 - 115).  Sums and factors in fp32; t is rounded for `total` only.
// Rows of any finite magnitude: where squares pass the range of fp32 they are taken of the row times a power of two.
//
// Backward, from g (gradient of out) and h (of t), means over a row:
//   u = g weight,  dt = r2 (u - n2 mean(u n2)) + h,   dweight = sum over rows of g n2
//   dresidual = dt scale,  dscale = sum of dt residual,  dgate = sum over a run of dt m
//   e = dt gate,  dpost = sum of e n1,  s = e post,  dx = r1 (s - n1 mean(s n1))   (without the norm dx = e)
// n1 and n2 are at most the root of the columns: nothing but the gradients themselves can pass fp32's range.  t is formed again, as
// its rounding would show in the sums over rows.
#include <stddef.h>

#include <type_traits>

#include "sc_dense.h"

namespace geo_sc {
namespace {

struct NormArgs {
    const void *x, *residual, *weight, *post, *gate, *scale;   // post, gate, scale: or NULL
    int64_t rows, cols, x_stride, residual_stride, run;        // run: rows that share a gate
    float eps;
    void *out, *total;   // T
    float* rstd;         // [rows][2]: r1, r2; or NULL
    int8_t* q;           // instead of out
    int64_t q_stride;
    float* q_scale;
    void* values;
    int values_dtype;
    bool streamed;       // out, total, values
    int64_t first_row;   // of a launch
};

// threadIdx.y: of a row of whole waves it is the wave's, and so are the row's addresses and factors.
template <int LANES>
__device__ __forceinline__ uint32_t row_in_block()
{
    if constexpr (LANES == 64) return (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.y);
    else return threadIdx.y;
}

// Sum, or sum and largest, over a row's lanes: LANES 32 (two rows in a wave) or 64, then over its waves.
template <int LANES>
__device__ __forceinline__ void reduce_row(float& sum, uint32_t& most, int waves, RowSlots& slots, int& turn)
{
    if constexpr (LANES == 32) {
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) {
            sum += __shfl_xor(sum, d);
            most = max(most, (uint32_t)__shfl_xor((int)most, d));
        }
    } else {
        row_reduce(sum, most, waves, slots, turn++);
    }
}
template <int LANES>
__device__ __forceinline__ void reduce_row(float& sum, int waves, RowSlots& slots, int& turn)
{
#pragma unroll
    for (int d = LANES / 2; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
    if (LANES == 32 || waves == 1) return;
    if ((threadIdx.x & 63) == 0) slots.sum[turn & 1][threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.f;
    for (int k = 0; k < waves; ++k) sum += slots.sum[turn & 1][k];
    ++turn;
}

// (rows are counted in 31 bits; a division of 64 takes as long as a row's sums)
__device__ __forceinline__ int64_t run_of(int64_t row, int64_t run) { return (uint32_t)row / (uint32_t)run; }

// The factor of a norm: n = v up factor, r = unit.  `up` is 1 but where the squares of v pass fp32's range.
struct Root {
    float up, factor, unit;
};
__device__ __forceinline__ Root root_of(float squares, int64_t cols, float eps)
{
    const float r = 1.f / sqrtf(squares / (float)cols + eps);
    return {1.f, r, r};
}
// whether the sum of squares lost nothing to infinity or zero (rows of zeros count as if it had)
__device__ __forceinline__ bool in_range(float squares, int64_t cols, float eps)
{
    return squares < __uint_as_float(kInfinityBits) && squares + eps * (float)cols > 0x1p-64f;
}
// the same from the squares of v up
__device__ __forceinline__ Root root_of_scaled(float squares, float up, int64_t cols, float eps)
{
    const float e = eps * up * up;
    if (e < 0x1p100f) {
        const float f = 1.f / sqrtf(squares / (float)cols + e);
        return {up, f, f * up};
    }
    const float r = 1.f / sqrtf(eps);   // eps alone counts
    return {up, r * (1.f / up), r};
}

// A chunk as it lies in memory.  (An array of 16-bit elements takes a register for each of them.)  keep(): what is formed from it is
// formed behind this, not ahead into registers of its own.
template <typename T>
struct Raw {
    uint32_t words[kChunk * sizeof(T) / 4];
    template <bool ONCE>
    __device__ __forceinline__ void fetch(const void* row, int64_t c, int64_t cols)
    {
        T v[kChunk];
        if (c + kChunk <= cols) {   // (either way into whole registers by itself)
            fetch_whole<ONCE>((const T*)row + c, v);
            __builtin_memcpy(words, v, sizeof words);
            return;
        }
        fetch_chunk<ONCE>((const T*)row, c, cols, v);
        __builtin_memcpy(words, v, sizeof words);
        keep();
    }
    __device__ __forceinline__ void set(float v)
    {
        T one[kChunk];
#pragma unroll
        for (int j = 0; j < kChunk; ++j) one[j] = (T)v;
        __builtin_memcpy(words, one, sizeof words);
    }
    __device__ __forceinline__ void fetch_or_ones(const void* row, int64_t c, int64_t cols)
    {
        if (row) fetch<false>(row, c, cols);
        else set(1.f);
    }
    __device__ __forceinline__ void keep()
    {
#pragma unroll
        for (int i = 0; i < (int)(sizeof words / 4); ++i) asm volatile("" : "+v"(words[i]));
    }
    __device__ __forceinline__ float operator[](int j) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(words[j]);
        else if constexpr (std::is_same_v<T, bf16>) return __uint_as_float(j & 1 ? words[j / 2] & 0xffff0000u : words[j / 2] << 16);
        else return (float)__builtin_bit_cast(f16, (uint16_t)(words[j / 2] >> (16 * (j & 1))));
    }
};

// fp32 numbers from here on.  (A product or multiply-add whose result goes into fp16 is one instruction with one rounding, where the compiler
// takes it: 401 of 4097 x 2056 outputs were others for rows at odd addresses.)
__device__ __forceinline__ void rounded(float (&v)[kChunk])
{
#pragma unroll
    for (int j = 0; j < kChunk; ++j) asm volatile("" : "+v"(v[j]));
}

// ROWS rows per threadIdx.y: their blockDim.x threads hold ITEMS chunks of eight columns of each.  Two rows at once read what belongs to
// the channels once, four vectors of a row's length out of L2 beside a row's four, and share the exchanges.  (Fused multiply-adds by name: the
// compiler's choice is another in every instance, and outputs and totals are the same bits in all of them.)
template <int ROWS>
struct ManySlots {
    float sum[2][ROWS][16];
};
template <typename T, int ROWS, int ITEMS, int LANES, bool ONCE, bool EIGHT>
__global__ __launch_bounds__(1024) void k_gated_norm(NormArgs a)
{
    __shared__ RowSlots slots;
    __shared__ ManySlots<ROWS> many;
    const int threads = blockDim.x, t = threadIdx.x, waves = threads >> 6;   // (blocks of several rows have no more than a wave per row: no barrier)
    const int64_t row0 = a.first_row + ((int64_t)blockIdx.x * blockDim.y + row_in_block<LANES>()) * ROWS;
    if (row0 >= a.rows) return;
    const auto row_of = [&](int q) { return row0 + q < a.rows ? row0 + q : a.rows - 1; };   // (one too many is the last one again, and not stored)
    int turn = 0;
    const auto column = [&](int i) { return ((int64_t)i * threads + t) * kChunk; };
    const auto reduce_all = [&](float (&sum)[ROWS]) {
#pragma unroll
        for (int q = 0; q < ROWS; ++q)
#pragma unroll
            for (int d = LANES / 2; d >= 1; d >>= 1) sum[q] += __shfl_xor(sum[q], d);
        if (LANES == 32 || waves == 1) return;
        if ((t & 63) == 0)
#pragma unroll
            for (int q = 0; q < ROWS; ++q) many.sum[turn & 1][q][t >> 6] = sum[q];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            sum[q] = 0.f;
            for (int k = 0; k < waves; ++k) sum[q] += many.sum[turn & 1][q][k];
        }
        ++turn;
    };
    // the sums of squares of what is held, and their roots; again from v times a power of two where that is needed
    const auto roots_of = [&](const float (&v)[ROWS][ITEMS][kChunk], Root (&root)[ROWS]) {
        float squares[ROWS];
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            squares[q] = 0.f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int j = 0; j < kChunk; ++j) squares[q] = fmaf(v[q][i][j], v[q][i][j], squares[q]);
        }
        reduce_all(squares);
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            root[q] = root_of(squares[q], a.cols, a.eps);
            if (__builtin_expect(in_range(squares[q], a.cols, a.eps), true)) continue;   // (all threads of a row alike)
            uint32_t peak = 0;
            float none = 0.f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int j = 0; j < kChunk; ++j) peak = max(peak, magnitude_bits(v[q][i][j]));
            reduce_row<LANES>(none, peak, waves, slots, turn);
            if (peak == 0 || peak >= kInfinityBits) continue;
            const float up = power_up(peak);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int j = 0; j < kChunk; ++j) sum = fmaf(v[q][i][j] * up, v[q][i][j] * up, sum);
            reduce_row<LANES>(sum, waves, slots, turn);
            root[q] = root_of_scaled(sum, up, a.cols, a.eps);
        }
    };
    Raw<T> raw[ROWS][ITEMS], also[ROWS][ITEMS];
    float v[ROWS][ITEMS][kChunk];
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if (column(i) < a.cols) {
                raw[q][i].template fetch<ONCE>((const T*)a.x + row_of(q) * a.x_stride, column(i), a.cols);
                also[q][i].template fetch<ONCE>((const T*)a.residual + row_of(q) * a.residual_stride, column(i), a.cols);
            } else {
                raw[q][i].set(0.f);
                also[q][i].set(0.f);
            }
        }
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < kChunk; ++j) v[q][i][j] = raw[q][i][j];
    Root first[ROWS], second[ROWS];
#pragma unroll
    for (int q = 0; q < ROWS; ++q) first[q] = {1.f, 1.f, 1.f};
    if (a.post) roots_of(v, first);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (column(i) < a.cols) {
            float f[kChunk];
            if (a.post) {
                load_chunk((const T*)a.post, column(i), a.cols, 0.f, f);
#pragma unroll
                for (int q = 0; q < ROWS; ++q)
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) v[q][i][j] = v[q][i][j] * first[q].up * first[q].factor * f[j];
            }
            if (a.gate) {
#pragma unroll
                for (int q = 0; q < ROWS; ++q) {
                    load_chunk((const T*)a.gate + run_of(row_of(q), a.run) * a.cols, column(i), a.cols, 0.f, f);
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) v[q][i][j] *= f[j];
                }
            }
#pragma unroll
            for (int j = 0; j < kChunk; ++j) f[j] = 1.f;
            if (a.scale) load_chunk((const T*)a.scale, column(i), a.cols, 0.f, f);
#pragma unroll
            for (int q = 0; q < ROWS; ++q) {
                also[q][i].keep();
#pragma unroll
                for (int j = 0; j < kChunk; ++j) v[q][i][j] = fmaf(f[j], also[q][i][j], v[q][i][j]);
                rounded(v[q][i]);
                if (row0 + q < a.rows) store_chunk((T*)a.total + (row0 + q) * a.cols, column(i), a.cols, v[q][i], a.streamed);
            }
        }
    roots_of(v, second);
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
        if (t == 0 && a.rstd && row0 + q < a.rows) {
            a.rstd[2 * (row0 + q)] = first[q].unit;
            a.rstd[2 * (row0 + q) + 1] = second[q].unit;
        }
    uint32_t most[ROWS] = {};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (column(i) < a.cols) {
            float w[kChunk];
            load_chunk((const T*)a.weight, column(i), a.cols, 0.f, w);
#pragma unroll
            for (int q = 0; q < ROWS; ++q) {
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    v[q][i][j] = v[q][i][j] * second[q].up * second[q].factor * w[j];
                    most[q] = max(most[q], magnitude_bits(v[q][i][j]));
                }
                if constexpr (!EIGHT) rounded(v[q][i]);
                if constexpr (!EIGHT)
                    if (row0 + q < a.rows) store_chunk((T*)a.out + (row0 + q) * a.cols, column(i), a.cols, v[q][i], a.streamed);
            }
        }
    if constexpr (EIGHT) {
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            float none = 0.f;
            reduce_row<LANES>(none, most[q], waves, slots, turn);
            if (row0 + q >= a.rows) continue;
            const int64_t row = row0 + q;
            const RowScale rs = row_scale(most[q], 1.f, true);
            if (t == 0) a.q_scale[row] = rs.scale;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (column(i) < a.cols) {
                    float values[kChunk];
                    store_eight(a.q + row * a.q_stride, column(i), a.cols, rs, v[q][i], values);
                    if (a.values) store_chunk(a.values, a.values_dtype, row * a.cols, column(i), a.cols, values, a.streamed);
                }
        }
    }
}

// t of a chunk, and x
template <typename T>
__device__ __forceinline__ void form_total(const NormArgs& a, int64_t row, int64_t c, const Root& first, float (&t)[kChunk])
{
    float f[kChunk];
    load_chunk((const T*)a.x + row * a.x_stride, c, a.cols, 0.f, t);
    if (a.post) {
        load_chunk((const T*)a.post, c, a.cols, 0.f, f);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) t[j] = t[j] * first.up * first.factor * f[j];
    }
    if (a.gate) {
        load_chunk((const T*)a.gate + run_of(row, a.run) * a.cols, c, a.cols, 0.f, f);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) t[j] *= f[j];
    }
#pragma unroll
    for (int j = 0; j < kChunk; ++j) f[j] = 1.f;
    if (a.scale) load_chunk((const T*)a.scale, c, a.cols, 0.f, f);
    float r[kChunk];
    load_chunk((const T*)a.residual + row * a.residual_stride, c, a.cols, 0.f, r);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) t[j] = fmaf(f[j], r[j], t[j]);
    rounded(t);
}

// Rows that do not fit into a workgroup's registers: read again, out of L2, after each exchange.
template <typename T, bool EIGHT>
__global__ __launch_bounds__(1024) void k_gated_norm_long(NormArgs a)
{
    __shared__ RowSlots slots;
    const int64_t row = a.first_row + blockIdx.x, begin = (int64_t)threadIdx.x * kChunk, step = (int64_t)blockDim.x * kChunk;
    const int waves = blockDim.x >> 6;
    int turn = 0;
    float v[kChunk];
    const auto root_of_row = [&](auto take) {
        float squares = 0.f;
        for (int64_t c = begin; c < a.cols; c += step) {
            take(c);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) squares = fmaf(v[j], v[j], squares);
        }
        reduce_row<64>(squares, waves, slots, turn);
        if (__builtin_expect(in_range(squares, a.cols, a.eps), true)) return root_of(squares, a.cols, a.eps);
        uint32_t peak = 0;
        float none = 0.f;
        for (int64_t c = begin; c < a.cols; c += step) {
            take(c);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) peak = max(peak, magnitude_bits(v[j]));
        }
        reduce_row<64>(none, peak, waves, slots, turn);
        if (peak == 0 || peak >= kInfinityBits) return root_of(squares, a.cols, a.eps);
        const float up = power_up(peak);
        squares = 0.f;
        for (int64_t c = begin; c < a.cols; c += step) {
            take(c);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) squares = fmaf(v[j] * up, v[j] * up, squares);
        }
        reduce_row<64>(squares, waves, slots, turn);
        return root_of_scaled(squares, up, a.cols, a.eps);
    };
    Root first = {1.f, 1.f, 1.f};
    if (a.post) first = root_of_row([&](int64_t c) { load_chunk((const T*)a.x + row * a.x_stride, c, a.cols, 0.f, v); });
    const Root second = root_of_row([&](int64_t c) { form_total<T>(a, row, c, first, v); });
    if (threadIdx.x == 0 && a.rstd) {
        a.rstd[2 * row] = first.unit;
        a.rstd[2 * row + 1] = second.unit;
    }
    const auto normed = [&](int64_t c, bool write_total) {
        float w[kChunk];
        form_total<T>(a, row, c, first, v);
        if (write_total) store_chunk((T*)a.total + row * a.cols, c, a.cols, v, a.streamed);
        load_chunk((const T*)a.weight, c, a.cols, 0.f, w);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) v[j] = v[j] * second.up * second.factor * w[j];
        rounded(v);
    };
    uint32_t most = 0;
    for (int64_t c = begin; c < a.cols; c += step) {
        normed(c, true);
        if constexpr (!EIGHT) store_chunk((T*)a.out + row * a.cols, c, a.cols, v, a.streamed);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) most = max(most, magnitude_bits(v[j]));
    }
    if constexpr (EIGHT) {
        float none = 0.f;
        reduce_row<64>(none, most, waves, slots, turn);
        const RowScale rs = row_scale(most, 1.f, true);
        if (threadIdx.x == 0) a.q_scale[row] = rs.scale;
        for (int64_t c = begin; c < a.cols; c += step) {
            float values[kChunk];
            normed(c, false);
            store_eight(a.q + row * a.q_stride, c, a.cols, rs, v, values);
            if (a.values) store_chunk(a.values, a.values_dtype, row * a.cols, c, a.cols, values, a.streamed);
        }
    }
}

// Two chunks a thread, in 16 bits two rows at once, where rows are many and more than a wave's: the channels' vectors are read once for
// both.  One chunk / two, us: bf16 2048 x 1024 9.3 / 11.1, 4096 x 1024 14.1 / 14.5, 16384 x 1024 41.3 / 36.5, 1024 x 4096 14.0 / 15.1, 2048 x 4096
// 22.3 / 21.0, 8192 x 4096 73.3 / 70.0, 4096 x 8192 87.3 / 76.2; fp32 within a twentieth either way (4096 x 8192 137 / 131, 8192 x 4096 124 / 132).
template <typename T, bool EIGHT>
int run_norm(NormArgs a, int dtype, hipStream_t s)
{
    const bool once = reads_once(dtype, a.x, a.x_stride) && reads_once(dtype, a.residual, a.residual_stride);
    a.streamed = streams(a.rows * a.cols * ((int64_t)sizeof(T) + (EIGHT ? a.values ? dtype_bytes(a.values_dtype) : 0 : (int64_t)sizeof(T))));
    const int64_t chunks = (a.cols + kChunk - 1) / kChunk;
    const int threads = chunks <= 32 ? 32 : threads_of_row(chunks, a.rows >= 2048 && chunks > 64 ? 2 : 1);
    const int64_t items = (chunks + threads - 1) / threads;
    const bool two = sizeof(T) == 2 && a.rows >= 2048 && items == 2;
    const int per_block = threads <= 64 ? 256 / threads : 1, rows_per_block = per_block * (two ? 2 : 1);
    const dim3 block(threads, per_block);
    in_launches((a.rows + rows_per_block - 1) / rows_per_block, threads * per_block, [&](int64_t first, uint32_t grid) {
        a.first_row = first * rows_per_block;
        const auto held = [&](auto rows, auto count, auto lanes) {
            if (once) k_gated_norm<T, rows(), count(), lanes(), true, EIGHT><<<grid, block, 0, s>>>(a);
            else k_gated_norm<T, rows(), count(), lanes(), false, EIGHT><<<grid, block, 0, s>>>(a);
        };
        const std::integral_constant<int, 64> wave;
        const std::integral_constant<int, 1> one;
        const std::integral_constant<int, 2> pair;
        if (threads == 32) held(one, one, std::integral_constant<int, 32>());
        else if (items <= 1) held(one, one, wave);
        else if (two) held(pair, pair, wave);
        else if (items <= 2) held(one, pair, wave);
        else if (items <= 4) held(one, std::integral_constant<int, 4>(), wave);
        else k_gated_norm_long<T, EIGHT><<<grid, block, 0, s>>>(a);
    });
    return hipGetLastError() == hipSuccess ? GEO_SC_OK : GEO_SC_ERR_LAUNCH;
}

// ---------------------------------------------------------------- backward
//
// Rows are dealt out in `units` of `each` consecutive ones.  A unit keeps its columns' sums over its rows in registers and leaves
// them as one partial sum each for dweight, dpost and dscale.  A run's gate gradient is written by the unit that has all of the run's
// rows; of a run that is cut between units each leaves its part: in place 0 where the run holds its first row, else in place 1 (a unit
// has no third, a run that neither begins nor ends in it being its first).  k_join adds in a fixed order: no atomics.

struct BackArgs {
    NormArgs n;
    const void *grad, *grad_total;   // grad_total: or NULL
    int64_t grad_stride, grad_total_stride;
    void *dx, *dresidual;
    void *dweight, *dpost, *dgate, *dscale;   // or NULL
    int64_t units, each;
    float* partial;       // [units][3][cols], then [units][2][cols]; NULL: no sums over rows are wanted
    float* means;         // [rows][2] of the long rows: mean(u n2), mean(s n1)
    bool streamed;        // dx, dresidual
};
enum { kWeight, kPost, kScale, kSums };

__device__ __forceinline__ float* gate_part(const BackArgs& a, int64_t unit, int place)
{
    return a.partial + (a.units * kSums + unit * 2 + place) * a.n.cols;
}
// the sum over a run's rows in [first, last)
template <typename T>
__device__ __forceinline__ void put_gate(const BackArgs& a, int64_t unit, int64_t first, int64_t last, int64_t run, int64_t c, const float (&d)[kChunk])
{
    if (!a.dgate) return;
    if (run * a.n.run >= first && (run + 1) * a.n.run <= last) store_chunk((T*)a.dgate + run * a.n.cols, c, a.n.cols, d);
    else store_chunk(gate_part(a, unit, run == first / a.n.run ? 0 : 1), c, a.n.cols, d);
}
template <typename T>
__device__ __forceinline__ void load_or_ones(const void* p, int64_t c, int64_t cols, float (&v)[kChunk])
{
    if (p) {
        load_chunk((const T*)p, c, cols, 0.f, v);
    } else {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) v[j] = 1.f;
    }
}

// The row and two of the channels' numbers are held as they lie in memory and formed anew on either side of an exchange; gate and post
// come as their product only, and of their two sums over rows one is kept, sum dt n1 over a run, which post and the run's gate multiply where
// the run ends.  That leaves two waves on a SIMD with two chunks a thread: 8192 x 4096 in workgroups of 256, two on a compute unit.  402 MB
// and 25 MB of partial sums in 105 us (4.1 TB/s), joined in 9.
template <typename T, int ITEMS, int LANES, bool ONCE>
__global__ __launch_bounds__(512, 2) void k_gated_back(BackArgs a)
{
    __shared__ RowSlots slots;
    const NormArgs& n = a.n;
    const int threads = blockDim.x, t = threadIdx.x, waves = threads >> 6;
    const int64_t unit = (int64_t)blockIdx.x * blockDim.y + row_in_block<LANES>(), first = unit * a.each;
    const int64_t last = first + a.each < n.rows ? first + a.each : n.rows;
    if (unit >= a.units) return;
    const auto column = [&](int i) { return ((int64_t)i * threads + t) * kChunk; };
    Raw<T> weight[ITEMS], scale[ITEMS];
    float branch[ITEMS][kChunk];   // gate post
    float dweight[ITEMS][kChunk], dscale[ITEMS][kChunk], sum[ITEMS][kChunk];   // sum: of dt n1 over a run
    int64_t run = n.gate ? run_of(first, n.run) : 0, run_end = n.gate ? (run + 1) * n.run : n.rows;
    const auto gate_of_run = [&]() { return n.gate ? (const T*)n.gate + run * n.cols : nullptr; };
    const auto begin_run = [&](int i) {
        float gate[kChunk];
        load_or_ones<T>(n.post, column(i), n.cols, branch[i]);
        load_or_ones<T>(gate_of_run(), column(i), n.cols, gate);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            branch[i][j] *= gate[j];
            sum[i][j] = 0.f;
        }
    };
    bool some = false;   // runs of this unit have ended
    const auto end_run = [&](int i) {
        float v[kChunk], d[kChunk];
        if (a.dgate) {
            load_or_ones<T>(n.post, column(i), n.cols, v);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) d[j] = sum[i][j] * v[j];
            put_gate<T>(a, unit, first, last, run, column(i), d);
        }
        if (a.dpost) {
            float* to = a.partial + (unit * kSums + kPost) * n.cols;
            load_or_ones<T>(gate_of_run(), column(i), n.cols, v);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) d[j] = 0.f;
            if (some) load_chunk(to, column(i), n.cols, 0.f, d);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) d[j] += sum[i][j] * v[j];
            store_chunk(to, column(i), n.cols, d);
        }
    };
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) dweight[i][j] = dscale[i][j] = 0.f;
        if (column(i) < n.cols) {
            weight[i].fetch_or_ones(n.weight, column(i), n.cols);
            scale[i].fetch_or_ones(n.scale, column(i), n.cols);
            begin_run(i);
        }
    }
    int turn = 0;
    // (the next row is on its way while one is worked on)
    Raw<T> x_next[ITEMS], residual_next[ITEMS], g_next[ITEMS], also_next[ITEMS];
    const auto ask = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (column(i) < n.cols) {
                x_next[i].template fetch<ONCE>((const T*)n.x + row * n.x_stride, column(i), n.cols);
                residual_next[i].template fetch<ONCE>((const T*)n.residual + row * n.residual_stride, column(i), n.cols);
                g_next[i].template fetch<ONCE>((const T*)a.grad + row * a.grad_stride, column(i), n.cols);
                if (a.grad_total) also_next[i].template fetch<ONCE>((const T*)a.grad_total + row * a.grad_total_stride, column(i), n.cols);
                else also_next[i].set(0.f);
            }
    };
    ask(first);
    for (int64_t row = first; row < last; ++row) {
        if (row == run_end) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (column(i) < n.cols) end_run(i);
            some = true;
            ++run;
            run_end += n.run;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (column(i) < n.cols) begin_run(i);
        }
        const float r1 = n.rstd[2 * row], r2 = n.rstd[2 * row + 1];
        Raw<T> x[ITEMS], residual[ITEMS], g[ITEMS], also[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) x[i] = x_next[i], residual[i] = residual_next[i], g[i] = g_next[i], also[i] = also_next[i];
        if (row + 1 < last) ask(row + 1);
        const auto keep_all = [&](int i) { x[i].keep(), residual[i].keep(), g[i].keep(), also[i].keep(), weight[i].keep(), scale[i].keep(); };
        const auto form_n2 = [&](int i, int j, float n1) { return (scale[i][j] * residual[i][j] + branch[i][j] * n1) * r2; };
        float along = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (column(i) < n.cols) {
                keep_all(i);
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    const float n2 = form_n2(i, j, x[i][j] * r1);
                    dweight[i][j] += g[i][j] * n2;
                    along += g[i][j] * weight[i][j] * n2;
                }
            }
        reduce_row<LANES>(along, waves, slots, turn);
        const float back = along / (float)n.cols;
        float s[ITEMS][kChunk];
        along = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (column(i) < n.cols) {
                float d[kChunk];
                keep_all(i);
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    const float n1 = x[i][j] * r1, dt = r2 * (g[i][j] * weight[i][j] - form_n2(i, j, n1) * back) + also[i][j];
                    d[j] = dt * scale[i][j];
                    dscale[i][j] += dt * residual[i][j];
                    sum[i][j] += dt * n1;
                    s[i][j] = dt * branch[i][j];
                    along += s[i][j] * n1;
                }
                store_chunk((T*)a.dresidual + row * n.cols, column(i), n.cols, d, a.streamed);
            }
        float through = 0.f;
        if (n.post) {
            reduce_row<LANES>(along, waves, slots, turn);
            through = along / (float)n.cols;
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (column(i) < n.cols) {
                float d[kChunk];
#pragma unroll
                for (int j = 0; j < kChunk; ++j) d[j] = n.post ? r1 * (s[i][j] - x[i][j] * r1 * through) : s[i][j];
                store_chunk((T*)a.dx + row * n.cols, column(i), n.cols, d, a.streamed);
            }
    }
    if (!a.partial) return;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (column(i) < n.cols) {
            float* to = a.partial + unit * kSums * n.cols;
            if (a.dweight) store_chunk(to + kWeight * n.cols, column(i), n.cols, dweight[i]);
            if (a.dscale) store_chunk(to + kScale * n.cols, column(i), n.cols, dscale[i]);
            end_run(i);
        }
}

// What the backward has of a chunk before and after mean(u n2) is known.
template <typename T>
struct Terms {
    float x[kChunk], residual[kChunk], g[kChunk], weight[kChunk], post[kChunk], scale[kChunk], gate[kChunk], n1[kChunk], n2[kChunk], dt[kChunk];
    __device__ __forceinline__ void load(const BackArgs& a, int64_t row, int64_t c, float r1, float r2)
    {
        const NormArgs& n = a.n;
        load_chunk((const T*)n.x + row * n.x_stride, c, n.cols, 0.f, x);
        load_chunk((const T*)n.residual + row * n.residual_stride, c, n.cols, 0.f, residual);
        load_chunk((const T*)a.grad + row * a.grad_stride, c, n.cols, 0.f, g);
        load_chunk((const T*)n.weight, c, n.cols, 0.f, weight);
        load_or_ones<T>(n.post, c, n.cols, post);
        load_or_ones<T>(n.scale, c, n.cols, scale);
        load_or_ones<T>(n.gate ? (const T*)n.gate + run_of(row, n.run) * n.cols : nullptr, c, n.cols, gate);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            n1[j] = x[j] * r1;
            n2[j] = (scale[j] * residual[j] + gate[j] * (n1[j] * post[j])) * r2;
        }
    }
    __device__ __forceinline__ void total_gradient(const BackArgs& a, int64_t row, int64_t c, float r2, float back)
    {
        float h[kChunk] = {};
        if (a.grad_total) load_chunk((const T*)a.grad_total + row * a.grad_total_stride, c, a.n.cols, 0.f, h);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) dt[j] = r2 * (g[j] * weight[j] - n2[j] * back) + h[j];
    }
};

// Rows that do not fit into a workgroup's registers: dresidual and dx row by row, read again after each exchange; the sums over rows by
// columns, in k_gated_back_columns.
template <typename T>
__global__ __launch_bounds__(512) void k_gated_back_long(BackArgs a)
{
    __shared__ RowSlots slots;
    const NormArgs& n = a.n;
    const int waves = blockDim.x >> 6;
    const int64_t row = n.first_row + blockIdx.x, begin = (int64_t)threadIdx.x * kChunk, step = (int64_t)blockDim.x * kChunk;
    const float r1 = n.rstd[2 * row], r2 = n.rstd[2 * row + 1];
    int turn = 0;
    Terms<T> v;
    float along = 0.f;
    for (int64_t c = begin; c < n.cols; c += step) {
        v.load(a, row, c, r1, r2);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) along += v.g[j] * v.weight[j] * v.n2[j];
    }
    reduce_row<64>(along, waves, slots, turn);
    const float back = along / (float)n.cols;
    along = 0.f;
    for (int64_t c = begin; c < n.cols; c += step) {
        float d[kChunk];
        v.load(a, row, c, r1, r2);
        v.total_gradient(a, row, c, r2, back);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            d[j] = v.dt[j] * v.scale[j];
            along += v.dt[j] * v.gate[j] * v.post[j] * v.n1[j];
        }
        store_chunk((T*)a.dresidual + row * n.cols, c, n.cols, d, a.streamed);
        if (!n.post) {
#pragma unroll
            for (int j = 0; j < kChunk; ++j) d[j] = v.dt[j] * v.gate[j];
            store_chunk((T*)a.dx + row * n.cols, c, n.cols, d, a.streamed);
        }
    }
    float through = 0.f;
    if (n.post) {
        reduce_row<64>(along, waves, slots, turn);
        through = along / (float)n.cols;
        for (int64_t c = begin; c < n.cols; c += step) {
            float d[kChunk];
            v.load(a, row, c, r1, r2);
            v.total_gradient(a, row, c, r2, back);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) d[j] = r1 * (v.dt[j] * v.gate[j] * v.post[j] - v.n1[j] * through);
            store_chunk((T*)a.dx + row * n.cols, c, n.cols, d, a.streamed);
        }
    }
    if (threadIdx.x == 0) a.means[row] = back;
}
template <typename T>
__global__ __launch_bounds__(256) void k_gated_back_columns(BackArgs a)
{
    const NormArgs& n = a.n;
    const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * kChunk, unit = blockIdx.y, first = unit * a.each;
    const int64_t last = first + a.each < n.rows ? first + a.each : n.rows;
    if (c >= n.cols) return;
    float dweight[kChunk] = {}, dpost[kChunk] = {}, dscale[kChunk] = {}, dgate[kChunk] = {};
    int64_t run = n.gate ? run_of(first, n.run) : 0, run_end = n.gate ? (run + 1) * n.run : n.rows;
    for (int64_t row = first; row < last; ++row) {
        if (row == run_end) {
            put_gate<T>(a, unit, first, last, run, c, dgate);
            ++run;
            run_end += n.run;
#pragma unroll
            for (int j = 0; j < kChunk; ++j) dgate[j] = 0.f;
        }
        Terms<T> v;
        v.load(a, row, c, n.rstd[2 * row], n.rstd[2 * row + 1]);
        v.total_gradient(a, row, c, n.rstd[2 * row + 1], a.means[row]);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            dweight[j] += v.g[j] * v.n2[j];
            dscale[j] += v.dt[j] * v.residual[j];
            dgate[j] += v.dt[j] * (v.n1[j] * v.post[j]);
            dpost[j] += v.dt[j] * v.gate[j] * v.n1[j];
        }
    }
    float* to = a.partial + unit * kSums * n.cols;
    if (a.dweight) store_chunk(to + kWeight * n.cols, c, n.cols, dweight);
    if (a.dpost) store_chunk(to + kPost * n.cols, c, n.cols, dpost);
    if (a.dscale) store_chunk(to + kScale * n.cols, c, n.cols, dscale);
    put_gate<T>(a, unit, first, last, run, c, dgate);
}

// The sums over the units: COLS columns by SHARES shares of the units in a workgroup.  blockIdx.y: dweight, dpost, dscale, then the runs that may
// be cut: all of them, or one for each border between units where those are fewer.
template <typename T, int COLS, int SHARES>
__global__ __launch_bounds__(COLS * SHARES) void k_join(BackArgs a, bool by_border)
{
    __shared__ float sums[SHARES][COLS];
    const int64_t cols = a.n.cols, c = (int64_t)blockIdx.x * COLS + threadIdx.x;
    float s = 0.f;
    T* to;
    if (blockIdx.y < kSums) {
        to = (T*)(blockIdx.y == kWeight ? a.dweight : blockIdx.y == kPost ? a.dpost : a.dscale);
        if (!to) return;
        if (c < cols) {
#pragma unroll 16
            for (int64_t u = threadIdx.y; u < a.units; u += SHARES) s += a.partial[(u * kSums + blockIdx.y) * cols + c];
        }
    } else {
        if (!a.dgate) return;
        int64_t run = blockIdx.y - kSums;
        if (by_border) {
            const int64_t border = (run + 1) * a.each;
            run = border / a.n.run;
            // a border between runs cuts none; of several in a run the first one's workgroups join it
            if (border % a.n.run == 0 || border - a.each > run * a.n.run) return;
        }
        const int64_t from = run * a.n.run / a.each, to_unit = ((run + 1) * a.n.run - 1) / a.each;
        if (from == to_unit) return;   // written by its unit
        to = (T*)a.dgate + run * cols;
        if (c < cols)
            for (int64_t u = from + threadIdx.y; u <= to_unit; u += SHARES) s += gate_part(a, u, u * a.each / a.n.run == run ? 0 : 1)[c];
    }
    sums[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < cols) {
        s = 0.f;
#pragma unroll 16
        for (int k = 0; k < SHARES; ++k) s += sums[k][threadIdx.x];
        to[c] = (T)s;
    }
}

constexpr int kBackThreads = 512;
constexpr int64_t kHeldBackCols = 2 * kBackThreads * kChunk;   // columns that a workgroup's registers hold in the backward

// Threads of a row: two chunks each where there are rows to fill the compute units so.  1009 x 1111 fp16 20 us with two, 15 with one.
int back_threads(int64_t rows, int64_t cols)
{
    const int64_t chunks = (cols + kChunk - 1) / kChunk;
    return chunks <= 32 ? 32 : threads_of_row(chunks, chunks > 512 || (chunks > 64 && rows >= 2048) ? 2 : 1);
}

// Rows go to as many units as are on the GPU at once, eight waves of them on a compute unit (their registers; with one chunk each
// twelve).  (One more and they go round twice: 8192 x 4100 bf16 both passes in 409 units 363 us, in 256 298.)
struct Units {
    int64_t count, each;
};
Units units_of(int64_t rows, int64_t cols)
{
    const int threads = back_threads(rows, cols);
    const int waves = (cols + kChunk - 1) / kChunk > threads ? 8 : 12;
    const int64_t most = cols > kHeldBackCols ? 64 : (int64_t)256 * (threads == 32 ? 16 : threads == 64 ? 8 : waves / (threads / 64));
    const int64_t each = (rows + most - 1) / most;
    return {(rows + each - 1) / each, each};
}

template <typename T>
int run_back(BackArgs a, int dtype, hipStream_t s)
{
    const NormArgs& n = a.n;
    const int64_t chunks = (n.cols + kChunk - 1) / kChunk;
    a.streamed = streams(2 * n.rows * n.cols * (int64_t)sizeof(T));
    if (n.cols > kHeldBackCols) {
        in_launches(n.rows, kBackThreads, [&](int64_t first, uint32_t count) {
            BackArgs b = a;
            b.n.first_row = first;
            k_gated_back_long<T><<<dim3(count), dim3(kBackThreads), 0, s>>>(b);
        });
        if (a.partial)
            k_gated_back_columns<T><<<dim3((uint32_t)((chunks + 255) / 256), (uint32_t)a.units), dim3(256), 0, s>>>(a);
    } else {
        const bool once = reads_once(dtype, n.x, n.x_stride) && reads_once(dtype, n.residual, n.residual_stride) &&
                          reads_once(dtype, a.grad, a.grad_stride) && (!a.grad_total || reads_once(dtype, a.grad_total, a.grad_total_stride));
        const int threads = back_threads(n.rows, n.cols);
        const int per_block = threads <= 64 ? 256 / threads : 1;
        const dim3 block(threads, per_block), grid((uint32_t)((a.units + per_block - 1) / per_block));
        const auto held = [&](auto count, auto lanes) {
            if (once) k_gated_back<T, count(), lanes(), true><<<grid, block, 0, s>>>(a);
            else k_gated_back<T, count(), lanes(), false><<<grid, block, 0, s>>>(a);
        };
        const std::integral_constant<int, 64> wave;
        if (threads == 32) held(std::integral_constant<int, 1>(), std::integral_constant<int, 32>());
        else if (chunks <= threads) held(std::integral_constant<int, 1>(), wave);
        else held(std::integral_constant<int, 2>(), wave);
    }
    if (a.partial) {
        const int64_t runs = a.dgate ? n.rows / n.run : 0;
        const bool by_border = runs > a.units - 1;
        const auto join = [&](auto columns, auto shares) {
            const dim3 grid((uint32_t)((n.cols + columns() - 1) / columns()), (uint32_t)(kSums + (by_border ? a.units - 1 : runs)));
            k_join<T, columns(), shares()><<<grid, dim3(columns(), shares()), 0, s>>>(a, by_border);
        };
        // Few columns by many shares of the units, or whole lines where the columns are workgroups enough.  8 x 128 / 32 x 16, us: 16384 x 256 fp32
        // 18 / 107, 8192 x 1024 bf16 22 / 54, 1009 x 1111 fp16 17 / 28, 8192 x 2048 22 / 28, 8192 x 3000 16.6 / 18.4, 8192 x 3500 20.1 / 19.2,
        // 8192 x 4096 22.8 / 16.1 (all four sums).
        if (n.cols <= 3000) join(std::integral_constant<int, 8>(), std::integral_constant<int, 128>());
        else join(std::integral_constant<int, 32>(), std::integral_constant<int, 16>());
    }
    return hipGetLastError() == hipSuccess ? GEO_SC_OK : GEO_SC_ERR_LAUNCH;
}

// what a description must have, whichever call it is for
int check(const geo_sc_gated_norm_desc* d, NormArgs* n)
{
    if (!d || (d->struct_bytes != sizeof *d && d->struct_bytes != offsetof(geo_sc_gated_norm_desc, rstd)) || !dtype_known(d->dtype) ||
        d->rows < 0 || d->cols < 1 || d->rows > 0x7fffffff || d->cols > 0x7fffffff || d->x_stride < 0 || d->residual_stride < 0 || !(d->eps >= 0.f) || (d->gate && (d->rows_per_gate < 1 || d->rows % d->rows_per_gate)))
        return GEO_SC_ERR_INVALID_ARGUMENT;
    if (d->rows && (!d->x || !d->residual || !d->weight)) return GEO_SC_ERR_INVALID_ARGUMENT;
    *n = {};
    n->x = d->x;
    n->residual = d->residual;
    n->weight = d->weight;
    n->post = d->post_weight;
    n->gate = d->gate;
    n->scale = d->residual_scale;
    n->rows = d->rows;
    n->cols = d->cols;
    n->x_stride = d->x_stride;
    n->residual_stride = d->residual_stride;
    n->run = d->gate ? d->rows_per_gate : 1;
    n->eps = d->eps;
    return GEO_SC_OK;
}

template <bool EIGHT>
int run_forward(const NormArgs& n, int dtype, hipStream_t s)
{
    if (dtype == GEO_SC_F32) return run_norm<f32, EIGHT>(n, dtype, s);
    if (dtype == GEO_SC_BF16) return run_norm<bf16, EIGHT>(n, dtype, s);
    return run_norm<f16, EIGHT>(n, dtype, s);
}

}  // namespace
}  // namespace geo_sc

using namespace geo_sc;

extern "C" {

int geo_sc_gated_norm(const geo_sc_gated_norm_desc* desc, void* out, void* total, float* rstd, geo_sc_stream_t stream)
{
    NormArgs n;
    if (const int rc = check(desc, &n)) return rc;
    if (n.rows == 0) return GEO_SC_OK;
    if (!out || !total) return GEO_SC_ERR_INVALID_ARGUMENT;
    n.out = out;
    n.total = total;
    n.rstd = rstd;
    return run_forward<false>(n, desc->dtype, (hipStream_t)stream);
}

int geo_sc_gated_norm_q8(const geo_sc_gated_norm_desc* desc, int8_t* q, int64_t q_stride, float* scale, void* total, void* values,
                         int values_dtype, geo_sc_stream_t stream)
{
    NormArgs n;
    if (const int rc = check(desc, &n)) return rc;
    if (q_stride < n.cols || (values && !dtype_known(values_dtype))) return GEO_SC_ERR_INVALID_ARGUMENT;
    if (n.rows == 0) return GEO_SC_OK;
    if (!q || !scale || !total) return GEO_SC_ERR_INVALID_ARGUMENT;
    n.total = total;
    n.q = q;
    n.q_stride = q_stride;
    n.q_scale = scale;
    if (desc->struct_bytes == sizeof *desc) n.rstd = desc->rstd;
    n.values = values;
    n.values_dtype = values_dtype;
    return run_forward<true>(n, desc->dtype, (hipStream_t)stream);
}

int geo_sc_gated_norm_backward_workspace_size(int64_t rows, int64_t cols, size_t* bytes)
{
    if (!bytes || rows < 1 || cols < 1 || rows > 0x7fffffff || cols > 0x7fffffff) return GEO_SC_ERR_INVALID_ARGUMENT;
    *bytes = ((size_t)units_of(rows, cols).count * (kSums + 2) * (size_t)cols + (size_t)rows) * sizeof(float);
    return GEO_SC_OK;
}

int geo_sc_gated_norm_backward(const geo_sc_gated_norm_desc* desc, const void* grad, int64_t grad_stride, const void* grad_total,
                               int64_t grad_total_stride, const float* rstd, void* dx, void* dresidual, void* dweight, void* dpost, void* dgate,
                               void* dscale, void* workspace, size_t workspace_bytes, geo_sc_stream_t stream)
{
    BackArgs a = {};
    if (const int rc = check(desc, &a.n)) return rc;
    if (a.n.rows < 1 || grad_stride < 0 || grad_total_stride < 0 || !grad || !rstd || !dx || !dresidual || (dpost && !a.n.post) ||
        (dgate && !a.n.gate) || (dscale && !a.n.scale))
        return GEO_SC_ERR_INVALID_ARGUMENT;
    size_t need = 0;
    geo_sc_gated_norm_backward_workspace_size(a.n.rows, a.n.cols, &need);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 4) return GEO_SC_ERR_WORKSPACE;
    const Units units = units_of(a.n.rows, a.n.cols);
    a.n.rstd = const_cast<float*>(rstd);
    a.grad = grad;
    a.grad_stride = grad_stride;
    a.grad_total = grad_total;
    a.grad_total_stride = grad_total_stride;
    a.dx = dx;
    a.dresidual = dresidual;
    a.dweight = dweight;
    a.dpost = dpost;
    a.dgate = dgate;
    a.dscale = dscale;
    a.units = units.count;
    a.each = units.each;
    a.partial = dweight || dpost || dgate || dscale ? (float*)workspace : nullptr;
    a.means = (float*)workspace + units.count * (kSums + 2) * a.n.cols;
    hipStream_t s = (hipStream_t)stream;
    if (desc->dtype == GEO_SC_F32) return run_back<f32>(a, desc->dtype, s);
    if (desc->dtype == GEO_SC_BF16) return run_back<bf16>(a, desc->dtype, s);
    return run_back<f16>(a, desc->dtype, s);
}

}  // extern "C"
