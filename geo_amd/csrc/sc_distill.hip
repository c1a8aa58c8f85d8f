// Distillation from a teacher's top logits: the divergence of the student's softmax over all columns from the teacher's
// softmax over its top entries, both at temperature T, and its gradient.
//
//   p_k = softmax over the row's entries of t_k / T,   q = softmax over the columns of z / T
//   loss = T^2 sum_k p_k (log p_k - log q[index_k])
//   dz_j = g T (q_j - sum_{k: index_k = j} p_k),   g: gradient of the row's loss
//
// An entry whose index is outside the columns is absent; a row without entries (or with entries of weight zero only) has loss 0 and gradient 0.
// Forward: one pass over z with the running maximum m and s = sum exp((z - m) / T).  Backward: one more read of z, one write of
// dz.  The row's m, 1 / s and the teacher's maximum and 1 / sum pass from one to the other (kStats floats per row).
//
// exp((z - m) / T) is taken as 2^((z - m) c) with c = log2(e) / T: the difference is formed first, so that the rounding of the product
// weighs by the distance from the maximum and not by the size of the logits.
#include <type_traits>

#include "sc_dense.h"

namespace geo_sc {
namespace {

constexpr int kStats = 4;
constexpr int kMaxTop = 4096;
constexpr float kMinusInfinity = -__builtin_huge_valf();

struct DistillArgs {
    const void *z, *top_logits, *top_index;
    int top_dtype, index64, top;
    int64_t rows, cols, z_stride;
    float temperature;
    int splits;
    int64_t per_split;   // columns of a split, whole chunks
    float *partial;      // [rows][splits][2]: m and s
    float *loss, *stats;
    const float* grad;   // of the loss: one, or one per row
    int grad_per_row;
    float factor;        // of the rows' losses in the result
    void* dz;
    bool streamed;       // dz
};

__device__ __forceinline__ float exp_scaled(float difference, float c) { return __builtin_amdgcn_exp2f(difference * c); }
__device__ __forceinline__ float log2e_over(float temperature) { return 1.44269504088896340736f / temperature; }
// a maximum to subtract: 0 where there is none yet, so that exp(-inf - m) is 0 and not NaN
__device__ __forceinline__ float finite_base(float m) { return m == kMinusInfinity ? 0.f : m; }

__device__ __forceinline__ float wave_max_float(float v)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

// joins (m, s) of the lanes; every lane receives the result
__device__ __forceinline__ void wave_join(float& m, float& s, float c)
{
    const float all = wave_max_float(m), base = finite_base(all);
    s = wave_sum(s * exp_scaled(finite_base(m) - base, c));
    m = all;
}

__device__ __forceinline__ int64_t entry_index(const DistillArgs& a, int64_t row, int k)
{
    const int64_t at = row * a.top + k;
    const int64_t j = a.index64 ? ((const int64_t*)a.top_index)[at] : (int64_t)((const int32_t*)a.top_index)[at];
    return j >= 0 && j < a.cols ? j : -1;
}
__device__ __forceinline__ float entry_logit(const DistillArgs& a, int64_t row, int k)
{
    const int64_t at = row * a.top + k;
    if (a.top_dtype == GEO_SC_F32) return ((const f32*)a.top_logits)[at];
    if (a.top_dtype == GEO_SC_BF16) return (float)((const bf16*)a.top_logits)[at];
    return (float)((const f16*)a.top_logits)[at];
}

// A lane's first entry, asked for before the row is read: by itself it is three ways to memory, one after the other.
struct Entry {
    int64_t j;
    float t, z;
};
template <typename T>
__device__ __forceinline__ Entry entry_of(const DistillArgs& a, int64_t row, int k)
{
    Entry e = {-1, 0.f, 0.f};
    if (k < a.top) {
        e.j = entry_index(a, row, k);
        e.t = entry_logit(a, row, k);
        if (e.j >= 0) e.z = (float)((const T*)a.z)[row * a.z_stride + e.j];
    }
    return e;
}

// The row's loss from m and s, by one wave.
template <typename T>
__device__ __forceinline__ void finish_row(const DistillArgs& a, int64_t row, float m, float s, const Entry& mine)
{
    const int lane = threadIdx.x & 63;
    const float c = log2e_over(a.temperature), inverse_t = 1.f / a.temperature;
    float most = mine.j >= 0 ? mine.t : kMinusInfinity;
    for (int k = lane + 64; k < a.top; k += 64)
        if (entry_index(a, row, k) >= 0) most = fmaxf(most, entry_logit(a, row, k));
    most = wave_max_float(most);
    const float base = finite_base(most);
    float total = mine.j >= 0 ? exp_scaled(mine.t - base, c) : 0.f;
    for (int k = lane + 64; k < a.top; k += 64)
        if (entry_index(a, row, k) >= 0) total += exp_scaled(entry_logit(a, row, k) - base, c);
    total = wave_sum(total);
    const bool empty = total == 0.f;
    const float inverse = empty ? 0.f : 1.f / total, log_total = logf(total), log_s = logf(s), m0 = finite_base(m);
    float loss = 0.f;
    const auto add = [&](const Entry& e) {
        const float t = e.t - base, p = exp_scaled(t, c) * inverse;
        if (e.j >= 0 && !empty && p != 0.f) loss += p * ((t - (e.z - m0)) * inverse_t - log_total + log_s);
    };
    add(mine);
    for (int k = lane + 64; k < a.top; k += 64) add(entry_of<T>(a, row, k));
    loss = wave_sum(loss) * a.temperature * a.temperature;
    if (lane == 0) {
        a.loss[row] = loss;
        float* st = a.stats + row * kStats;
        st[0] = m0;
        st[1] = 1.f / s;
        st[2] = base;
        st[3] = inverse;
    }
}

// m and s of the columns [from, to) of a row, by blockDim.x threads; every lane of the first wave receives them
template <typename T, bool ONCE>
__device__ __forceinline__ void scan_row(const DistillArgs& a, int64_t row, int64_t from, int64_t to, float& m_out, float& s_out)
{
    __shared__ float ms[16], ss[16];
    const float c = log2e_over(a.temperature);
    const T* z = (const T*)a.z + row * a.z_stride;
    const int threads = blockDim.x, waves = threads >> 6;
    float m = kMinusInfinity, s = 0.f;
    const auto add = [&](const float(&v)[kChunk]) {
        float top = m;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) top = fmaxf(top, v[j]);
        const float base = finite_base(top);
        float e = 0.f;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) e += exp_scaled(v[j] - base, c);
        s = s * exp_scaled(finite_base(m) - base, c) + e;
        m = top;
    };
    constexpr int kAhead = 4;
    int64_t at = from + (int64_t)threadIdx.x * kChunk;
    const int64_t step = (int64_t)threads * kChunk;
    for (; at + (kAhead - 1) * step + kChunk <= to; at += kAhead * step) {
        float v[kAhead][kChunk];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) load_chunk<ONCE>(z + at + i * step, v[i]);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) add(v[i]);
    }
    for (; at < to; at += step) {
        float v[kChunk];
        load_chunk(z, at, to, kMinusInfinity, v);
        add(v);
    }
    wave_join(m, s, c);
    if (waves > 1) {
        if ((threadIdx.x & 63) == 0) {
            ms[threadIdx.x >> 6] = m;
            ss[threadIdx.x >> 6] = s;
        }
        __syncthreads();
        m = kMinusInfinity;
        for (int k = 0; k < waves; ++k) m = fmaxf(m, ms[k]);
        const float base = finite_base(m);
        s = 0.f;
        for (int k = 0; k < waves; ++k) s += ss[k] * exp_scaled(finite_base(ms[k]) - base, c);
    }
    m_out = m;
    s_out = s;
}

// One row per threadIdx.y (several rows only where a row has one wave).  Bound by memory: 4096 x 32768 bf16 in 60 us (4.5 TB/s; read
// through the caches 82).
template <typename T, bool ONCE>
__global__ __launch_bounds__(1024) void k_distill_rows(DistillArgs a)
{
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= a.rows) return;
    const Entry mine = entry_of<T>(a, row, threadIdx.x < 64 ? (int)threadIdx.x : a.top);
    float m, s;
    scan_row<T, ONCE>(a, row, 0, a.cols, m, s);
    if (threadIdx.x < 64) finish_row<T>(a, row, m, s, mine);
}

// A share of the columns of a long row, of which there are too few for the compute units; k_distill_join puts the shares together.
// 19 x 100003 bf16 5.4 and 3.6 us: a launch and a way to memory each.
template <typename T>
__global__ __launch_bounds__(1024) void k_distill_split(DistillArgs a)
{
    const int64_t row = blockIdx.y, from = (int64_t)blockIdx.x * a.per_split;
    const int64_t to = from + a.per_split < a.cols ? from + a.per_split : a.cols;
    float m, s;
    scan_row<T, false>(a, row, from, to, m, s);
    if (threadIdx.x == 0) {
        float* p = a.partial + (row * a.splits + blockIdx.x) * 2;
        p[0] = m;
        p[1] = s;
    }
}
template <typename T>
__global__ __launch_bounds__(64) void k_distill_join(DistillArgs a)
{
    const int64_t row = blockIdx.x;
    float m = kMinusInfinity, s = 0.f;
    if ((int)threadIdx.x < a.splits) {   // (at most 64 splits)
        const float* p = a.partial + (row * a.splits + threadIdx.x) * 2;
        m = p[0];
        s = p[1];
    }
    const Entry mine = entry_of<T>(a, row, threadIdx.x);
    wave_join(m, s, log2e_over(a.temperature));
    finish_row<T>(a, row, m, s, mine);
}

// the rows' losses in a fixed order, by one workgroup: 4.6 us for 4096 rows
__global__ __launch_bounds__(1024) void k_sum_losses(const float* rows_loss, int64_t rows, float factor, float* loss)
{
    __shared__ float sums[16];
    float s = 0.f;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) s += rows_loss[r];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.f;
        for (int k = 0; k < 16; ++k) s += sums[k];
        *loss = s * factor;
    }
}

// Bound by memory: 4096 x 32768 bf16 reads and writes 537 MB in 118 us behind a forward that read past the caches (98 behind one
// that left them its last rows, and took 22 more itself).
template <typename T>
__global__ __launch_bounds__(1024) void k_distill_back(DistillArgs a)
{
    extern __shared__ int32_t columns[];   // the entries' columns of each row of the block
    // From the last rows on: what the forward, which commonly ran just before, read last is still in the caches (4096 x 32768 fp32,
    // both passes, 329 us, in the order of the rows 350).
    const int64_t group = gridDim.y - 1 - blockIdx.y, row = group * blockDim.y + threadIdx.y, from = (int64_t)blockIdx.x * a.per_split;
    const int64_t to = from + a.per_split < a.cols ? from + a.per_split : a.cols;
    const bool live = row < a.rows;
    const T* z = (const T*)a.z + row * a.z_stride;
    T* dz = (T*)a.dz + row * a.cols;
    int32_t* column = columns + threadIdx.y * a.top;
    const float c = log2e_over(a.temperature);
    float m = 0.f, inverse_s = 0.f, top_m = 0.f, top_inverse = 0.f, scale = 0.f;
    Entry mine = {};
    if (live) {
        const float* st = a.stats + row * kStats;
        m = st[0];
        inverse_s = st[1];
        top_m = st[2];
        top_inverse = st[3];
        scale = a.grad[a.grad_per_row ? row : 0] * a.factor * a.temperature;
        mine = entry_of<T>(a, row, threadIdx.x);
        for (int k = threadIdx.x; k < a.top; k += blockDim.x) column[k] = (int32_t)entry_index(a, row, k);
        const bool empty = top_inverse == 0.f;
        const float k = scale * inverse_s;
        const int64_t step = (int64_t)blockDim.x * kChunk;
        const auto gradient = [&](float(&v)[kChunk]) {
#pragma unroll
            for (int j = 0; j < kChunk; ++j) v[j] = empty ? 0.f : exp_scaled(v[j] - m, c) * k;
        };
        constexpr int kAhead = 8;
        int64_t at = from + (int64_t)threadIdx.x * kChunk;
        for (; at + (kAhead - 1) * step + kChunk <= to; at += kAhead * step) {
            float v[kAhead][kChunk];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) load_chunk(z + at + i * step, v[i]);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                gradient(v[i]);
                store_chunk(dz, at + i * step, to, v[i], a.streamed);
            }
        }
        for (; at < to; at += step) {
            float v[kChunk];
            load_chunk(z, at, to, 0.f, v);
            gradient(v);
            store_chunk(dz, at, to, v, a.streamed);
        }
    }
    // The entries' columns are written again, each by one thread: the one of the entry that names the column first,
    // which sums the weights of all that name it.
    __syncthreads();
    if (!live || top_inverse == 0.f) return;
    for (int k = threadIdx.x; k < a.top; k += blockDim.x) {
        const Entry e = k == (int)threadIdx.x ? mine : entry_of<T>(a, row, k);
        if (e.j < from || e.j >= to) continue;
        bool owner = true;
        float p = exp_scaled(e.t - top_m, c) * top_inverse;
        for (int f = 0; f < k; ++f) owner = owner && column[f] != (int32_t)e.j;
        if (!owner) continue;
        for (int f = k + 1; f < a.top; ++f)
            if (column[f] == (int32_t)e.j) p += exp_scaled(entry_logit(a, row, f) - top_m, c) * top_inverse;
        dz[e.j] = (T)(scale * (exp_scaled(e.z - m, c) * inverse_s - p));
    }
}

constexpr int64_t kSplitLeast = 8192;   // columns that a split of a row has at least

// Long rows, when there are few (fewer than `groups`, so that they fit the grid's second dimension), are cut: enough workgroups for the
// compute units, at most 64 shares (the join is one wave).
void cut_rows(DistillArgs& a, int64_t groups)
{
    int64_t splits = (groups + a.rows - 1) / a.rows;
    const int64_t most = (a.cols + kSplitLeast - 1) / kSplitLeast;
    if (splits > most) splits = most;
    if (splits > 64) splits = 64;
    const int64_t chunks = (a.cols + kChunk - 1) / kChunk;
    a.per_split = (chunks + splits - 1) / splits * kChunk;
    a.splits = (int)((a.cols + a.per_split - 1) / a.per_split);
}
int threads_of(int64_t cols)
{
    int threads = 64;
    while (threads < 256 && threads * kChunk * 2 < cols) threads *= 2;
    return threads;
}

// the rows from `first` on, of what forward and backward have in common
template <typename T>
DistillArgs rows_from(DistillArgs a, int64_t first)
{
    a.rows -= first;
    a.z = (const T*)a.z + first * a.z_stride;
    a.stats += first * kStats;
    a.top_logits = (const char*)a.top_logits + first * a.top * dtype_bytes(a.top_dtype);
    a.top_index = (const char*)a.top_index + first * a.top * (a.index64 ? 8 : 4);
    return a;
}

template <typename T>
int run_distill(const DistillArgs& a, int reduction, float* result, hipStream_t s)
{
    const int threads = threads_of(a.per_split), per_block = threads == 64 ? 4 : 1;
    if (a.splits == 1) {
        const dim3 block(threads, per_block);
        in_launches((a.rows + per_block - 1) / per_block, threads, [&](int64_t first, uint32_t grid) {
            DistillArgs b = rows_from<T>(a, first * per_block);
            b.loss = a.loss + first * per_block;
            // (fp32 gains nothing: 4096 x 32768 with the gradient 339 us, read like any other 329)
            if constexpr (std::is_same_v<T, f32>) k_distill_rows<T, false><<<grid, block, 0, s>>>(b);
            else if (reads_once(GEO_SC_BF16, a.z, a.z_stride)) k_distill_rows<T, true><<<grid, block, 0, s>>>(b);
            else k_distill_rows<T, false><<<grid, block, 0, s>>>(b);
        });
    } else {
        k_distill_split<T><<<dim3((uint32_t)a.splits, (uint32_t)a.rows), dim3(threads), 0, s>>>(a);
        k_distill_join<T><<<dim3((uint32_t)a.rows), dim3(64), 0, s>>>(a);
    }
    if (reduction != GEO_SC_REDUCE_NONE) k_sum_losses<<<1, 1024, 0, s>>>(a.loss, a.rows, a.factor, result);
    return hipGetLastError() == hipSuccess ? GEO_SC_OK : GEO_SC_ERR_LAUNCH;
}

template <typename T>
int run_distill_back(const DistillArgs& a, hipStream_t s)
{
    const int threads = threads_of(a.per_split), per_block = threads == 64 ? 4 : 1;
    for (int64_t r = 0; r < a.rows; r += 65535 * (int64_t)per_block) {   // rows are the grid's second dimension
        DistillArgs b = rows_from<T>(a, r);
        if (b.rows > 65535 * (int64_t)per_block) b.rows = 65535 * (int64_t)per_block;
        b.dz = (T*)a.dz + r * a.cols;
        b.grad = a.grad + (a.grad_per_row ? r : 0);
        k_distill_back<T><<<dim3((uint32_t)a.splits, (uint32_t)((b.rows + per_block - 1) / per_block)), dim3(threads, per_block),
                            (size_t)per_block * a.top * sizeof(int32_t), s>>>(b);
    }
    return hipGetLastError() == hipSuccess ? GEO_SC_OK : GEO_SC_ERR_LAUNCH;
}

bool distill_sizes_fit(int64_t rows, int64_t cols, int top)
{
    return rows >= 1 && rows <= 0x3fffffff && cols >= 1 && cols <= 0x7fffffff && top >= 1 && top <= kMaxTop;
}
// The loss takes T^2 as a factor; where that is a number above zero, so are 1 / T and log2(e) / T.
bool temperature_fits(float t) { return t > 0.f && t * t > 0.f && t * t <= 3.402823466e38f; }
constexpr int64_t kGroups = 1024;   // workgroups that few long rows are cut into
float factor_of(int reduction, int64_t rows) { return reduction == GEO_SC_REDUCE_MEAN ? 1.f / (float)rows : 1.f; }

}  // namespace
}  // namespace geo_sc

using namespace geo_sc;

extern "C" {

int geo_sc_distill_topk_workspace_size(int64_t rows, int64_t cols, size_t* bytes)
{
    if (!bytes || !distill_sizes_fit(rows, cols, 1)) return GEO_SC_ERR_INVALID_ARGUMENT;
    DistillArgs a = {};
    a.rows = rows;
    a.cols = cols;
    cut_rows(a, kGroups);
    *bytes = (size_t)rows * sizeof(float) + (a.splits > 1 ? (size_t)rows * a.splits * 2 * sizeof(float) : 0);
    return GEO_SC_OK;
}

int geo_sc_distill_topk(const void* logits, int dtype, int64_t logits_stride, const void* top_logits, int top_dtype,
                        const void* top_index, int index_bytes, int64_t rows, int64_t cols, int top, float temperature, int reduction,
                        float* loss, float* stats, void* workspace, size_t workspace_bytes, geo_sc_stream_t stream)
{
    if (!distill_sizes_fit(rows, cols, top) || !dtype_known(dtype) || !dtype_known(top_dtype) || (index_bytes != 4 && index_bytes != 8) ||
        logits_stride < 0 || !temperature_fits(temperature) || reduction < GEO_SC_REDUCE_NONE || reduction > GEO_SC_REDUCE_MEAN || !logits ||
        !top_logits || !top_index || !loss || !stats)
        return GEO_SC_ERR_INVALID_ARGUMENT;
    DistillArgs a = {};
    a.z = logits;
    a.top_logits = top_logits;
    a.top_index = top_index;
    a.top_dtype = top_dtype;
    a.index64 = index_bytes == 8;
    a.top = top;
    a.rows = rows;
    a.cols = cols;
    a.z_stride = logits_stride;
    a.temperature = temperature;
    a.factor = factor_of(reduction, rows);
    cut_rows(a, kGroups);
    size_t need = 0;
    geo_sc_distill_topk_workspace_size(rows, cols, &need);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 4) return GEO_SC_ERR_WORKSPACE;
    a.loss = reduction == GEO_SC_REDUCE_NONE ? loss : (float*)workspace;
    a.partial = (float*)workspace + rows;
    a.stats = stats;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == GEO_SC_F32) return run_distill<f32>(a, reduction, loss, s);
    if (dtype == GEO_SC_BF16) return run_distill<bf16>(a, reduction, loss, s);
    return run_distill<f16>(a, reduction, loss, s);
}

int geo_sc_distill_topk_backward(const float* grad, int reduction, const void* logits, int dtype, int64_t logits_stride,
                                 const void* top_logits, int top_dtype, const void* top_index, int index_bytes, int64_t rows,
                                 int64_t cols, int top, float temperature, const float* stats, void* dlogits, geo_sc_stream_t stream)
{
    if (!distill_sizes_fit(rows, cols, top) || !dtype_known(dtype) || !dtype_known(top_dtype) || (index_bytes != 4 && index_bytes != 8) ||
        logits_stride < 0 || !temperature_fits(temperature) || reduction < GEO_SC_REDUCE_NONE || reduction > GEO_SC_REDUCE_MEAN || !grad ||
        !logits || !top_logits || !top_index || !stats || !dlogits)
        return GEO_SC_ERR_INVALID_ARGUMENT;
    DistillArgs a = {};
    a.z = logits;
    a.top_logits = top_logits;
    a.top_index = top_index;
    a.top_dtype = top_dtype;
    a.index64 = index_bytes == 8;
    a.top = top;
    a.rows = rows;
    a.cols = cols;
    a.z_stride = logits_stride;
    a.temperature = temperature;
    a.factor = factor_of(reduction, rows);
    a.stats = const_cast<float*>(stats);
    a.grad = grad;
    a.grad_per_row = reduction == GEO_SC_REDUCE_NONE;
    a.dz = dlogits;
    a.streamed = streams(rows * cols * dtype_bytes(dtype));
    cut_rows(a, kGroups);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == GEO_SC_F32) return run_distill_back<f32>(a, s);
    if (dtype == GEO_SC_BF16) return run_distill_back<bf16>(a, s);
    return run_distill_back<f16>(a, s);
}

}  // extern "C"
