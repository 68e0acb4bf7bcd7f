// The join of a block's output with the residual stream and the norm behind it:
//   x' = x + scale * gate * Npost(y),  h = Npre(x'),
// Npost and Npre each LayerNorm, RMSNorm or nothing, the gate a row of its own for
// every rows_per_gate rows. y may be missing (x' = x), x' or h may be left out.
//
// What bounds it: HBM, x and y read once, x' and h written once. A row's values stay
// in registers between the reading and the second norm, so both norms' sums (a mean,
// then the sum of squared differences from it) run over registers; h is formed from
// x' before its rounding. A row takes 16, 64, 256 or 1024 threads by its width: the
// fewest that hold it, since beyond a wave every sum costs two barriers. x is read with
// y, ahead of y's sums (57600 x 1536 in bf16: 142 us, behind them 152).
// Measured, both norms and a gate, 708 MB: bf16 57600 x 1536 132-138 us (5.1-5.4 TB/s),
// x 1024 134, x 2048 134, x 4096 140, x 8192 139; fp32 x 144 130, x 1024 131; rows
// that allow 4-byte moves only (1002 wide) 161, single elements (1001) 182. A large copy
// reaches 5.2-5.8 TB/s here.
#include "types.h"

using namespace hatk;

// The sum over a row's TPR threads, the same in each, added in a fixed order.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* lds)
{
#pragma unroll
    for (int o = TPR < 64 ? TPR / 2 : 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (TPR > 64) {
        __syncthreads();  // the last sum's values have been read
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) v += lds[w];
    }
    return v;
}

// A row of p.width elements: moves at the thread's vectors i * TPR + t. Rows that a whole
// wave shares go through a buffer descriptor that ends with the row (zeros past it, no
// branch); rows of 16 threads through pointers and a check a vector.
template <class T, int TPR, int V>
struct Row {
    T* p;
    __amdgpu_buffer_rsrc_t r;
    int width, t;
    __device__ __forceinline__ Row(const void* base, long long offset, int w, int thread) : width(w), t(thread)
    {
        p = (T*)base + offset;
        if constexpr (TPR >= 64) r = buffer_of(p, w * (int)sizeof(T));
    }
    __device__ __forceinline__ void load(int i, float (&v)[V]) const
    {
        if constexpr (TPR >= 64) {
            constexpr int part = sizeof(T) * V > 16 ? 16 / (int)sizeof(T) : V;
#pragma unroll
            for (int h = 0; h < V; h += part) {
                float u[part];
                buffer_load_vec<T, part>(r, t * V * (int)sizeof(T), (i * TPR * V + h) * (int)sizeof(T), u);
#pragma unroll
                for (int j = 0; j < part; ++j) v[h + j] = u[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = 0.0f;
            if ((i * TPR + t) * V < width) load_vec<T, V>(p + (i * TPR + t) * V, v);
        }
    }
    __device__ __forceinline__ typename Vec<T, V>::type raw(int i) const
    {
        if constexpr (TPR >= 64)
            return buffer_load_raw<T, V>(r, t * V * (int)sizeof(T), i * TPR * V * (int)sizeof(T));
        else
            return (i * TPR + t) * V < width ? *(const typename Vec<T, V>::type*)(p + (i * TPR + t) * V)
                                             : (typename Vec<T, V>::type)(T)0.0f;
    }
    __device__ __forceinline__ void store(int i, const float (&v)[V]) const
    {
        if constexpr (TPR >= 64) {
            buffer_store_vec<T, V>(r, t * V * (int)sizeof(T), i * TPR * V * (int)sizeof(T), v);
        } else {
            if ((i * TPR + t) * V < width) store_vec<T, V>(p + (i * TPR + t) * V, v);
        }
    }
};

// v = N(v) over the row's p.width values; zeros stay past the width.
template <int TPR, int V, int NV>
__device__ __forceinline__ void row_norm(float (&v)[NV][V], int kind, const float* w, const float* b, float eps,
                                         int width, int t, float* lds)
{
    // The mean is 0 for RMSNorm and taken off all the same: with the subtraction under the
    // condition the compiler lost the values on the other path (f16, one vector a thread).
    float mean = 0.0f;
    if (kind == NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[i][j];
        mean = row_sum<TPR>(s, lds) / (float)width;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const float m = (i * TPR + t) * V < width ? mean : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] -= m;
    }
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) q = __builtin_fmaf(v[i][j], v[i][j], q);
    const float r = 1.0f / sqrtf(row_sum<TPR>(q, lds) / (float)width + eps);
    const Row<float, TPR, V> rw(w, 0, width, t), rb(b, 0, width, t);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[V], a[V];
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = 1.0f, a[j] = 0.0f;
        if (w) rw.load(i, f);
        if (b) rb.load(i, a);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = __builtin_fmaf(v[i][j] * r, f[j], a[j]);
    }
}

// THREADS a block, TPR of them a row, NV vectors of V elements a thread.
template <class T, int THREADS, int TPR, int V, int NV>
__device__ __forceinline__ void resnorm_body(const ResNormArgs& p)
{
    __shared__ float lds[THREADS / 64];
    const int t = threadIdx.x % TPR;
    int in_block = threadIdx.x / TPR;
    if constexpr (TPR >= 64) in_block = __builtin_amdgcn_readfirstlane(in_block);
    const long long row = (long long)blockIdx.x * (THREADS / TPR) + in_block;
    if (row >= p.rows) return;  // whole rows leave; with more than a wave a row, whole blocks
    float v[NV][V];
    const Row<T, TPR, V> x(p.x, row * p.xs, p.width, t), xo(p.xo, row * p.xos, p.width, t);
    // x is read before y's sums, as it came: its loads run under them
    typename Vec<T, V>::type xr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) xr[i] = x.raw(i);
    if (p.y) {
        const Row<T, TPR, V> y(p.y, row * p.ys, p.width, t);
#pragma unroll
        for (int i = 0; i < NV; ++i) y.load(i, v[i]);
        if (p.post != NORM_NONE) row_norm<TPR, V, NV>(v, p.post, p.post_w, p.post_b, p.post_eps, p.width, t, lds);
        if (p.gate) {
            const Row<T, TPR, V> g(p.gate, (p.rows_per_gate == p.rows ? 0 : row / p.rows_per_gate) * p.gs, p.width, t);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float f[V];
                g.load(i, f);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] *= f[j];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float u[V];
        to_float<T, V>(xr[i], u);
        if (p.y) {
#pragma unroll
            for (int j = 0; j < V; ++j) u[j] = __builtin_fmaf(p.scale, v[i][j], u[j]);
        }
        if (p.xo) xo.store(i, u);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = u[j];
    }
    if (!p.h) return;
    if (p.pre != NORM_NONE) row_norm<TPR, V, NV>(v, p.pre, p.pre_w, p.pre_b, p.pre_eps, p.width, t, lds);
    const Row<T, TPR, V> h(p.h, row * p.hs, p.width, t);
#pragma unroll
    for (int i = 0; i < NV; ++i) h.store(i, v[i]);
}

// NV: the most vectors a thread. The body is compiled for fewer as well, since moves past
// the row's end cost their issue (86400 rows of 1024 in bf16: 178 us with two of four
// vectors in use, 134 with two compiled).
template <class T, int THREADS, int TPR, int V, int NV>
__device__ __forceinline__ void resnorm_kernel(const ResNormArgs& p)
{
    const int n = (p.width + TPR * V - 1) / (TPR * V);
    if constexpr (NV >= 8) {
        if (n <= NV / 4)
            resnorm_body<T, THREADS, TPR, V, NV / 4>(p);
        else if (n <= NV / 2)
            resnorm_body<T, THREADS, TPR, V, NV / 2>(p);
        else
            resnorm_body<T, THREADS, TPR, V, NV>(p);
    } else {
        if (n == 1)
            resnorm_body<T, THREADS, TPR, V, 1>(p);
        else if (n == 2)
            resnorm_body<T, THREADS, TPR, V, 2>(p);
        else if (NV == 4 && n == 3)
            resnorm_body<T, THREADS, TPR, V, 3>(p);
        else
            resnorm_body<T, THREADS, TPR, V, NV>(p);
    }
}

#define RESNORM_INST(NAME, T, THREADS, TPR, V, NV) \
    extern "C" __global__ __launch_bounds__(THREADS) void NAME(ResNormArgs p) { resnorm_kernel<T, THREADS, TPR, V, NV>(p); }

// by the bytes of a move (16; 4 or one element where the rows' alignment or width allow
// no more) and the threads a row
RESNORM_INST(hat_resnorm_f32_16, float, 256, 16, 4, 3)
RESNORM_INST(hat_resnorm_f32_64, float, 256, 64, 4, 4)
RESNORM_INST(hat_resnorm_f32_256, float, 256, 256, 4, 4)
RESNORM_INST(hat_resnorm_f32_1024, float, 1024, 1024, 4, 4)
RESNORM_INST(hat_resnorm_f32_64e, float, 256, 64, 1, 16)
RESNORM_INST(hat_resnorm_f32_256e, float, 256, 256, 1, 16)
RESNORM_INST(hat_resnorm_f32_1024e, float, 1024, 1024, 1, 16)
RESNORM_INST(hat_resnorm_f16_16, f16, 256, 16, 8, 2)
RESNORM_INST(hat_resnorm_f16_64, f16, 256, 64, 8, 4)
RESNORM_INST(hat_resnorm_f16_256, f16, 256, 256, 8, 4)
RESNORM_INST(hat_resnorm_f16_1024, f16, 1024, 1024, 8, 2)
RESNORM_INST(hat_resnorm_f16_64h, f16, 256, 64, 2, 8)
RESNORM_INST(hat_resnorm_f16_256h, f16, 256, 256, 2, 8)
RESNORM_INST(hat_resnorm_f16_1024h, f16, 1024, 1024, 2, 8)
RESNORM_INST(hat_resnorm_f16_64e, f16, 256, 64, 1, 16)
RESNORM_INST(hat_resnorm_f16_256e, f16, 256, 256, 1, 16)
RESNORM_INST(hat_resnorm_f16_1024e, f16, 1024, 1024, 1, 16)
RESNORM_INST(hat_resnorm_bf16_16, bf16, 256, 16, 8, 2)
RESNORM_INST(hat_resnorm_bf16_64, bf16, 256, 64, 8, 4)
RESNORM_INST(hat_resnorm_bf16_256, bf16, 256, 256, 8, 4)
RESNORM_INST(hat_resnorm_bf16_1024, bf16, 1024, 1024, 8, 2)
RESNORM_INST(hat_resnorm_bf16_64h, bf16, 256, 64, 2, 8)
RESNORM_INST(hat_resnorm_bf16_256h, bf16, 256, 256, 2, 8)
RESNORM_INST(hat_resnorm_bf16_1024h, bf16, 1024, 1024, 2, 8)
RESNORM_INST(hat_resnorm_bf16_64e, bf16, 256, 64, 1, 16)
RESNORM_INST(hat_resnorm_bf16_256e, bf16, 256, 256, 1, 16)
RESNORM_INST(hat_resnorm_bf16_1024e, bf16, 1024, 1024, 1, 16)
