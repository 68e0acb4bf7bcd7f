// Rotary positions with several axes: every pair (a, b) of a head's rotated dims is
// turned by its axis's coordinate times its own frequency,
//   a' = a cos t - b sin t,  b' = b cos t + a sin t,
// q and k in one launch; dims past the rotated ones are copied.
//
// What bounds it: HBM, each element read and written once. The angles are shared by
// all heads of a token, so a block computes those of its tokens once into LDS and
// then streams the heads.
//
// The angle is formed in double, in revolutions: position * turn keeps 2^-22 of a
// revolution at positions of 2^31 where fp32 has lost it at 2^20, and only the
// fraction goes on in fp32.
#include "types.h"

using namespace hatk;

#define ROT_THREADS 256
#define ROT_ANGLES 4096  // cos and sin values a block keeps (32 KB)

// n / d for n < 2^20 by d's reciprocal: the error of (n + 1/2) / d is below 2^-2 / d.
__device__ __forceinline__ int div_small(int n, float inv) { return (int)(((float)n + 0.5f) * inv); }

template <class T, int V>
__device__ __forceinline__ void rotary_body(const RotaryArgs& p)
{
    __shared__ __attribute__((aligned(16))) float cs[ROT_ANGLES], sn[ROT_ANGLES];
    const long long first = (long long)blockIdx.x * p.per;
    const long long all = p.tokens * p.batch;
    const int n = (int)(all - first < p.per ? all - first : p.per);
    for (int e = threadIdx.x; e < n * p.pairs; e += ROT_THREADS) {
        const int t = div_small(e, p.inv_pairs), i = e - t * p.pairs;
        const long long b = (first + t) / p.tokens, tok = first + t - b * p.tokens;
        int axis = 0;
#pragma unroll
        for (int a = 0; a < ROT_AXES - 1; ++a) axis += i >= p.ends[a];
        const double turns = (double)p.pos[b * p.pb + tok * p.pt + axis * p.pa] * p.turn[i];
        float s, c;
        sincospif(2.0f * (float)(turns - __builtin_rint(turns)), &s, &c);
        cs[e] = c;
        sn[e] = s;
    }
    __syncthreads();
    const int turned = p.neighbours && V > 1 ? 2 * p.pairs / V : p.pairs / V;
    const int per_token = p.chunks * (p.heads[0] + p.heads[1]);
    for (int e = threadIdx.x; e < n * per_token; e += ROT_THREADS) {
        const int t = div_small(e, p.inv_items), r = e - t * per_token;
        int head = div_small(r, p.inv_chunks);
        const int c = r - head * p.chunks;
        const int w = head >= p.heads[0];
        head -= w ? p.heads[0] : 0;
        const long long b = (first + t) / p.tokens, tok = first + t - b * p.tokens;
        const T* x = (const T*)p.x[w] + b * p.xb[w] + tok * p.xt[w] + head * p.xh[w];
        T* y = (T*)p.y[w] + b * p.yb[w] + tok * p.yt[w] + head * p.yh[w];
        if (c >= turned) {  // behind the rotated dims
            const int d = 2 * p.pairs + (c - turned) * V;
            *(typename Vec<T, V>::type*)(y + d) = *(const typename Vec<T, V>::type*)(x + d);
        } else if (!p.neighbours) {
            const int i = c * V;
            float u[V], v[V], uo[V], vo[V];
            load_vec<T, V>(x + i, u);
            load_vec<T, V>(x + i + p.pairs, v);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float cj = cs[t * p.pairs + i + j], sj = sn[t * p.pairs + i + j];
                uo[j] = u[j] * cj - v[j] * sj;
                vo[j] = v[j] * cj + u[j] * sj;
            }
            store_vec<T, V>(y + i, uo);
            store_vec<T, V>(y + i + p.pairs, vo);
        } else if constexpr (V > 1) {
            const int d = c * V;
            float u[V], o[V];
            load_vec<T, V>(x + d, u);
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float cj = cs[t * p.pairs + (d + j) / 2], sj = sn[t * p.pairs + (d + j) / 2];
                o[j] = u[j] * cj - u[j + 1] * sj;
                o[j + 1] = u[j + 1] * cj + u[j] * sj;
            }
            store_vec<T, V>(y + d, o);
        } else {
            const float u = (float)x[2 * c], v = (float)x[2 * c + 1], cj = cs[t * p.pairs + c], sj = sn[t * p.pairs + c];
            y[2 * c] = (T)(u * cj - v * sj);
            y[2 * c + 1] = (T)(v * cj + u * sj);
        }
    }
}

#define ROTARY_INST(NAME, T, V) \
    extern "C" __global__ __launch_bounds__(ROT_THREADS) void NAME(RotaryArgs p) { rotary_body<T, V>(p); }

ROTARY_INST(hat_rotary_f32_v4, float, 4)
ROTARY_INST(hat_rotary_f32_v2, float, 2)
ROTARY_INST(hat_rotary_f32_v1, float, 1)
ROTARY_INST(hat_rotary_f16_v8, f16, 8)
ROTARY_INST(hat_rotary_f16_v4, f16, 4)
ROTARY_INST(hat_rotary_f16_v1, f16, 1)
ROTARY_INST(hat_rotary_bf16_v8, bf16, 8)
ROTARY_INST(hat_rotary_bf16_v4, bf16, 4)
ROTARY_INST(hat_rotary_bf16_v1, bf16, 1)
