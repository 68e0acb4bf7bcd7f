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
#define ROT_TOKENS 64    // tokens a block takes at most
#define ROT_AHEAD 4

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
    // where the block's tokens lie in x and y
    __shared__ long long at[4][ROT_TOKENS];
    for (int t = threadIdx.x; t < n; t += ROT_THREADS) {
        const long long b = (first + t) / p.tokens, tok = first + t - b * p.tokens;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            at[w][t] = b * p.xb[w] + tok * p.xt[w];
            at[2 + w][t] = b * p.yb[w] + tok * p.yt[w];
        }
    }
    __syncthreads();
    const int turned = p.neighbours && V > 1 ? 2 * p.pairs / V : p.pairs / V;
    const int per_token = p.chunks * (p.heads[0] + p.heads[1]);
    const int all_items = n * per_token;
    typedef typename Vec<T, V>::type vec;
    // ROT_AHEAD items a thread at a time, their loads issued before the first is used
    for (int e0 = threadIdx.x; e0 < all_items; e0 += ROT_THREADS * ROT_AHEAD) {
        vec u[ROT_AHEAD], v[ROT_AHEAD];
        T* y[ROT_AHEAD];
        int c[ROT_AHEAD], angle[ROT_AHEAD];  // c < 0: no item
#pragma unroll
        for (int k = 0; k < ROT_AHEAD; ++k) {
            const int e = e0 + k * ROT_THREADS;
            c[k] = -1;
            if (e >= all_items) continue;
            const int t = div_small(e, p.inv_items), r = e - t * per_token;
            int head = div_small(r, p.inv_chunks);
            c[k] = r - head * p.chunks;
            angle[k] = t * p.pairs;
            const int w = head >= p.heads[0];
            head -= w ? p.heads[0] : 0;
            const T* x = (const T*)p.x[w] + at[w][t] + head * p.xh[w];
            y[k] = (T*)p.y[w] + at[2 + w][t] + head * p.yh[w];
            if (V == 1 && p.neighbours && c[k] < turned) {
                u[k] = *(const vec*)(x + 2 * c[k]);
                v[k] = *(const vec*)(x + 2 * c[k] + 1);
            } else {
                const int d = c[k] < turned ? c[k] * V : 2 * p.pairs + (c[k] - turned) * V;
                u[k] = *(const vec*)(x + d);
                if (!p.neighbours && c[k] < turned) v[k] = *(const vec*)(x + d + p.pairs);
            }
        }
#pragma unroll
        for (int k = 0; k < ROT_AHEAD; ++k) {
            if (c[k] < 0) continue;
            if (c[k] >= turned) {  // behind the rotated dims
                *(vec*)(y[k] + 2 * p.pairs + (c[k] - turned) * V) = u[k];
            } else if (!p.neighbours || V == 1) {
                const int i = c[k] * V;
                float uo[V], vo[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float a, b;
                    if constexpr (V == 1)
                        a = (float)u[k], b = (float)v[k];
                    else
                        a = (float)u[k][j], b = (float)v[k][j];
                    const float cj = cs[angle[k] + i + j], sj = sn[angle[k] + i + j];
                    uo[j] = a * cj - b * sj;
                    vo[j] = b * cj + a * sj;
                }
                store_vec<T, V>(y[k] + (V == 1 && p.neighbours ? 2 * i : i), uo);
                store_vec<T, V>(y[k] + (V == 1 && p.neighbours ? 2 * i + 1 : i + p.pairs), vo);
            } else if constexpr (V > 1) {
                const int d = c[k] * V;
                float o[V];
#pragma unroll
                for (int j = 0; j < V; j += 2) {
                    const float a = (float)u[k][j], b = (float)u[k][j + 1];
                    const float cj = cs[angle[k] + (d + j) / 2], sj = sn[angle[k] + (d + j) / 2];
                    o[j] = a * cj - b * sj;
                    o[j + 1] = b * cj + a * sj;
                }
                store_vec<T, V>(y[k] + d, o);
            }
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
