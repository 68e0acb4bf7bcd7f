// Rotary positions with several axes: every pair (a, b) of a head's rotated dims is
// turned by its axis's coordinate times its own frequency,
//   a' = a cos t - b sin t,  b' = b cos t + a sin t,
// q and k in one launch; dims past the rotated ones are copied.
//
// What bounds it: HBM, each element read and written once. The angles are shared by
// all heads of a token, so a block computes those of its tokens once into LDS and
// then streams the heads, consecutive lanes on consecutive moves of a token.
// Measured, 57600 tokens of 12 + 12 heads in fp16: dims of 64 72-75 us (4.7-4.9 TB/s), of 80
// with 64 turned 92 (4.8), of 72 with 64 turned 85-88 (4.5-4.7), with 56 turned in 8-byte
// moves 90 (4.4); a large copy reaches 5.2-5.8 TB/s. A small call is its launch: 256 tokens
// of 6 + 6 heads of 24 take 4.0 us.
//
// The angle is formed in double, in revolutions: position * turn keeps 2^-22 of a
// revolution at positions of 2^31 where fp32 has lost it at 2^20, and only the
// fraction goes on in fp32.
#include "types.h"

using namespace hatk;

#define ROT_THREADS 256
#define ROT_ANGLES 4096  // cos and sin values a block keeps (32 KB)
#define ROT_TOKENS 64    // tokens a block takes at most

// n / d for n < 2^20 by d's reciprocal: the error of (n + 1/2) / d is below 2^-2 / d.
__device__ __forceinline__ int div_small(int n, float inv) { return (int)(((float)n + 0.5f) * inv); }

template <class T, int V>
__device__ __forceinline__ void rotary_body(const RotaryArgs& p)
{
    __shared__ __attribute__((aligned(16))) f32x2 cs[ROT_ANGLES];  // (cos, sin)
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
        cs[e] = (f32x2){c, s};
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
    // An item is two moves of V elements: the halves of V pairs, two neighbouring runs, or
    // two runs of the dims behind the rotated ones. All take the same path, as a branch
    // would cost a wave both: the runs without an angle keep their bits at the end.
    const int turned = p.neighbours ? (2 * p.pairs / V + 1) / 2 : p.pairs / V;
    const int rest = p.dim / V - 2 * p.pairs / V;  // moves behind the rotated dims
    const int per_token = p.chunks * (p.heads[0] + p.heads[1]);
    const int all_items = n * per_token;
    typedef typename Vec<T, V>::type vec;
    // items a thread loads before it stores the first: 57600 tokens, 24 heads of 64 in 16-byte
    // moves 77 us by one, 72 by two, 75 by four; of 72 in 8-byte moves 112, 95, 89 (six: 92)
    constexpr int ROT_AHEAD = sizeof(T) * V >= 16 ? 2 : 4;
    for (int e0 = threadIdx.x; e0 < all_items; e0 += ROT_THREADS * ROT_AHEAD) {
        vec u[ROT_AHEAD], v[ROT_AHEAD];
        T* y[ROT_AHEAD];
        int d0[ROT_AHEAD], d1[ROT_AHEAD], angle[ROT_AHEAD];  // angle < 0: a copy; d0 < 0: no item
#pragma unroll
        for (int k = 0; k < ROT_AHEAD; ++k) {
            const int e = e0 + k * ROT_THREADS;
            d0[k] = -1;
            if (e >= all_items) continue;
            const int t = div_small(e, p.inv_items), r = e - t * per_token;
            int head = div_small(r, p.inv_chunks);
            const int c = r - head * p.chunks;
            const int w = head >= p.heads[0];
            head -= w ? p.heads[0] : 0;
            const T* x = (const T*)p.x[w] + at[w][t] + head * p.xh[w];
            y[k] = (T*)p.y[w] + at[2 + w][t] + head * p.yh[w];
            if (c >= turned) {
                const int i = c - turned, j = i + (rest + 1) / 2;
                d0[k] = 2 * p.pairs + i * V;
                d1[k] = 2 * p.pairs + (j < rest ? j : i) * V;  // an odd one twice
                angle[k] = -1;
            } else if (p.neighbours) {
                d0[k] = 2 * c * V;
                d1[k] = d0[k] + V < 2 * p.pairs ? d0[k] + V : d0[k];
                angle[k] = t * p.pairs;
            } else {
                d0[k] = c * V;
                d1[k] = d0[k] + p.pairs;
                angle[k] = t * p.pairs + d0[k];
            }
            u[k] = *(const vec*)(x + d0[k]);
            v[k] = *(const vec*)(x + d1[k]);
        }
#pragma unroll
        for (int k = 0; k < ROT_AHEAD; ++k) {
            if (d0[k] < 0) continue;
            const bool copy = angle[k] < 0;
            vec uo, vo;
            if constexpr (V == 1) {
                // neighbours too are a pair: turned counts pairs here
                const f32x2 a = cs[copy ? 0 : p.neighbours ? angle[k] + d0[k] / 2 : angle[k]];
                const float f = (float)u[k], g = (float)v[k];
                uo = (T)(f * a[0] - g * a[1]);
                vo = (T)(g * a[0] + f * a[1]);
            } else if (p.neighbours) {
#pragma unroll
                for (int j = 0; j < V; j += 2) {
                    const f32x2 a = cs[copy ? 0 : angle[k] + (d0[k] + j) / 2], b = cs[copy ? 0 : angle[k] + (d1[k] + j) / 2];
                    const float f = (float)u[k][j], g = (float)u[k][j + 1], h = (float)v[k][j], i = (float)v[k][j + 1];
                    uo[j] = (T)(f * a[0] - g * a[1]);
                    uo[j + 1] = (T)(g * a[0] + f * a[1]);
                    vo[j] = (T)(h * b[0] - i * b[1]);
                    vo[j + 1] = (T)(i * b[0] + h * b[1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const f32x2 a = cs[(copy ? 0 : angle[k]) + j];
                    const float f = (float)u[k][j], g = (float)v[k][j];
                    uo[j] = (T)(f * a[0] - g * a[1]);
                    vo[j] = (T)(g * a[0] + f * a[1]);
                }
            }
            *(vec*)(y[k] + d0[k]) = copy ? u[k] : uo;
            *(vec*)(y[k] + d1[k]) = copy ? v[k] : vo;
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
