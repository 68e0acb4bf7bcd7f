// Attention over sequences of any length on device tensors:
//   s(i, j) = cap tanh(scale q_i . k_j / cap) - slope_head * distance(i, j)
//   o_i = sum_j e^s(i, j) v_j / sum_j e^s(i, j)  over the keys j that query i sees,
// zeros where it sees none. Every query sees the keys below a limit of its own:
// its sequence's length, the causal edge, or the prefix where that reaches further,
// so one number a row is the whole mask.
#include "types.h"

using namespace hatk;

// A sequence's place in the tensors.
struct SeqView {
    int s, lq, lk;            // its number, queries and keys in use
    int q0, k0;               // token index of its first query and key (packed tensors)
    long long bq, bk;         // batch index of the q and k tensors (0 where packed)
};

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Offsets and lengths come from device memory: clamped, so that no value of theirs
// leads outside the tensors.
__device__ __forceinline__ SeqView seq_view(const SeqAttnArgs& p, int s)
{
    SeqView v;
    v.s = s;
    if (p.cu_q) {
        v.q0 = clamp_int(p.cu_q[s], 0, p.q_tokens);
        v.lq = clamp_int(p.cu_q[s + 1], v.q0, p.q_tokens) - v.q0;
        v.bq = 0;
    } else {
        v.q0 = 0;
        v.lq = p.q_lens ? clamp_int(p.q_lens[s], 0, p.q_tokens) : p.q_tokens;
        v.bq = s;
    }
    if (p.cu_k) {
        v.k0 = clamp_int(p.cu_k[s], 0, p.k_tokens);
        v.lk = clamp_int(p.cu_k[s + 1], v.k0, p.k_tokens) - v.k0;
        v.bk = 0;
    } else {
        v.k0 = 0;
        v.lk = p.k_lens ? clamp_int(p.k_lens[s], 0, p.k_tokens) : p.k_tokens;
        v.bk = s;
    }
    return v;
}

// The first key that query i does not see; prefix: the sequence's, or 0.
__device__ __forceinline__ int row_limit(const SeqAttnArgs& p, const SeqView& v, int i, int prefix)
{
    if (!p.causal) return v.lk;
    const int edge = i + v.lk - v.lq + 1;
    return clamp_int(edge > prefix ? edge : prefix, 0, v.lk);
}

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

__device__ __forceinline__ float lane_value(float v, int lane)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// One row by one wave, in fp32 throughout, every product of its own: keys that the
// row does not see are not touched, whatever they hold.
template <class T>
__device__ void attn_row(const SeqAttnArgs& p, const SeqView& v, int i, int head, int limit)
{
    const int lane = threadIdx.x & 63;
    const int D = p.dim, kvh = head / p.group;
    const T* q = (const T*)p.q + v.bq * p.qb + (long long)(v.q0 + i) * p.qt + head * p.qh;
    const T* k = (const T*)p.k + v.bk * p.kb + (long long)v.k0 * p.kt + kvh * p.kh;
    const T* vv = (const T*)p.v + v.bk * p.vb + (long long)v.k0 * p.vt + kvh * p.vh;
    const float qa = lane < D ? (float)q[lane] : 0.0f, qc = lane + 64 < D ? (float)q[lane + 64] : 0.0f;
    const float slope = p.slopes ? p.slopes[head] * HAT_LOG2E : 0.0f;
    float m = -INFINITY, l = 0.0f, oa = 0.0f, oc = 0.0f;
    for (int j0 = 0; j0 < limit; j0 += 64) {
        const int j = j0 + lane;
        // every lane takes part, those past the limit on the last key: a lane's value
        // is read by all (v_readlane), so it must be computed by all
        const int jr = j < limit ? j : limit - 1;
        const T* kr = k + (long long)jr * p.kt;
        float s = 0.0f;
        for (int d = 0; d < D && d < 64; ++d) s = __builtin_fmaf(lane_value(qa, d), (float)kr[d], s);
        for (int d = 64; d < D; ++d) s = __builtin_fmaf(lane_value(qc, d - 64), (float)kr[d], s);
        s *= p.scale;
        if (p.cap > 0.0f) s = p.cap * tanhf(s * p.inv_cap);
        s *= HAT_LOG2E;
        if (p.slopes) {
            float far;
            if (p.pos_q) {
                const int* a = p.pos_q + v.bq * p.pqb + (long long)(v.q0 + i) * p.pqt;
                const int* b = p.pos_k + v.bk * p.pkb + (long long)(v.k0 + jr) * p.pkt;
                far = 0.0f;
                for (int x = 0; x < p.axes; ++x) far += fabsf((float)(a[x * p.pqa] - b[x * p.pka]));
            } else {
                far = fabsf((float)(i + v.lk - v.lq - jr));
            }
            s = __builtin_fmaf(-slope, far, s);
        }
        s = j < limit ? s : -INFINITY;
        const float mn = fmaxf(m, wave_max(s));
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float e = j < limit ? fast_exp2(s - base) : 0.0f;
        const float corr = fast_exp2(m - base);
        l = l * corr + wave_sum(e);
        oa *= corr;
        oc *= corr;
        const int n = limit - j0 < 64 ? limit - j0 : 64;
        for (int t = 0; t < n; ++t) {
            const float pt = lane_value(e, t);
            const T* vr = vv + (long long)(j0 + t) * p.vt;
            if (lane < D) oa = __builtin_fmaf(pt, (float)vr[lane], oa);
            if (lane + 64 < D) oc = __builtin_fmaf(pt, (float)vr[lane + 64], oc);
        }
        m = mn;
    }
    T* o = (T*)p.o + v.bq * p.ob + (long long)(v.q0 + i) * p.ot + head * p.oh;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (lane < D) o[lane] = (T)(oa * inv);
    if (lane + 64 < D) o[lane + 64] = (T)(oc * inv);
}

// A wave a row, four rows a block.
template <class T>
__device__ __forceinline__ void attn_rows_body(const SeqAttnArgs& p)
{
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int head = (int)(row % p.q_heads);
    const long long tok = row / p.q_heads;
    int s, i;
    if (p.cu_q) {
        if (tok >= p.q_tokens) return;
        int lo = 0, hi = p.n_seq;  // the first sequence that ends behind the token
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (p.cu_q[mid + 1] > tok)
                hi = mid;
            else
                lo = mid + 1;
        }
        s = lo;
        if (s == p.n_seq) return;
        i = (int)tok - clamp_int(p.cu_q[s], 0, p.q_tokens);
    } else {
        s = (int)(tok / p.q_tokens);
        i = (int)(tok - (long long)s * p.q_tokens);
        if (s >= p.n_seq) return;
    }
    const SeqView v = seq_view(p, s);
    if (i < 0 || i >= v.lq) return;
    attn_row<T>(p, v, i, head, row_limit(p, v, i, p.prefix ? p.prefix[s] : 0));
}

#define SEQ_ROWS_INST(NAME, T) \
    extern "C" __global__ __launch_bounds__(256) void NAME(SeqAttnArgs p) { attn_rows_body<T>(p); }

SEQ_ROWS_INST(hat_attnseq_rows_f32, float)
SEQ_ROWS_INST(hat_attnseq_rows_f16, f16)
SEQ_ROWS_INST(hat_attnseq_rows_bf16, bf16)
