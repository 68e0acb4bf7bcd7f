// Attention over sequences of any length on device tensors:
//   s(i, j) = cap tanh(scale q_i . k_j / cap) - slope_head * distance(i, j)
//   o_i = sum_j e^s(i, j) v_j / sum_j e^s(i, j)  over the keys j that query i sees,
// zeros where it sees none. Every query sees the keys below a limit of its own:
// its sequence's length, the causal edge, or the prefix where that reaches further,
// so one number a row is the whole mask, and only the stages that a limit of the wave
// crosses compare with it. The query heads that share a key head are rows of one tile:
// K and V are read once for all of them.
//
// Three forms, by rows (query, head of the group) a key head and by type; the host's
// rules and both sides' times are at attn_plan:
// - many rows (seq_body; fp32: seq32_body): a block of four waves, 32 rows each, walks the
//   keys. Scores are formed transposed, S^T = K Q^T, so that a lane holds 16 scores of
//   one row: the softmax needs one exchange with the other half of the wave, and the
//   probabilities are MFMA's B operand for O^T += V^T P^T where they lie. V^T comes
//   from LDS by the transposing read.
// - few rows (seq_split_body): the keys are split over a block's waves and over blocks.
// - fp32 with up to eight rows (seq_few_body): four rows at a time.
//
// What bounds the first: issue. MFMA and vector instructions take turns on a SIMD: at 16-bit
// head_dim 128, 64 keys x 32 rows cost a wave 1024 cycles of MFMA and about 680 of the
// softmax (32 exponentials of 8 cycles, 105 instructions of 4), 1930 measured: 53% MFMA
// busy, LDS 53%. Two and more waves a SIMD cover each other's waits: with 64 rows a wave
// and one wave a SIMD 787 TFLOP/s where this has 1060. The next stage's scores formed
// under the present one's softmax gained 2% at 128 dims and lost 4% at 64: not kept.
// Measured: bf16 16384 x 16384, 8 heads of 128 1.00-1.10 ms (1.0-1.1 PFLOP/s; the library's
// 8192-cubed product 1.11); fp16 2 x 12 heads of 64, 4096 keys 133-149 us (700-770
// TFLOP/s), with a bias by distance 160-169; the cap at 128 dims, causal, 2 x 16 heads, 8192
// keys 626 us (880 TFLOP/s of the seen pairs); 256 windows of 256 tokens, 6 heads of 24,
// bias over two axes: fp16 60-64 us, fp32 110-123.
#include "types.h"

using namespace hatk;

// A sequence's place in the tensors.
struct SeqView {
    int s, lq, lk;            // its number, queries and keys in use
    int q0, k0;               // token index of its first query and key (packed tensors)
    long long bq, bk;         // batch index of the q and k tensors (0 where packed)
};

// Shapes. A stage of keys sits in LDS as rows of DP = 32 DT elements in 16-byte
// chunks; chunk c of row r lies at slot c ^ swizzle(r), so that the reads down the
// rows (K: 8 rows of one chunk at a time; 16-bit V: four rows of two chunks) meet
// every bank once. fp32 V is read along its rows and needs none.
template <class T, int DT>
struct SeqShape {
    static constexpr int DP = 32 * DT;
    static constexpr int E = 16 / (int)sizeof(T);  // elements a chunk
    static constexpr int CH = DP / E;              // chunks a row
    static constexpr int KS = CH / 2;              // MFMA steps of q . k: two chunks each, one a lane half
    static constexpr int ROW = DP * (int)sizeof(T);
    __device__ static __forceinline__ int kswz(int r) { return CH % 8 ? (r >> 1) & 3 : r & 7; }
    __device__ static __forceinline__ int vswz(int r)
    {
        return sizeof(T) == 4 ? 0 : CH % 8 ? (r & 2) : (r & 3) << 1;
    }
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

// Keys [j0, j1) of one row by one wave, in fp32 throughout, every product of its own:
// keys that the row does not see are not touched, whatever they hold. m: the largest
// score (log2 units), l: the sum of 2^(s - m), oa, oc: dims lane and lane + 64 of the
// sum of 2^(s - m) v.
template <class T>
__device__ void attn_row(const SeqAttnArgs& p, const SeqView& v, int i, int head, int j0, int j1, float& m, float& l,
                         float& oa, float& oc)
{
    const int lane = threadIdx.x & 63;
    const int D = p.dim, kvh = head / p.group;
    const T* q = (const T*)p.q + v.bq * p.qb + (long long)(v.q0 + i) * p.qt + head * p.qh;
    const T* k = (const T*)p.k + v.bk * p.kb + (long long)v.k0 * p.kt + kvh * p.kh;
    const T* vv = (const T*)p.v + v.bk * p.vb + (long long)v.k0 * p.vt + kvh * p.vh;
    const float qa = lane < D ? (float)q[lane] : 0.0f, qc = lane + 64 < D ? (float)q[lane + 64] : 0.0f;
    const float slope = p.slopes ? p.slopes[head] * HAT_LOG2E : 0.0f;
    m = -INFINITY, l = oa = oc = 0.0f;
    for (; j0 < j1; j0 += 64) {
        const int j = j0 + lane;
        // every lane takes part, those past the end on the last key: a lane's value
        // is read by all (v_readlane), so it must be computed by all
        const int jr = j < j1 ? j : j1 - 1;
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
        s = j < j1 ? s : -INFINITY;
        const float mn = fmaxf(m, wave_max(s));
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float e = j < j1 ? fast_exp2(s - base) : 0.0f;
        const float corr = fast_exp2(m - base);
        l = l * corr + wave_sum(e);
        oa *= corr;
        oc *= corr;
        const int n = j1 - j0 < 64 ? j1 - j0 : 64;
        for (int t = 0; t < n; ++t) {
            const float pt = lane_value(e, t);
            const T* vr = vv + (long long)(j0 + t) * p.vt;
            if (lane < D) oa = __builtin_fmaf(pt, (float)vr[lane], oa);
            if (lane + 64 < D) oc = __builtin_fmaf(pt, (float)vr[lane + 64], oc);
        }
        m = mn;
    }
}

__device__ __forceinline__ float join_scale(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

__device__ __forceinline__ float swap_max(float v)  // over a lane and its twin in the other half
{
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    const unsigned b = __float_as_uint(v);
    const u2 r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float swap_sum(float v)
{
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    const unsigned b = __float_as_uint(v);
    const u2 r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ f32x16 mma16(u32x4 a, u32x4 b, f32x16 c, f16) { return mfma_f16(a, b, c); }
__device__ __forceinline__ f32x16 mma16(u32x4 a, u32x4 b, f32x16 c, bf16)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ unsigned pack16(float a, float b, f16)
{
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){a, b}, f16x2));
}
__device__ __forceinline__ unsigned pack16(float a, float b, bf16) { return pk_bf16(a, b); }

// s plus both values of a packed pair: the sum is over the probabilities that the
// product with v sees.
__device__ __forceinline__ float add_pair(unsigned w, float s, f16)
{
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), (f16x2){(_Float16)1.0f, (_Float16)1.0f}, s, false);
}
__device__ __forceinline__ float add_pair(unsigned w, float s, bf16)
{
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), (bf16x2){(__bf16)1.0f, (__bf16)1.0f}, s, false);
}

// 16 bytes of elements from element `at` of a buffer, zeros from the `left`th on, in moves
// of 4 bytes (wide == 1) or of an element.
template <class T>
__device__ __forceinline__ u32x4 load_chunk(__amdgpu_buffer_rsrc_t r, int at, int left, int wide)
{
    u32x4 u;
    if (sizeof(T) == 4 || wide) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int x = e * 4 / (int)sizeof(T);
            u[e] = __builtin_amdgcn_raw_buffer_load_b32(r, x < left ? (at + x) * (int)sizeof(T) : 0x80000000u, 0, 0);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned lo = __builtin_amdgcn_raw_buffer_load_b16(r, 2 * e < left ? (at + 2 * e) * 2 : 0x80000000u, 0, 0);
            const unsigned hi =
                __builtin_amdgcn_raw_buffer_load_b16(r, 2 * e + 1 < left ? (at + 2 * e + 1) * 2 : 0x80000000u, 0, 0);
            u[e] = (lo & 0xffffu) | hi << 16;
        }
    }
    return u;
}

// The rows of K or V of one stage into LDS, by THREADS threads (a block, or one wave on
// its own): R rows from row `first` of n, zeros past the last and past the head's dims.
// Chunks go straight to LDS through a buffer descriptor that ends with the last row,
// whose range check supplies the zeros without a branch.
template <class T, int DT, int R, int THREADS, bool V>
struct Stage {
    using S = SeqShape<T, DT>;
    static constexpr int N = R * S::CH / THREADS;
    static_assert(R * S::CH % THREADS == 0, "whole moves a thread");
    const T* base;     // the sequence's first row, this head
    long long stride;  // of rows
    int n, dim;
    unsigned off[N];   // the lane's byte offset from the stage's first row, per move
    __device__ __forceinline__ void init(const T* b, long long st, int rows, int d, int tid)
    {
        base = b, stride = st, n = rows, dim = d;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = j * THREADS + tid, r = c / S::CH, lc = (c % S::CH) ^ (V ? S::vswz(r) : S::kswz(r));
            off[j] = lc * S::E < dim ? (unsigned)(r * (int)stride * (int)sizeof(T) + lc * 16) : 0x80000000u;
        }
    }
    __device__ __forceinline__ void issue(unsigned char* lds, int first, int tid, int wide) const
    {
        const int left = n - first;
        const int rows = left < R ? left : R;
        const auto rsrc = buffer_of(base + (long long)first * stride,
                                    rows <= 0 ? 0 : ((rows - 1) * (int)stride + dim) * (int)sizeof(T));
        if (wide == 2) {
            unsigned char* to = lds + (THREADS > 64 ? __builtin_amdgcn_readfirstlane(tid >> 6) : 0) * 1024;
#pragma unroll
            for (int j = 0; j < N; ++j)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rsrc, (__attribute__((address_space(3))) void*)(to + j * THREADS * 16), 16, off[j], 0, 0, 0);
        } else {
#pragma unroll 1  // the registers are needed elsewhere
            for (int j = 0; j < N; ++j) {
                const int c = j * THREADS + tid, r = c / S::CH, d0 = ((c % S::CH) ^ (V ? S::vswz(r) : S::kswz(r))) * S::E;
                *(u32x4*)(lds + c * 16) = load_chunk<T>(rsrc, r * (int)stride + d0, dim - d0, wide);
            }
        }
    }
};

// What a lane knows of its row: row r of a (sequence, key head) pair is query r / group,
// head r % group of the pair's heads.
struct SeqRow {
    int i, head;
    bool live;
};

__device__ __forceinline__ SeqRow seq_row(const SeqAttnArgs& p, int r, int rows, int kvh)
{
    const int i = r / p.group;
    return {i, kvh * p.group + r - i * p.group, r < rows};
}

template <class T>
__device__ __forceinline__ const T* row_of(const SeqAttnArgs& p, const SeqView& v, const SeqRow& r)
{
    return (const T*)p.q + v.bq * p.qb + (long long)(v.q0 + r.i) * p.qt + r.head * p.qh;
}

// 16 bytes of elements from p + d0, zeros from the `left`th on; elements past the end are
// read at the row's start instead, without a branch.
template <class T>
__device__ __forceinline__ u32x4 row_chunk(const T* p, int d0, int left, int wide)
{
    u32x4 u;
    if (sizeof(T) == 4 || wide) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int x = e * 4 / (int)sizeof(T);
            const unsigned w = *(const unsigned*)(p + (x < left ? d0 + x : 0));
            u[e] = x < left ? w : 0u;
        }
    } else {
        const unsigned short* q = (const unsigned short*)p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned lo = q[2 * e < left ? d0 + 2 * e : 0], hi = q[2 * e + 1 < left ? d0 + 2 * e + 1 : 0];
            u[e] = (2 * e < left ? lo : 0u) | (2 * e + 1 < left ? hi << 16 : 0u);
        }
    }
    return u;
}

// The lane's q as the B operand of K Q^T: step ks holds the lane half's chunk 2 ks + h.
template <class T, int DT>
__device__ __forceinline__ void load_q(const SeqAttnArgs& p, const SeqView& v, const SeqRow& r,
                                       u32x4 (&q)[SeqShape<T, DT>::KS])
{
    using S = SeqShape<T, DT>;
    const int h = (threadIdx.x >> 5) & 1;
    const auto row = row_of<T>(p, v, r);
    const bool flip = p.scale < 0.0f;
#pragma unroll
    for (int ks = 0; ks < S::KS; ++ks) {
        const int d0 = (2 * ks + h) * S::E;
        u32x4 u = {0, 0, 0, 0};
        if (p.wide == 2) {
            if (r.live && d0 < p.dim) u = *(const u32x4*)(row + d0);
        } else if (r.live) {
            u = row_chunk<T>(row, d0, p.dim - d0, p.wide);
        }
        if (flip) {  // c1 is positive
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] ^= sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
        }
        q[ks] = u;
    }
}

// The same from fp32, split: eight dims a step and lane half.
template <int DT>
__device__ __forceinline__ void load_q32(const SeqAttnArgs& p, const SeqView& v, const SeqRow& r, u32x4 (&q)[2 * DT][3])
{
    const int h = (threadIdx.x >> 5) & 1;
    const float* row = (const float*)p.q + v.bq * p.qb + (long long)(v.q0 + r.i) * p.qt + r.head * p.qh;
    const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int ks = 0; ks < 2 * DT; ++ks) {
        float f[8];
#pragma unroll
        for (int x = 0; x < 8; x += 4) {
            const int d0 = (2 * ks + h) * 8 + x;
            f32x4 u = {0.f, 0.f, 0.f, 0.f};
            if (p.wide == 2) {
                if (r.live && d0 < p.dim) u = *(const f32x4*)(row + d0);
            } else if (r.live) {
                u = __builtin_bit_cast(f32x4, row_chunk<float>(row, d0, p.dim - d0, 1));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) f[x + e] = u[e] * sign;
        }
        split3_x8(f, q[ks]);
    }
}

// One lane's running softmax over the keys of its row.
template <class T, int DT>
struct SeqAcc {
    f32x16 o[DT];
    float m, l;
    __device__ __forceinline__ void init()
    {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
        m = -1e30f, l = 0.0f;  // finite: 2^(-inf - m) is 0, not NaN
    }
};

// What stands between q . k and the softmax, compiled apart: every instruction a score
// costs counts, as the vector and the matrix unit take turns.
enum SeqMode {
    SEQ_PLAIN,  // nothing
    SEQ_BIAS,   // the bias, which MFMA's accumulator starts from (in units of q . k)
    SEQ_CAP,    // the cap: scores held as r = 1 / (e^2x + 1), tanh x = 1 - 2 r
    SEQ_BOTH,   // whatever the arguments say, in log2 units
};

// The bias of a lane's row.
struct SeqBias {
    float slope;      // SEQ_BIAS: in units of q . k; SEQ_BOTH: in log2 units
    int at;           // i + Lk - Lq
    unsigned pos[4];  // positions, offset to order as unsigned
};

__device__ __forceinline__ SeqBias seq_bias(const SeqAttnArgs& p, const SeqView& v, const SeqRow& r, bool raw)
{
    SeqBias b;
    b.slope = p.slopes && r.live ? p.slopes[r.head] * HAT_LOG2E : 0.0f;
    if (raw) b.slope /= p.c1;
    b.at = r.i + v.lk - v.lq;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        b.pos[a] = 0;
        if (p.pos_q && r.live && a < p.axes)
            b.pos[a] = (unsigned)p.pos_q[v.bq * p.pqb + (long long)(v.q0 + r.i) * p.pqt + a * p.pqa] ^ 0x80000000u;
    }
    return b;
}

// c + |a - b|: one instruction, which the compiler does not form by itself.
__device__ __forceinline__ unsigned sad(unsigned a, unsigned b, unsigned c)
{
    unsigned d;
    asm("v_sad_u32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

// s[r] -= slope * distance for 32 keys by their positions in LDS (pk, one row of `pstride`
// an axis). Register r is key 8 (r / 4) + 4 h + r % 4.
__device__ __forceinline__ void pos_bias(const SeqAttnArgs& p, const SeqBias& b, f32x16& s, const unsigned* pk, int pstride)
{
    const unsigned* k = pk + 4 * ((threadIdx.x >> 5) & 1);
    unsigned far[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) far[r] = 0;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        if (a < p.axes) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const u32x4 x = *(const u32x4*)(k + a * pstride + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) far[4 * g + e] = sad(b.pos[a], x[e], far[4 * g + e]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(-b.slope, (float)far[r], s[r]);
}

__device__ __forceinline__ void index_bias(const SeqBias& b, f32x16& s, int k0)
{
    const float at = (float)(b.at - k0 - 4 * (int)((threadIdx.x >> 5) & 1));
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(-b.slope, fabsf(at - (float)(8 * (r >> 2) + (r & 3))), s[r]);
}

// Where MFMA starts from for 32 keys from k0: s, and a row's constant beside it. By index,
// keys that lie on one side of all the wave's rows (at0 .. at1) have a bias that is linear
// in the key: a product with the key's place in the tile, the rest a constant of the row.
template <int MODE>
__device__ __forceinline__ float seq_start(const SeqAttnArgs& p, const SeqBias& b, f32x16& s, int k0, const unsigned* pk,
                                           int pstride, int at0, int at1)
{
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
    if constexpr (MODE != SEQ_BIAS) return 0.0f;
    if (p.pos_q) {
        pos_bias(p, b, s, pk, pstride);
        return 0.0f;
    }
    if (k0 + 31 <= at0 || k0 >= at1) {
        const float sl = k0 >= at1 ? -b.slope : b.slope;
        const float base = (float)(4 * (int)((threadIdx.x >> 5) & 1));
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = sl * (float)(8 * (r >> 2) + (r & 3));
        return sl * ((float)(k0 - b.at) + base);
    }
    index_bias(b, s, k0);
    return 0.0f;
}

// SEQ_BOTH: the scores of 32 keys from k0 in log2 units.
template <class T>
__device__ __forceinline__ void seq_scores(const SeqAttnArgs& p, const SeqBias& b, f32x16& s, int k0, const unsigned* pk,
                                           int pstride)
{
    if (p.cap > 0.0f) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = p.cap * HAT_LOG2E * tanhf(s[r] * fabsf(p.scale) * p.inv_cap);
        } else {
            // tanh x = 1 - 2 / (e^2x + 1): off by 2^-23 of the cap, which the
            // probabilities' rounding to 16 bits covers
            const float a = p.cap * HAT_LOG2E;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[r] = __builtin_fmaf(-2.0f * a, __builtin_amdgcn_rcpf(fast_exp2(s[r] * p.c1) + 1.0f), a);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= p.c1;
    }
    if (!p.slopes) return;
    if (p.pos_q)
        pos_bias(p, b, s, pk, pstride);
    else
        index_bias(b, s, k0);
}

// S^T = K Q^T of KT x 32 keys and 32 rows (A = 32 keys, B = the wave's q), so that
// a lane holds 16 scores of one row and, as probabilities, the B operand of O^T += V^T P^T
// without a move. s: where it starts from.
template <class T, int DT, int KT>
__device__ __forceinline__ void seq_qk(const unsigned char* K, const u32x4 (&q)[SeqShape<T, DT>::KS], f32x16 (&s)[KT])
{
    using S = SeqShape<T, DT>;
    const int lane = threadIdx.x & 63, ql = lane & 31, h = lane >> 5;
    const int krow = ql * S::ROW, ksw = S::kswz(ql);
#pragma unroll
    for (int ks = 0; ks < S::KS; ++ks) {
        const int at = krow + (((2 * ks + h) ^ ksw) << 4);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            const u32x4 a = *(const u32x4*)(K + at + kt * 32 * S::ROW);
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[kt] = mfma32(__uint_as_float(a[e]), __uint_as_float(q[ks][e]), s[kt]);
            } else {
                s[kt] = mma16(a, q[ks], s[kt], T());
            }
        }
    }
}

// How far (log2) above 1 the largest probability is held: fp16 has 2^15 above and little
// below, where thousands of small ones may add up (100000 of 2^-24 of the largest).
template <class T>
struct SeqUp {
    static constexpr float value = 0.0f;
};
template <>
struct SeqUp<f16> {
    static constexpr float value = 6.0f;
};

// The mask and the running base, SeqUp below the largest score: it moves only when a score
// passes it by 2^8, so the sums are seldom rescaled; P stays below 2^(8 + SeqUp). rc: the
// rows' constants (seq_start).
template <class T, int DT, int KT, int MODE>
__device__ __forceinline__ void seq_max(const SeqAttnArgs& p, const unsigned* pk, int pstride, f32x16 (&s)[KT],
                                        const float (&rc)[KT], SeqAcc<T, DT>& c, const SeqBias& bias, int limit, int k0,
                                        bool masked)
{
    const int h = (threadIdx.x >> 5) & 1;
    const float a = p.cap * HAT_LOG2E;
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        f32x16& x = s[kt];
        if constexpr (MODE == SEQ_BOTH) seq_scores<T>(p, bias, x, k0 + 32 * kt, pk + 32 * kt, pstride);
        if constexpr (MODE == SEQ_CAP) {
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_rcpf(fast_exp2(x[r] * p.c1) + 1.0f);
        }
        if (masked) {
            const float out = MODE == SEQ_CAP ? INFINITY : -INFINITY;
            const int left = limit - k0 - 32 * kt - 4 * h;
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = 8 * (r >> 2) + (r & 3) < left ? x[r] : out;
        }
        float m = x[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) m = MODE == SEQ_CAP ? fminf(m, x[r]) : fmaxf(m, x[r]);
        if constexpr (MODE == SEQ_CAP) m = __builtin_fmaf(-2.0f * a, m, a);
        if constexpr (MODE == SEQ_BIAS) m += rc[kt];
        mx = fmaxf(mx, m);
    }
    mx = swap_max(mx);
    if constexpr (MODE == SEQ_PLAIN || MODE == SEQ_BIAS) mx *= p.c1;
    if (__any(mx > c.m + (8.0f + SeqUp<T>::value))) {
        const float mn = fmaxf(c.m, mx - SeqUp<T>::value), corr = fast_exp2(c.m - mn);
        c.m = mn;
        c.l *= corr;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) c.o[d][r] *= corr;
    }
}

// The probabilities 2^(s - m), in place (fp32) or packed for the product (16-bit types).
template <class T, int DT, int KT, int MODE>
__device__ __forceinline__ void seq_exp(const SeqAttnArgs& p, f32x16 (&s)[KT], const float (&rc)[KT], SeqAcc<T, DT>& c,
                                        u32x4 (&pb)[KT][2])
{
    const float a = p.cap * HAT_LOG2E;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const float f = MODE == SEQ_CAP ? -2.0f * a : p.c1;
        const float m = MODE == SEQ_CAP ? a - c.m : MODE == SEQ_BIAS ? __builtin_fmaf(rc[kt], p.c1, -c.m) : -c.m;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[kt][r] = fast_exp2(MODE == SEQ_BOTH ? s[kt][r] + m : __builtin_fmaf(s[kt][r], f, m));
            if constexpr (sizeof(T) == 4) c.l += s[kt][r];
        }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const unsigned w = pack16(s[kt][r], s[kt][r + 1], T());
                pb[kt][r >> 3][(r & 7) >> 1] = w;
                c.l = add_pair(w, c.l, T());
            }
        }
    }
}

// V's 16-bit operand of one MFMA: two transposed reads, four keys each, `step` bytes apart.
__device__ __forceinline__ u32x4 read_v(const unsigned char* at, int step)
{
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    const u2 a = __builtin_bit_cast(
        u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
    const u2 b = __builtin_bit_cast(
        u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + step)));
    return (u32x4){a[0], a[1], b[0], b[1]};
}

// O^T += V^T P^T. With MFMA's key order within 16 (lane half h, slot j: keys 4 h + j,
// then 8 + 4 h + j - 4) V's 16-bit operand is two transposed reads of four keys each.
template <class T, int DT, int KT>
__device__ __forceinline__ void seq_pv(const unsigned char* V, const f32x16 (&s)[KT], const u32x4 (&pb)[KT][2],
                                       SeqAcc<T, DT>& c)
{
    using S = SeqShape<T, DT>;
    const int lane = threadIdx.x & 63, ql = lane & 31, h = lane >> 5;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const unsigned char* row = V + (32 * kt + 8 * (r >> 2) + 4 * h + (r & 3)) * S::ROW + ql * 4;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const float a = *(const float*)(row + d * 128);
                    c.o[d] = mfma32(a, s[kt][r], c.o[d]);
                }
            }
    } else {
        const int x = lane & 15, kr = 4 * h + (x >> 2);
        const int row = kr * S::ROW + (x & 1) * 8;
        const int lc = 2 * ((lane >> 4) & 1) + ((x & 3) >> 1), vsw = S::vswz(kr);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const u32x4 a = read_v(V + row + ((lc + 4 * d) ^ vsw) * 16 + (32 * kt + 16 * st) * S::ROW, 8 * S::ROW);
                    c.o[d] = mma16(a, pb[kt][st], c.o[d], T());
                }
    }
}

// Whether a lane's row came out finite (l and every o).
template <class T, int DT>
__device__ __forceinline__ bool seq_finite(const SeqAcc<T, DT>& c)
{
    float z = c.l * 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) z = __builtin_fmaf(c.o[d][r], 0.0f, z);
    return z == 0.0f;
}

// The sequence of slot `at` where sequence s owns the slots from cu[s] * mul / per + s
// on: enough for ceil(length * mul / per) each, whatever the lengths, so the host needs
// only the totals. All lanes look at 64 sequences at a time; -1: none.
__device__ __forceinline__ int find_sequence(const int* cu, int n, int total, int mul, int per, int at, int& first)
{
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;  // the last s with slot(s) <= at lies in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64;
        const int s = lo + lane * step;
        bool ok = false;
        if (s < hi) ok = (long long)clamp_int(cu[s], 0, total) * mul / per + s <= at;
        const int c = __popcll(__ballot(ok));
        if (c == 0) return -1;
        lo += (c - 1) * step;
        if (lo + step < hi) hi = lo + step;
    }
    first = (int)((long long)clamp_int(cu[lo], 0, total) * mul / per) + lo;
    return first <= at ? lo : -1;
}

__device__ __forceinline__ SeqView uniform(const SeqView& v)
{
    SeqView w;
    w.s = __builtin_amdgcn_readfirstlane(v.s);
    w.lq = __builtin_amdgcn_readfirstlane(v.lq);
    w.lk = __builtin_amdgcn_readfirstlane(v.lk);
    w.q0 = __builtin_amdgcn_readfirstlane(v.q0);
    w.k0 = __builtin_amdgcn_readfirstlane(v.k0);
    w.bq = v.bq ? w.s : 0;
    w.bk = v.bk ? w.s : 0;
    return w;
}

// A block's tile of 128 rows, and its waves' shares: 32 rows each.
struct SeqTile {
    SeqView v;
    int kvh, rows, prefix;
    int row0;         // the wave's first row
    int end;          // the block's keys
    int least, most;  // the least and the largest limit of the wave's rows (limits rise with the row)
    int at0, at1;     // i + Lk - Lq of its first and last row
};

__device__ __forceinline__ bool seq_tile(const SeqAttnArgs& p, SeqTile& w)
{
    constexpr int BQ = 128;
    const int pairs = p.cu_q ? p.kv_heads : p.kv_heads * p.n_seq;
    const int pair = blockIdx.x % pairs;
    int tile = blockIdx.x / pairs, sq;
    if (p.cu_q) {
        int first = 0;
        w.kvh = pair;
        sq = find_sequence(p.cu_q, p.n_seq, p.q_tokens, p.group, BQ, tile, first);
        if (sq < 0) return false;
        tile -= first;
    } else {
        sq = pair / p.kv_heads;
        w.kvh = pair - sq * p.kv_heads;
    }
    const SeqView v = w.v = uniform(seq_view(p, __builtin_amdgcn_readfirstlane(sq)));
    tile = __builtin_amdgcn_readfirstlane(tile);
    w.rows = v.lq * p.group;
    const int tiles = (w.rows + BQ - 1) / BQ;
    if (tile >= tiles) return false;
    // Under the causal mask a tile's work grows with its number: the longest first, and
    // where all blocks run at once (p.fold) the second half from the shortest on, so that
    // the CUs, which take blocks in turn, get a long and a short one each.
    if (p.causal) {
        const int half = (tiles + 1) / 2;
        tile = p.fold && tile >= half ? tile - half : tiles - 1 - tile;
    }
    w.prefix = p.prefix ? __builtin_amdgcn_readfirstlane(p.prefix[v.s]) : 0;
    w.row0 = tile * BQ + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 32;
    const int block_last = tile * BQ + BQ - 1 < w.rows ? tile * BQ + BQ - 1 : w.rows - 1;
    w.end = row_limit(p, v, block_last / p.group, w.prefix);
    w.least = 0x7fffffff, w.most = 0;
    if (w.row0 < w.rows) {
        w.least = row_limit(p, v, w.row0 / p.group, w.prefix);
        const int last = w.row0 + 31 < w.rows ? w.row0 + 31 : w.rows - 1;
        w.most = row_limit(p, v, last / p.group, w.prefix);
    }
    w.at0 = w.row0 / p.group + v.lk - v.lq, w.at1 = (w.row0 + 31) / p.group + v.lk - v.lq;
    return true;
}

// The 32 rows from row0 written out.
template <class T, int DT>
__device__ __forceinline__ void seq_finish(const SeqAttnArgs& p, const SeqTile& w, const SeqRow& row, int row0,
                                           SeqAcc<T, DT>& c)
{
    const SeqView& v = w.v;
    const int lane = threadIdx.x & 63;
    c.l = swap_sum(c.l);
    // A probability of 0 does not keep out a NaN or an infinity of an unseen key in
    // a tile that holds seen ones: such rows are done again, key by key.
    const bool bad = row.live && !seq_finite(c);
    T* o = (T*)p.o + v.bq * p.ob + (long long)(v.q0 + row.i) * p.ot + row.head * p.oh;
    const unsigned long long all = __ballot(bad);
    unsigned redo = (unsigned)(all | all >> 32);
    const bool mine = (redo >> (lane & 31)) & 1;
    if (row.live && !mine) {
        const float inv = join_scale(c.l);
        const int h = lane >> 5;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at = 32 * d + 8 * g + 4 * h;
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = c.o[d][4 * g + e] * inv;
                if (p.wide_out) {
                    if (at < p.dim) store_vec<T, 4>(o + at, f);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at + e < p.dim) o[at + e] = (T)f[e];
                }
            }
    }
    while (redo) {
        const int x = __builtin_ctz(redo);
        redo &= redo - 1;
        const SeqRow r = seq_row(p, row0 + x, w.rows, w.kvh);
        float m, l, oa, oc;
        attn_row<T>(p, v, r.i, r.head, 0, row_limit(p, v, r.i, w.prefix), m, l, oa, oc);
        T* ro = (T*)p.o + v.bq * p.ob + (long long)(v.q0 + r.i) * p.ot + r.head * p.oh;
        if (lane < p.dim) ro[lane] = (T)(oa * join_scale(l));
        if (lane + 64 < p.dim) ro[lane + 64] = (T)(oc * join_scale(l));
    }
}

// ---- many rows: a block of four waves, 32 rows each, walks the keys in stages of
// KT x 32, two in LDS: the next one's copy runs under the present one's products.
template <class T, int DT, int KT, int MODE>
__device__ __forceinline__ void seq_body(const SeqAttnArgs& p, unsigned char* K0, unsigned char* K1, unsigned char* V0,
                                         unsigned char* V1, unsigned* P0, unsigned* P1)
{
    constexpr int BK = 32 * KT;
    SeqTile w;
    if (!seq_tile(p, w)) return;
    const SeqView& v = w.v;
    const int tid = threadIdx.x, lane = tid & 63;
    const SeqRow row = seq_row(p, w.row0 + (lane & 31), w.rows, w.kvh);
    const int limit = row.live ? row_limit(p, v, row.i, w.prefix) : 0x7fffffff;
    u32x4 q[SeqShape<T, DT>::KS];
    load_q<T, DT>(p, v, row, q);
    SeqBias bias;
    if constexpr (MODE == SEQ_BIAS || MODE == SEQ_BOTH) bias = seq_bias(p, v, row, MODE == SEQ_BIAS);
    SeqAcc<T, DT> acc;
    acc.init();

    Stage<T, DT, BK, 256, false> sk;
    Stage<T, DT, BK, 256, true> sv;
    sk.init((const T*)p.k + v.bk * p.kb + (long long)v.k0 * p.kt + w.kvh * p.kh, p.kt, v.lk, p.dim, tid);
    sv.init((const T*)p.v + v.bk * p.vb + (long long)v.k0 * p.vt + w.kvh * p.vh, p.vt, v.lk, p.dim, tid);
    const int* pos_k = p.pos_k + v.bk * p.pkb + (long long)v.k0 * p.pkt;
    const auto stage = [&](const unsigned char* K, const unsigned char* V, const unsigned* P, int k0) {
        if (k0 >= w.most) return;
        f32x16 s[KT];
        float rc[KT];
        u32x4 pb[KT][2];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
            rc[kt] = seq_start<MODE>(p, bias, s[kt], k0 + 32 * kt, P + 32 * kt, BK, w.at0, w.at1);
        seq_qk<T, DT, KT>(K, q, s);
        seq_max<T, DT, KT, MODE>(p, P, BK, s, rc, acc, bias, limit, k0, k0 + BK > w.least);
        seq_exp<T, DT, KT, MODE>(p, s, rc, acc, pb);
        seq_pv<T, DT, KT>(V, s, pb, acc);
    };
    // The positions of a stage's keys, one a thread: read with the stage's copies, put into
    // LDS behind the present stage's products.
    const bool has_pos = (MODE == SEQ_BIAS || MODE == SEQ_BOTH) && p.pos_q && tid < p.axes * BK;
    unsigned pos = 0;
    const auto issue = [&](unsigned char* K, unsigned char* V, int k0) {
        if (has_pos && k0 + tid % BK < v.lk)
            pos = (unsigned)pos_k[(long long)(k0 + tid % BK) * p.pkt + tid / BK * p.pka] ^ 0x80000000u;
        sk.issue(K, k0, tid, p.wide);
        sv.issue(V, k0, tid, p.wide);
    };
    const auto put_pos = [&](unsigned* P) {
        if (has_pos) P[tid] = pos;
    };
    if (w.end > 0) {
        issue(K0, V0, 0);
        put_pos(P0);
        __syncthreads();
        for (int k0 = 0; k0 < w.end; k0 += 2 * BK) {
            issue(K1, V1, k0 + BK);  // past the last key: zeros
            stage(K0, V0, P0, k0);
            put_pos(P1);
            __syncthreads();
            if (k0 + BK >= w.end) break;
            issue(K0, V0, k0 + 2 * BK);
            stage(K1, V1, P1, k0 + BK);
            put_pos(P0);
            __syncthreads();
        }
    }
    seq_finish<T, DT>(p, w, row, w.row0, acc);
}

// ---- fp32 with many rows: the same walk on the BF16 matrix path at fp32 accuracy. Every
// operand enters as three bf16 parts and a product as the six terms of order <= 2 (common.h),
// 192 cycles of MFMA for 32 x 32 x 16 where FP32 MFMA takes 512. bf16 keeps fp32's range,
// so no operand needs a scale (two f16 parts would need one: k and v have no bound here).
// K and V go through registers, where a block splits them once for its four waves. On FP32
// MFMA -> here, 4 x 2048 x 2048: 8 heads of 128 550 -> 340-357 us, of 64 288 -> 201; 256
// windows of 256 tokens, 6 heads of 24, bias over two axes: 153 -> 110-123. What is left at 24
// dims is vector work: 13 instructions a score, 5.5 of them the probabilities' split.
template <int DT, int KT>
struct Seq32Shape {
    using S = SeqShape<bf16, DT>;
    static constexpr int BK = 32 * KT;
    static constexpr int PLANE = BK * S::ROW;          // bytes of one part of K or V
    static constexpr int CHUNKS = BK * S::CH;          // eight elements each
    static constexpr int N = (CHUNKS + 255) / 256;     // a thread's
};

// A thread's chunks of a stage's K or V rows, in fp32.
template <int DT, int KT, bool V>
struct Stage32 {
    using X = Seq32Shape<DT, KT>;
    using S = SeqShape<bf16, DT>;
    const float* base;
    long long stride;
    int n, dim;
    unsigned off[X::N][2];
    f32x4 u[X::N][2];
    __device__ __forceinline__ int row_of(int c) const { return c / S::CH; }
    __device__ __forceinline__ int dim_of(int c) const
    {
        return ((c % S::CH) ^ (V ? S::vswz(row_of(c)) : S::kswz(row_of(c)))) * 8;
    }
    __device__ __forceinline__ void init(const float* b, long long st, int rows, int d, int tid)
    {
        base = b, stride = st, n = rows, dim = d;
#pragma unroll
        for (int j = 0; j < X::N; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int c = j * 256 + tid, at = dim_of(c) + 4 * x;
                off[j][x] = c < X::CHUNKS && at < dim ? (unsigned)(row_of(c) * (int)stride + at) * 4 : 0x80000000u;
            }
    }
    __device__ __forceinline__ void load(int first, int tid, int wide)
    {
        const int left = n - first;
        const int rows = left < X::BK ? left : X::BK;
        const auto rsrc =
            buffer_of(base + (long long)first * stride, rows <= 0 ? 0 : ((rows - 1) * (int)stride + dim) * 4);
#pragma unroll
        for (int j = 0; j < X::N; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (wide == 2) {
                    u[j][x] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off[j][x], 0, 0));
                } else {
                    const int c = j * 256 + tid, d0 = dim_of(c) + 4 * x;
                    u[j][x] = __builtin_bit_cast(
                        f32x4, load_chunk<float>(rsrc, row_of(c) * (int)stride + d0, c < X::CHUNKS ? dim - d0 : 0, 1));
                }
            }
    }
    __device__ __forceinline__ void put(unsigned char* planes, int tid) const
    {
#pragma unroll
        for (int j = 0; j < X::N; ++j) {
            const int c = j * 256 + tid;
            if (X::CHUNKS % 256 && c >= X::CHUNKS) break;
            const float v[8] = {u[j][0][0], u[j][0][1], u[j][0][2], u[j][0][3], u[j][1][0], u[j][1][1], u[j][1][2], u[j][1][3]};
            u32x4 w[3];
            split3_x8(v, w);
#pragma unroll
            for (int pl = 0; pl < 3; ++pl) *(u32x4*)(planes + pl * X::PLANE + c * 16) = w[pl];
        }
    }
};

__device__ __forceinline__ f32x16 mfma6(const u32x4 (&a)[3], const u32x4 (&b)[3], f32x16 c)
{
    c = mma16(a[2], b[0], c, bf16());
    c = mma16(a[1], b[1], c, bf16());
    c = mma16(a[0], b[2], c, bf16());
    c = mma16(a[1], b[0], c, bf16());
    c = mma16(a[0], b[1], c, bf16());
    return mma16(a[0], b[0], c, bf16());
}

template <int DT, int KT, int MODE>
__device__ __forceinline__ void seq32_body(const SeqAttnArgs& p, unsigned char* Kp, unsigned char* Vp, unsigned* P)
{
    using X = Seq32Shape<DT, KT>;
    using S = SeqShape<bf16, DT>;
    SeqTile w;
    if (!seq_tile(p, w)) return;
    const SeqView& v = w.v;
    const int tid = threadIdx.x, lane = tid & 63, ql = lane & 31, h = lane >> 5;
    const SeqRow row = seq_row(p, w.row0 + ql, w.rows, w.kvh);
    u32x4 q[S::KS][3];
    load_q32<DT>(p, v, row, q);
    SeqAcc<float, DT> acc;
    acc.init();
    SeqBias bias;
    if constexpr (MODE != SEQ_PLAIN) bias = seq_bias(p, v, row, MODE == SEQ_BIAS);
    const int limit = row.live ? row_limit(p, v, row.i, w.prefix) : 0x7fffffff;
    Stage32<DT, KT, false> sk;
    Stage32<DT, KT, true> sv;
    sk.init((const float*)p.k + v.bk * p.kb + (long long)v.k0 * p.kt + w.kvh * p.kh, p.kt, v.lk, p.dim, tid);
    sv.init((const float*)p.v + v.bk * p.vb + (long long)v.k0 * p.vt + w.kvh * p.vh, p.vt, v.lk, p.dim, tid);
    const int* pos_k = p.pos_k + v.bk * p.pkb + (long long)v.k0 * p.pkt;
    const bool has_pos = MODE != SEQ_PLAIN && p.pos_q && tid < p.axes * X::BK;
    unsigned pos = 0;
    const auto load = [&](int k0) {
        if (has_pos && k0 + tid % X::BK < v.lk)
            pos = (unsigned)pos_k[(long long)(k0 + tid % X::BK) * p.pkt + tid / X::BK * p.pka] ^ 0x80000000u;
        sk.load(k0, tid, p.wide);
        sv.load(k0, tid, p.wide);
    };
    if (w.end > 0) load(0);
    for (int k0 = 0; k0 < w.end; k0 += X::BK) {
        sk.put(Kp, tid);
        sv.put(Vp, tid);
        if (has_pos) P[tid] = pos;
        __syncthreads();
        load(k0 + X::BK);  // past the last key: zeros
        if (k0 < w.most) {
            f32x16 s[KT];
            float rc[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
                rc[kt] = seq_start<MODE>(p, bias, s[kt], k0 + 32 * kt, P + 32 * kt, X::BK, w.at0, w.at1);
#pragma unroll
            for (int ks = 0; ks < S::KS; ++ks) {
                const int at = ql * S::ROW + (((2 * ks + h) ^ S::kswz(ql)) << 4);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    u32x4 a[3];
#pragma unroll
                    for (int pl = 0; pl < 3; ++pl) a[pl] = *(const u32x4*)(Kp + pl * X::PLANE + at + kt * 32 * S::ROW);
                    s[kt] = mfma6(a, q[ks], s[kt]);
                }
            }
            seq_max<float, DT, KT, MODE>(p, P, X::BK, s, rc, acc, bias, limit, k0, k0 + X::BK > w.least);
            u32x4 none[KT][2];
            seq_exp<float, DT, KT, MODE>(p, s, rc, acc, none);
            const int x = lane & 15, kr = 4 * h + (x >> 2);
            const int vrow = kr * S::ROW + (x & 1) * 8;
            const int lc = 2 * ((lane >> 4) & 1) + ((x & 3) >> 1), vsw = S::vswz(kr);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    float f[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = s[kt][8 * st + j];
                    u32x4 b[3];
                    split3_x8(f, b);
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        u32x4 a[3];
#pragma unroll
                        for (int pl = 0; pl < 3; ++pl)
                            a[pl] = read_v(Vp + pl * X::PLANE + vrow + ((lc + 4 * d) ^ vsw) * 16 + (32 * kt + 16 * st) * S::ROW,
                                           8 * S::ROW);
                        acc.o[d] = mfma6(a, b, acc.o[d]);
                    }
                }
        }
        __syncthreads();  // the stage has been read
    }
    seq_finish<float, DT>(p, w, row, w.row0, acc);
}

// ---- few rows a sequence (a token each, say) against many keys: the keys go over blocks
// in chunks and over a block's W waves in tiles of 32, each wave with LDS and a pipeline of
// its own; the waves' sums are joined in LDS, the chunks' by hat_attnseq_join.
template <class T, int DT, int W>
struct SplitShape {
    static constexpr int TILE = 32 * SeqShape<T, DT>::ROW;  // a wave's stage of K or V
    static constexpr int XROW = 36;                         // floats of a joined row's 32 dims
    static constexpr int BYTES = W * TILE > W * 32 * XROW * 4 ? W * TILE : W * 32 * XROW * 4;
};

// Partial results of a (chunk slot, key head): rows of dim values, rows of (m, l).
__device__ __forceinline__ long long part_row(const SeqAttnArgs& p, int slot, int kvh, int r)
{
    return ((long long)slot * p.kv_heads + kvh) * ((long long)p.q_tokens * p.group) + r;
}

// A block's part of the split form: a tile of TILE rows and a chunk of keys.
struct SplitTile {
    SeqView v;
    int kvh, slot, rows, prefix;
    int row0;
    int c0, c1;       // the chunk's keys, cut at the last row's limit
    int least;        // the first row's limit
};

template <int TILE>
__device__ __forceinline__ bool split_tile(const SeqAttnArgs& p, SplitTile& w)
{
    int tile, sq, chunk = 0, first = 0;
    w.slot = 0;
    if (p.cu_q) {  // b = tile slot * kv_heads + kvh, all keys in one chunk
        w.kvh = blockIdx.x % p.kv_heads;
        tile = blockIdx.x / p.kv_heads;
        sq = find_sequence(p.cu_q, p.n_seq, p.q_tokens, p.group, TILE, tile, first);
        if (sq < 0) return false;
        tile = __builtin_amdgcn_readfirstlane(tile - first);
    } else {  // b = (chunk slot * kv_heads + kvh) * tiles + tile
        tile = blockIdx.x % p.tiles;
        w.kvh = blockIdx.x / p.tiles % p.kv_heads;
        w.slot = blockIdx.x / p.tiles / p.kv_heads;
        if (p.cu_k) {
            sq = find_sequence(p.cu_k, p.n_seq, p.k_tokens, 1, p.chunk, w.slot, first);
            if (sq < 0) return false;
            chunk = w.slot - first;
        } else {
            sq = w.slot / p.slots;
            chunk = w.slot - sq * p.slots;
        }
    }
    const SeqView v = w.v = uniform(seq_view(p, __builtin_amdgcn_readfirstlane(sq)));
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    w.rows = v.lq * p.group;
    w.row0 = tile * TILE;
    if (w.row0 >= w.rows) return false;
    w.prefix = p.prefix ? __builtin_amdgcn_readfirstlane(p.prefix[v.s]) : 0;
    const int last = w.row0 + TILE - 1 < w.rows ? w.row0 + TILE - 1 : w.rows - 1;
    w.least = row_limit(p, v, w.row0 / p.group, w.prefix);
    const int end = row_limit(p, v, last / p.group, w.prefix);
    w.c0 = chunk * p.chunk;
    if (w.c0 >= end && chunk > 0) return false;  // no row's join asks for it; chunk 0 writes the empty rows
    w.c1 = end - w.c0 < p.chunk ? end : w.c0 + p.chunk;
    return true;
}

// A row of the chunk done again key by key (as in seq_finish), by one wave.
template <class T>
__device__ __forceinline__ void split_again(const SeqAttnArgs& p, const SplitTile& w, int r)
{
    const SeqView& v = w.v;
    const int lane = threadIdx.x & 63;
    const SeqRow sr = seq_row(p, w.row0 + r, w.rows, w.kvh);
    int to = row_limit(p, v, sr.i, w.prefix);
    to = to < w.c1 ? to : w.c1;
    float m, l, oa, oc;
    attn_row<T>(p, v, sr.i, sr.head, w.c0, to, m, l, oa, oc);
    if (!p.part) {
        T* out = (T*)p.o + v.bq * p.ob + (long long)(v.q0 + sr.i) * p.ot + sr.head * p.oh;
        if (lane < p.dim) out[lane] = (T)(oa * join_scale(l));
        if (lane + 64 < p.dim) out[lane + 64] = (T)(oc * join_scale(l));
    } else {
        const long long pr = part_row(p, w.slot, w.kvh, w.row0 + r);
        if (lane < p.dim) p.part[pr * p.dim + lane] = oa;
        if (lane + 64 < p.dim) p.part[pr * p.dim + lane + 64] = oc;
        if (lane == 0) p.part_ml[2 * pr] = m == -INFINITY ? -1e30f : m, p.part_ml[2 * pr + 1] = l;
    }
}

// WIDE: rows in 16-byte moves. Both ways in one loop make the copies in flight depend on
// the path, and the compiler waits for all of them (1023 keys, 2 heads of 64: 11.7 us
// against 10.3).
template <class T, int DT, int W, bool WIDE>
__device__ __forceinline__ void seq_split_body(const SeqAttnArgs& p, unsigned char* B0, unsigned char* B1,
                                               unsigned char* B2, unsigned char* B3, unsigned* P0, unsigned* P1,
                                               float* ml, unsigned* flags)
{
    using X = SplitShape<T, DT, W>;
    constexpr int DP = 32 * DT;
    SplitTile w;
    if (!split_tile<32>(p, w)) return;
    const SeqView& v = w.v;
    const int kvh = w.kvh, slot = w.slot, rows = w.rows, row0 = w.row0, c0 = w.c0, c1 = w.c1, least = w.least,
              prefix = w.prefix;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    u32x4 q[SeqShape<T, DT>::KS];
    const SeqRow row = seq_row(p, row0 + (lane & 31), rows, kvh);
    load_q<T, DT>(p, v, row, q);
    int limit = row.live ? row_limit(p, v, row.i, prefix) : 0x7fffffff;
    limit = limit < c1 ? limit : c1;  // keys behind the chunk lie in another
    const SeqBias bias = seq_bias(p, v, row, false);
    SeqAcc<T, DT> c;
    c.init();

    Stage<T, DT, 32, 64, false> sk;
    Stage<T, DT, 32, 64, true> sv;
    sk.init((const T*)p.k + v.bk * p.kb + (long long)v.k0 * p.kt + kvh * p.kh, p.kt, c1, p.dim, lane);
    sv.init((const T*)p.v + v.bk * p.vb + (long long)v.k0 * p.vt + kvh * p.vh, p.vt, c1, p.dim, lane);
    const int* pos_k = p.pos_k + v.bk * p.pkb + (long long)v.k0 * p.pkt;
    const int lds = wave * X::TILE;
    constexpr int MOVES = 2 * Stage<T, DT, 32, 64, false>::N;
    const auto issue = [&](unsigned char* K, unsigned char* V, int k0) {
        if (!WIDE && k0 >= c1) return;  // nothing to wait for by count
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this buffer's reads are done
        sk.issue(K + lds, k0, lane, WIDE ? 2 : p.wide & 1);
        sv.issue(V + lds, k0, lane, WIDE ? 2 : p.wide & 1);
    };
    // The positions of a tile's keys, two axes a register: read with the tile's copies, put
    // into LDS when the tile's turn comes.
    unsigned pos[2] = {0, 0};
    const auto read_pos = [&](int k0) {
        const int j = k0 + (lane & 31);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int a = 2 * x + (lane >> 5);
            if (p.pos_q && a < p.axes && j < c1) pos[x] = (unsigned)pos_k[(long long)j * p.pkt + a * p.pka] ^ 0x80000000u;
        }
    };
    const auto put_pos = [&](unsigned* P) {
        if (!p.pos_q) return;
        P[wave * 128 + lane] = pos[0];
        P[wave * 128 + 64 + lane] = pos[1];
    };
    const auto stage = [&](const unsigned char* K, const unsigned char* V, const unsigned* P, int k0) {
        // the other buffer's moves may still be under way
        if (WIDE) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MOVES) : "memory");
        f32x16 s[1];
        const float rc[1] = {0.0f};
        u32x4 pb[1][2];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[0][r] = 0.0f;
        seq_qk<T, DT, 1>(K + lds, q, s);
        seq_max<T, DT, 1, SEQ_BOTH>(p, P + wave * 128, 32, s, rc, c, bias, limit, k0, k0 + 32 > least || k0 + 32 > c1);
        seq_exp<T, DT, 1, SEQ_BOTH>(p, s, rc, c, pb);
        seq_pv<T, DT, 1>(V + lds, s, pb, c);
    };
    int k0 = c0 + 32 * wave;
    read_pos(k0);
    issue(B0, B2, k0);
    while (k0 < c1) {
        put_pos(P0);
        read_pos(k0 + 32 * W);
        issue(B1, B3, k0 + 32 * W);
        stage(B0, B2, P0, k0);
        k0 += 32 * W;
        if (k0 >= c1) break;
        put_pos(P1);
        read_pos(k0 + 32 * W);
        issue(B0, B2, k0 + 32 * W);
        stage(B1, B3, P1, k0);
        k0 += 32 * W;
    }

    // the waves' sums side by side: 32 dims of each row in a buffer
    c.l = swap_sum(c.l);
    if (tid == 0) *flags = 0;
    __syncthreads();  // every wave is through its stages, and its moves have arrived
    const int h = lane >> 5, ql = lane & 31;
    unsigned char* buf[4] = {B0, B1, B2, B3};
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *(f32x4*)((float*)buf[d] + (wave * 32 + ql) * X::XROW + 8 * g + 4 * h) =
                (f32x4){c.o[d][4 * g], c.o[d][4 * g + 1], c.o[d][4 * g + 2], c.o[d][4 * g + 3]};
    if (h == 0) ml[(wave * 32 + ql) * 2] = c.m, ml[(wave * 32 + ql) * 2 + 1] = c.l;
    __syncthreads();
    constexpr int N = 32 * DP / (64 * W);  // values a thread: one dim of every (64 W / 32)th row
    const int x = tid & 31;
    float o[N], m[N / DT], l[N / DT];
#pragma unroll
    for (int n = 0; n < N / DT; ++n) {
        const int r = (tid >> 5) + n * 2 * W;
        m[n] = ml[r * 2];
#pragma unroll
        for (int w = 1; w < W; ++w) m[n] = fmaxf(m[n], ml[(w * 32 + r) * 2]);
        l[n] = 0.0f;
        float f[W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            f[w] = fast_exp2(ml[(w * 32 + r) * 2] - m[n]);
            l[n] += f[w] * ml[(w * 32 + r) * 2 + 1];
        }
        float z = l[n] * 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) sum = __builtin_fmaf(f[w], ((const float*)buf[d])[(w * 32 + r) * X::XROW + x], sum);
            o[n * DT + d] = sum;
            z = __builtin_fmaf(sum, 0.0f, z);
        }
        if (row0 + r < rows && !(z == 0.0f)) atomicOr(flags, 1u << r);
    }
    __syncthreads();
    const unsigned bad = *flags;  // rows to do again key by key, as in seq_body
    const bool whole = p.part == nullptr;
#pragma unroll
    for (int n = 0; n < N / DT; ++n) {
        const int r = (tid >> 5) + n * 2 * W;
        if (row0 + r >= rows || ((bad >> r) & 1)) continue;
        const SeqRow sr = seq_row(p, row0 + r, rows, kvh);
        T* out = (T*)p.o + v.bq * p.ob + (long long)(v.q0 + sr.i) * p.ot + sr.head * p.oh;
        const long long pr = part_row(p, slot, kvh, row0 + r);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int at = 32 * d + x;
            if (at < p.dim) {
                if (whole)
                    out[at] = (T)(o[n * DT + d] * join_scale(l[n]));
                else
                    p.part[pr * p.dim + at] = o[n * DT + d];
            }
        }
        if (!whole && x == 0) p.part_ml[2 * pr] = m[n], p.part_ml[2 * pr + 1] = l[n];
    }
    for (int r = wave; r < 32; r += W)
        if ((bad >> r) & 1) split_again<T>(p, w, r);
}

// ---- fp32 with at most a few rows a sequence: four rows at a time on the 4 x 4 x 1 matrix
// instruction, sixteen of them side by side. The tiles of 32 rows above spend 8192 cycles of
// FP32 MFMA on 32 keys of 128 dims whatever the rows; this takes 2048 on 64. A wave has 64
// keys, a lane one: K goes through LDS to the lane that owns the key (read straight from
// memory the rows' lines were fetched eight times over: 31 us for 3 sequences of 6819 keys, 4
// heads of 128), V comes with a dim a lane.
//   scores: A = q, four rows, one block of lanes for each of 16 dims, picked and broadcast to
//           the other blocks by the instruction (cbsz, abid); B = K, a dim of every lane's key.
//   output: A = P, transposed within each four lanes so that block b holds keys 4 b .. + 3,
//           picked the same way; B = V, a key's dims over the lanes.
// It is then as fast as K and V arrive.
template <int ABID>
__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_4x4x1f32(a, b, c, 4, ABID, 0);
}

template <int X>
__device__ __forceinline__ float quad_xor(float v)  // the lane's neighbour at lane ^ X within four
{
    constexpr int perm = X == 1 ? 0xb1 : X == 2 ? 0x4e : 0x1b;
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), perm, 0xf, 0xf, true));
}

// t[i] of lane j of four <- t[j] of lane i: two rounds of swaps with the neighbours.
__device__ __forceinline__ void quad_transpose(float (&t)[4])
{
    const int j = threadIdx.x & 3;
    {
        const float a = j & 1 ? t[0] : t[1], c = j & 1 ? t[2] : t[3];
        const float x = quad_xor<1>(a), y = quad_xor<1>(c);
        t[0] = j & 1 ? x : t[0], t[1] = j & 1 ? t[1] : x;
        t[2] = j & 1 ? y : t[2], t[3] = j & 1 ? t[3] : y;
    }
    const float a = j & 2 ? t[0] : t[2], c = j & 2 ? t[1] : t[3];
    const float x = quad_xor<2>(a), y = quad_xor<2>(c);
    t[0] = j & 2 ? x : t[0], t[2] = j & 2 ? t[2] : x;
    t[1] = j & 2 ? y : t[1], t[3] = j & 2 ? t[3] : y;
}

template <int DT, int W>
__device__ __forceinline__ void seq_few_body(const SeqAttnArgs& p, unsigned char* K, float* xo, float* ml)
{
    constexpr int DP = 32 * DT, SETS = (DP + 63) / 64;  // of 64 dims
    SplitTile w;
    if (!split_tile<4>(p, w)) return;
    const SeqView& v = w.v;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c1 = w.c1;

    float q[2 * DT];  // lane 4 b + i: row i, dim 16 j + b
    {
        const SeqRow r = seq_row(p, w.row0 + (lane & 3), w.rows, w.kvh);
        const float* row = row_of<float>(p, v, r);
        const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) {
            const int d = 16 * j + (lane >> 2);
            q[j] = r.live && d < p.dim ? row[d] * sign : 0.0f;
        }
    }
    int limit[4];
    float slope[4], m[4], l[4];
    unsigned pq[4][4];
    int at[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const SeqRow sr = seq_row(p, w.row0 + r, w.rows, w.kvh);
        limit[r] = sr.live ? row_limit(p, v, sr.i, w.prefix) : 0;
        limit[r] = limit[r] < c1 ? limit[r] : c1;
        const SeqBias b = seq_bias(p, v, sr, false);
        slope[r] = b.slope, at[r] = b.at;
#pragma unroll
        for (int a = 0; a < 4; ++a) pq[r][a] = b.pos[a];
        m[r] = -1e30f, l[r] = 0.0f;
    }
    f32x4 o[SETS];
#pragma unroll
    for (int s = 0; s < SETS; ++s) o[s] = (f32x4){0.f, 0.f, 0.f, 0.f};

    const float* kb = (const float*)p.k + v.bk * p.kb + (long long)v.k0 * p.kt + w.kvh * p.kh;
    const float* vb = (const float*)p.v + v.bk * p.vb + (long long)v.k0 * p.vt + w.kvh * p.vh;
    const int* pos_k = p.pos_k + v.bk * p.pkb + (long long)v.k0 * p.pkt;
    const auto rows_of = [&](const float* b, long long stride, int k0) {
        const int rows = c1 - k0 < 64 ? c1 - k0 : 64;
        return buffer_of(b + (long long)k0 * stride, rows <= 0 ? 0 : ((rows - 1) * (int)stride + p.dim) * 4);
    };
    using S = SeqShape<float, DT>;
    unsigned char* kl = K + wave * 64 * S::ROW;
    Stage<float, DT, 64, 64, false> sk;
    sk.init(kb, p.kt, c1, p.dim, lane);
    int k0 = w.c0 + 64 * wave;
    if (k0 < c1) sk.issue(kl, k0, lane, p.wide);
    for (; k0 < c1; k0 += 64 * W) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // K has arrived
        float vv[64][SETS];
        const auto rv = rows_of(vb, p.vt, k0);
#pragma unroll
        for (int j = 0; j < 64; ++j)
#pragma unroll
            for (int s = 0; s < SETS; ++s)
                vv[j][s] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                    rv, lane + 64 * s < p.dim ? (lane + 64 * s) * 4 : 0x80000000u, j * (int)p.vt * 4, 0));
        f32x4 k[S::CH];
#pragma unroll
        for (int j = 0; j < S::CH; ++j) k[j] = *(const f32x4*)(kl + lane * S::ROW + ((j ^ S::kswz(lane)) << 4));
        const int key = k0 + lane;
        unsigned pk[4] = {0, 0, 0, 0};
        if (p.pos_q) {
#pragma unroll
            for (int a = 0; a < 4; ++a)
                if (a < p.axes && key < c1) pk[a] = (unsigned)pos_k[(long long)key * p.pkt + a * p.pka] ^ 0x80000000u;
        }
        f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;  // two chains
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) {
#define FEW_QK(B, S) S = mfma4<B>(q[j], k[4 * j + B / 4][B % 4], S);
            FEW_QK(0, s0) FEW_QK(1, s1) FEW_QK(2, s0) FEW_QK(3, s1) FEW_QK(4, s0) FEW_QK(5, s1) FEW_QK(6, s0) FEW_QK(7, s1)
            FEW_QK(8, s0) FEW_QK(9, s1) FEW_QK(10, s0) FEW_QK(11, s1) FEW_QK(12, s0) FEW_QK(13, s1) FEW_QK(14, s0) FEW_QK(15, s1)
#undef FEW_QK
        }
        if (k0 + 64 * W < c1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K has been read
            sk.issue(kl, k0 + 64 * W, lane, p.wide);
        }
        float t[4];
        bool need = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float x = s0[r] + s1[r];
            if (p.cap > 0.0f)
                x = p.cap * HAT_LOG2E * tanhf(x * fabsf(p.scale) * p.inv_cap);
            else
                x *= p.c1;
            if (p.slopes) {
                float far = fabsf((float)(at[r] - key));
                if (p.pos_q) {
                    unsigned u = 0;
#pragma unroll
                    for (int a = 0; a < 4; ++a) u = a < p.axes ? sad(pq[r][a], pk[a], u) : u;
                    far = (float)u;
                }
                x = __builtin_fmaf(-slope[r], far, x);
            }
            t[r] = key < limit[r] ? x : -INFINITY;
            need |= t[r] > m[r] + 8.0f;
        }
        if (__any(need)) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float mn = fmaxf(m[r], wave_max(t[r])), corr = fast_exp2(m[r] - mn);
                m[r] = mn;
                l[r] *= corr;
#pragma unroll
                for (int s = 0; s < SETS; ++s) o[s][r] *= corr;
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            t[r] = fast_exp2(t[r] - m[r]);
            l[r] += t[r];
        }
        quad_transpose(t);  // t[i] of lane 4 b + j: row j, key 4 b + i
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
#define FEW_PV(B)                                                                                            \
    o[s] = mfma4<B>(t[0], vv[4 * B][s], o[s]), o[s] = mfma4<B>(t[1], vv[4 * B + 1][s], o[s]),                \
    o[s] = mfma4<B>(t[2], vv[4 * B + 2][s], o[s]), o[s] = mfma4<B>(t[3], vv[4 * B + 3][s], o[s]);
            FEW_PV(0) FEW_PV(1) FEW_PV(2) FEW_PV(3) FEW_PV(4) FEW_PV(5) FEW_PV(6) FEW_PV(7)
            FEW_PV(8) FEW_PV(9) FEW_PV(10) FEW_PV(11) FEW_PV(12) FEW_PV(13) FEW_PV(14) FEW_PV(15)
#undef FEW_PV
        }
    }

    // the waves' sums side by side
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        l[r] = wave_sum(l[r]);
        if (lane == 0) ml[(wave * 4 + r) * 2] = m[r], ml[(wave * 4 + r) * 2 + 1] = l[r];
#pragma unroll
        for (int s = 0; s < SETS; ++s) xo[(wave * 4 + r) * (64 * SETS) + 64 * s + lane] = o[s][r];
    }
    __syncthreads();
    // wave x of W joins rows x, x + W, ...
    float jo[4 / W][SETS], jm[4 / W], jl[4 / W];
#pragma unroll
    for (int n = 0; n < 4 / W; ++n) {
        const int r = wave + n * W;
        float mx = ml[r * 2];
#pragma unroll
        for (int x = 1; x < W; ++x) mx = fmaxf(mx, ml[(x * 4 + r) * 2]);
        float sum = 0.0f, z = 0.0f;
#pragma unroll
        for (int s = 0; s < SETS; ++s) jo[n][s] = 0.0f;
#pragma unroll
        for (int x = 0; x < W; ++x) {
            const float f = fast_exp2(ml[(x * 4 + r) * 2] - mx);
            sum = __builtin_fmaf(f, ml[(x * 4 + r) * 2 + 1], sum);
#pragma unroll
            for (int s = 0; s < SETS; ++s) jo[n][s] = __builtin_fmaf(f, xo[(x * 4 + r) * (64 * SETS) + 64 * s + lane], jo[n][s]);
        }
        jm[n] = mx, jl[n] = sum;
        z = sum * 0.0f;
#pragma unroll
        for (int s = 0; s < SETS; ++s) z = __builtin_fmaf(jo[n][s], 0.0f, z);
        if (w.row0 + r >= w.rows) continue;
        if (__any(!(z == 0.0f))) {  // as in seq_finish
            split_again<float>(p, w, r);
            continue;
        }
        const SeqRow sr = seq_row(p, w.row0 + r, w.rows, w.kvh);
        float* out = (float*)p.o + v.bq * p.ob + (long long)(v.q0 + sr.i) * p.ot + sr.head * p.oh;
        const long long pr = part_row(p, w.slot, w.kvh, w.row0 + r);
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
            const int d = 64 * s + lane;
            if (d < p.dim) {
                if (!p.part)
                    out[d] = jo[n][s] * join_scale(jl[n]);
                else
                    p.part[pr * p.dim + d] = jo[n][s];
            }
        }
        if (p.part && lane == 0) p.part_ml[2 * pr] = jm[n], p.part_ml[2 * pr + 1] = jl[n];
    }
}

// The join of a row's chunks, a wave a row: o = sum 2^(m_c - m) o_c / sum 2^(m_c - m) l_c.
template <class T>
__device__ __forceinline__ void seq_join_body(const SeqAttnArgs& p)
{
    const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long long per = (long long)p.q_tokens * p.group;
    const long long pair = at / per;
    const int r = (int)(at - pair * per), lane = threadIdx.x & 63;
    const int sq = (int)(pair / p.kv_heads), kvh = (int)(pair - (long long)sq * p.kv_heads);
    if (sq >= p.n_seq) return;
    const SeqView v = seq_view(p, sq);
    if (r >= v.lq * p.group) return;
    const SeqRow row = seq_row(p, r, v.lq * p.group, kvh);
    const int limit = row_limit(p, v, row.i, p.prefix ? p.prefix[sq] : 0);
    const int n = (int)(((long long)limit + p.chunk - 1) / p.chunk);
    const int slot = p.cu_k ? v.k0 / p.chunk + sq : sq * p.slots;
    // a lane a chunk for the weights, then the chunks' rows eight at a time
    float m = -1e30f;
    for (int c = lane; c < n; c += 64) m = fmaxf(m, p.part_ml[2 * part_row(p, slot + c, kvh, r)]);
    m = wave_max(m);
    float l = 0.0f, oa = 0.0f, oc = 0.0f;
    for (int c0 = 0; c0 < n; c0 += 64) {
        const long long mine = 2 * part_row(p, slot + (c0 + lane < n ? c0 + lane : 0), kvh, r);
        const float f = c0 + lane < n ? fast_exp2(p.part_ml[mine] - m) : 0.0f;
        l += wave_sum(f * p.part_ml[mine + 1]);
        const int here = n - c0 < 64 ? n - c0 : 64;
        for (int x = 0; x < here; x += 8) {
            float a[8], b[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float* pr = p.part + part_row(p, slot + c0 + (x + e < here ? x + e : 0), kvh, r) * p.dim;
                a[e] = pr[lane < p.dim ? lane : 0];
                b[e] = pr[lane + 64 < p.dim ? lane + 64 : 0];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // a chunk past the last has the weight of none, and may hold anything
                const float w = lane_value(f, x + e < here ? x + e : 0);
                oa = x + e < here ? __builtin_fmaf(w, a[e], oa) : oa;
                oc = x + e < here ? __builtin_fmaf(w, b[e], oc) : oc;
            }
        }
    }
    T* o = (T*)p.o + v.bq * p.ob + (long long)(v.q0 + row.i) * p.ot + row.head * p.oh;
    if (lane < p.dim) o[lane] = (T)(oa * join_scale(l));
    if (lane + 64 < p.dim) o[lane + 64] = (T)(oc * join_scale(l));
}

#define SEQ_INST(NAME, T, DT, KT, MODE, WPS)                                                                 \
    extern "C" __global__ __launch_bounds__(256, WPS) void NAME(SeqAttnArgs p)                               \
    {                                                                                                        \
        constexpr int B = 32 * KT * SeqShape<T, DT>::ROW;                                                    \
        constexpr int PB = MODE == SEQ_BIAS || MODE == SEQ_BOTH ? 128 * KT : 4;                              \
        __shared__ __attribute__((aligned(16))) unsigned char K0[B], K1[B], V0[B], V1[B];                    \
        __shared__ __attribute__((aligned(16))) unsigned P0[PB], P1[PB];                                     \
        seq_body<T, DT, KT, MODE>(p, K0, K1, V0, V1, P0, P1);                                                \
    }

SEQ_INST(hat_attnseq_f16_d1, f16, 1, 2, SEQ_PLAIN, 3)
SEQ_INST(hat_attnseq_f16_d2, f16, 2, 2, SEQ_PLAIN, 3)
SEQ_INST(hat_attnseq_f16_d3, f16, 3, 2, SEQ_PLAIN, 2)
SEQ_INST(hat_attnseq_f16_d4, f16, 4, 2, SEQ_PLAIN, 2)
SEQ_INST(hat_attnseq_f16_d1_bias, f16, 1, 2, SEQ_BIAS, 3)
SEQ_INST(hat_attnseq_f16_d2_bias, f16, 2, 2, SEQ_BIAS, 2)
SEQ_INST(hat_attnseq_f16_d3_bias, f16, 3, 2, SEQ_BIAS, 2)
SEQ_INST(hat_attnseq_f16_d4_bias, f16, 4, 2, SEQ_BIAS, 2)
SEQ_INST(hat_attnseq_f16_d1_cap, f16, 1, 2, SEQ_CAP, 3)
SEQ_INST(hat_attnseq_f16_d2_cap, f16, 2, 2, SEQ_CAP, 3)
SEQ_INST(hat_attnseq_f16_d3_cap, f16, 3, 2, SEQ_CAP, 2)
SEQ_INST(hat_attnseq_f16_d4_cap, f16, 4, 2, SEQ_CAP, 2)
SEQ_INST(hat_attnseq_f16_d1_both, f16, 1, 2, SEQ_BOTH, 2)
SEQ_INST(hat_attnseq_f16_d2_both, f16, 2, 2, SEQ_BOTH, 2)
SEQ_INST(hat_attnseq_f16_d3_both, f16, 3, 2, SEQ_BOTH, 2)
SEQ_INST(hat_attnseq_f16_d4_both, f16, 4, 2, SEQ_BOTH, 2)
SEQ_INST(hat_attnseq_bf16_d1, bf16, 1, 2, SEQ_PLAIN, 3)
SEQ_INST(hat_attnseq_bf16_d2, bf16, 2, 2, SEQ_PLAIN, 3)
SEQ_INST(hat_attnseq_bf16_d3, bf16, 3, 2, SEQ_PLAIN, 2)
SEQ_INST(hat_attnseq_bf16_d4, bf16, 4, 2, SEQ_PLAIN, 2)
SEQ_INST(hat_attnseq_bf16_d1_bias, bf16, 1, 2, SEQ_BIAS, 3)
SEQ_INST(hat_attnseq_bf16_d2_bias, bf16, 2, 2, SEQ_BIAS, 2)
SEQ_INST(hat_attnseq_bf16_d3_bias, bf16, 3, 2, SEQ_BIAS, 2)
SEQ_INST(hat_attnseq_bf16_d4_bias, bf16, 4, 2, SEQ_BIAS, 2)
SEQ_INST(hat_attnseq_bf16_d1_cap, bf16, 1, 2, SEQ_CAP, 3)
SEQ_INST(hat_attnseq_bf16_d2_cap, bf16, 2, 2, SEQ_CAP, 3)
SEQ_INST(hat_attnseq_bf16_d3_cap, bf16, 3, 2, SEQ_CAP, 2)
SEQ_INST(hat_attnseq_bf16_d4_cap, bf16, 4, 2, SEQ_CAP, 2)
SEQ_INST(hat_attnseq_bf16_d1_both, bf16, 1, 2, SEQ_BOTH, 2)
SEQ_INST(hat_attnseq_bf16_d2_both, bf16, 2, 2, SEQ_BOTH, 2)
SEQ_INST(hat_attnseq_bf16_d3_both, bf16, 3, 2, SEQ_BOTH, 2)
SEQ_INST(hat_attnseq_bf16_d4_both, bf16, 4, 2, SEQ_BOTH, 2)
#define SEQ_FP_INST(NAME, DT, KT, MODE, WPS)                                                                   \
    extern "C" __global__ __launch_bounds__(256, WPS) void NAME(SeqAttnArgs p)                               \
    {                                                                                                        \
        constexpr int B = 3 * Seq32Shape<DT, KT>::PLANE;                                                     \
        __shared__ __attribute__((aligned(16))) unsigned char K[B], V[B];                                    \
        __shared__ __attribute__((aligned(16))) unsigned P[MODE == SEQ_PLAIN ? 4 : 128 * KT];                \
        seq32_body<DT, KT, MODE>(p, K, V, P);                                                                \
    }

SEQ_FP_INST(hat_attnseq_f32_d1, 1, 2, SEQ_PLAIN, 2)
SEQ_FP_INST(hat_attnseq_f32_d1_bias, 1, 2, SEQ_BIAS, 2)
SEQ_FP_INST(hat_attnseq_f32_d1_both, 1, 2, SEQ_BOTH, 2)
SEQ_FP_INST(hat_attnseq_f32_d2, 2, 2, SEQ_PLAIN, 2)
SEQ_FP_INST(hat_attnseq_f32_d2_bias, 2, 2, SEQ_BIAS, 2)
SEQ_FP_INST(hat_attnseq_f32_d2_both, 2, 1, SEQ_BOTH, 2)
SEQ_FP_INST(hat_attnseq_f32_d3, 3, 1, SEQ_PLAIN, 2)
SEQ_FP_INST(hat_attnseq_f32_d3_bias, 3, 1, SEQ_BIAS, 2)
SEQ_FP_INST(hat_attnseq_f32_d3_both, 3, 1, SEQ_BOTH, 2)
SEQ_FP_INST(hat_attnseq_f32_d4, 4, 1, SEQ_PLAIN, 2)
SEQ_FP_INST(hat_attnseq_f32_d4_bias, 4, 1, SEQ_BIAS, 2)
SEQ_FP_INST(hat_attnseq_f32_d4_both, 4, 1, SEQ_BOTH, 2)

#define SPLIT_INST(NAME, T, DT, W)                                                                           \
    extern "C" __global__ __launch_bounds__(64 * W, 1) void NAME(SeqAttnArgs p)                              \
    {                                                                                                        \
        constexpr int B = SplitShape<T, DT, W>::BYTES;                                                       \
        __shared__ __attribute__((aligned(16))) unsigned char B0[B], B1[B], B2[B], B3[B];                    \
        __shared__ __attribute__((aligned(16))) unsigned P0[W * 128], P1[W * 128];                           \
        __shared__ float ml[W * 64];                                                                         \
        __shared__ unsigned flags;                                                                           \
        if (p.wide == 2)                                                                                     \
            seq_split_body<T, DT, W, true>(p, B0, B1, B2, B3, P0, P1, ml, &flags);                           \
        else                                                                                                 \
            seq_split_body<T, DT, W, false>(p, B0, B1, B2, B3, P0, P1, ml, &flags);                          \
    }

SPLIT_INST(hat_attnseq_f16_d1_split, f16, 1, 8)
SPLIT_INST(hat_attnseq_f16_d2_split, f16, 2, 8)
SPLIT_INST(hat_attnseq_f16_d3_split, f16, 3, 4)
SPLIT_INST(hat_attnseq_f16_d4_split, f16, 4, 4)
SPLIT_INST(hat_attnseq_bf16_d1_split, bf16, 1, 8)
SPLIT_INST(hat_attnseq_bf16_d2_split, bf16, 2, 8)
SPLIT_INST(hat_attnseq_bf16_d3_split, bf16, 3, 4)
SPLIT_INST(hat_attnseq_bf16_d4_split, bf16, 4, 4)
SPLIT_INST(hat_attnseq_f32_d1_split, float, 1, 8)
SPLIT_INST(hat_attnseq_f32_d2_split, float, 2, 4)
SPLIT_INST(hat_attnseq_f32_d3_split, float, 3, 2)
SPLIT_INST(hat_attnseq_f32_d4_split, float, 4, 2)

#define SEQ_FEW_INST(NAME, DT)                                                                               \
    extern "C" __global__ __launch_bounds__(256, 1) void NAME(SeqAttnArgs p)                                 \
    {                                                                                                        \
        __shared__ __attribute__((aligned(16))) unsigned char K[4 * 64 * 128 * DT];                          \
        __shared__ float xo[4 * 4 * 64 * ((DT + 1) / 2)], ml[4 * 4 * 2];                                     \
        seq_few_body<DT, 4>(p, K, xo, ml);                                                                    \
    }

SEQ_FEW_INST(hat_attnseq_f32_d1_few, 1)
SEQ_FEW_INST(hat_attnseq_f32_d2_few, 2)
SEQ_FEW_INST(hat_attnseq_f32_d3_few, 3)
SEQ_FEW_INST(hat_attnseq_f32_d4_few, 4)

#define JOIN_INST(NAME, T) \
    extern "C" __global__ __launch_bounds__(256) void NAME(SeqAttnArgs p) { seq_join_body<T>(p); }

JOIN_INST(hat_attnseq_join_f32, float)
JOIN_INST(hat_attnseq_join_f16, f16)
JOIN_INST(hat_attnseq_join_bf16, bf16)
