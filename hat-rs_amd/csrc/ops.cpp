#include "ops.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "hip_rt.h"
#include "kargs.h"

namespace hat {

using namespace hatk;

namespace {

constexpr long long MAX_STRIDE = 1ll << 40;  // elements: every offset stays far inside 64 bits
constexpr double LOG2E = 1.4426950408889634;

size_t element(int dtype) { return dtype == HAT_F32 ? 4 : 2; }

const char* type_name(int dtype) { return dtype == HAT_F32 ? "f32" : dtype == HAT_F16 ? "f16" : "bf16"; }

void check_dtype(const char* op, int dtype)
{
    if (dtype != HAT_F32 && dtype != HAT_F16 && dtype != HAT_BF16)
        throw Error(std::string(op) + ": type " + std::to_string(dtype) + " is none of HAT_F32, HAT_F16, HAT_BF16");
}

void check_range(const char* op, const char* what, long long v, long long lo, long long hi)
{
    if (v < lo || v > hi)
        throw Error(std::string(op) + ": " + what + " " + std::to_string(v) + " is out of range (" + std::to_string(lo) +
                    " to " + std::to_string(hi) + ")");
}

void check_pointer(const char* op, const char* what, const void* p, size_t align)
{
    if (!p) throw Error(std::string(op) + ": " + what + " is null");
    if ((uintptr_t)p % align) throw Error(std::string(op) + ": " + what + " is not aligned to its elements");
}

void check_stride(const char* op, const char* what, long long v)
{
    if (v < 0 || v > MAX_STRIDE) throw Error(std::string(op) + ": " + what + " has a stride of " + std::to_string(v));
}

void check_heads(const char* op, const char* what, const hat_heads& t, int dtype)
{
    check_pointer(op, what, t.data, element(dtype));
    check_stride(op, what, t.batch_stride);
    check_stride(op, what, t.token_stride);
    check_stride(op, what, t.head_stride);
}

// An output's rows lie apart: an axis of more than one entry moves at least a row on.
void check_rows_apart(const char* op, const char* what, const hat_heads& t, long long batch, long long tokens, int heads, int dim)
{
    if ((batch > 1 && t.batch_stride < dim) || (tokens > 1 && t.token_stride < dim) || (heads > 1 && t.head_stride < dim))
        throw Error(std::string(op) + ": " + what + " has rows on top of one another");
}

void check_replaces(const char* op, const char* what, const hat_heads& in, const hat_heads& out)
{
    if (in.data == out.data && (in.batch_stride != out.batch_stride || in.token_stride != out.token_stride ||
                                in.head_stride != out.head_stride))
        throw Error(std::string(op) + ": " + what + " overlaps its input with other strides");
}

void check_positions(const char* op, const hat_positions& p)
{
    check_pointer(op, "positions", p.data, 4);
    check_stride(op, "positions", p.batch_stride);
    check_stride(op, "positions", p.token_stride);
    check_stride(op, "positions", p.axis_stride);
}

// The caller's stream, refused where it is another device's.
hipStream_t check_stream(const char* op, void* stream)
{
    if (stream) {
        hipDevice_t dev = -1;
        const Runtime& rt = Runtime::get();
        rt.check(rt.api().StreamGetDevice((hipStream_t)stream, &dev), "hipStreamGetDevice");
        if (dev != 0) throw Error(std::string(op) + ": the stream belongs to device " + std::to_string(dev) + ", not 0");
    }
    return (hipStream_t)stream;
}

// Whether rows at these offsets from data can be moved `bytes` at a time.
bool aligned(const hat_heads& t, int dtype, size_t bytes)
{
    const size_t e = element(dtype);
    return ((uintptr_t)t.data | (size_t)t.batch_stride * e | (size_t)t.token_stride * e | (size_t)t.head_stride * e) % bytes == 0;
}

unsigned grid_of(const char* op, long long blocks)
{
    if (blocks > 0x7fffffffll) throw Error(std::string(op) + ": too large");
    return (unsigned)blocks;
}

}  // namespace

// ---------------------------------------------------------------------------

void op_rotary(const hat_rotary* a, void* stream)
{
    const char* op = "rotary";
    if (!a) throw Error("rotary: null argument");
    check_dtype(op, a->dtype);
    check_range(op, "head_dim", a->head_dim, 1, 2 * ROT_PAIRS);
    check_range(op, "axes", a->axes, 1, ROT_AXES);
    check_range(op, "batch", a->batch, 0, 1 << 30);
    check_range(op, "tokens", a->tokens, 0, 1ll << 31);
    check_range(op, "q_heads", a->q_heads, 1, 1 << 12);
    check_range(op, "k_heads", a->k_heads, a->k.data || a->k_out.data ? 1 : 0, 1 << 12);
    if (!(a->base > 0.0) || !std::isfinite(a->base)) throw Error("rotary: base must be positive");
    int pairs = 0;
    RotaryArgs p{};
    for (int x = 0; x < ROT_AXES; ++x) {
        if (x < a->axes) {
            check_range(op, "section", a->sections[x], 0, ROT_PAIRS);
            pairs += a->sections[x];
        }
        p.ends[x] = pairs;
    }
    if (pairs < 1 || 2 * pairs > a->head_dim)
        throw Error("rotary: sections of " + std::to_string(pairs) + " pairs do not fit a head_dim of " +
                    std::to_string(a->head_dim));
    if (a->batch == 0 || a->tokens == 0) return;
    const bool two = a->k.data || a->k_out.data;
    const hat_heads* in[2] = {&a->q, &a->k};
    const hat_heads* out[2] = {&a->q_out, &a->k_out};
    const int heads[2] = {a->q_heads, two ? a->k_heads : 0};
    bool in_place = true;
    for (int w = 0; w < (two ? 2 : 1); ++w) {
        check_heads(op, w ? "k" : "q", *in[w], a->dtype);
        check_heads(op, w ? "k_out" : "q_out", *out[w], a->dtype);
        check_rows_apart(op, w ? "k_out" : "q_out", *out[w], a->batch, a->tokens, heads[w], a->head_dim);
        check_replaces(op, w ? "k_out" : "q_out", *in[w], *out[w]);
        in_place = in_place && in[w]->data == out[w]->data;
    }
    check_positions(op, a->pos);

    // The widest move that every row, the pairs' halves and the copied rest allow (57600
    // tokens, 24 heads of 64 in fp16: 72 us in 16-byte moves, 76 in 8-byte ones).
    const int size = (int)element(a->dtype);
    const int widths[2] = {16 / size, 8 / size};
    int V = 1;
    for (int v : widths) {
        bool ok = a->head_dim % v == 0 && (a->neighbours ? 2 * pairs : pairs) % v == 0;
        for (int w = 0; ok && w < (two ? 2 : 1); ++w)
            ok = aligned(*in[w], a->dtype, v * size) && aligned(*out[w], a->dtype, v * size);
        if (ok) {
            V = v;
            break;
        }
    }
    for (int w = 0; w < 2; ++w) {
        p.x[w] = in[w]->data, p.y[w] = out[w]->data;
        p.xb[w] = in[w]->batch_stride, p.xt[w] = in[w]->token_stride, p.xh[w] = in[w]->head_stride;
        p.yb[w] = out[w]->batch_stride, p.yt[w] = out[w]->token_stride, p.yh[w] = out[w]->head_stride;
        p.heads[w] = heads[w];
    }
    p.pos = a->pos.data, p.pb = a->pos.batch_stride, p.pt = a->pos.token_stride, p.pa = a->pos.axis_stride;
    p.tokens = a->tokens, p.batch = a->batch;
    p.dim = a->head_dim, p.pairs = pairs, p.neighbours = a->neighbours != 0;
    const int turned = a->neighbours ? (2 * pairs / V + 1) / 2 : pairs / V;
    const int rest = in_place ? 0 : (a->head_dim - 2 * pairs) / V;  // in place they are there already
    p.chunks = turned + (rest + 1) / 2;
    const int items = p.chunks * (heads[0] + heads[1]);
    int n = 0;
    for (int x = 0; x < a->axes; ++x)
        for (int i = 0; i < a->sections[x]; ++i, ++n) {
            const double ladder = a->joint ? (double)n / pairs : (double)i / a->sections[x];
            const double turn = std::pow(a->base, -ladder) / (2.0 * M_PI);
            p.turn[n] = a->inverse ? -turn : turn;
        }
    // Tokens a block: about eight items a thread, fewer while the grid would not
    // fill the device, and within the angles' LDS and div_small's range.
    const long long all = a->tokens * a->batch;
    int per = std::max(1, std::min({2048 / items, 4096 / pairs, 64}));
    while (per > 1 && all / per < 2048) per = (per + 1) / 2;
    p.per = per;
    p.blocks = (all + per - 1) / per;
    p.inv_chunks = 1.0f / p.chunks, p.inv_items = 1.0f / items, p.inv_pairs = 1.0f / pairs;
    if ((long long)per * items >= 1 << 20) throw Error("rotary: too many heads");
    const DeviceScope scope;
    hipStream_t s = check_stream(op, stream);
    const std::string name = std::string("hat_rotary_") + type_name(a->dtype) + "_v" + std::to_string(V);
    launch(s, name.c_str(), grid_of(op, p.blocks), 1, 1, 256, p);
}

// ---------------------------------------------------------------------------

namespace {

void check_attention(const hat_attention* a)
{
    const char* op = "attention";
    if (!a) throw Error("attention: null argument");
    check_dtype(op, a->dtype);
    check_range(op, "head_dim", a->head_dim, 1, 128);
    check_range(op, "n_seq", a->n_seq, 0, 1 << 24);
    check_range(op, "kv_heads", a->kv_heads, 1, 1 << 12);
    check_range(op, "q_heads", a->q_heads, 1, 1 << 12);
    if (a->q_heads % a->kv_heads)
        throw Error("attention: " + std::to_string(a->q_heads) + " query heads do not divide over " +
                    std::to_string(a->kv_heads) + " key heads");
    check_range(op, "q_tokens", a->q_tokens, 0, (1ll << 31) - 1024);
    check_range(op, "k_tokens", a->k_tokens, 0, (1ll << 31) - 1024);
    check_range(op, "q_tokens times heads", a->q_tokens * (a->q_heads / a->kv_heads), 0, (1ll << 31) - 1024);
    if (!std::isfinite(a->scale)) throw Error("attention: scale must be finite");
    if (!(a->cap >= 0.0f) || !std::isfinite(a->cap)) throw Error("attention: cap must be 0 or positive");
    if (a->cap > 0.0f && !(a->cap >= 1e-6f && std::fabs(a->scale) / a->cap <= 1e6f))
        throw Error("attention: cap is next to nothing beside 1e-6 and a millionth of the scale");
    if ((a->cu_q && a->q_lens) || (a->cu_k && a->k_lens))
        throw Error("attention: a packed tensor has offsets, not lengths");
    if (a->prefix && !a->causal) throw Error("attention: a prefix belongs to the causal mask");
    // (tensors without tokens may have no address)
    if (a->q_tokens && a->k_tokens && (a->pos_q.data != nullptr) != (a->pos_k.data != nullptr))
        throw Error("attention: positions of queries and keys go together");
    if (a->pos_q.data && !a->slopes) throw Error("attention: positions without slopes");
    if (a->pos_q.data) check_range(op, "axes", a->axes, 1, 4);
}

}  // namespace

namespace {

// How a call runs, from its sizes alone.
struct AttnPlan {
    bool split;       // keys in chunks over blocks and waves
    bool few;         // fp32, four rows at a time
    int tiles;        // of rows: a sequence's (batch) or all sequences' slots (packed)
    int chunk, slots; // split: keys a chunk; a sequence's chunks (batch) or all slots (packed)
    long long blocks, join_rows;  // join_rows > 0: partial results and their join
    size_t workspace;
};

int dim_tiles(const hat_attention* a) { return (a->head_dim + 31) / 32; }

// Waves a block of the split kernels (SPLIT_INST): as many as their LDS allows.
int split_waves(const hat_attention* a)
{
    const int dt = dim_tiles(a);
    return a->dtype == HAT_F32 ? (dt == 1 ? 8 : dt == 2 ? 4 : 2) : dt <= 2 ? 8 : 4;
}

AttnPlan attn_plan(const hat_attention* a)
{
    AttnPlan p{};
    const int group = a->q_heads / a->kv_heads;
    const long long rows = a->q_tokens * group;
    const auto tiles = [&](int per) { return a->cu_q ? rows / per + a->n_seq : (rows + per - 1) / per; };
    const long long pairs = (long long)a->kv_heads * (a->cu_q ? 1 : a->n_seq);
    p.tiles = (int)tiles(128);
    p.blocks = tiles(128) * pairs;
    // Tiles of 32 rows whose keys the waves (and blocks) share, where tiles of 128 leave CUs
    // without a block: fewer than 128 of them, or up to 256 with few rows each and keys
    // enough to share. Split against not, us:
    //   120 tiles (3 x 2504 queries, 2 heads of 80, fp16, bias over two axes) 80, 86; 128 (2048
    //   queries, 8 heads of 128, fp32) 318, 274; 792 (2 x 4099, 12 heads of 64, fp16) 233, 146;
    //   4 queries each, 8 heads of 64 / 128, fp16: 192 tiles of 256 keys 8.6, 7.5 / 10.9, 11.2, of
    //   4096 36, 55 / 81, 112; 384 of 1024 26, 19 / 42, 35, of 4096 95, 82 / 168, 161;
    //   1024 x 64 queries and keys, 6 heads of 32 262, 37.
    const double keys_each = (double)a->k_tokens / (a->cu_k ? std::max(a->n_seq, 1) : 1);
    // fp32 with up to eight rows goes by fours, whose cost follows the rows: 4 queries each, 8
    // heads of 128, by fours against tiles of 128: 192 of 4096 keys 142, 659, 640 of 256 keys 44,
    // 94; 6144 of 8 rows and 256 keys 673, 706 at 128 dims, 185, 113 at 32; 3 sequences
    // of 6819 keys, 4 heads of 128, one row 20 against 49 by tiles of 32.
    p.few = a->dtype == HAT_F32 && !a->cu_q && rows <= 8 && (dim_tiles(a) >= 3 || p.blocks <= 512);
    p.split = p.few || p.blocks < 128 || (!a->cu_q && rows <= 64 && p.blocks <= 256 && keys_each >= 512);
    if (!p.split) return p;
    const int per = p.few ? 4 : 32, waves = p.few ? 4 : split_waves(a);
    p.tiles = (int)tiles(per);
    if (a->cu_q) {
        p.blocks = tiles(per) * a->kv_heads;
        p.chunk = 1 << 30;
        return p;
    }
    // Chunks of keys. A block fills a CU's LDS, so 256 blocks are a round; with lengths that
    // the host does not know some stay empty, so they get two rounds. (16 sequences of
    // 16384 keys, 8 heads of 128: 182 us in 256 blocks, 188 in 512, 200 in 1024; lengths of
    // 8192 to 16384: 164 us in 512, 196 in 2048.) Up to 128 keys a wave one chunk costs less
    // than the join's launch (1023 keys, 2 heads of 64: 9.4 us against 7 + 4).
    const double keys = (double)a->k_tokens * (a->cu_k ? 1 : a->n_seq);
    const double work = keys * a->kv_heads * p.tiles;  // keys times blocks that read them
    const long long blocks = a->cu_k || a->k_lens ? 512 : 256, whole = 128 * waves;
    const long long even = (long long)std::min(work / blocks, 1e9);
    p.chunk = (int)std::max<long long>(p.few ? 512 : 256, (even + 127) / 128 * 128);
    if (a->k_tokens <= whole) p.chunk = (int)whole;
    const long long n = (a->k_tokens + p.chunk - 1) / p.chunk;
    const long long slots = a->cu_k ? a->k_tokens / p.chunk + a->n_seq : std::max<long long>(n, 1) * a->n_seq;
    p.slots = (int)(a->cu_k ? slots : std::max<long long>(n, 1));
    p.blocks = slots * a->kv_heads * p.tiles;
    if (n > 1) {
        p.join_rows = rows * a->kv_heads * a->n_seq;
        p.workspace = (size_t)(slots * a->kv_heads * rows) * (a->head_dim + 2) * sizeof(float);
    }
    return p;
}

}  // namespace

size_t op_attention_workspace(const hat_attention* a)
{
    check_attention(a);
    return a->n_seq == 0 || a->q_tokens == 0 ? 0 : attn_plan(a).workspace;
}

void op_attention(const hat_attention* a, void* stream)
{
    const char* op = "attention";
    check_attention(a);
    if (a->n_seq == 0 || a->q_tokens == 0) return;
    check_heads(op, "q", a->q, a->dtype);
    check_heads(op, "out", a->out, a->dtype);
    check_rows_apart(op, "out", a->out, a->cu_q ? 1 : a->n_seq, a->q_tokens, a->q_heads, a->head_dim);
    check_replaces(op, "out", a->q, a->out);
    if (a->k_tokens) {
        check_heads(op, "k", a->k, a->dtype);
        check_heads(op, "v", a->v, a->dtype);
        // a stage of 64 rows lies within a buffer descriptor's 31 bits
        check_range(op, "k's token stride", a->k.token_stride, 0, (1 << 22) - 1);
        check_range(op, "v's token stride", a->v.token_stride, 0, (1 << 22) - 1);
        if (a->pos_q.data) {
            check_positions(op, a->pos_q);
            check_positions(op, a->pos_k);
        }
    }
    for (const void* i : {(const void*)a->cu_q, (const void*)a->cu_k, (const void*)a->q_lens, (const void*)a->k_lens,
                          (const void*)a->prefix, (const void*)a->slopes})
        if (i) check_pointer(op, "an int32 or fp32 argument", i, 4);
    const AttnPlan plan = attn_plan(a);
    if (plan.workspace) {
        if (!a->workspace || a->workspace_bytes < plan.workspace)
            throw Error("attention: a workspace of " + std::to_string(plan.workspace) + " bytes is needed");
        if ((uintptr_t)a->workspace % 16) throw Error("attention: the workspace is not aligned to 16 bytes");
    }
    SeqAttnArgs p{};
    p.q = a->q.data, p.k = a->k.data, p.v = a->v.data, p.o = a->out.data;
    p.qb = a->q.batch_stride, p.qt = a->q.token_stride, p.qh = a->q.head_stride;
    p.kb = a->k.batch_stride, p.kt = a->k.token_stride, p.kh = a->k.head_stride;
    p.vb = a->v.batch_stride, p.vt = a->v.token_stride, p.vh = a->v.head_stride;
    p.ob = a->out.batch_stride, p.ot = a->out.token_stride, p.oh = a->out.head_stride;
    p.cu_q = a->cu_q, p.cu_k = a->cu_k, p.q_lens = a->q_lens, p.k_lens = a->k_lens, p.prefix = a->prefix;
    p.slopes = a->slopes;
    if (a->pos_q.data && a->k_tokens) {
        p.pos_q = a->pos_q.data, p.pos_k = a->pos_k.data, p.axes = a->axes;
        p.pqb = a->pos_q.batch_stride, p.pqt = a->pos_q.token_stride, p.pqa = a->pos_q.axis_stride;
        p.pkb = a->pos_k.batch_stride, p.pkt = a->pos_k.token_stride, p.pka = a->pos_k.axis_stride;
    }
    p.n_seq = a->n_seq, p.q_heads = a->q_heads, p.kv_heads = a->kv_heads, p.group = a->q_heads / a->kv_heads;
    p.dim = a->head_dim;
    p.q_tokens = (int)a->q_tokens, p.k_tokens = (int)a->k_tokens;
    p.causal = a->causal != 0;
    const int size = (int)element(a->dtype);
    for (int bytes : {16, 4}) {
        if (a->head_dim * size % bytes == 0 && aligned(a->q, a->dtype, bytes) && aligned(a->k, a->dtype, bytes) &&
            aligned(a->v, a->dtype, bytes)) {
            p.wide = bytes == 16 ? 2 : 1;
            break;
        }
    }
    p.wide_out = a->head_dim % 4 == 0 && aligned(a->out, a->dtype, 4 * size);
    p.scale = a->scale;
    p.cap = a->cap, p.inv_cap = a->cap > 0.0f ? 1.0f / a->cap : 0.0f;
    // positive (the sign goes into q), so that the largest score is the largest product
    const double c = std::max(std::fabs((double)a->scale), 1e-37) * LOG2E;
    p.c1 = (float)(a->cap > 0.0f ? 2.0 * c / a->cap : c);
    p.tiles = plan.tiles, p.chunk = plan.chunk, p.slots = plan.slots;
    if (plan.join_rows) {
        p.part = (float*)a->workspace;
        p.part_ml = p.part + plan.workspace / sizeof(float) / (a->head_dim + 2) * a->head_dim;
    }
    const DeviceScope scope;
    hipStream_t s = check_stream(op, stream);
    const std::string type = type_name(a->dtype);
    std::string name = "hat_attnseq_" + type + "_d" + std::to_string(dim_tiles(a));
    // The bias as MFMA's starting value needs it in units of q . k: not where the scale is
    // next to nothing. fp32 has no kernel for the cap alone: its tanh is computed in full.
    if (plan.few)
        name += "_few";
    else if (plan.split)
        name += "_split";
    else if (a->cap > 0.0f)
        name += a->slopes || a->dtype == HAT_F32 ? "_both" : "_cap";
    else if (a->slopes)
        name += p.c1 > 1e-6f ? "_bias" : "_both";
    // Causal tiles in one order from the longest, or folded (attnseq.hip): 512 blocks 129 and
    // 123 us, 792 152 and 146, 2048 629 and 680.
    p.fold = p.causal && !a->cu_q && plan.blocks <= 1024;
    const int threads = plan.split && !plan.few ? 64 * split_waves(a) : 256;
    launch(s, name.c_str(), grid_of(op, plan.blocks), 1, 1, threads, p);
    if (plan.join_rows)
        launch(s, ("hat_attnseq_join_" + type).c_str(), grid_of(op, (plan.join_rows + 3) / 4), 1, 1, 256, p);
}

// ---------------------------------------------------------------------------

void op_residual_norm(const hat_residual_norm* a, void* stream)
{
    const char* op = "residual_norm";
    if (!a) throw Error("residual_norm: null argument");
    check_dtype(op, a->dtype);
    check_range(op, "width", a->width, 1, 16384);
    check_range(op, "rows", a->rows, 0, 1ll << 40);
    check_range(op, "post", a->post, HAT_NORM_NONE, HAT_NORM_RMS);
    check_range(op, "pre", a->pre, HAT_NORM_NONE, HAT_NORM_RMS);
    if (!a->y && (a->post != HAT_NORM_NONE || a->gate)) throw Error("residual_norm: a norm or a gate of no y");
    if (a->post == HAT_NORM_NONE && (a->post_w || a->post_b)) throw Error("residual_norm: weights of no norm");
    if (a->pre == HAT_NORM_NONE && (a->pre_w || a->pre_b)) throw Error("residual_norm: weights of no norm");
    if (!std::isfinite(a->scale) || !(a->post_eps >= 0.0f) || !(a->pre_eps >= 0.0f))
        throw Error("residual_norm: scale must be finite, eps 0 or positive");
    if (a->gate) check_range(op, "rows_per_gate", a->rows_per_gate, 1, 1ll << 40);
    if (a->rows == 0) return;  // tensors without rows may have no address
    if (!a->x_out && !a->h) throw Error("residual_norm: no output");
    const size_t e = element(a->dtype);
    const struct {
        const char* what;
        const void* p;
        long long stride;
        bool out;
    } rows[] = {{"x", a->x, a->x_stride, false},
                {"y", a->y, a->y_stride, false},
                {"gate", a->gate, a->gate_stride, false},
                {"x_out", a->x_out, a->x_out_stride, true},
                {"h", a->h, a->h_stride, true}};
    if (!a->x) throw Error("residual_norm: x is null");
    size_t move = 16;  // bytes a move: 16, 4 or one element
    while ((size_t)a->width * e % move) move /= 4;
    for (const auto& r : rows) {
        if (!r.p) continue;
        check_pointer(op, r.what, r.p, e);
        check_stride(op, r.what, r.stride);
        if (r.out && a->rows > 1 && r.stride < a->width)
            throw Error(std::string("residual_norm: ") + r.what + " has rows on top of one another");
        while (((uintptr_t)r.p | (size_t)r.stride * e) % move) move /= 4;
    }
    for (int i = 0; i < 2; ++i)
        for (int o = 3; o < 5; ++o)
            if (rows[i].p && rows[i].p == rows[o].p && rows[i].stride != rows[o].stride && a->rows > 1)
                throw Error(std::string("residual_norm: ") + rows[o].what + " overlaps its input with other strides");
    if (a->x_out && a->x_out == a->h) throw Error("residual_norm: x_out and h are the same rows");
    for (const float* w : {a->post_w, a->post_b, a->pre_w, a->pre_b}) {
        if (!w) continue;
        check_pointer(op, "a norm's weight", w, 4);
        if ((uintptr_t)w % 16 && move == 16) move = 4;
    }
    ResNormArgs p{};
    p.x = a->x, p.y = a->y, p.gate = a->gate, p.xo = a->x_out, p.h = a->h;
    p.post_w = a->post_w, p.post_b = a->post_b, p.pre_w = a->pre_w, p.pre_b = a->pre_b;
    p.xs = a->x_stride, p.ys = a->y_stride, p.gs = a->gate_stride, p.xos = a->x_out_stride, p.hs = a->h_stride;
    p.rows = a->rows, p.rows_per_gate = a->gate ? a->rows_per_gate : 1;
    p.width = a->width, p.post = a->post, p.pre = a->pre;
    p.scale = a->scale, p.post_eps = a->post_eps, p.pre_eps = a->pre_eps;
    // The fewest threads a row whose registers hold it (resnorm.hip): no barrier up to a
    // wave, and a 1024-thread block costs twice a 256-thread one (8192 in bf16: 257 us
    // against 135).
    const int W = a->width;
    const bool vec = move == 16;
    std::string form;
    int per = 1, threads = 256;
    if (vec && W <= (e == 4 ? 192 : 256))
        form = "16", per = 16;
    else if (W <= (vec ? 64 * 4 * 16 / (int)e : 1024))
        form = "64", per = 4;
    else if (W <= (vec ? 256 * 4 * 16 / (int)e : 4096))
        form = "256";
    else
        form = "1024", threads = 1024;
    if (!vec) form += move > e ? "h" : "e";
    const DeviceScope scope;
    hipStream_t s = check_stream(op, stream);
    const std::string name = std::string("hat_resnorm_") + type_name(a->dtype) + "_" + form;
    launch(s, name.c_str(), grid_of(op, (a->rows + per - 1) / per), 1, 1, threads, p);
}

}  // namespace hat
