/*
 * hat.h - the C ABI of the MI355X HAT backend (libhat.so).
 *
 * A drop-in for the reference's GPU backend (jacobsparts/hat-rs). Every entry
 * point names the reference interface it replaces. Plain pointers and sizes
 * only; no GPU runtime types cross this boundary. Errors: functions returning
 * int give 0 on success (or a count, where stated) and a negative value on
 * failure; functions returning a pointer give NULL on failure. In both cases
 * hat_last_error() holds the message (thread-local), the counterpart of the
 * reference's `Result<_, String>` printed as `hat: <msg>` (src/main.rs:189-195).
 */
#ifndef HAT_H
#define HAT_H
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct hat_weights hat_weights;
typedef struct hat_backend hat_backend;

/* Library version string (the reference's hat::VERSION, src/lib.rs). */
const char *hat_version(void);

/* The last error message on this thread, or "" (main.rs:189-195). */
const char *hat_last_error(void);

/* ---- Weights (src/weights.rs) ------------------------------------------ */

/* Weights::load (weights.rs:60-129): mmap a converted .safetensors file, read
 * the architecture from __metadata__, validate every tensor shape
 * (weights.rs:133-265). */
hat_weights *hat_weights_open(const char *path);
void hat_weights_close(hat_weights *w);

/* The architecture fields of `Weights` (weights.rs:28-57). */
typedef struct {
    int scale, window, owin, embed, heads, head_dim, mlp_ratio;
    int n_stages;
    int depths[32];
    int compressed, squeezed, head_feat;
    float conv_scale, img_range;
    float mean[3];
} hat_model_info;
int hat_weights_info(const hat_weights *w, hat_model_info *out);

/* The checkpoint's `variant` metadata and its size in bytes (Weights.variant,
 * Weights.bytes, weights.rs:28-57; main.rs:205-206 prints both). */
const char *hat_weights_variant(const hat_weights *w);
unsigned long long hat_weights_file_bytes(const hat_weights *w);

/* Tensor listing and access (weights.rs:270-272 `t`, `--list-weights`). */
int hat_weights_count(const hat_weights *w);
const char *hat_weights_name(const hat_weights *w, int i);
/* F32 tensor data (owned by the weights object) and its element count. */
const float *hat_weights_tensor(const hat_weights *w, const char *name, size_t *numel);
/* Weights::i64 (weights.rs:331-346): copies up to n int64 values; returns the
 * element count. */
long hat_weights_index_i64(const hat_weights *w, const char *name, long long *out, size_t n);

/* A seeded checkpoint in tools/convert.py's format (convert.py:205-250): every
 * weight, bias and bias table ~ N(0, 0.02), LayerNorm weight 1 / bias 0, the
 * int64 relative-position index buffers from their closed forms. `variant` is
 * "hat-s", "hat" or "hat-l"; `depths` (may be NULL) overrides the variant's
 * per-stage block counts. No reference counterpart: the reference ships
 * converted checkpoints, and this writes the synthetic ones the benchmarks
 * and parity tests use. */
int hat_weights_generate(const char *path, const char *variant, int scale, unsigned long long seed,
                         const int *depths, int n_depths);

/* ---- Backend (src/backend.rs:29-36, src/gpu.rs:372-803) ------------------ */

/* 1 if the HIP runtime and a device can be brought up, else 0 (the probe
 * behind main.rs:148-174 `resolve_device`). Never fails. */
int hat_gpu_available(void);

/* Gpu::new (gpu.rs:372-386): brings up the runtime, checks that every kernel
 * resolves (cuda.rs:558-563) and uploads every weight. `device` must be "gpu"
 * (or NULL): this library has no CPU path, and asking for one is an error
 * rather than a silent fallback. The weights must outlive the backend. */
hat_backend *hat_backend_new(const hat_weights *w, const char *device);
/* Backend::name (backend.rs:30). */
const char *hat_backend_name(const hat_backend *b);
/* Backend::forward (backend.rs:32-35): in = [3][h][w] in [0,1] host memory;
 * out = caller-allocated [3][h*scale][w*scale] host memory. Synchronous. */
int hat_backend_forward(hat_backend *b, size_t h, size_t w, const float *in, float *out);
/* The same pass on device-resident buffers (from hat_device_alloc);
 * asynchronous on the backend's stream until hat_backend_synchronize. */
int hat_backend_forward_device(hat_backend *b, size_t h, size_t w, const float *d_in, float *d_out);
int hat_backend_synchronize(hat_backend *b);
/* hat_backend_forward_device without allocating: no reference counterpart. It
 * is for callers that cannot call hipMalloc (code under graph capture, serving
 * loops that forbid allocation). Every per-plan buffer of the pass is carved
 * from one fixed 256 MiB device array the library holds from load to process
 * exit (enough for HAT-S or HAT x4 up to 128 x 128 input pixels); a larger
 * plan is refused with an error and nothing runs. The caller passes device
 * input and output as for hat_backend_forward_device; the pass is asynchronous
 * on the backend's stream. All calls in a process share the one array: calls
 * that overlap on the GPU (two backends, two streams, two threads) race. */
int hat_backend_forward_noalloc(hat_backend *b, size_t h, size_t w, const float *d_in, float *d_out);
/* One HAB of the backend's network, `hab` (gpu.rs:469-520; HAB.forward,
 * hat_arch.py:266-309): x' = x + W-MSA(norm1 x) + conv_scale * CAB(norm1 x),
 * out = x' + MLP(norm2 x'), for layers.<stage>.residual_group.blocks.<block>,
 * shifted and masked when the block is odd. x/out: host token-major
 * [hp*wp][embed] on a plane whose sides are window multiples. iters > 0: *ms
 * (if non-NULL) = mean device time of the block over that many further runs. */
int hat_backend_hab(hat_backend *b, int stage, int block, size_t hp, size_t wp, const float *x,
                    float *out, int iters, float *ms);
/* Device bytes of the per-plan buffers and of the uploaded weights
 * (Acts/footprint, gpu.rs:78-290). */
size_t hat_backend_acts_bytes(const hat_backend *b);
size_t hat_backend_weight_bytes(const hat_backend *b);
void hat_backend_free(hat_backend *b);

/* ---- Batching, tiling and memory admission (src/tile.rs, src/memguard.rs) */

/* n images of one size through the backend: in = host [n][3][h][w], out =
 * host [n][3][h*scale][w*scale]. Up to 4 images are in flight at once, each on
 * its own stream with its own per-plan buffers, so the kernels of several
 * small images fill the device together (the single-GPU part of multi-image
 * batching). Synchronous; results identical to n calls of hat_backend_forward. */
int hat_backend_forward_batch(hat_backend *b, size_t n, size_t h, size_t w, const float *in, float *out);

/* tile::Tiling (tile.rs:34-45). */
typedef struct {
    size_t tile, margin, scale, tiles, largest_h, largest_w;
} hat_tiling;
/* tile::forward (tile.rs:50-107): the image in window-aligned cores of `tile`
 * input pixels, each run with a halo of `margin` pixels (both rounded up to
 * the window) on every side that is not the image's edge; only the cores are
 * copied to out. info (may be NULL) reports what ran. */
int hat_tile_forward(hat_backend *b, size_t h, size_t w, const float *in, float *out, size_t tile,
                     size_t margin, hat_tiling *info);
/* tile::auto_tile (tile.rs:140-184): the largest window-multiple core whose
 * sub-image (core plus both margins) fits budget_bytes at per_pixel_floats per
 * pixel plus constant_floats; 0 when not even one window fits (None). */
size_t hat_auto_tile(size_t h, size_t w, size_t win, unsigned long long budget_bytes,
                     unsigned long long per_pixel_floats, unsigned long long constant_floats, size_t margin);
/* memguard::Plan (memguard.rs:46-58). */
typedef struct {
    unsigned long long activations, weights, base, need, avail;
    int have_avail;
} hat_mem_plan;
/* memguard::gpu_plan (memguard.rs:147-160): the per-plan device buffers of an
 * h x w pass, the checkpoint's bytes and 128 MiB of runtime, with 5% slack,
 * against free device memory (have_avail = 0 when no device answers). The
 * backend refuses a plan that does not fit, with the reference's message
 * (memguard.rs:162-190), before allocating it. */
int hat_gpu_plan(const hat_weights *w, size_t h, size_t wd, hat_mem_plan *out);
/* main.rs:115-140 gpu_auto_tile: the tile a run without --tile/--mem uses,
 * halved from the larger image side until hat_gpu_plan fits. */
long hat_gpu_auto_tile(const hat_weights *w, size_t h, size_t wd);

/* ---- PNG I/O (src/image.rs) ------------------------------------------- */

/* image::load_rgb (image.rs:43-99): decode an 8- or 16-bit grey, grey+alpha,
 * RGB or RGBA PNG into planar [3][h][w] floats in [0,1]. Sets *w and *h; with
 * out non-NULL also writes the planes (cap >= 3*w*h floats). */
int hat_png_load(const char *path, size_t *w, size_t *h, float *out, size_t cap);
/* image::save_rgb of Image::to_rgb8 (image.rs:30-41,101-114): planar [3][h][w]
 * floats, clamped to [0,1], scaled by 255, rounded half up, as 8-bit RGB. */
int hat_png_save(const char *path, size_t w, size_t h, const float *planes);

/* Weights::shape (weights.rs:275-280, `--list-weights`): writes up to cap
 * dimensions of the named tensor; returns its rank. */
int hat_weights_shape(const hat_weights *w, const char *name, size_t *dims, int cap);

/* ---- Contracts (src/main.rs:312-326, src/selftest.rs:437-523) ----------- */

/* `--verify`: load a HATF v1 fixture (fixture.rs:44-78), run the backend,
 * print "  verify worst |diff| ... at (y, x, ch), mean |diff| ..." and return
 * 0 if the worst difference is within 1e-4, 1 if it is not, -1 on error. */
int hat_verify(const hat_weights *w, const char *device, const char *fixture_path);

/* `--cuda-selftest`: every gfx950 kernel against a host twin; prints
 * "  ok  <name>" per check and returns the number passed, or -1. */
int hat_gpu_selftest(void);

/* ---- Isolated ops (benchmark configs 2 and 3; host buffers) -------------- */

/* Shifted-window self-attention, the attention branch of HAB.forward
 * (hat_arch.py:266-309; cpu.rs:1117-1130): gather with the cyclic shift,
 * qkv linear, attention with relative-position bias and (shift > 0) the
 * SW-MSA mask, proj linear, scatter. x/out are token-major [hp*wp][c]; table is
 * [961][heads]. `iters` > 0 times that many extra runs: *ms = mean device time
 * of the op, *attn_ms = of its attention kernel alone (either may be NULL). */
int hat_op_swmsa(const float *x, float *out, int hp, int wp, int c, int heads, int shift,
                 const float *qkv_w, const float *qkv_b, const float *proj_w, const float *proj_b,
                 const float *table, int iters, float *ms, float *attn_ms);

/* The OCAB block (hat_arch.py:392-438; cpu.rs:1170-1198): norm1, qkv,
 * 24x24 unfold (stride 16, pad 4), attention with the [1521][heads] bias on
 * all 576 keys, proj + shortcut, norm2, GELU MLP + residual. */
int hat_op_ocab(const float *x, float *out, int hp, int wp, int c, int heads, int mlp_ratio,
                const float *n1w, const float *n1b, const float *qkv_w, const float *qkv_b,
                const float *proj_w, const float *proj_b, const float *table, const float *n2w,
                const float *n2b, const float *fc1_w, const float *fc1_b, const float *fc2_w,
                const float *fc2_b, int iters, float *ms, float *attn_ms);

/* ---- Operators on device tensors ------------------------------------------
 *
 * The transformer block around image and video tokens: rotary positions on
 * several axes, attention over sequences, and the join with the residual stream
 * (no reference counterpart; hat_op_swmsa and hat_op_ocab above are the
 * network's own attention). Tensors are device memory of device 0 (from
 * hat_device_alloc or another allocator of the process); strides count
 * elements and the last axis always has stride 1. Types: HAT_F32, HAT_F16,
 * HAT_BF16, one for all of a call's tensors; sums, softmax and norms are held
 * in fp32 and every result is rounded once.
 *
 * A call checks its arguments, enqueues its kernels on `stream` (a hipStream_t
 * of device 0; NULL: the default stream, as hat_device_copy) and returns; it
 * neither allocates nor waits, so it can be captured into a graph. Outputs
 * may be the inputs they replace (the same pointer and strides) where stated
 * and must otherwise not overlap them. */
enum { HAT_F32 = 0, HAT_F16 = 1, HAT_BF16 = 2 };

/* [batch][token][head][dim] */
typedef struct {
    void *data;
    long long batch_stride, token_stride, head_stride;
} hat_heads;
/* int32 [batch][token][axis]; batch_stride 0: one set for every batch entry. */
typedef struct {
    const int *data;
    long long batch_stride, token_stride, axis_stride;
} hat_positions;

/* Rotary positions: pair i of axis a (0 <= i < sections[a]) of every head is
 * turned by pos[token][a] * base^(-i / sections[a]), or, joint, by
 * pos[token][a] * base^(-n / S) with n the pair's index over all axes and S
 * their sum: (u, v) -> (u cos - v sin, v cos + u sin). Pair n is dims (n,
 * n + S), or (2n, 2n + 1) with `neighbours`; dims from 2 S on are copied.
 * inverse: by the negative angle, which is also the gradient. q and k are
 * turned in one launch (k.data NULL: q alone); q_out, k_out may be q, k.
 * head_dim <= 256. */
typedef struct {
    int dtype, batch, q_heads, k_heads, head_dim, axes;
    long long tokens; /* of a batch entry */
    int sections[4];
    int joint, neighbours, inverse;
    double base;
    hat_positions pos;
    hat_heads q, q_out, k, k_out;
} hat_rotary;
int hat_op_rotary(const hat_rotary *a, void *stream);

/* Attention over n_seq sequences. Query head h reads key head
 * h / (q_heads / kv_heads).
 *   s(i, j) = c tanh(scale q_i . k_j / c) - slopes[h] * distance(i, j)
 *   out_i   = sum_j e^s(i, j) v_j / sum_j e^s(i, j)
 * over the keys that query i sees; zeros where it sees none (or where every
 * weight is zero). cap 0: no tanh; else at least 1e-6, and scale / 1e6.
 * distance: |i + Lk - Lq - j| in a sequence of Lq queries and Lk keys, or with
 * positions the sum over the axes of |pos_q[i] - pos_k[j]| (below 2^31).
 * Sequences: entry s of a batch, its first q_lens[s] queries and k_lens[s] keys
 * (NULL: all q_tokens, k_tokens); or, with cu_q / cu_k (n_seq + 1 rising
 * offsets), rows cu[s] .. cu[s + 1) of a packed tensor of q_tokens / k_tokens
 * rows (its batch_stride is not used), which is the document mask. Lengths and
 * offsets are int32 in device memory, clamped to the tensors. Rows of out that
 * belong to no query keep what they hold.
 * causal: query i sees keys j <= i + Lk - Lq, and keys below prefix[s] (NULL:
 * none). Keys that a query does not see have no influence, whatever they hold.
 * head_dim <= 128; k's and v's token_stride below 2^22; out may be q. workspace: hat_op_attention_workspace bytes,
 * 16-byte aligned, in use until the call's kernels end: calls (and captured
 * graphs) that may run at the same time need one each. */
typedef struct {
    int dtype, n_seq, q_heads, kv_heads, head_dim, axes;
    long long q_tokens, k_tokens;
    hat_heads q, k, v, out;
    const int *cu_q, *cu_k, *q_lens, *k_lens, *prefix;
    int causal;
    float scale, cap;
    const float *slopes; /* [q_heads] in device memory, or NULL */
    hat_positions pos_q, pos_k; /* data NULL: distance by index */
    void *workspace;
    size_t workspace_bytes;
} hat_attention;
/* Reads sizes only: pointers count as set or NULL. (size_t)-1 on error. */
size_t hat_op_attention_workspace(const hat_attention *a);
int hat_op_attention(const hat_attention *a, void *stream);

/* The join with the residual stream and the norms before and after it, row by
 * row of `width` values (<= 16384):
 *   x' = x + scale * gate * Npost(y),   h = Npre(x')   (x' before its rounding)
 * N: HAT_NORM_NONE, HAT_NORM_LAYER (v - mean) / sqrt(var + eps) * w + b, or
 * HAT_NORM_RMS v / sqrt(mean v^2 + eps) * w + b; w, b fp32 [width] or NULL (ones,
 * zeros). gate: rows of `width` values, row r / rows_per_gate for row r (NULL:
 * ones). y NULL: x' = x. x_out or h may be NULL; x_out and h may be x or y. */
enum { HAT_NORM_NONE = 0, HAT_NORM_LAYER = 1, HAT_NORM_RMS = 2 };
typedef struct {
    int dtype, width, post, pre;
    long long rows, rows_per_gate;
    const void *x, *y, *gate;
    void *x_out, *h;
    long long x_stride, y_stride, gate_stride, x_out_stride, h_stride; /* of rows */
    const float *post_w, *post_b, *pre_w, *pre_b;
    float scale, post_eps, pre_eps;
} hat_residual_norm;
int hat_op_residual_norm(const hat_residual_norm *a, void *stream);

/* ---- Device memory and timing (lightgpu::vm DevBuf, src/cuda.rs:528-555) -- */
void *hat_device_alloc(size_t bytes);
int hat_device_free(void *p);
int hat_memcpy_h2d(void *dst, const void *src, size_t bytes);
int hat_memcpy_d2h(void *dst, const void *src, size_t bytes);
/* Device-to-device copy with the library's plain copy kernel (bytes a multiple
 * of 16, 16-byte aligned pointers); asynchronous on the library's stream. It is
 * also the HBM reference point the benchmark scales traffic counters by. */
int hat_device_copy(void *dst, const void *src, size_t bytes);
int hat_device_synchronize(void);
/* Free and total device memory in bytes (hipMemGetInfo): the measured side
 * of the working-set figures (the reference's free-VRAM delta,
 * examples/bench.rs:110-184). */
int hat_device_mem_info(size_t *free_bytes, size_t *total_bytes);
/* Device name and compute-unit count; "" / 0 when no device. */
const char *hat_device_name(void);
int hat_device_cu_count(void);

/* Per-kernel HIP-event timing of every launch between begin and end, on the
 * stream each kernel is launched on. hat_profile_get returns 0 and fills the
 * i-th kernel's name, launch count and total milliseconds. */
int hat_profile_begin(void);
int hat_profile_end(void);
int hat_profile_count(void);
int hat_profile_get(int i, char *name, int cap, long *count, double *total_ms);

#ifdef __cplusplus
}
#endif
#endif
