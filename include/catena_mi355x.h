/*
 * catena_mi355x.h -- C ABI of the MI355X-native catena hot path.
 *
 * Two layers, both plain C (pointers, sizes, status codes; no torch types):
 *
 *  1. The program ABI that catena's generated module exports and that its
 *     runtime calls through libffi (catena-lang/src/runtime/executor.rs:47-106,
 *     signature table catena-lang/src/runtime/signature.rs:18-72, emitted by
 *     catena-lang/src/codegen/gpu.rs:235-285).  Symbols are
 *     `program_` + the source name with every non-alphanumeric mapped to `_`
 *     (catena-lang/src/codegen/mod.rs:379-388); inputs by value, outputs as
 *     pointers, return void, and assertion / GPU failures are fail-stop
 *     (message on stderr, then a trap: catena-lang/src/codegen/prelude.rs:38-55).
 *
 *  2. The kernel ABI those programs lower to ("catena_mi355x_*"), which
 *     returns a status and never traps, plus the device buffer pool that
 *     replaces the reference's per-buffer managed allocation
 *     (catena-lang/src/runtime/mem.rs:152-171, hipFree on drop :119-125).
 *
 *  3. The runtime mirror ("catena_runtime_*") of Runtime::from_sources /
 *     Runtime::exec / Value (catena-lang/src/runtime/runtime.rs:104-247,
 *     catena-lang/src/runtime/value.rs:5-49).
 *
 * Everything runs on one device and one library-owned HIP stream.  Kernel
 * ABI calls are stream-ordered (asynchronous); program ABI calls and
 * catena_runtime_exec synchronise before returning, like the generated host
 * wrapper (catena-lang/src/codegen/ops/materializec.rs:123-141).
 */
#ifndef CATENA_MI355X_H
#define CATENA_MI355X_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* catena_mem_t: by-value fat pointer, len in BYTES.
 * Reference: catena-lang/src/codegen/prelude.rs:28-31 and
 * catena-lang/src/runtime/executor.rs:14-19 (CatenaMem).  Here `data` is a
 * device pointer owned by the pool; len == 0 means data == NULL
 * (catena-lang/src/codegen/ops/materializec.rs:114). */
typedef struct catena_mem {
  void *data;
  uint64_t len;
} catena_mem_t;

typedef enum catena_status {
  CATENA_OK = 0,
  CATENA_ERR_INVALID_ARGUMENT = 1,
  CATENA_ERR_UNSUPPORTED = 2,
  CATENA_ERR_HIP = 3,
  CATENA_ERR_OUT_OF_MEMORY = 4,
  CATENA_ERR_NOT_INITIALIZED = 5,
  CATENA_ERR_LOAD = 6
} catena_status_t;

/* ------------------------------------------------------------------ */
/* library / device                                                     */

/* Select the device, create the library stream, load the gfx950 code
 * objects (hipModuleLoad) that sit next to this library.  Idempotent.
 * Replaces GpuRuntime::load (catena-lang/src/runtime/mem.rs:134-150) and the
 * per-Runtime hipcc + dlopen of catena-lang/src/runtime/artifact.rs:44-103. */
int catena_mi355x_init(int device);
/* Orderly teardown before the process exits: waits for the library
 * stream, returns the library's own device memory (split-K workspace,
 * completion counters, cached pool blocks), unloads the code objects and
 * destroys the stream.  Buffers the caller still holds stay allocated and
 * may still be freed with catena_mem_free.  A later call re-initialises on
 * demand.  The reference instead keeps its generated library resident for
 * the process lifetime (RTLD_NODELETE, catena-lang/src/runtime/runtime.rs:
 * 249-263); here nothing is left for the runtime's own exit to tear down. */
int catena_mi355x_shutdown(void);
/* Message of the last failing call on this thread ("" if none). */
const char *catena_mi355x_last_error(void);
/* The hipStream_t every launch goes to (for events / interop). */
void *catena_mi355x_stream(void);
int catena_mi355x_synchronize(void);

/* ------------------------------------------------------------------ */
/* device buffer pool                                                    */

/* Allocate len bytes of device memory (size-classed, cached free lists).
 * Replaces Mem allocation (catena-lang/src/runtime/mem.rs:152-171). */
int catena_mem_alloc(uint64_t len, catena_mem_t *out);
/* Return a buffer to the pool and null the handle.  Stream-ordered: work
 * already queued on the library stream may still use it.  Replaces
 * Mem::drop -> hipFree (catena-lang/src/runtime/mem.rs:119-125). */
int catena_mem_free(catena_mem_t *mem);
/* Host <-> device copies (synchronous).  catena_mem_read replaces the raw
 * host dereference of managed memory in Mem::to_f32_vec / to_u64_vec
 * (catena-lang/src/runtime/mem.rs:44-70). */
int catena_mem_write(catena_mem_t mem, uint64_t offset, const void *src, uint64_t len);
int catena_mem_read(catena_mem_t mem, uint64_t offset, void *dst, uint64_t len);
int catena_pool_stats(uint64_t *bytes_live, uint64_t *bytes_cached, uint64_t *device_allocs);
/* Release every cached (free) block, and the scratch memory that bf16 products
 * of ragged or unaligned operands have taken, back to the device. */
int catena_pool_trim(void);

/* ------------------------------------------------------------------ */
/* kernel ABI (device pointers; stream-ordered)                         */

/* C[n x m] = A[n x k] * B[k x m], f32, row-major, each cell the
 * k-ascending fold acc = acc + A*B from +0.0 with no FMA: bitwise the
 * reference's f32.matmul.row-major.materialize
 * (catena-lang/stdlib/matrix.hex:236-327, lowered by
 * catena-lang/src/codegen/ops/materializec.rs:36-82 and
 * catena-lang/src/codegen/ops/reducec.rs:73-130). */
int catena_mi355x_gemm_f32_exact(const float *a, const float *b, float *c, uint64_t n,
                                 uint64_t m, uint64_t k);

/* C[n x m] = A[n x k] * B[k x m] on bf16 inputs (raw bf16 bits), f32
 * accumulation on MFMA in a fixed order, output bf16 (RNE) or f32 when
 * out_f32 != 0.  Same contraction as above, extended to bf16 (no reference
 * counterpart: catena has no bf16, catena-lang/src/codegen/lower_types.rs:13-22).
 * n <= 16 (decode shape) uses the weight-streaming kernel (both outputs) when
 * m % 8 == 0, k % 8 == 0 and the pointers are 16-byte aligned.  Any other
 * product is one ascending fold of 32-k MFMA steps per element, or, where few
 * output tiles meet a deep k, a few such folds over consecutive k ranges whose
 * f32 sums are added in ascending order (catena_mi355x_gemm_bf16_plan); its
 * bits do not depend on the pointers or on whether the call is captured into
 * a graph. */
int catena_mi355x_gemm_bf16(const uint16_t *a, const uint16_t *b, void *c, uint64_t n,
                            uint64_t m, uint64_t k, int out_f32);

/* How catena_mi355x_gemm_bf16 folds a product that is not the weight-streaming
 * kernel's: the number of k groups (1: one fold), the k of each group but the
 * last, and the rows and columns of the output tile a workgroup owns (0 when
 * the aligned 256-row tile kernels or, for m or k past 2^22, the kernel with
 * 64-bit addressing takes it).  A function of (n, m, k) alone; needs no
 * device.  No reference counterpart. */
int catena_mi355x_gemm_bf16_plan(uint64_t n, uint64_t m, uint64_t k, uint32_t *k_groups,
                                 uint64_t *group_k, uint32_t *tile_rows, uint32_t *tile_cols);

/* The k split of the decode-shape GEMM (1 <= n <= 16, m % 8 == 0, k % 8 ==
 * 0): the number of k groups whose f32 partials are added in ascending
 * order, and the bytes of those partials (0 when k is not split).  A function
 * of (n, m, k) alone -- never of the device -- so the decode GEMM's bits
 * depend only on the shape and the inputs.  Needs no device.  No reference
 * counterpart (the reference's fold is one sequential chain per cell). */
int catena_mi355x_gemm_bf16_decode_plan(uint64_t n, uint64_t m, uint64_t k, uint32_t *k_groups,
                                        uint64_t *partials_bytes);

/* Allocation-free form of catena_mi355x_gemm_bf16 for decode shapes
 * (1 <= n <= 16, m % 8 == 0, k % 8 == 0, k > 0; 16-byte aligned pointers):
 * the same kernels and the same bits, with the split-K partials in a fixed
 * 4 MiB device array the library holds on each device from load to exit,
 * instead of a workspace it grows with hipMalloc.  No reference counterpart:
 * for callers that cannot allocate device memory (code under HIP graph
 * capture, serving loops, harnesses that forbid hipMalloc).  Needs a prior
 * catena_mi355x_init (returns CATENA_ERR_NOT_INITIALIZED otherwise; it never
 * initialises, since init allocates); shapes whose partials exceed 4 MiB
 * (see catena_mi355x_gemm_bf16_decode_plan) return CATENA_ERR_UNSUPPORTED.
 * Calls share the device's array: calls that overlap on one device race. */
int catena_mi355x_gemm_bf16_decode_noalloc(const uint16_t *a, const uint16_t *b, void *c,
                                           uint64_t n, uint64_t m, uint64_t k, int out_f32);

/* LM head of a decode step in one launch: c = a * b as the decode shape of
 * catena_mi355x_gemm_bf16 computes it (f32 c[n][m]), and idx[r] =
 * tensor.argmax-f32 of row r of c (catena-lang/stdlib/tensor.hex:204-227:
 * the first maximum after the last NaN, or the last NaN when it is the
 * final element).  1 <= n <= 16, m % 8 == 0, k % 8 == 0, k > 0, m < 2^31,
 * n * ceil(m / 128) <= 57,344 (the per-block summaries' buffer); 16-byte
 * aligned a, b, c.  No reference counterpart (the decoder's greedy step). */
int catena_mi355x_gemm_bf16_argmax(const uint16_t *a, const uint16_t *b, float *c, uint32_t *idx,
                                   uint64_t n, uint64_t m, uint64_t k);

/* Decode attention, one query per (batch, head): q[B][H][D], k/v[B][H][L][D]
 * bf16, lens[B] (device u32, each <= L), o[B][H][D] f32.  Bitwise the
 * sequential composition of cell-dot, nn.softmax and cell-dot
 * (catena-lang/stdlib/matrix.hex:236-256, catena-lang/stdlib/nn.hex:93-122,
 * catena-lang/stdlib/math.hex:148-199).  No reference counterpart (catena
 * has no attention primitive).  head_dim must be 128. */
int catena_mi355x_attn_decode_bf16(const uint16_t *q, const uint16_t *k, const uint16_t *v,
                                   const uint32_t *lens, float *o, uint32_t batch,
                                   uint32_t heads, uint32_t max_len, uint32_t head_dim,
                                   float scale);

/* nn.softmax over `rows` contiguous vectors of length n (bitwise the
 * reference's fold order; catena-lang/stdlib/nn.hex:93-122).  y may equal x. */
int catena_mi355x_softmax_f32(const float *x, float *y, uint64_t rows, uint64_t n);

/* math.exp-approx elementwise (catena-lang/stdlib/math.hex:185-199). */
int catena_mi355x_exp_approx_f32(const float *x, float *y, uint64_t n);

/* The scalar stdlib programs elementwise, bitwise the reference's op order
 * (each is one generated __host__ __device__ function in the reference,
 * rendered from these hexpr sources).  y may equal x. */
typedef enum catena_map_op {
  CATENA_MAP_EXP_APPROX = 0,     /* math.exp-approx, catena-lang/stdlib/math.hex:185-199 */
  CATENA_MAP_SQRT = 1,           /* math.sqrt, catena-lang/stdlib/math.hex:235-272 */
  CATENA_MAP_SIGMOID = 2,        /* nn.sigmoid, catena-lang/stdlib/nn.hex:1-12 */
  CATENA_MAP_SILU = 3,           /* nn.silu, catena-lang/stdlib/nn.hex:15-21 */
  CATENA_MAP_SIN_APPROX = 4,     /* math.sin-approx, catena-lang/stdlib/math.hex:1-23 */
  CATENA_MAP_COS_APPROX = 5,     /* math.cos-approx, catena-lang/stdlib/math.hex:25-47 */
  CATENA_MAP_SIN_APPROX_FULL = 6 /* math.sin-approx-full, catena-lang/stdlib/math.hex:49-103 */
} catena_map_op_t;
int catena_mi355x_map_f32(uint32_t op, const float *x, float *y, uint64_t n);

/* Seeded synthetic inputs (counter-based splitmix64; see fill.hip). */
int catena_mi355x_fill_normal_bf16(uint16_t *out, uint64_t n, uint64_t seed, uint64_t stream,
                                   float scale);
int catena_mi355x_fill_uniform_f32(float *out, uint64_t n, uint64_t seed, uint64_t stream);
/* Device-to-device copy kernel (16-byte aligned pointers, n % 16 == 0); also
 * the known-size reference for calibrating HBM traffic counters. */
int catena_mi355x_copy_bytes(void *dst, const void *src, uint64_t n);

/* -- decoder-block pieces (the callers on either side of the two hot ops) -- */

/* Causal KV-cache attention for Tq queries per sequence (prefill, or
 * several tokens per step): q[B][Tq][H][D], k/v[B][H][L][D] bf16,
 * lens[B] (device u32: positions in the cache after the append, <= L),
 * o[B][Tq][H][D] f32 (out_f32 != 0) or bf16 RNE.  Query tq of sequence b
 * attends to the first lens[b] - (Tq - 1 - tq) positions, each exactly as
 * catena_mi355x_attn_decode_bf16 (Tq = 1 is that call).  No reference
 * counterpart.  head_dim must be 128. */
int catena_mi355x_attn_causal_bf16(const uint16_t *q, const uint16_t *k, const uint16_t *v,
                                   const uint32_t *lens, void *o, uint32_t batch, uint32_t tq,
                                   uint32_t heads, uint32_t max_len, uint32_t head_dim,
                                   float scale, int out_f32);

/* nn.rmsnorm over `rows` contiguous vectors of length n
 * (catena-lang/stdlib/nn.hex:154-182 with math.sqrt,
 * catena-lang/stdlib/math.hex:235-272): bitwise the reference's fold order.
 * n % 4 == 0; y may not alias x. */
int catena_mi355x_rmsnorm_f32(const float *x, float *y, uint64_t rows, uint64_t n);

/* Residual add in front of nn.rmsnorm, bf16 output: for output row i with
 * src = row_index ? row_index[i] : i, h = x[src] + resid[src] (h = x[src]
 * when resid is NULL), written to h_out[i] when h_out is not NULL; then
 * y[i] = bf16(nn.rmsnorm(h)).  No reference counterpart (the decoder's fused
 * form of f32.add and nn.rmsnorm).  n % 4 == 0. */
int catena_mi355x_residual_rmsnorm_bf16(const float *x, const float *resid,
                                        const uint32_t *row_index, float *h_out, uint16_t *y,
                                        uint64_t rows, uint64_t n);

/* Token embedding: x[r][:] = widen(table[tokens[r]][:]) for r < rows;
 * table[vocab][d] bf16, x f32; a token >= vocab gives a row of NaN.
 * d % 8 == 0.  No reference counterpart. */
int catena_mi355x_embed_bf16(const uint32_t *tokens, const uint16_t *table, float *x,
                             uint64_t rows, uint32_t vocab, uint32_t d);

/* RoPE inverse frequencies on the host: out[i] = (float)(1 / base^(2i/d))
 * in double precision, i < head_dim / 2.  No reference counterpart. */
int catena_mi355x_rope_inv_freq(float *out_host, uint32_t head_dim, double base);

/* RoPE + KV-cache append on a fused projection qkv[B*Tq][3*H*D] f32
 * (columns: q heads | k heads | v heads; row b*Tq + tq at position
 * lens[b] - Tq + tq).  Pairs (i, i + D/2) rotate by theta = pos *
 * inv_freq[i] with sin = math.sin-approx-full
 * (catena-lang/stdlib/math.hex:52-103) and cos the same reduction with the
 * quadrant advanced by one.  Writes q[B*Tq][H*D] bf16 and the bf16 rotated
 * k and v rows into k_cache/v_cache[B][H][L][D].  No reference counterpart. */
int catena_mi355x_rope_qkv_bf16(const float *qkv, const float *inv_freq, const uint32_t *lens,
                                uint16_t *q, uint16_t *k_cache, uint16_t *v_cache,
                                uint32_t batch, uint32_t tq, uint32_t heads, uint32_t head_dim,
                                uint32_t max_len);

/* The rotation table of catena_mi355x_rope_qkv_bf16 for positions 0 ..
 * positions - 1: tab[pos][i] = (cos, sin) of theta = (f32)pos * inv_freq[i],
 * i < head_dim / 2, f32 pairs -- the values that call computes per row.
 * positions <= 65535.  No reference counterpart. */
int catena_mi355x_rope_table_f32(const float *inv_freq, float *tab, uint32_t positions,
                                 uint32_t head_dim);

/* The decoder's prefill q / k / v projection in one kernel:
 * catena_mi355x_gemm_bf16(a, w, qkv, batch * tq, 3 * heads * 128, k, out_f32 = 1)
 * followed by catena_mi355x_rope_qkv_bf16(qkv, ..., head_dim = 128), bitwise,
 * without writing the f32 product.  a[batch * tq][k], w[k][3 * heads * 128]
 * bf16; rope_tab from catena_mi355x_rope_table_f32 with at least max_len
 * positions.  Rows whose position lens[b] - tq + t falls outside [0, max_len)
 * write q (rotated at position 0) and no cache row.  Needs batch * tq % 256
 * == 0, k % 128 == 0, k <= 2^22, 16-byte aligned pointers; other shapes
 * return CATENA_ERR_UNSUPPORTED.  No reference counterpart. */
int catena_mi355x_gemm_bf16_rope_qkv(const uint16_t *a, const uint16_t *w, const float *rope_tab,
                                     const uint32_t *lens, uint16_t *q, uint16_t *k_cache,
                                     uint16_t *v_cache, uint32_t batch, uint32_t tq, uint32_t heads,
                                     uint32_t max_len, uint64_t k);

/* bf16 GEMM as f32 k-split partials (the decoder's prefill W_down):
 * parts[z][n][m] = the product over k in [z k / splits, (z + 1) k / splits),
 * each folded as catena_mi355x_gemm_bf16 folds a product; a consumer adds
 * them in ascending z.  Needs 1 <= splits <= 64, n % 256 == 0, m % 256 == 0,
 * k % (128 splits) == 0, k <= 2^22, 16-byte aligned pointers.  No reference
 * counterpart. */
int catena_mi355x_gemm_bf16_ksplit_f32(const uint16_t *a, const uint16_t *b, float *parts,
                                       uint64_t n, uint64_t m, uint64_t k, uint32_t splits);

/* SwiGLU gate: gu[rows][2F] f32 -> out[rows][F] = bf16(nn.silu(gate) * up)
 * (catena-lang/stdlib/nn.hex:1-21).  group = 0: columns gate | up; group =
 * G: gate and up interleaved in groups of G columns (gate 0..G-1, up
 * 0..G-1, gate G..2G-1, ...), the decoder's W_gu layout (G = 64).
 * F % 4 == 0, G % 4 == 0, F % G == 0.  No reference counterpart. */
int catena_mi355x_silu_mul_bf16(const float *gu, uint16_t *out, uint64_t rows, uint32_t ffn,
                                uint32_t group);

/* bf16 GEMM with the SwiGLU gate fused into its epilogue (the decoder's
 * W_gu projection in prefill): act[n][m/2] = bf16(nn.silu(gate) * up) of the
 * f32 product A[n][k] x B[k][m], whose columns are gate and up interleaved in
 * groups of 64 (catena_mi355x_silu_mul_bf16 with group 64).  Bitwise the same
 * as catena_mi355x_gemm_bf16(..., out_f32 = 1) followed by that call, without
 * writing the f32 product.  Needs the 32-k tile kernels: n % 256 == 0, m % 128
 * == 0, k > 0 with k % 128 == 0, k <= 2^22, m <= 2^24, 16-byte aligned
 * pointers; other shapes return CATENA_ERR_UNSUPPORTED (n == 0 or m == 0 is a
 * no-op).  No reference counterpart. */
int catena_mi355x_gemm_bf16_silu(const uint16_t *a, const uint16_t *b, uint16_t *act, uint64_t n,
                                 uint64_t m, uint64_t k);

/* -- a key-value cache in pages -- */

/* A cache whose slots live in pages: k / v [num_pages][kv_heads][page_size]
 * [head_dim] bf16, table[rows][max_pages] (device u32): slot j of a row is
 * place j % page_size of page table[row][j / page_size].  page_size is a power
 * of two from 16 to 1024, head_dim 64 or 128, max_pages * page_size < 2^31;
 * k and v are 16-byte aligned.  A page number >= num_pages names no page: its
 * slots are read as absent and written nowhere.  The struct itself is read by
 * the call and not kept.  No reference counterpart. */
typedef struct catena_paged_kv {
  uint16_t *k;
  uint16_t *v;
  const uint32_t *table;
  uint32_t num_pages;
  uint32_t page_size;
  uint32_t rows;
  uint32_t max_pages; /* table entries per row */
  uint32_t kv_heads;
  uint32_t head_dim;
} catena_paged_kv_t;

/* How catena_mi355x_attn_paged_bf16 deals out its work -- into `parts` equal
 * parts of all rows' slots, joined by a second kernel, or (0) a row and kv head
 * at a time -- and the bytes of workspace that it takes (0: none).  A function
 * of the sizes alone (k, v and table are not looked at); needs no device. */
int catena_mi355x_attn_paged_plan(const catena_paged_kv_t *kv, uint32_t heads, int weights,
                                  uint32_t *parts, uint64_t *workspace_bytes);

/* Attention of one new token per row over a cache in pages: q[rows][heads]
 * [head_dim] bf16, lens[rows] (device u32: slots in use, the new token's among
 * them; a length past the table counts as the table's), o[rows][heads]
 * [head_dim] f32 (out_f32 != 0) or bf16 RNE.  Query head h reads kv head
 * h / (heads / kv_heads); o = sum_j p_j v_j, p = softmax(scale * q . k_j) with
 * the exponential itself (not math.exp-approx), sums in f32 that finite values of
 * any size do not overflow (p to 24 bits for an f32 o, to 2^-16 for a bf16 one).
 * A row of no slots gives 0, a row whose pages are all unknown NaN.  What the
 * cache holds past a row's slots is never used.
 * acc_in / acc_out[rows][kv_heads][max_pages * page_size] f32 (both or
 * neither, may be the same): acc_out[j] = acc_in[j] + the sum of p_j over the
 * query heads of a kv head, for the slots in use; others are left as they are.
 * The result depends on the sizes and the inputs alone, bit by bit; where the work
 * is cut follows from the lengths of all rows, so a row's last bits may differ
 * beside other rows.
 * workspace: 16-byte aligned, as many bytes as the plan says, used until the
 * call's work has run; calls that may overlap (two captured graphs) take one
 * each.  q and o 16-byte aligned.  Allocates nothing; may be captured. */
int catena_mi355x_attn_paged_bf16(const catena_paged_kv_t *kv, const uint16_t *q,
                                  const uint32_t *lens, void *o, uint32_t heads, float scale,
                                  int out_f32, const float *acc_in, float *acc_out,
                                  void *workspace, uint64_t workspace_bytes);

/* RoPE + append into pages, catena_mi355x_rope_qkv_bf16's twin for a cache in
 * pages and grouped heads: qkv[rows * tq][(heads + 2 kv_heads) * head_dim] f32
 * (columns: q heads | k heads | v heads), rope_tab[table_positions]
 * [head_dim / 2] (cos, sin) f32 (catena_mi355x_rope_table_f32's, or any).
 * lens[rows] (device u32) counts a row's slots after the append: token t goes
 * to slot lens[row] - tq + t.  seen[rows] counts its positions after the
 * append, given-up ones among them: token t is at position seen[row] - tq + t;
 * NULL: as lens.  Writes q[rows * tq][heads * head_dim] bf16 (rotated) and the
 * bf16 rotated k and v into the slots.  acc and slot_pos ([rows][kv_heads]
 * [max_pages * page_size] f32 and u32, both or neither): the new slots' weight
 * 0 and their position.  A token whose slot lies outside the table or whose
 * position outside rope_tab writes q (rotated by rope_tab's first position)
 * and nothing else, and so do all tokens of a row whose lens or seen is below tq;
 * one whose page does not exist writes q alone.  No two tokens of a call go to
 * the same slot of a page; rows may share pages, so that the tokens of prompts of
 * different lengths are rows of one token each, whose tables are their prompt's
 * (acc and slot_pos belong to a row: NULL there).  qkv, rope_tab and q 16-byte
 * aligned.  No reference counterpart. */
int catena_mi355x_rope_qkv_paged_bf16(const catena_paged_kv_t *kv, const float *qkv,
                                      const float *rope_tab, uint32_t table_positions,
                                      const uint32_t *lens, const uint32_t *seen, uint16_t *q,
                                      uint32_t tq, uint32_t heads, float *acc, uint32_t *slot_pos);

/* Bytes of workspace that catena_mi355x_kv_evict_paged_bf16 takes (0: none).
 * A function of the sizes alone; needs no device. */
int catena_mi355x_kv_evict_paged_plan(const catena_paged_kv_t *kv, uint32_t budget,
                                      uint64_t *workspace_bytes);

/* Bounds a cache in pages: per (row, kv head), of the lens[row] slots in use
 * min(lens[row], budget) are kept -- those of the last `recent` of the
 * seen[row] positions (the newest where they are more than the budget), then
 * those of the largest accumulated weight, the lower slot where two are equal, a
 * NaN weight behind every number -- and become the
 * first slots: the i-th slot given up below the budget takes K, V, weight and
 * position of the i-th slot kept from the budget on; the others stay where
 * they are.  (Attention does not depend on the order of slots; RoPE is applied
 * before the append.)  lens_out[rows] is the new length.  acc_in / acc_out and
 * slot_pos_in / slot_pos_out ([rows][kv_heads][max_pages * page_size]) are each
 * two buffers or the same one, 16-byte aligned; entries past the new length are
 * left as they are.  lens_out is neither lens nor seen.  The pages must be the
 * row's own (one that catena_mi355x_beam_reorder_paged_bf16 shares changes for
 * all its rows); K and V of a slot without a page are not moved.
 * workspace as for catena_mi355x_attn_paged_bf16.  No reference counterpart. */
int catena_mi355x_kv_evict_paged_bf16(const catena_paged_kv_t *kv, const uint32_t *lens,
                                      const uint32_t *seen, const float *acc_in,
                                      const uint32_t *slot_pos_in, uint32_t *lens_out,
                                      float *acc_out, uint32_t *slot_pos_out, uint32_t budget,
                                      uint32_t recent, void *workspace, uint64_t workspace_bytes);

/* Row r of a cache in pages goes on as row parents[r] was (beam search): the
 * pages that the parent has filled are shared, the partly filled one is copied
 * into page spare[r].  kv gives the sizes and the table (k and v are not
 * used); pools[n_pools] (host array of device pointers, 16-byte aligned) are
 * the K and V pools of every layer, all under this table.  lens[rows],
 * parents[rows] (row numbers), spare[rows] (device u32).  table_out[rows]
 * [max_pages]: the parent's filled pages, then spare[r] where a page was
 * copied, then r's own; lens_out[rows]; spare_out[rows]: r's own partly filled
 * page where spare[r] took its place, else spare[r].  A row that is its own
 * parent keeps its pages and copies nothing.  So rows that begin with
 * max_pages pages and one spare page of their own need no allocator: filled
 * pages are never written again, and the page that a row writes next is its
 * own.  A row whose parent does not exist, has another length than the row, or
 * one past the table comes out with length 0 and page numbers 0xFFFFFFFF.  A
 * partly filled page of the parent that does not exist is passed on as it is (and
 * r keeps spare[r]); one that was to go into a spare page that does not exist is
 * absent.
 * The outputs are not the inputs; spare pages are distinct and in no table.
 * No reference counterpart. */
int catena_mi355x_beam_reorder_paged_bf16(const catena_paged_kv_t *kv, uint16_t *const *pools,
                                          uint32_t n_pools, const uint32_t *lens,
                                          const uint32_t *parents, const uint32_t *spare,
                                          uint32_t *table_out, uint32_t *lens_out,
                                          uint32_t *spare_out);

/* -- a step over requests of different lengths -- */

/* The step's tokens form one list, row after row (a row: a request's place in the
 * table); row r's new ones are starts[r] .. starts[r + 1] - 1.  In order:
 * catena_mi355x_kv_admit_paged finds their places, catena_mi355x_rope_packed_bf16
 * (or _q4) writes them, catena_mi355x_attn_prompt_bf16 lets them attend; rows of
 * one token each also catena_mi355x_attn_paged_bf16 or catena_mi355x_attn_paged_q4.
 * All of it may be captured: lists have a length that the call names, and what lies
 * behind the last token is marked as no token. */

/* Pages for a step.  kv gives the sizes (k, v and table are not used); table[rows]
 * [max_pages] is written in place: row r has lens[r] slots in the pages table[r]
 * [0 .. held[r] - 1] and asks for want[r] more slots.  free_pages[0 .. *free_count - 1]
 * (of num_pages entries at most) is a stack of free pages, its top the last one.
 * A row asks for its tokens if lens[r] + want[r] slots fit the table (else for none),
 * and for the pages that they need and it does not hold.  It is admitted where the
 * tokens asked for by the rows up to it are at most max_tokens, and it needs no page
 * or the pages asked for by the rows up to it are at most *free_count.  So the rows
 * that are refused are behind the admitted ones (but for rows that ask for no page, or
 * do not fit the table), and take nothing.  What a refused row asks for stays in the sums: one
 * that asks for more pages than are free stops all rows behind it that need a page,
 * step after step, until it asks for less; one that asks for more tokens than are left, all
 * rows behind it that ask for any.  So requests that have begun stand in front of those
 * that wait, or a want that is not met is taken back: starts[rows] below the sum
 * of want says that there is one, lens_out[r] == lens[r] with want[r] > 0 which.
 * Admitted rows enter their pages into the table behind those that they hold, the lowest row
 * from the top of the stack.
 * Writes lens_out, held_out (both [rows]), starts[rows + 1], *free_count_out, and for
 * each of the max_tokens places of the list its position token_pos and its slot
 * slot_map = page * page_size + place in the page: token t of row r has position
 * lens[r] + t (seen[r] + t where seen is given, which counts given-up positions too,
 * as in catena_mi355x_rope_qkv_paged_bf16; seen_out[r] then counts the new ones) and
 * goes to slot lens[r] + t.  Places behind the last token have position 0 and slot
 * 0xFFFFFFFFFFFFFFFF, which names no place; so has a token whose page does not exist.
 * The free pages themselves stay as they are.  No output is an input; table entries
 * that are handed out are the only ones written.  No reference counterpart. */
int catena_mi355x_kv_admit_paged(const catena_paged_kv_t *kv, uint32_t *table, const uint32_t *lens,
                                 const uint32_t *held, const uint32_t *want,
                                 const uint32_t *free_pages, const uint32_t *free_count,
                                 uint32_t *lens_out, uint32_t *held_out, uint32_t *starts,
                                 uint32_t *free_count_out, uint32_t *token_pos, uint64_t *slot_map,
                                 uint32_t max_tokens, const uint32_t *seen, uint32_t *seen_out);

/* Rows with finished[r] != 0 have ended: their pages table[r][0 .. held[r] - 1] go
 * onto the stack, in the order of rows and entries, those entries become 0xFFFFFFFF,
 * lens_out[r] and held_out[r] 0; other rows keep theirs.  free_pages is written in
 * place behind *free_count (it has num_pages entries; what would not fit is dropped).
 * The pages must be the row's own.  No output but free_pages and table is an input.
 * No reference counterpart. */
int catena_mi355x_kv_release_paged(const catena_paged_kv_t *kv, uint32_t *table,
                                   const uint32_t *lens, const uint32_t *held,
                                   const uint32_t *finished, uint32_t *free_pages,
                                   const uint32_t *free_count, uint32_t *lens_out,
                                   uint32_t *held_out, uint32_t *free_count_out);

/* Frequencies of rotary positions on the host, in double: out_host[i], i <
 * rotary_dim / 2, from f_i = base^(-2 i / rotary_dim):
 *   PLAIN   f_i
 *   LINEAR  f_i / factor (positions stretched)
 *   BASE    f_i with base * factor^(rotary_dim / (rotary_dim - 2)): the lowest
 *           frequency is divided by factor, the highest kept
 *   PARTS   by the turns f_i makes in the trained length, trained * f_i / (2 pi):
 *           kept from `high` turns on, divided by factor up to `low` turns, a linear
 *           mix of both between
 * No reference counterpart. */
typedef enum catena_rope_scaling {
  CATENA_ROPE_PLAIN = 0,
  CATENA_ROPE_LINEAR = 1,
  CATENA_ROPE_BASE = 2,
  CATENA_ROPE_PARTS = 3
} catena_rope_scaling_t;
int catena_mi355x_rope_inv_freq_scaled(double *out_host, uint32_t rotary_dim, double base,
                                       uint32_t kind, double factor, double trained, double low,
                                       double high);

/* tab[i][j] = mscale * (cos, sin) of (first + i) * inv_freq[j], i < positions, j <
 * rotary_dim / 2, f32: angles, sines and the product in double (inv_freq too, on the
 * device), so that far positions are as good as near ones.  (mscale: the factor that
 * some scalings put on q and k.)  No reference counterpart;
 * catena_mi355x_rope_table_f32 has the reference's sine. */
int catena_mi355x_rope_table_scaled_f32(const double *inv_freq, float *tab, uint32_t first,
                                        uint32_t positions, uint32_t rotary_dim, double mscale);

/* Rotation of a list of tokens and their append: qkv[tokens][(heads + 2 kv_heads) *
 * head_dim] (columns: q heads | k heads | v heads; f32 where qkv_f32 != 0, else bf16).
 * Of each q and k head the first rotary_dim values (a multiple of 16) turn by
 * rope_tab[token_pos][rotary_dim / 2] (cos, sin), in pairs (i, i + rotary_dim / 2), or
 * (2 i, 2 i + 1) where interleaved != 0, each operation rounded to f32 and the results to
 * bf16; the others are rounded alone.  Writes q[tokens][heads][head_dim], k and v into
 * slot slot_map[token] of kv's pools (page * page_size + place; the table is not used),
 * and k_out / v_out[tokens][kv_heads][head_dim] (both or neither).  slot_map may be NULL:
 * no token has a slot.  A token whose slot names no place, or whose position is not
 * below table_positions (it turns by rope_tab's first position), writes q and the
 * copies alone.  No two tokens have the same slot.  qkv, rope_tab, q, k_out and v_out
 * 16-byte aligned.  No reference counterpart. */
int catena_mi355x_rope_packed_bf16(const catena_paged_kv_t *kv, const void *qkv, int qkv_f32,
                                   const float *rope_tab, uint32_t table_positions,
                                   uint32_t rotary_dim, int interleaved, const uint32_t *token_pos,
                                   const uint64_t *slot_map, uint16_t *q, uint64_t tokens,
                                   uint32_t heads, uint16_t *k_out, uint16_t *v_out);

/* Causal attention of packed sequences over a cache in pages: q[tokens][heads]
 * [head_dim] bf16, starts[rows + 1] (device u32), lens[rows] (device u32: a row's
 * slots with the new tokens' among them; past the table: the table's).  Token t of row
 * r's n = starts[r + 1] - starts[r] sees the row's first lens[r] - n + t + 1 slots, n
 * = 1 alone all of them, so prompts, later parts of prompts and single tokens may stand
 * beside each other.  Query head h reads kv head h / (heads / kv_heads).  o[tokens]
 * [heads][head_dim] bf16 RNE: scores, sums and o in f32, p rounded to bf16 (2^-8 of
 * it) in the sum over v and in its own; as catena_mi355x_attn_paged_bf16 has it, to
 * 2^-16, where a row's n tokens are up to 64 query rows of a kv head (n * heads / kv_heads),
 * or the last of them up to 64 behind a multiple of 256.  The same call gives the same bits; where long
 * rows are cut, a row's last bits depend on the rows beside it.  A token that sees no
 * slot gives 0; slots without a page are not seen, and a token whose slots all have none
 * gives NaN.  What lies in slots that a token does not see never reaches it, infinities
 * and NaN included.  Sums of finite values do not overflow (a mean within 2^-8 of the
 * type's largest may); of n slots that a token sees values below n^2 2^-105 lose bits (o is
 * off by n^2 2^-113 more).  An infinity in v makes o infinite where its p is 2^-60 of the
 * largest or more; a smaller p may be 0 beside it, which gives NaN.  starts past `tokens` are cut there, rows that end before they
 * begin have no tokens; places of q and o that belong to no row are not touched.
 * No two rows' tokens overlap.  o is not q, k or v.
 * workspace as for catena_mi355x_attn_paged_bf16, of attn_prompt_plan's size, which is
 * a function of the sizes alone and needs no device (0 for few tokens over tables of up to
 * 1024 slots, else up to 136 MB at 128 columns, 69 at 64, and 64 bytes for every row and
 * 256 query rows).  q and o 16-byte aligned.
 * Allocates nothing; may be captured.  No reference counterpart. */
int catena_mi355x_attn_prompt_plan(const catena_paged_kv_t *kv, uint64_t tokens, uint32_t heads,
                                   uint64_t *workspace_bytes);
int catena_mi355x_attn_prompt_bf16(const catena_paged_kv_t *kv, const uint16_t *q,
                                   const uint32_t *starts, const uint32_t *lens, uint16_t *o,
                                   uint64_t tokens, uint32_t heads, float scale, void *workspace,
                                   uint64_t workspace_bytes);

/* The same over packed keys and values, of prompts with nothing before them: k, v
 * [tokens][kv_heads][head_dim] bf16, token after token kv_stride elements apart (0:
 * kv_heads * head_dim; a multiple of 8, up to 2^25), 16-byte aligned; token t of a row
 * sees the row's tokens 0 .. t.  head_dim 64 or 128.  No reference counterpart
 * (catena_mi355x_attn_causal_bf16 has the reference's exponential and equal lengths). */
int catena_mi355x_attn_packed_plan(uint32_t rows, uint64_t tokens, uint32_t heads,
                                   uint32_t kv_heads, uint32_t head_dim, uint64_t *workspace_bytes);
int catena_mi355x_attn_packed_bf16(const uint16_t *q, const uint16_t *k, const uint16_t *v,
                                   const uint32_t *starts, uint16_t *o, uint32_t rows,
                                   uint64_t tokens, uint32_t heads, uint32_t kv_heads,
                                   uint32_t head_dim, uint64_t kv_stride, float scale,
                                   void *workspace, uint64_t workspace_bytes);

/* A cache in pages held in 4 bits: e2m1 values (code 0 .. 7: 0, .5, 1, 1.5, 2, 3, 4, 6;
 * 8 more: negative), two a byte, the first in the lower half.
 *   k       [num_pages][kv_heads][page_size][head_dim / 2] bytes
 *   k_scale [num_pages][kv_heads][head_dim / 32][page_size] bytes: 32 neighbouring
 *           values of a slot count 2^(byte - 127) each, 255: NaN
 *   v       [num_pages][kv_heads][head_dim / 2][page_size] bytes: byte (i, j) holds
 *           values 2 i and 2 i + 1 of slot j
 *   v_scale [num_pages][kv_heads][page_size] bf16: what a slot's values count
 * Sizes and table as in catena_paged_kv_t; all pools 16-byte aligned.  A slot takes
 * head_dim + head_dim / 32 + 2 bytes a head, 0.26 of bf16's (head_dim 128). */
typedef struct catena_paged_kv4 {
  uint8_t *k;
  uint8_t *v;
  uint8_t *k_scale;
  uint16_t *v_scale;
  const uint32_t *table;
  uint32_t num_pages;
  uint32_t page_size;
  uint32_t rows;
  uint32_t max_pages; /* table entries per row */
  uint32_t kv_heads;
  uint32_t head_dim;
} catena_paged_kv4_t;

/* catena_mi355x_rope_packed_bf16 into a cache in 4 bits.  The bf16 k and v are cut to
 * codes: a block of keys counts the smallest power of two, 2^-127 at least, of which
 * its largest |x| is at most 6; a head's values count a sixth of their largest |x|,
 * rounded up to bf16; each code is the nearest, of two the even one.  A block with an
 * infinity or NaN becomes NaN (and |k| above 3.5 * 2^126 counts 2^128, which bf16 does not
 * hold: an infinity in k_out).  k_out and v_out are the values that the codes stand for, so that a prompt
 * attends to what later steps will: k's exactly, v's, products of a code and a bf16
 * scale, rounded to bf16 (2^-8 of them at most; catena_mi355x_attn_paged_q4 takes them
 * whole).
 * kv_heads <= 128. */
int catena_mi355x_rope_packed_q4(const catena_paged_kv4_t *kv, const void *qkv, int qkv_f32,
                                 const float *rope_tab, uint32_t table_positions,
                                 uint32_t rotary_dim, int interleaved, const uint32_t *token_pos,
                                 const uint64_t *slot_map, uint16_t *q, uint64_t tokens,
                                 uint32_t heads, uint16_t *k_out, uint16_t *v_out);

/* Attention of one new token per row over a cache in 4 bits, as
 * catena_mi355x_attn_paged_bf16 has it: lens, absent pages, rows of no slots, scores
 * and sums in f32 (p to 2^-16), o[rows][heads][head_dim] bf16 RNE; workspace of
 * attn_paged_q4_plan's size.  No reference counterpart. */
int catena_mi355x_attn_paged_q4_plan(const catena_paged_kv4_t *kv, uint32_t heads, uint32_t *parts,
                                     uint64_t *workspace_bytes);
int catena_mi355x_attn_paged_q4(const catena_paged_kv4_t *kv, const uint16_t *q,
                                const uint32_t *lens, uint16_t *o, uint32_t heads, float scale,
                                void *workspace, uint64_t workspace_bytes);

/* Bytes of workspace that catena_mi355x_beam_select_f32 takes.  A function of
 * the sizes alone; needs no device. */
int catena_mi355x_beam_select_plan(uint32_t groups, uint32_t beams, uint32_t vocab,
                                   uint64_t *workspace_bytes);

/* Beam search's selection: of logits[groups][beams][vocab] f32 and scores
 * [groups][beams] f32 (log probabilities so far) the `beams` largest
 *   scores[w] + logits[w][v] - log sum_u exp(logits[w][u])
 * over a group's beams w and tokens v, larger first; equal scores (of two beams:
 * to 2^-42 of them): the lower beam, then the larger logit, then the lower token.
 * A beam's log sum is off by up to 3e-6: its exponentials and their sums by 16 are
 * f32, all further sums f64.  So a beam's own tokens come in the order of their
 * logits, but continuations of two beams that are less than 6e-6 apart may
 * come in either order, and scores_out is off by as much and its rounding to f32.
 * done[groups][beams] u32 (NULL: none): a beam that is not 0 there offers only
 * token eos, at its own score.  Writes per place tokens, parents (rows:
 * group * beams + w), scores_out and done_out (may be NULL): 1 where the
 * parent was done or the token is eos.  eos 0xFFFFFFFF: no token ends a beam
 * (done must then be NULL).  A continuation whose score is not finite is not
 * offered; NaN or +inf among a beam's logits take all of them.  A place that
 * nothing fills has its own row as parent, token 0, score -inf and done 0.
 * For the first step after a prompt give all beams but a group's first the
 * score -inf.  scores_out may be scores, done_out may be done.  1 <= beams <=
 * 32, 1 <= vocab <= 2^26.  workspace as for catena_mi355x_attn_paged_bf16.  No
 * reference counterpart (catena_mi355x_argmax_f32 is the greedy choice). */
int catena_mi355x_beam_select_f32(const float *logits, const float *scores, const uint32_t *done,
                                  uint32_t *tokens, uint32_t *parents, float *scores_out,
                                  uint32_t *done_out, uint32_t groups, uint32_t beams,
                                  uint32_t vocab, uint32_t eos, void *workspace,
                                  uint64_t workspace_bytes);

/* tensor.argmax-f32 per row (catena-lang/stdlib/tensor.hex:204-227):
 * idx[r] = first index of the maximum with the reference's NaN behaviour;
 * n = 0 gives 0xFFFFFFFF (the reference asserts n != 0). */
int catena_mi355x_argmax_f32(const float *x, uint32_t *idx, uint64_t rows, uint64_t n);

/* -- buffer producers and folds (materializec / reducec programs) -- */

/* tensor.broadcast-f32 body (catena-lang/stdlib/tensor.hex:1-21): out[i] = value. */
int catena_mi355x_broadcast_f32(float *out, uint64_t n, float value);
/* tensor.arange-f32 body (catena-lang/stdlib/tensor.hex:23-46): out[i] =
 * u64.to-f32(i), round to nearest even. */
int catena_mi355x_arange_f32(float *out, uint64_t n);
/* Element copy behind tensor.slice-f32 / tensor.concat-f32
 * (catena-lang/stdlib/tensor.hex:48-168); any 4-byte alignment. */
int catena_mi355x_copy_f32(float *dst, const float *src, uint64_t n);
/* sum-f32 / mean-f32 / max-f32 per row (catena-lang/stdlib/sum.hex:29-101):
 * the reference's sequential folds (sum from +0, max-env from -inf),
 * bitwise.  sum / mean: n <= 0xFFFFF800 (longer rows return
 * CATENA_ERR_UNSUPPORTED); max: n < 2^31. */
int catena_mi355x_sum_f32(const float *x, float *out, uint64_t rows, uint64_t n);
int catena_mi355x_mean_f32(const float *x, float *out, uint64_t rows, uint64_t n);
int catena_mi355x_max_f32(const float *x, float *out, uint64_t rows, uint64_t n);
/* sum-u64 / dot-u64 per row (catena-lang/tests/cases/reducec/basic.hex):
 * wrapping u64 arithmetic. */
int catena_mi355x_sum_u64(const uint64_t *x, uint64_t *out, uint64_t rows, uint64_t n);
int catena_mi355x_dot_u64(const uint64_t *a, const uint64_t *b, uint64_t *out, uint64_t rows,
                          uint64_t n);

/* ------------------------------------------------------------------ */
/* program ABI (generated-module symbols; synchronous; fail-stop)        */

/* tests/cases/matrix/matmul.hex:1-63 "matmul-2x2-via-mem":
 * (mem A, mem B, n, m, k, nk, km, nm) -> (mem C).  Asserts nk == len(A)/4 and
 * km == len(B)/4 like the reference, and additionally n*k == nk, k*m == km,
 * n*m == nm (the reference leaves those to its type checker). */
void program_matmul_2x2_via_mem(catena_mem_t a, catena_mem_t b, uint64_t n, uint64_t m,
                                uint64_t k, uint64_t nk, uint64_t km, uint64_t nm,
                                catena_mem_t *out);
/* tests/cases/matrix/matmul.hex:65-106 / :108-147: A * I and I * A. */
void program_matmul_right_identity_2x2_via_mem(catena_mem_t a, uint64_t n, uint64_t nn,
                                               catena_mem_t *out);
void program_matmul_left_identity_2x2_via_mem(catena_mem_t a, uint64_t n, uint64_t nn,
                                              catena_mem_t *out);
/* catena-lang/stdlib/nn.hex:93-122 "nn.softmax": (mem) -> (mem). */
void program_nn_softmax(catena_mem_t x, catena_mem_t *out);
/* catena-lang/stdlib/math.hex:185-199 "math.exp-approx": (f32) -> (f32). */
void program_math_exp_approx(float x, float *out);
/* The scalar stdlib programs, (f32) -> (f32) each, as the reference's
 * generated module exports them (catena-lang/src/codegen/gpu.rs:235-285):
 *   "math.sqrt"            catena-lang/stdlib/math.hex:235-272
 *   "nn.sigmoid"           catena-lang/stdlib/nn.hex:1-12
 *   "nn.silu"              catena-lang/stdlib/nn.hex:15-21
 *   "math.sin-approx"      catena-lang/stdlib/math.hex:1-23
 *   "math.cos-approx"      catena-lang/stdlib/math.hex:25-47
 *   "math.sin-approx-full" catena-lang/stdlib/math.hex:49-103 */
void program_math_sqrt(float x, float *out);
void program_nn_sigmoid(float x, float *out);
void program_nn_silu(float x, float *out);
void program_math_sin_approx(float x, float *out);
void program_math_cos_approx(float x, float *out);
void program_math_sin_approx_full(float x, float *out);
/* bf16 analogue of matmul-2x2-via-mem (no reference counterpart):
 * (mem A bf16, mem B bf16, n, m, k, nk, km, nm) -> (mem C bf16). */
void program_bf16_matmul_via_mem(catena_mem_t a, catena_mem_t b, uint64_t n, uint64_t m,
                                 uint64_t k, uint64_t nk, uint64_t km, uint64_t nm,
                                 catena_mem_t *out);
/* Decode attention as a program (no reference counterpart):
 * (mem q, mem k, mem v, mem lens u32, batch, heads, max_len, head_dim, f32 scale)
 * -> (mem o f32). */
void program_attn_decode_via_mem(catena_mem_t q, catena_mem_t k, catena_mem_t v,
                                 catena_mem_t lens, uint64_t batch, uint64_t heads,
                                 uint64_t max_len, uint64_t head_dim, float scale,
                                 catena_mem_t *out);

/* catena-lang/stdlib/nn.hex:154-182 "nn.rmsnorm": (mem) -> (mem). */
void program_nn_rmsnorm(catena_mem_t x, catena_mem_t *out);
/* catena-lang/stdlib/tensor.hex:204-227 "tensor.argmax-f32": (mem) -> (u64);
 * traps on an empty input like the reference's u64.assert-nz. */
void program_tensor_argmax_f32(catena_mem_t x, uint64_t *out);

/* catena-lang/stdlib/tensor.hex producers: (f32 value, u64 len) -> (mem);
 * (u64 len) -> (mem); (mem, u64 start, u64 len) -> (mem), trapping unless
 * start + len <= len(input); (mem, mem) -> (mem). */
void program_tensor_broadcast_f32(float value, uint64_t len, catena_mem_t *out);
void program_tensor_arange_f32(uint64_t len, catena_mem_t *out);
void program_tensor_slice_f32(catena_mem_t input, uint64_t start, uint64_t len, catena_mem_t *out);
void program_tensor_concat_f32(catena_mem_t a, catena_mem_t b, catena_mem_t *out);
/* catena-lang/stdlib/sum.hex folds: (mem) -> (f32). */
void program_sum_f32(catena_mem_t x, float *out);
void program_mean_f32(catena_mem_t x, float *out);
void program_max_f32(catena_mem_t x, float *out);
/* catena-lang/tests/cases/reducec/basic.hex: (mem) -> (u64); (mem, mem) ->
 * (u64), trapping unless the lengths are equal. */
void program_sum_u64(catena_mem_t x, uint64_t *out);
void program_dot_u64(catena_mem_t a, catena_mem_t b, uint64_t *out);

/* ------------------------------------------------------------------ */
/* decoder (Llama-style blocks composed from the ops above)              */

/* No reference counterpart: the model the two hot contractions serve.
 * Per layer, rows r of the residual stream x (f32):
 *   xn  = bf16(rmsnorm(x));  qkv = xn * W_qkv (f32);  RoPE + cache append;
 *   o   = bf16(attention);   h = x + o * W_o;  hn = bf16(rmsnorm(h));
 *   gu  = hn * W_gu (f32);   a = bf16(silu(gate) * up);  x' = h + a * W_down.
 * Then bf16(rmsnorm(x)) of each sequence's last row times W_lm gives f32
 * logits and greedy argmax the next token.  Weights bf16, row-major NN:
 * W_qkv[d][3d] (columns q heads | k heads | v heads), W_o[d][d],
 * W_gu[d][2F] (gate and up columns interleaved in groups of 64),
 * W_down[F][d], W_lm[d][vocab]; embedding[vocab][d]. */
typedef struct catena_decoder catena_decoder_t;
typedef struct catena_decoder_config {
  uint32_t d_model;  /* = n_heads * head_dim */
  uint32_t n_heads;
  uint32_t head_dim; /* 128 */
  uint32_t ffn_dim;  /* SwiGLU width F */
  uint32_t n_layers;
  uint32_t vocab;
  uint32_t max_batch; /* <= 4096 */
  uint32_t max_len;   /* cache positions per sequence; the attention holds one
                         f32 score per position in LDS: <= 36,720 on gfx950
                         ((163,840 - 16,960) / 4) */
  float rope_base;
} catena_decoder_config_t;
/* create() rejects (CATENA_ERR_UNSUPPORTED) n_heads or n_layers > 4096,
 * ffn_dim > 2^24, vocab > 2^26, d_model > 20,476 (the RMSNorm holds a row
 * and its squares in LDS: 16 + 8 * d_model <= 163,840 B on gfx950) and the
 * limits above. */

typedef enum catena_decoder_tensor {
  CATENA_DEC_EMBED = 0, /* [vocab][d] bf16 */
  CATENA_DEC_W_QKV,     /* per layer [d][3d] bf16 */
  CATENA_DEC_W_O,       /* per layer [d][d] bf16 */
  CATENA_DEC_W_GU,      /* per layer [d][2F] bf16, gate / up interleaved by 64 */
  CATENA_DEC_W_DOWN,    /* per layer [F][d] bf16 */
  CATENA_DEC_W_LM,      /* [d][vocab] bf16 */
  CATENA_DEC_K_CACHE,   /* per layer [max_batch][H][max_len][D] bf16 */
  CATENA_DEC_V_CACHE,   /* per layer, same */
  CATENA_DEC_INV_FREQ,  /* [D/2] f32 */
  /* activations of the last forward call (rows = batch * tokens per
   * sequence; the last layer's values when n_layers > 1) */
  CATENA_DEC_X,         /* [rows][d] f32: residual stream into the last layer */
  CATENA_DEC_XN,        /* [rows][d] bf16 */
  CATENA_DEC_QKV,       /* [rows][3d] f32; not written by a prefill of rows % 256 == 0
                         * (its projection applies RoPE and fills q and the caches in its
                         * epilogue) */
  CATENA_DEC_Q,         /* [rows][d] bf16 (rotated) */
  CATENA_DEC_ATTN,      /* [rows][d] bf16 */
  CATENA_DEC_ATTN_PROJ, /* [rows][d] f32 */
  CATENA_DEC_H,         /* [rows][d] f32 */
  CATENA_DEC_HN,        /* [rows][d] bf16 */
  CATENA_DEC_GU,        /* [rows][2F] f32, gate / up interleaved by 64; not written by a
                         * prefill of rows % 256 == 0 (the SwiGLU gate runs in the GEMM's
                         * epilogue) */
  CATENA_DEC_ACT,       /* [rows][F] bf16 */
  CATENA_DEC_FFN_OUT,   /* [rows][d] f32; after a prefill whose W_down runs as k-half
                         * partials (rows % 256 == 0, d % 256 == 0, d_ff % 256 == 0, at
                         * most 128 tiles of 256 x 256) only the rows the final norm reads
                         * (each sequence's last) hold the sum */
  CATENA_DEC_FINAL_H,   /* [batch][d] f32: residual stream at the last rows */
  CATENA_DEC_FINAL_XN,  /* [batch][d] bf16 */
  CATENA_DEC_LOGITS,    /* [batch][vocab] f32 */
  CATENA_DEC_LENS,      /* [batch] u32: cache positions per sequence */
  /* [vocab + 1][d] bf16: bf16(rmsnorm(widen(embed[t]))) for every token t,
   * row vocab all NaN (the row of a token out of range); rebuilt by
   * init_weights and, once decoder_tensor(CATENA_DEC_EMBED) has handed out
   * the embedding (which the caller may then write through at any time), at
   * the start of every prefill and generate call (one pass over vocab rows
   * per call, not per step).  A decode step
   * gathers layer 0's normalized input from it, so in a decode step layer
   * 0 writes neither CATENA_DEC_X nor CATENA_DEC_XN. */
  CATENA_DEC_EMBED_NORM,
  CATENA_DEC_TENSOR_COUNT
} catena_decoder_tensor_t;

int catena_mi355x_decoder_create(const catena_decoder_config_t *cfg, catena_decoder_t **out);
void catena_mi355x_decoder_destroy(catena_decoder_t *dec);
/* Device memory owned by the decoder (weights can be written through it). */
int catena_mi355x_decoder_tensor(catena_decoder_t *dec, uint32_t which, uint32_t layer,
                                 catena_mem_t *out);
/* Every weight ~ N(0, std) in bf16 from the seeded counter generator. */
int catena_mi355x_decoder_init_weights(catena_decoder_t *dec, uint64_t seed, float std);
/* Prefill `tokens` (device u32 [batch][t]) into an empty cache, then write
 * each sequence's greedy next token to next (device u32 [batch]). */
int catena_mi355x_decoder_prefill(catena_decoder_t *dec, const uint32_t *tokens,
                                  uint32_t batch, uint32_t t, uint32_t *next);
/* `steps` greedy decode steps after a prefill: step s appends tokens
 * out[s-1] (out[-1] = the prefill's next) and writes out[s][batch].  out is
 * device u32 [steps][batch].  Fails when the cache would overflow. */
int catena_mi355x_decoder_generate(catena_decoder_t *dec, uint32_t steps, uint32_t *out);

/* ------------------------------------------------------------------ */
/* runtime mirror                                                         */

/* ValueKind, catena-lang/src/runtime/value.rs:15-21 */
typedef enum catena_value_kind {
  CATENA_VALUE_BOOL = 0,
  CATENA_VALUE_U32 = 1,
  CATENA_VALUE_U64 = 2,
  CATENA_VALUE_F32 = 3,
  CATENA_VALUE_MEM = 4
} catena_value_kind_t;

/* Value, catena-lang/src/runtime/value.rs:5-12 */
typedef struct catena_value {
  catena_value_kind_t kind;
  union {
    uint8_t b;
    uint32_t u32;
    uint64_t u64;
    float f32;
    catena_mem_t mem;
  } as;
} catena_value_t;

/* ExecError / InitError kinds, catena-lang/src/runtime/runtime.rs:36-102 */
typedef enum catena_exec_status {
  CATENA_EXEC_OK = 0,
  CATENA_EXEC_UNKNOWN_SOURCE_FUNCTION = 1,
  CATENA_EXEC_INPUT_ARITY_MISMATCH = 2,
  CATENA_EXEC_OUTPUT_ARITY_MISMATCH = 3,
  CATENA_EXEC_TYPE_MISMATCH = 4,
  CATENA_INIT_PARSE = 10,
  CATENA_INIT_NO_LOWERING = 11,
  CATENA_INIT_SIGNATURE_MISMATCH = 12,
  CATENA_INIT_DIALECT = 13,
  CATENA_INIT_DEVICE = 14,
  /* not reference error kinds: host memory ran out while reading sources;
   * a NULL runtime, name, source list, argument or output array */
  CATENA_INIT_HOST_MEMORY = 15,
  CATENA_EXEC_BAD_CALL = 20
} catena_exec_status_t;

typedef struct catena_runtime catena_runtime_t;

/* Runtime::from_sources (catena-lang/src/runtime/runtime.rs:115-121).
 * `dialect` is "hip" (the only accepted GpuDialect here).  Sources are
 * scanned for `(def program NAME : TYPE = ...)` forms; every declared
 * program with a native lowering becomes executable, its signature taken
 * from the declared type. */
int catena_runtime_from_sources(const char *const *sources, size_t n_sources,
                                const char *dialect, catena_runtime_t **out);
void catena_runtime_destroy(catena_runtime_t *rt);
/* Runtime::exec (catena-lang/src/runtime/runtime.rs:175-236): validation in
 * the reference's order (unknown name, input arity, output arity, kinds);
 * outputs are written to outs[0..n_outs). */
int catena_runtime_exec(catena_runtime_t *rt, const char *name, const catena_value_t *args,
                        size_t n_args, catena_value_t *outs, size_t n_outs);
/* Details of the last runtime error on this thread (index / expected /
 * actual for TypeMismatch, expected / actual counts for arity errors). */
int catena_runtime_last_error_detail(int64_t *index, int64_t *expected, int64_t *actual);
/* Number of executable programs and their names (for listing). */
size_t catena_runtime_program_count(const catena_runtime_t *rt);
const char *catena_runtime_program_name(const catena_runtime_t *rt, size_t i);
/* Runtime::mem_u64 / mem_f32 (catena-lang/src/runtime/runtime.rs:166-172). */
int catena_runtime_mem_u64(catena_runtime_t *rt, const uint64_t *values, size_t n,
                           catena_value_t *out);
int catena_runtime_mem_f32(catena_runtime_t *rt, const float *values, size_t n,
                           catena_value_t *out);

#ifdef __cplusplus
}
#endif
#endif
