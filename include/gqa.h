/*
 * gqa.h -- C ABI of libgqa.so, the MI355X (gfx950) GQA streaming-attention engine.
 *
 * The library replaces the PS->PL hardware boundary of the LARA KV260 accelerator
 * (CSR block + AXI-Stream K/V/Q sink + O source) with device-resident K/V caches in
 * HBM and hand-written HIP kernels.  Every entry point below names the reference
 * interface it stands in for (paths are relative to the reference repository).
 *
 * Conventions
 *   - bf16 tensors cross the boundary as raw IEEE bf16 words (uint16_t), exactly the
 *     words sw/attn_driver.py:88-98 (fp32_to_bf16_u16) produces.
 *   - Host buffers are caller-owned; the library never frees or retains them.
 *   - Every function returns a status code: 0 = OK, otherwise one of GQA_ERR_*.
 *     Codes 0x01..0x12 keep the values of error_code_t (hw/rtl/pkg/attn_pkg.sv:279-286).
 *   - Calls on one context are serialised by the caller (one transaction at a time,
 *     like the reference's start_ready handshake).  Separate contexts are independent.
 *   - K/V cache layout in HBM: [B][H_kv][L_cap][D] bf16, row stride D*2 bytes, where
 *     L_cap = max_seq_len rounded up to a multiple of 64.  Element (b, h, t, d) lives at
 *     ((b*H_kv + h)*L_cap + t)*D + d -- per (b, h) this is the token*HEAD_DIM + dim
 *     addressing of hw/rtl/mem/kv_cache_ram.sv:77-83.
 */
#ifndef LARA_GQA_H
#define LARA_GQA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---------------------------------------------------------- */
#define GQA_OK                 0x00
#define GQA_ERR_BAD_CFG        0x01 /* ERR_BAD_CFG    attn_pkg.sv:281 */
#define GQA_ERR_BUSY_START     0x02 /* ERR_BUSY_START attn_pkg.sv:282 */
#define GQA_ERR_STREAM_LEN     0x10 /* ERR_STREAM_LEN attn_pkg.sv:283: payload size mismatch */
#define GQA_ERR_STREAM_DEST    0x11 /* ERR_STREAM_DEST attn_pkg.sv:284: bad destination/index */
#define GQA_ERR_RESULT_LEN     0x12 /* ERR_RESULT_LEN attn_pkg.sv:285: output size mismatch */
#define GQA_ERR_HIP            0x20 /* a HIP runtime call failed */
#define GQA_ERR_OOM            0x21 /* device, pinned or host allocation failed, or sizes past any memory */
#define GQA_ERR_NO_DEVICE      0x22 /* no usable gfx950 device */
#define GQA_ERR_NULL           0x23 /* required pointer argument is NULL */
#define GQA_ERR_RANGE          0x24 /* length / position outside the configured capacity */
#define GQA_ERR_TIMEOUT        0x25 /* gqa_wait deadline expired */
#define GQA_ERR_NO_TRANSACTION 0x26 /* start/wait/read with nothing submitted */
#define GQA_ERR_UNSUPPORTED    0x27 /* shape with no compiled kernel (head_dim, group) */
#define GQA_ERR_SCRATCH        0x28 /* plan exceeds GQA_NOALLOC_SCRATCH_BYTES (gqa_decode_append_noalloc) */

/* STATUS word bits returned by gqa_status (CSR_STATUS, attn_driver.py:51-57). */
#define GQA_STATUS_START_READY (1u << 0)
#define GQA_STATUS_BUSY        (1u << 1)
#define GQA_STATUS_DONE        (1u << 2)
#define GQA_STATUS_ERROR       (1u << 3)

/* Per-kernel timer slots reported by gqa_kernel_times. */
#define GQA_TIMER_APPEND  0 /* rows into the cache; E4M3: also its rows read back (gqa_read_kv, prefill) */
#define GQA_TIMER_DECODE  1
#define GQA_TIMER_COMBINE 2 /* log-sum-exp merge launch of split-KV decode or segmented prefill */
#define GQA_TIMER_PREFILL 3
#define GQA_TIMER_NORM    4 /* layer stage: RMSNorm (gqa_layer_qkv_device) */
#define GQA_TIMER_PROJECTION 5 /* layer stage: the QKV projection's hipBLASLt kernels, between two recorded events;
                                  gqa_w4_project_device */
#define GQA_TIMER_ROPE    6 /* layer stage: RoPE + scatter; gqa_qk_norm_rope_device, _step_device */
#define GQA_TIMER_COUNT   7

/* Tunables for gqa_set_option. */
#define GQA_OPT_DECODE_CHUNK 1 /* keys per split-KV work-group (a multiple of 64 giving at most max(l_cap / 256,
                                  the automatic plan's) splits; a last split of <= chunk/4 keys joins the one
                                  before it; 0 = auto: about 8 waves per CU, whole 16-key rounds per wave, or,
                                  for K/V of at most 16 MiB, in 64-key steps about 112 work-groups per 256 CUs
                                  that merge in the decode launch).
                                  The automatic plan does not split a (sequence, kv head) whose K/V take
                                  at most 128 KiB (256 KiB from 32 of them on).  Work-groups have 8 waves, or
                                  4 when the 8-wave plan has at most 8 work-groups (the automatic chunk is
                                  then planned for 4).
                                  E4M3 contexts: rounded up to a power of two of 256 .. 2^30 keys, and no split
                                  where that gives more than 16 pieces per CU (the pieces are then shared out in
                                  equal runs, two per CU).  0: one work-group for a (sequence, kv head) whose K/V
                                  take at most 128 KiB (256 KiB from 32 of them on, 640 KiB from half as many as
                                  CUs on); else pieces for up to one work-group per CU while there are at most a
                                  quarter as many as CUs, else equal runs.  The device forms and prepared steps plan
                                  with max_seq_len for the length: a few short sequences in a large context take
                                  longer than in one of their own size (decode_kv8.hip has figures) */
#define GQA_OPT_PROFILE      2 /* 1 = time every kernel launch with a HIP event pair bound to the launch
                                  (hipExtLaunchKernel; restarts the record).  Binding adds no GPU work
                                  between launches, but each timed launch costs the host several us,
                                  so launches run back to back only if queued ahead of the GPU */
#define GQA_OPT_PREFILL_WGS  3 /* prefill work-groups the KV segmentation aims for (0 = auto: one per CU, 1 = none) */
#define GQA_OPT_NUMERICS     4 /* GQA_NUMERICS_*: arithmetic of prefill / transactions (decode: EXACT only) */
#define GQA_OPT_DECODE_MERGE 5 /* GQA_DECODE_MERGE_*: how split-KV decode merges a sequence's splits */
#define GQA_OPT_PREFILL_KERNEL 6 /* GQA_PREFILL_KERNEL_*: decomposition of prefill / transaction launches */
#define GQA_OPT_LAYER        7 /* layered paged context: the cache layer every entry point reads and writes
                                  (0 .. n_layers-1; gqa_create_paged_layers) */

/* Prefill decomposition (GQA_OPT_PREFILL_KERNEL).  SHARED: a work-group per kv head and 8 tasks of 32
 * (query row, head) pairs shares each K/V tile over its GQA group; launches smaller than the GPU are
 * cut into KV segments merged by a second launch (GQA_OPT_PREFILL_WGS).  ROWS: a work-group per
 * (query head, or two of them where one each would take several rounds of the CUs; 32-row block) whose
 * waves split the keys and merge in LDS (one launch, no segments).
 * PAIRED: SHARED whose work-groups each own a long and a short causal row block (last and first),
 * the short one's waves moving to the long one's keys once theirs end, so the work-groups of a causal
 * launch carry equal work (causal launches of group 4 with more than one row block, always planned in
 * one KV segment; others as SHARED).
 * AUTO (default, no segment target set): PAIRED (one segment) for a causal prompt whose rows see no
 * keys before its own and whose SHARED grid holds half to one work-group per CU (a single dispatch
 * round, which longest-first dispatch cannot balance); else, when the SHARED grid without segments has
 * fewer work-groups than the GPU has CUs, ROWS or, where its estimate is the shorter (few rows after
 * thousands of earlier keys), SHARED in one or more KV segments (several not under a capture, not in caches
 * of at most 1024 rows, and on one stream at a time: the first that needs the segments' workspace, then one
 * that asks for it a second time without a launch of that stream in between); else SHARED -- paired when
 * that grid is exactly one work-group per CU (for instance a causal 2048-row chunk after earlier keys at
 * 32q/8kv on 256 CUs), unpaired when larger.  gqa_last_prefill_plan reports the decomposition a launch took.
 * Launches in several segments under a forced decomposition or segment target share a workspace of their own,
 * which these options allocate (a forced decomposition without memory for it takes one segment): the caller
 * orders them among each other (streams, replayed graphs); AUTO's may be in flight beside them. */
#define GQA_PREFILL_KERNEL_AUTO   0
#define GQA_PREFILL_KERNEL_SHARED 1
#define GQA_PREFILL_KERNEL_ROWS   2
#define GQA_PREFILL_KERNEL_PAIRED 3

/* Split merge of the decode (GQA_OPT_DECODE_MERGE).  FUSED: the last split of a (sequence, kv head) to
 * finish merges the others' partials inside the decode launch (agent-scope atomics and a per-unit
 * arrival counter; one launch per step).  LAUNCH: a second, log-sum-exp merge launch.  AUTO (default):
 * FUSED while the split grid (sequences x kv heads x splits) is at most half the GPU's CU count and a
 * sequence has at most 16 splits (32 in the automatic plan's 64-key steps) -- every split ends with an L2
 * write-back of its XCD and an increment of its sequence's counter, which saves the launch for short steps
 * but slows the streaming of larger grids more than a launch costs -- else LAUNCH.  An automatic plan of the
 * shortest splits (one round of every wave) that would need the merge launch takes splits twice as long
 * where that lets AUTO fuse.
 * Both fold the splits in the same order (the same output words).  E4M3 contexts: equal runs always take LAUNCH, and
 * AUTO fuses while the split grid is at most half the GPU's CU count. */
#define GQA_DECODE_MERGE_AUTO   0
#define GQA_DECODE_MERGE_LAUNCH 1
#define GQA_DECODE_MERGE_FUSED  2

/* Numerics of the attention kernels (GQA_OPT_NUMERICS).
 * EXACT: fp32 scores, softmax, sums and accumulation, exact divide; the P.V product takes each
 *        softmax weight rounded to bf16 (RNE; the board truncates it, attn_top.sv:653-658) while
 *        l sums the fp32 weights.  Each output element is within 2 bf16 ulp of its row's largest
 *        |output| of exact attention plus 2^-8 of exact attention over |V| at that element
 *        (sum_k p_k |v_k[d]| / l); the second term matters only where V rows cancel -- otherwise
 *        it lies within the first.
 * KV260: the deployed KV260 datapath bit for bit -- sequential fp32 sums of exact bf16 products,
 *        the 1024-entry interpolated exp table (softmax_engine.sv:570-706), P truncated to bf16
 *        for PV (attn_top.sv:653-658), reciprocal-table normalisation (output_buffer.sv:192-286),
 *        16-key sub-blocks in the board's tile order (attn_core.sv:107-154); for comparing with
 *        board results word for word.  Transactions with q_len == kv_len follow the board's
 *        contract exactly; other shapes use the same walk over their own lengths. */
#define GQA_NUMERICS_EXACT 0
#define GQA_NUMERICS_KV260 1

typedef struct gqa_config {
    int32_t batch;       /* B: sequences resident in the cache                         */
    int32_t n_q_heads;   /* H_q  (N_Q_HEADS, attn_driver.py:65)                         */
    int32_t n_kv_heads;  /* H_kv (N_KV_HEADS, attn_driver.py:66); H_q % H_kv == 0        */
    int32_t head_dim;    /* D    (HEAD_DIM, attn_driver.py:63): 64 or 128               */
    int32_t max_seq_len; /* cache rows per (b, kv head), 1 .. 2^30 (MAX_SEQ_LEN generalised) */
    int32_t max_q_len;   /* largest prefill chunk / transaction length, 1 .. 2^30       */
    float   scale;       /* softmax scale; 0 selects fp32(1/sqrt(D)) (attn_pkg.sv:241)   */
    int32_t device;      /* HIP device ordinal                                          */
} gqa_config;

typedef struct gqa_ctx gqa_ctx;

/* ---- lifetime ---------------------------------------------------------------
 * gqa_create replaces AttentionAccelerator.__init__'s overlay/buffer set-up
 * (sw/attn_driver.py:251-288): it allocates the HBM K/V cache, staging and split-KV
 * workspace and a HIP stream.  gqa_destroy replaces close() (attn_driver.py:324-331). */
int gqa_create(const gqa_config* cfg, gqa_ctx** out_ctx);
int gqa_destroy(gqa_ctx* ctx);
int gqa_get_config(const gqa_ctx* ctx, gqa_config* out_cfg);
int gqa_set_option(gqa_ctx* ctx, int32_t option, int64_t value);
const char* gqa_status_string(int32_t code);
int gqa_device_count(int32_t* out_count);

/* ---- paged K/V cache --------------------------------------------------------
 * No reference counterpart: the KV260 reloads its cache on every transaction
 * (kv_cache_ram.sv:77-91, attn_driver.py:418-422), so it has no cache manager.  A paged
 * context keeps K and V in pools of n_pages pages of page_size rows (a power of two >= 64;
 * layout [n_pages][H_kv][page_size][D]) and one block table per sequence (page of each
 * page_size-row run of token rows, -1 = unmapped).  Every entry point works as on a
 * contiguous context, reading and writing through the tables; host-pointer forms return
 * GQA_ERR_RANGE when a row they touch is unmapped, device forms read unmapped rows as
 * zeros and skip writes to them.  KV260 numerics are not available on a paged context.
 * gqa_paged_reserve maps pages so rows [0, n_rows) of sequence b are backed (GQA_ERR_OOM,
 * changing nothing, when the pool is short); gqa_paged_release returns a sequence's pages;
 * gqa_paged_evict_lru releases whole sequences, least recently used first (reserve, load,
 * prefill and host-pointer decode calls count as uses) and skipping the n_pinned sequence
 * indices in pinned, until n_free_pages pages are free, writing up to max_evicted evicted
 * sequence indices (GQA_ERR_OOM, releasing nothing, if that cannot be reached).  Reserve,
 * release and evict synchronise the context stream; launches on other streams that read a
 * sequence must finish before its pages are released.  gqa_cache_pointers returns the
 * pools and page_size as l_cap. */
int gqa_create_paged(const gqa_config* cfg, int32_t page_size, int32_t n_pages, gqa_ctx** out_ctx);
int gqa_paged_reserve(gqa_ctx* ctx, int32_t b, int32_t n_rows);
int gqa_paged_release(gqa_ctx* ctx, int32_t b);
int gqa_paged_evict_lru(gqa_ctx* ctx, int32_t n_free_pages, const int32_t* pinned, int32_t n_pinned,
                        int32_t* evicted, int32_t max_evicted, int32_t* n_evicted);
int gqa_paged_info(gqa_ctx* ctx, int32_t* page_size, int32_t* n_pages, int32_t* n_free,
                   int32_t* max_pages);
int gqa_paged_table(gqa_ctx* ctx, int32_t b, int32_t* out, int32_t n);

/* ---- multi-layer paged K/V cache ---------------------------------------------
 * No reference counterpart: the board runs one layer per transaction and reloads its cache each
 * time (attn_driver.py:552-586).  gqa_create_paged_layers is gqa_create_paged for a model of
 * n_layers attention layers (1 .. GQA_MAX_LAYERS) sharing one block table per sequence and one
 * page allocator: a page index names the same token rows in every layer, so reserve, release and
 * evict map and unmap a run of tokens for all layers at once.  Each layer has its own pools
 * (layout [n_layers][n_pages][H_kv][page_size][D], K and V apart).  GQA_OPT_LAYER selects the
 * layer that decode, prefill, append, load, read, the layer stage and gqa_cache_pointers address
 * (default 0); switching is a host-side pointer change, ordered with the launches already queued
 * (each launch keeps the pools it was given).  A transaction reads the layer that was active when
 * it was submitted; a captured graph, the layer active at capture.  gqa_paged_layers returns
 * n_layers and the active layer (GQA_ERR_UNSUPPORTED on a contiguous context; gqa_create_paged
 * contexts have one layer). */
#define GQA_MAX_LAYERS 1024
int gqa_create_paged_layers(const gqa_config* cfg, int32_t page_size, int32_t n_pages, int32_t n_layers,
                            gqa_ctx** out_ctx);
int gqa_paged_layers(gqa_ctx* ctx, int32_t* n_layers, int32_t* layer);

/* ---- E4M3 K/V cache -----------------------------------------------------------
 * No reference counterpart (the board's cache holds bf16 words).  gqa_create_kv8 is gqa_create (page_size 0, n_pages 0,
 * n_layers 1) or gqa_create_paged_layers (page_size >= 64) with a cache of one byte per value and one scale byte per row:
 * half the bytes, so about half a decode step's time.  A row is the D values of a token of a kv head, K and V apart;
 * its value is code * 2^(byte - 127), the code an E4M3 number (8 bits, OCP) and byte the least one with
 * 448 * 2^(byte - 127) >= the row's largest finite |x| (1 at the least).  Each value is rounded once, to nearest even:
 * by at most 2^-4 of itself, or 2^-10 * 2^(byte - 127) below 2^-6 * 2^(byte - 127); infinities and NaN become NaN, and
 * finite values beyond 1.875 * 2^127 that value.  Codes and scale bytes of a new context are zero.
 * Every entry point works as on a bf16 context, with bf16 rows crossing the boundary: the rows given to gqa_load_kv,
 * gqa_append_kv, gqa_decode_append, gqa_prefill_append and the layer stage are quantised as they are written (in the
 * same launch for the decode step), attention sees the stored values (those of rows appended by the call too), and
 * gqa_read_kv returns them as bf16, which holds them exactly (but below 2^-133, where only the heads' entry points write).  Device operands are 16-byte aligned, in
 * gqa_load_kv_device and gqa_append_kv_device too.  Differences:
 *   - decode takes every group of 1 .. 16 query heads per kv head; prefill the bf16 kernels' groups.  Decode's error
 *     against exact attention over the stored values is as of the bf16 cache.
 *   - prefill (and transactions) read all kv_len rows back into a bf16 workspace first, however few query rows there are
 *     (16 after 7900 keys of 8 kv heads of 128: 17.5 us, 9.7 over a bf16 cache); the layer stage and the host forms of
 *     load and read pass through it too.  It holds 4 * H_kv * D bytes for each row of the largest such call, rounded up to
 *     a power of two where that can be had; a call that grows it synchronises the device.  Uses of it on several
 *     streams follow each other, and prefill and the layer stage return GQA_ERR_UNSUPPORTED under a stream capture.
 *     Append, decode, the device forms of load and read and the heads' entry points below need no workspace.
 *   - decode in equal runs plans for batch * n_kv_heads * (ceil(max_seq_len / 256) + 1) up to 2^28 (in the host forms, with
 *     the longest length); GQA_ERR_UNSUPPORTED above (a paged context may be sized so without having the rows).
 *   - V rows whose largest magnitude lies outside 2^-100 .. 2^96 may lose accuracy or pass fp32 on their way through
 *     decode's sums (a weight is at most 2^8 before the division, times the row's scale).
 *   - KV260 numerics and gqa_decode_append_noalloc are for bf16 caches.
 * Decode launches of one context share its split partials, as on a bf16 cache: the caller orders them, replays of captured
 * ones among them.
 * gqa_cache_pointers returns the codes' pools; gqa_kv8_scales the active layer's scale bytes ([B][H_kv][L_cap], paged
 * [n_pages][H_kv][page_size]; GQA_ERR_UNSUPPORTED on a bf16 context). */
int gqa_create_kv8(const gqa_config* cfg, int32_t page_size, int32_t n_pages, int32_t n_layers, gqa_ctx** out_ctx);
int gqa_kv8_scales(gqa_ctx* ctx, void** k_scale, void** v_scale);

/* ---- K/V cache --------------------------------------------------------------
 * gqa_load_kv replaces the KV branch of _service_request + _transfer(DEST_K_CACHE /
 * DEST_V_CACHE) (attn_driver.py:378-422) and the cache write of kv_cache_ram.sv:77-83:
 * k, v are host [H_kv][n][D] bf16 words written to rows start_pos..start_pos+n-1 of
 * sequence b.  Bit-exact. */
int gqa_load_kv(gqa_ctx* ctx, int32_t b, int32_t start_pos, int32_t n,
                const uint16_t* k, const uint16_t* v);
/* gqa_append_kv: one new row per sequence (no reference counterpart: the KV260 reloads
 * the whole cache per transaction, attn_driver.py:418-422).  k_rows, v_rows are host
 * [B][H_kv][D]; positions[b] is the row index, or -1 to leave sequence b untouched. */
int gqa_append_kv(gqa_ctx* ctx, const uint16_t* k_rows, const uint16_t* v_rows,
                  const int32_t* positions);
/* gqa_read_kv: copy rows back to the host ([H_kv][n][D] each) for bit-exact checks. */
int gqa_read_kv(gqa_ctx* ctx, int32_t b, int32_t start_pos, int32_t n,
                uint16_t* k, uint16_t* v);

/* ---- attention, synchronous host-pointer forms --------------------------------
 * gqa_decode replaces run_attention (attn_driver.py:469-550) for one new query row per
 * sequence: q is host [B][H_q][D]; ctx_lens[b] keys (rows 0..len-1) are attended,
 * q_head h reads kv head h / (H_q/H_kv) (board_performance.py:182-191).  o is host
 * [B][H_q][D] bf16 words (RNE), lse (optional) is host [B][H_q] natural-log
 * log-sum-exp of the scaled scores.  A sequence with ctx_lens[b] == 0 outputs zeros
 * (output_buffer.sv:276-277 semantics) and lse = -inf. */
int gqa_decode(gqa_ctx* ctx, const uint16_t* q, const int32_t* ctx_lens,
               uint16_t* o, float* lse);
/* gqa_decode_append: one decode step as a single kernel launch -- append one K/V row per
 * sequence (k_rows, v_rows host [B][H_kv][D] at positions[b], -1 = none; the same write
 * gqa_append_kv makes, bit-exact) and attend rows 0..ctx_lens[b]-1, which may include the
 * row just appended.  Replaces the KV-load + run_attention pair of attn_driver.py:418-550
 * for one new token per sequence; outputs as gqa_decode. */
int gqa_decode_append(gqa_ctx* ctx, const uint16_t* q, const uint16_t* k_rows, const uint16_t* v_rows,
                      const int32_t* positions, const int32_t* ctx_lens, uint16_t* o, float* lse);
/* gqa_prefill replaces run_attention for a block of q_len query rows of sequence b
 * against cache rows 0..kv_len-1: q and o are host head-major [H_q][q_len][D]
 * (attn_driver.py:487-488, 464).  Query i sits at absolute position q_pos_base + i,
 * key j at kv_pos_base + j; with causal != 0 key j is valid iff its position <= the
 * query's (softmax_engine.sv:865-871).  Rows with no valid key output zeros, and -inf for lse; a score of NaN (a NaN in
 * the query or in a key that it sees) makes the row and its lse NaN, here and in decode.  A V row that holds an infinity
 * or NaN reaches rows of its 32-row block that the causal mask hides it from, too (their weight of 0 times it). */
int gqa_prefill(gqa_ctx* ctx, int32_t b, const uint16_t* q, int32_t q_len,
                int32_t q_pos_base, int32_t kv_len, int32_t kv_pos_base, int32_t causal,
                uint16_t* o, float* lse);

/* gqa_prefill_append: one chunk of a chunked prefill as a single launch -- place the chunk's
 * own K/V rows (k_rows, v_rows host [H_kv][n_new][D]) at cache rows kv_len-n_new .. kv_len-1 of
 * sequence b (bit-exact, as gqa_load_kv) and attend as gqa_prefill.  Replaces the per-transaction
 * K/V DMA + run_attention pair (attn_driver.py:418-550) when the cache grows chunk by chunk. */
int gqa_prefill_append(gqa_ctx* ctx, int32_t b, const uint16_t* q, const uint16_t* k_rows,
                       const uint16_t* v_rows, int32_t n_new, int32_t q_len, int32_t q_pos_base,
                       int32_t kv_len, int32_t kv_pos_base, int32_t causal, uint16_t* o, float* lse);

/* ---- transaction protocol (configure / start / status / wait_done / readback) -----
 * gqa_submit replaces configure() + the Q DMA (attn_driver.py:364-376, 423-432): it
 * validates the transaction and stages q (host head-major [H_q][q_len][D]) in HBM.
 * gqa_start replaces start() (attn_driver.py:434-437): it launches the kernels
 * asynchronously; GQA_ERR_BUSY_START if a transaction is still running.
 * gqa_status replaces status() (attn_driver.py:439-440) with the STATUS bits above.
 * gqa_wait replaces wait_done (attn_driver.py:442-456): timeout_ms < 0 waits forever.
 * gqa_read_output replaces readback_o (attn_driver.py:458-464); n_words must equal
 * H_q*q_len*D (else GQA_ERR_RESULT_LEN, like CSR_RESULT_LEN).
 * gqa_read_perf replaces read_perf (attn_driver.py:466-467): device-clock ticks of the
 * last transaction (total, kernel-only, copy-only) at clock_mhz. */
int gqa_submit(gqa_ctx* ctx, int32_t b, const uint16_t* q, int32_t q_len,
               int32_t q_pos_base, int32_t kv_len, int32_t kv_pos_base, int32_t causal);
int gqa_start(gqa_ctx* ctx);
int gqa_status(gqa_ctx* ctx, uint32_t* out_status);
int gqa_wait(gqa_ctx* ctx, int32_t timeout_ms);
int gqa_read_output(gqa_ctx* ctx, uint16_t* o, int64_t n_words);
int gqa_read_perf(gqa_ctx* ctx, uint64_t* total_ticks, uint64_t* kernel_ticks,
                  uint64_t* copy_ticks, double* clock_mhz);

/* ---- device-pointer forms (inputs already in HBM; stream may be NULL = ctx stream) --
 * Same semantics as the host forms; all pointers are device pointers.  They enqueue
 * and return without synchronising.  The context stream is a blocking HIP stream: work
 * on it is ordered both ways with the legacy default stream (handle 0, PyTorch's default
 * stream), so passing NULL from code that uses the default stream needs no extra sync.
 * A non-default caller stream gets no such ordering: pass that stream itself.
 * q, k_rows, v_rows and the prefill output o must be 16-byte aligned (the kernels move them
 * in 16-byte vectors; any hipMalloc or PyTorch allocation is), else GQA_ERR_RANGE. */
int gqa_append_kv_device(gqa_ctx* ctx, const void* k_rows, const void* v_rows,
                         const int32_t* positions, void* stream);
int gqa_decode_device(gqa_ctx* ctx, const void* q, const int32_t* ctx_lens,
                      void* o, float* lse, void* stream);
int gqa_decode_append_device(gqa_ctx* ctx, const void* q, const void* k_rows, const void* v_rows,
                             const int32_t* positions, const int32_t* ctx_lens, void* o, float* lse,
                             void* stream);
int gqa_prefill_device(gqa_ctx* ctx, int32_t b, const void* q, int32_t q_len,
                       int32_t q_pos_base, int32_t kv_len, int32_t kv_pos_base,
                       int32_t causal, void* o, float* lse, void* stream);
int gqa_prefill_append_device(gqa_ctx* ctx, int32_t b, const void* q, const void* k_rows,
                              const void* v_rows, int32_t n_new, int32_t q_len, int32_t q_pos_base,
                              int32_t kv_len, int32_t kv_pos_base, int32_t causal, void* o, float* lse,
                              void* stream);
/* gqa_load_kv_device: gqa_load_kv from device memory (k, v are [H_kv][n][D] in HBM). */
int gqa_load_kv_device(gqa_ctx* ctx, int32_t b, int32_t start_pos, int32_t n,
                       const void* k, const void* v, void* stream);
/* gqa_read_kv_device: gqa_read_kv into device memory (k, v are [H_kv][n][D] bf16 in HBM, 16-byte aligned), from a bf16 or
 * an E4M3 cache.  They must overlap neither each other nor the cache (GQA_ERR_RANGE). */
int gqa_read_kv_device(gqa_ctx* ctx, int32_t b, int32_t start_pos, int32_t n, void* k, void* v, void* stream);
/* Device addresses of the K and V caches ([B][H_kv][L_cap][D] bf16, or E4M3 codes) and L_cap. */
int gqa_cache_pointers(gqa_ctx* ctx, void** k_cache, void** v_cache, int32_t* l_cap);

/* ---- decode without allocation ------------------------------------------------------
 * No counterpart in the reference (the board has no allocator to avoid).  For callers that
 * cannot allocate device memory -- code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc: gqa_decode_append_device without a context.  The caller owns every
 * buffer: k_cache and v_cache are [B][H_kv][l_cap][D] bf16 in device memory (l_cap a multiple of
 * 64, >= cfg->max_seq_len; the layout of gqa_create's cache), q, k_rows, v_rows, positions,
 * ctx_lens, o and lse as for gqa_decode_append_device (k_rows = v_rows = positions = NULL:
 * attend only).  cfg supplies B, H_q, H_kv, D, max_seq_len, scale and device (max_q_len is
 * ignored).  The call allocates nothing: the split-KV partials of sequences longer than one split
 * live in a static device array of GQA_NOALLOC_SCRATCH_BYTES per device, held until the process
 * ends (its last 256 bytes are a zero K/V row); a plan that needs more returns GQA_ERR_SCRATCH
 * (the automatic plan needs at most about 9 MiB).  Every call on a device shares that array,
 * which keeps the last call's partials (each call writes every partial it reads): calls that
 * overlap on one device (other streams, other threads) race and must be serialised by the caller.
 * The first call on a device sets the array up (address lookup, zero row; it synchronises the
 * device) and returns GQA_ERR_UNSUPPORTED if `stream` is capturing: make one call before
 * capturing.  Same kernels and split plan as gqa_decode_append_device for the same cfg, so the
 * output words are the same. */
#define GQA_NOALLOC_SCRATCH_BYTES (16u << 20)
int gqa_decode_append_noalloc(const gqa_config* cfg, void* k_cache, void* v_cache, int32_t l_cap, const void* q,
                              const void* k_rows, const void* v_rows, const int32_t* positions,
                              const int32_t* ctx_lens, void* o, float* lse, void* stream);

/* ---- layer input stage (run_layer) -------------------------------------------------
 * Replace the host RMSNorm / QKV projection / RoPE / reshape_to_heads of
 * AttentionAccelerator.run_layer (attn_driver.py:552-576; the absent host_attention module;
 * hw/rtl/ext/rms_norm/rms_norm.sv:7-8, hw/rtl/ext/qkv_projection/qkv_projection.sv:7-8,
 * hw/rtl/core/rope_engine.sv:4-10).  x is [n_tokens][hidden] bf16; wq is
 * [H_q*D][hidden], wk and wv [H_kv*D][hidden] bf16 (out x in, Q = x Wq^T); rms_weight
 * (gamma, [hidden] bf16) may be NULL for no normalisation, else
 * y = x / sqrt(mean(x^2) + rms_eps) * gamma.  With rope != 0 the pair (2p, 2p+1) of each Q
 * head of token t is rotated by (q_pos_base + t) * theta_p and of each K head by
 * (kv_pos_base + t) * theta_p, theta_p = 10000^(-2p/D) in fp32 (hw/data/rope_theta.hex).
 * Positions must stay below 2^24.
 * gqa_submit_layer is gqa_submit for a layer: it uploads x and the weights, writes Q into
 * the transaction's staging and K/V into rows [0, n_tokens) of sequence b, and leaves a
 * transaction (q_len = kv_len = n_tokens) for gqa_start / gqa_wait / gqa_read_output.
 * gqa_layer_qkv_device does the same from device memory without a transaction: Q goes to
 * q_out ([H_q][n_tokens][D], 16-byte aligned, else GQA_ERR_RANGE), K/V to rows
 * [kv_row0, kv_row0 + n_tokens) of sequence b; it
 * allocates its workspace on first use.  The projection of a (token count, hidden) shape keeps
 * hipBLASLt's up to 8 best-ranked algorithms; the first call of the shape outside a stream capture
 * times them on the caller's operands (each run four times, the stream synchronised once per
 * algorithm: a few ms, once) and later calls use the fastest, while calls under a capture use the
 * best-ranked until such a call has run.  The context keeps the last 8 shapes.
 * Calls of up to 16 tokens (8 at hidden 8192) with hidden 1024, 2048, 4096 or 8192, 16-byte aligned
 * operands and outputs apart from them run as one launch of the library's own instead (no workspace, nothing
 * tuned), timed as the projection: the stages' other two times are then about zero.
 * gqa_layer_times returns the device time in us of
 * the RMSNorm, projection and RoPE stages (n <= 3; synchronises) of the last gqa_submit_layer
 * call (GQA_ERR_NO_TRANSACTION when there is none); gqa_layer_qkv_device calls made while
 * GQA_OPT_PROFILE is on record their stages in the GQA_TIMER_NORM / _PROJECTION / _ROPE slots of
 * gqa_kernel_times instead. */
int gqa_submit_layer(gqa_ctx* ctx, int32_t b, const uint16_t* x, int32_t n_tokens, int32_t hidden,
                     const uint16_t* wq, const uint16_t* wk, const uint16_t* wv,
                     const uint16_t* rms_weight, float rms_eps, int32_t q_pos_base,
                     int32_t kv_pos_base, int32_t causal, int32_t rope);
int gqa_layer_qkv_device(gqa_ctx* ctx, int32_t b, const void* x, int32_t n_tokens, int32_t hidden,
                         const void* wq, const void* wk, const void* wv, const void* rms_weight,
                         float rms_eps, int32_t q_pos_base, int32_t kv_pos_base, int32_t kv_row0,
                         int32_t rope, void* q_out, void* stream);
int gqa_layer_times(gqa_ctx* ctx, float* out_us, int32_t n);

/* ---- heads: norms, RoPE and scatter ---------------------------------------------------
 * No reference counterpart (the board's layer has no per-head norms).  For callers that project by themselves (or with
 * gqa_w4_project_device): qkv is [n_tokens][ld] bf16 in device memory, a row the Q heads, the K heads and the V heads of a
 * token, D columns each (ld >= (H_q + 2 H_kv) * D, a multiple of 8).  Each Q head is normalised with q_weight and each K
 * head with k_weight ([D] bf16; NULL: that side is not), y = h / sqrt(mean(h^2) + eps) * w over the head's D values, then
 * the pair (2p, 2p + 1) of each Q and K head is rotated by position * rope_base^(-2p/D) (rope_base 0: no rotation, else
 * > 1), then Q goes to q_out and K and V into the cache, bf16 or E4M3.  fp32 up to one rounding, angles in 64 bits (the
 * layer stage rounds the angle to fp32 as the board does: its rotations differ from these by up to 2^-24 of the angle).
 * gqa_qk_norm_rope_device: the tokens of sequence b; Q at positions q_pos_base .., K at kv_pos_base .., cache rows
 * kv_row0 ..; q_out is [H_q][n_tokens][D].
 * gqa_qk_norm_rope_step_device: one token of each sequence (n_tokens = batch): positions [B] and rows [B] in device
 * memory, rows NULL for rows = positions; q_out is [B][H_q][D].  A sequence with a negative position, or a row outside
 * 0 .. max_seq_len - 1, is left out: neither its Q nor its cache is written.  Positions of sequences that are not left
 * out stay below 2^30.
 * Sums of squares are fp32: a head with a magnitude above 2^60 may come out as zeros where it is normalised.
 * ld is a multiple of 8 below 2^31.  qkv, q_out and the cache must not overlap, nor the weights and q_out, and all
 * operands are 16-byte aligned (positions and rows 4-byte), else GQA_ERR_RANGE. */
int gqa_qk_norm_rope_device(gqa_ctx* ctx, int32_t b, const void* qkv, int64_t ld, int32_t n_tokens, const void* q_weight,
                            const void* k_weight, float eps, int32_t q_pos_base, int32_t kv_pos_base, int32_t kv_row0,
                            double rope_base, void* q_out, void* stream);
int gqa_qk_norm_rope_step_device(gqa_ctx* ctx, const void* qkv, int64_t ld, const void* q_weight, const void* k_weight,
                                 float eps, const int32_t* positions, const int32_t* rows, double rope_base, void* q_out,
                                 void* stream);

/* ---- 4-bit weights -----------------------------------------------------------------------
 * No reference counterpart.  The projection of a few tokens is the stream of its weights; 4-bit ones are a quarter of
 * it.  A matrix [rows][hidden] has codes c of 0 .. 15 and one bf16 scale s per row and group of `group` columns (32, 64 or
 * 128, dividing hidden; other groups: GQA_ERR_UNSUPPORTED): w = (c - 8) * s.  rows up to 2^20, hidden up to 2^16.
 * gqa_w4_pack_device lays codes [rows][hidden / 2] (a byte: the even column in its low four bits) and scales
 * [rows][hidden / group] out for the products, once; gqa_w4_bytes gives the sizes of the two results.
 * gqa_w4_project_device: y [n_tokens][ldy] bf16 (the first `rows` of each row) = norm(x) W^T for x [n_tokens][hidden] bf16,
 * norm(x) = x / sqrt(mean(x^2) + rms_eps) * rms_weight, or x with rms_weight NULL.  x * rms_weight is rounded to bf16,
 * sums are fp32, of (128 + c) x and -136 x before the scale: a token whose |x * rms_weight| passes 2^112, or that is
 * not finite, may give NaN in every row, and one with |x| above 2^55 zeros where it is normalised.  n_tokens up to GQA_W4_MAX_TOKENS, ldy below 2^31; a token's result does not
 * depend on the others of the call.
 * gqa_w4_unpack_device: the packed matrix as bf16 [rows][hidden], for long prompts (gqa_layer_qkv_device).
 * The context gives device and stream.  Operands are 16-byte aligned (codes any, scales and y 2-byte) and outputs must
 * not overlap inputs, else GQA_ERR_RANGE.  None of these calls allocates or synchronises. */
#define GQA_W4_MAX_TOKENS (1 << 16)
int gqa_w4_bytes(int32_t rows, int32_t hidden, int32_t group, int64_t* w_bytes, int64_t* scale_bytes);
int gqa_w4_pack_device(gqa_ctx* ctx, const void* codes, const void* scales, int32_t rows, int32_t hidden, int32_t group,
                       void* w, void* w_scales, void* stream);
int gqa_w4_unpack_device(gqa_ctx* ctx, const void* w, const void* w_scales, int32_t rows, int32_t hidden, int32_t group,
                         void* out, void* stream);
int gqa_w4_project_device(gqa_ctx* ctx, const void* x, int32_t n_tokens, int32_t hidden, const void* w,
                          const void* w_scales, int32_t group, int32_t rows, const void* rms_weight, float rms_eps, void* y,
                          int64_t ldy, void* stream);

/* ---- prepared decode steps ---------------------------------------------------------
 * No reference counterpart (the board's transaction is driven by CSR writes).  For serving loops
 * that replay one step shape over fixed device buffers.  gqa_graph_capture_decode_append plans one
 * gqa_decode_append_device step (k_rows = v_rows = positions = NULL: gqa_decode_device) over these
 * device pointers -- split plan sized for max_seq_len, kernel arguments bound -- and launches
 * nothing; gqa_graph_launch launches that step on `stream` (NULL = the context stream), reading q,
 * rows, positions and ctx_lens and writing o, lse and the cache at the bound addresses, so the
 * caller updates those buffers in place between launches.  A launch is the eager step's kernels
 * without the planning: no slower than gqa_decode_append_device.  (A HIP graph of the same step,
 * replayed back to back on this ROCm, cost 4.6 us more GPU time per replay and about 15 us of host
 * time per launch: B1 x 4097 keys 12.9 us against 8.3 eager.)  Callers that need a real HIP graph
 * capture gqa_decode_append_device or gqa_decode_append_noalloc in their own stream capture:
 * those calls enqueue only kernel launches (no allocation, synchronisation or memset).  A prepared
 * step must be destroyed before its context; profiling timers do not record its launches. */
typedef struct gqa_graph gqa_graph;
int gqa_graph_capture_decode_append(gqa_ctx* ctx, const void* q, const void* k_rows, const void* v_rows,
                                    const int32_t* positions, const int32_t* ctx_lens, void* o,
                                    float* lse, gqa_graph** out_graph);
int gqa_graph_launch(gqa_graph* graph, void* stream);
int gqa_graph_destroy(gqa_graph* graph);

/* ---- measurement -----------------------------------------------------------------
 * gqa_stream_read_device: no reference counterpart (the board harness reports against its own
 * measured PL clock, sw/board_performance.py:237-273).  Reads n_bytes (a multiple of 16) of device
 * memory at src the way the decode kernel streams its cache -- 16-byte nontemporal loads, 1 KiB
 * per wave instruction, `unroll` (1, 2, 4 or 8) loads in flight per thread, n_wgs work-groups of
 * 512 threads over contiguous shares -- and writes (almost) nothing (sink: n_wgs words): the
 * measured HBM read ceiling beside the 8 TB/s specification.  Enqueues on `stream` (NULL = the
 * legacy default stream) and returns. */
int gqa_stream_read_device(const void* src, int64_t n_bytes, int32_t n_wgs, int32_t unroll, uint32_t* sink,
                           void* stream);

/* ---- timing ---------------------------------------------------------------------
 * gqa_last_elapsed_us: elapsed time of the last synchronous call (HIP events on the ctx
 * stream).  With GQA_OPT_PROFILE on, every kernel launch is bracketed by HIP events on
 * the stream it runs on (up to 512 launches per kernel; setting the option again
 * restarts the record); gqa_kernel_times returns each kernel's AVERAGE duration in
 * microseconds, indexed by GQA_TIMER_* (0 when it did not run), and
 * gqa_kernel_launch_counts the number of launches averaged.  These replace the PL cycle
 * counters CSR_PERF_* (attn_pkg.sv:274-277) as the source of RunProfile timings. */
int gqa_last_elapsed_us(gqa_ctx* ctx, float* out_us);
int gqa_kernel_times(gqa_ctx* ctx, float* out_us, int32_t n);
int gqa_kernel_launch_counts(gqa_ctx* ctx, int32_t* out_counts, int32_t n);
/* gqa_kernel_durations: the duration (us) of each launch recorded in timer slot `slot` since
 * profiling was (re)started, in launch order, up to n of them (synchronises on them);
 * *n_out = the number recorded. */
int gqa_kernel_durations(gqa_ctx* ctx, int32_t slot, float* out_us, int32_t n, int32_t* n_out);
int gqa_synchronize(gqa_ctx* ctx);
/* gqa_last_prefill_plan: the decomposition (GQA_PREFILL_KERNEL_ROWS, _SHARED or _PAIRED) and the KV
 * segment count of the context's last prefill launch (gqa_prefill*, a transaction, run_layer's
 * attention); 0, 0 before any and after a KV260-numerics launch.  A diagnostic beside read_perf
 * (attn_driver.py:466-467): the board's tiling is fixed (attn_core.sv:107-154), the engine's is
 * chosen per launch, and tests use this to check which decomposition a launch took. */
int gqa_last_prefill_plan(gqa_ctx* ctx, int32_t* kernel, int32_t* n_segs);

/* gqa_last_prefill_row_heads: the query heads per work-group of that launch (1 or 2) where it was
 * GQA_PREFILL_KERNEL_ROWS, else 0. */
int gqa_last_prefill_row_heads(gqa_ctx* ctx, int32_t* heads);

#ifdef __cplusplus
}
#endif
#endif /* LARA_GQA_H */
