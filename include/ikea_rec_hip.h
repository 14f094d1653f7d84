/* C ABI of the MI355X-native GRU4Rec / BidirGRU4Rec / SQN / SMORL training path.
 *
 * Library: ikea-recommender-system_amd/recommenders/hip/libikea_rec_hip.so
 * (hipcc --offload-arch=gfx950; see ikea-recommender-system_amd/build.py).
 *
 * Conventions: every pointer is a device pointer unless documented as host;
 * every call is asynchronous on `stream` (a hipStream_t); return value is
 * 0 (RG_OK) or negative (RG_ERR_ARG -1, RG_ERR_LAUNCH -2, RG_ERR_SHAPE -3).
 * The Python shim (recommenders/hip/__init__.py) turns non-zero returns into
 * RuntimeError, mirroring the reference's exception-only error model.
 * The library owns no memory: callers (PyTorch-ROCm tensors) allocate
 * parameters, Adam moments and workspaces; pointers are borrowed per call.
 *
 * Each entry point names the reference interface it replaces
 * (paths relative to the reference repo root).
 */
#ifndef IKEA_REC_HIP_H
#define IKEA_REC_HIP_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void* rg_stream_t; /* hipStream_t */

/* ---- A4 ragged packing: replaces nn.utils.rnn.pack_padded_sequence(...,
 * enforce_sorted=False) at recommenders/models/GRU4Rec/model.py:70-72 (also
 * BidirGRU4Rec/model.py:79-81, SQN/sqn_gru.py:94-96, SMORL/smorl_gru.py:112-114).
 * lens: int64 (B).  unpacked=1 reproduces use_packed_seq=False (every row runs
 * all L steps, model.py:73-74).  Outputs: perm (B) sorted->original row,
 * lsort (B) lengths descending (stable), offs (B+1) CSR token offsets. */
int rg_pack(const int64_t* lens, int B, int L, int unpacked, int32_t* perm, int32_t* lsort, int32_t* offs,
            rg_stream_t stream);

/* ---- A3 embedding gather: replaces self.embedding(s) (nn.Embedding forward,
 * GRU4Rec/model.py:69,74).  Writes only the T valid tokens, packed (T, E), and
 * their int32 ids.  reverse=1: tokens of a row in reverse time order (the
 * backward direction of BidirGRU4Rec, BidirGRU4Rec/model.py:51-58).  Ids
 * outside [0, n_rows) (nn.Embedding raises) gather zeros, get tok_id -1 and
 * set *err |= 1 (err optional). */
int rg_gather(const int64_t* s, int B, int L, const int32_t* perm, const int32_t* lsort, const int32_t* offs,
              const float* emb, int64_t n_rows, int E, int reverse, int32_t* tok_id, float* X, int32_t* err,
              rg_stream_t stream);

/* ---- A3 embedding backward: replaces embedding_dense_backward (autograd of
 * nn.Embedding, incl. padding_idx masking when train_pad_embed=False,
 * GRU4Rec/model.py:36-47).  Deterministic, atomic-free scatter-add (csrc/segsum.hip): rows
 * i < *n_ptr (n_max the host bound) with a valid id != skip_id are added into a kept-zero
 * (n_rows, E) table G — keys sorted (stable radix sort), each row's contributions summed in
 * row order, so the result does not depend on scheduling — and tagged with `tag` for
 * rg_adam_rows.  Also the sampled head's row gradients.  work: rg_scatter_rows_work_bytes;
 * reuse_sort = 1 reuses the sorted order of the previous call on the same work buffer (same ids,
 * n_ptr, n_max, skip_id, n_rows): a second source over the same rows (the sampled head's bias).
 * Source row i is E floats at src + i·lds (lds >= E; 16-B aligned rows when E % 4 == 0). */
int64_t rg_scatter_rows_work_bytes(int n_max, int E, int64_t n_rows);
int rg_scatter_rows(const int32_t* ids, const float* src, int E, int lds, const int32_t* n_ptr, int n_max,
                    int skip_id, float* G, int64_t n_rows, int32_t* tags, int32_t tag, int reuse_sort, void* work,
                    int64_t work_bytes, rg_stream_t stream);

/* ---- A5 dense contractions of the GRU (input projection W_ih x + b_ih, its
 * input gradient, and the weight gradients of nn.GRU's backward).
 * C(m,n) = sum_k A(m,k) B(k,n) [+ bias(n)], A(m,k)=A[m*sam+k*sak],
 * B(k,n)=B[k*sbk+n*sbn]; Mptr/Kptr (device int, optional) override M/K;
 * splits>1 writes `splits` slabs of M*ldc (sum with rg_reduce_slabs). */
int rg_gemm_f32(const float* A, int64_t sam, int64_t sak, const float* B, int64_t sbk, int64_t sbn, float* C,
                int64_t ldc, const float* bias, int M, const int32_t* Mptr, int N, int K, const int32_t* Kptr,
                int splits, rg_stream_t stream);
int rg_reduce_slabs(const float* slabs, int nslab, int64_t n, float* out, const float* bias, int ncol, int accumulate,
                    rg_stream_t stream);
int rg_colsum(const float* X, int ncol, int rows, const int32_t* rows_ptr, int splits, float* slabs,
              rg_stream_t stream);
/* weight + bias gradient over packed tokens in one pass (nn.GRU backward's
 * dW_ih = dGi^T X, db_ih = sum dGi; dW_hh = dGh^T H_prev, db_hh = sum dGh):
 * dw_slabs (splits x M x N), db_slabs (splits x M); T read from *Tptr;
 * N in {16, 32, 64, 128, 256}, M % 4 == 0; the splits divide the device-side token count evenly. */
int rg_wgrad(const float* G, int M, const float* X, int N, int T_max, const int32_t* Tptr, int splits,
             float* dw_slabs, float* db_slabs, rg_stream_t stream);

/* ---- A5 GRU recurrence: replaces nn.GRU forward over the packed sequence and
 * `h = h[0, :, :]` (GRU4Rec/model.py:76-77; layer 0 only, the reference's
 * quirk).  Gi = packed input projections (T, 3H) incl. b_ih.  The final hidden
 * of each row is written to hout[orig_row*ldh + hoff + :H].  saved (optional,
 * 5 planes of plane floats) keeps h_prev, r, z, n, W_hn h + b_hn for BPTT.
 * H in {16, 32, 64, 128}. */
int rg_gru_fwd(const float* Gi, const float* Whh, const float* bhh, const int32_t* perm, const int32_t* lsort,
               const int32_t* offs, int B, int H, float* hout, int ldh, int hoff, float* saved, int64_t plane,
               rg_stream_t stream);
/* BPTT (autograd of nn.GRU): dh of the final hidden -> dGi (T, 3H) =
 * [da_r, da_z, da_n] and dGh (T, 3H) = [da_r, da_z, da_n*r]. */
int rg_gru_bwd(const float* saved, int64_t plane, const float* Whh, const int32_t* perm, const int32_t* lsort,
               const int32_t* offs, int B, int H, const float* dhout, int lddh, int dhoff, float* dGi, float* dGh,
               rg_stream_t stream);
/* every direction of a bidirectional layer (BidirGRU4Rec/model.py:51-58, 86-90) in ONE launch
 * (grid.y = direction): host arrays of ndir (1 or 2) device pointers; direction d reads / writes
 * columns hoff + d·H of hout (dhoff + d·H of dhout); the packing (perm / lsort / offs) is shared
 * (the backward direction's gather stored its rows time-reversed).  H in {16, 32, 64, 128}. */
int rg_gru_fwd_dirs(const float* const* Gi, const float* const* Whh, const float* const* bhh, float* const* saved,
                    int ndir, const int32_t* perm, const int32_t* lsort, const int32_t* offs, int B, int H,
                    float* hout, int ldh, int hoff, int64_t plane, rg_stream_t stream);
/* the same, also writing the final h as bf16 K-planes of the (B × ldh) matrix (rg_head_plane_bytes(B, ldh)
 * bytes, ldh in {32, 64, 128, 256}) for rg_sampled_logits' h_planes: the split happens once, where h is made. */
int rg_gru_fwd_dirs_planes(const float* const* Gi, const float* const* Whh, const float* const* bhh,
                           float* const* saved, int ndir, const int32_t* perm, const int32_t* lsort,
                           const int32_t* offs, int B, int H, float* hout, int ldh, int hoff, int64_t plane,
                           void* h_planes, rg_stream_t stream);
int rg_gru_bwd_dirs(float* const* saved, const float* const* Whh, float* const* dGi, float* const* dGh, int ndir,
                    int64_t plane, const int32_t* perm, const int32_t* lsort, const int32_t* offs, int B, int H,
                    const float* dhout, int lddh, int dhoff, rg_stream_t stream);

/* ---- A6/A7 full-softmax head: replaces self.output(h) (nn.Linear,
 * GRU4Rec/model.py:58-60,80) + nn.CrossEntropyLoss(mean) (:121,146).
 * Writes Z^T (A x ldz) when ZT != NULL and per-(32-item block, row)
 * (max, sum-exp, argmax) partials (nJ = ceil(A/rg_partial_block()) blocks x B).
 * HF in {16, 32, 64, 128, 256}. */
int rg_head_fwd(const float* h, const float* W, const float* bias, int B, int A, int HF, float* ZT, int64_t ldz,
                float* pmax, float* psum, int32_t* parg, int want_sum, rg_stream_t stream);
/* scratch bytes rg_head_fwd_x needs: B·HF·6 (h's bf16 planes) */
int64_t rg_head_work_bytes(int B, int HF);
/* rg_head_fwd on split-bf16 MFMAs (csrc/head_split.hip): terms = 9 (exact products, fp32
 * accumulation) or 6 (sub-ulp terms dropped); same Zᵀ and partial outputs.  B % 32 == 0,
 * HF in {32, 64, 128, 256}; work: rg_head_work_bytes(B, HF) bytes of device scratch. */
int rg_head_fwd_x(const float* h, const float* W, const float* bias, int B, int A, int HF, int terms, float* ZT,
                  int64_t ldz, float* pmax, float* psum, int32_t* parg, int want_sum, void* work,
                  rg_stream_t stream);
/* ---- A6/A7/A8 fused training head (csrc/head_flash.hip): the full-softmax
 * Linear + CrossEntropyLoss(mean) + Adam step of GRU4Rec/model.py:58-60, 80,
 * 121, 146, 149-153 without materialising the (B × A) logits, on split-bf16
 * MFMAs (terms 9: exact products, 6: sub-ulp terms dropped; 636 = precision
 * "f32x6d3": logits at 6 products, pass 1's O = P·W (-> dh) at the 3 leading
 * ones, dW at 6; rg_flash_amax_fwd reads it as its logits' 6).  HF in
 * {32, 64, 128, 256}; B % 32 == 0.  Multi-GPU item shards pass their first item `lo` and
 * merge lse over ranks between rg_flash_lse and rg_flash_rows.
 * rg_head_plane_bytes: bytes of one operand-plane buffer for `rows` rows.
 * rg_head_planes: X (rows × HF) -> K-planes / R-planes (either optional);
 *   with bias: bias_pad (rows rounded up to 32, -inf padded).
 * rg_flash_fwd: pass 1 — per (split, row) running max pm and Σexp pl (log2
 *   units) and O = Σ_j 2^(z_j − m)·W_j (nsplit × HF × B).
 * rg_flash_lse: lse (natural units) over the splits; zt = the target logit
 *   when the target is one of items [lo, lo + A), 0 when another shard holds
 *   it, NaN when it lies outside [0, A_full) (CrossEntropyLoss raises there).
 * rg_flash_rows: row records, B × 8 bytes, B % 32 == 0 (else RG_ERR_ARG): per 32-row chunk
 *   c, 64 floats — the 32 rows' lse·log2 e, then their targets − lo (int32 bits; -1 outside
 *   [0, A)).
 * rg_flash_dh: dh = gscale·(Σ_s 2^(m_s − lse)·O_s − W[target]) (B × HF).
 * rg_flash_dw_adam: pass 2 — dW = dZᵀ·h, db = Σ_b dZ, then Adam (adam6, host
 *   array) on W / bias / moments; with dW_out / db_out the raw gradients. */
int64_t rg_head_plane_bytes(int rows, int HF);
int rg_head_planes(const float* X, int rows, int HF, void* planes_k, void* planes_r, const float* bias,
                   float* bias_pad, rg_stream_t stream);
int rg_flash_fwd(const void* Hk, const void* Wk, const void* Wr, const float* bias_pad, int B, int A, int HF,
                 int terms, int nsplit, float* pm, float* pl, float* pO, rg_stream_t stream);
/* ---- fused top-k of the training head's logits (SMORL's diversity / novelty
 * rewards, smorl_gru.py:298-308 -> diversity.py:15-73 / novelty.py:12-47:
 * torch.topk(sup, k) of the supervised logits), no logits stored.
 * rg_flash_rows_per_block: rows of one pass-1 workgroup (row-block size).
 * rg_flash_fwd_top: rg_flash_fwd plus (optional, independent) per-split first maximum
 *   pbest/parg (nsplit × B, item local to the head) and every 32-item chunk's row
 *   maximum cmax (ceil(A/32) × B).  cmax alone is what rg_flash_topk needs, and skips the
 *   per-logit compare-and-select of the first maximum.
 * rg_flash_argmax: top-1 over the splits (first maximum), out = -1 for a row
 *   with no finite logit; out_max optional.
 * rg_flash_topk: canonical top-K (value desc, index asc; K <= 32) from cmax:
 *   candidate chunks are those whose maximum is >= tau - (tol_abs +
 *   tol_rel·|tau|), tau = the K-th largest chunk maximum; their items are
 *   rescored in fp32 (the native fp32 head's fmaf chain over HF, + bias: bitwise
 *   rg_head_fwd's logits).  tau comes from a chip-wide two-stage reduction of
 *   the chunk maxima.  Rows [0, B) of cmax (ceil(A/32) × ldc, ldc >= B: a
 *   ragged row chunk passes its valid rows as B).  cand: B × rg_flash_topk_cap()
 *   int32, ncand: B int32, work: rg_flash_topk_work_bytes(ldc, A, K) bytes.  A
 *   row with more candidate chunks than the cap (massive ties) is scanned whole
 *   (every item re-scored the same way, canonical top-K): the result is exact for
 *   every row; err (optional) counts the rows scanned. */
int rg_flash_rows_per_block(int HF);
/* zs (optional; B a multiple of rg_flash_rows_per_block(HF), else RG_ERR_SHAPE): pass 1
 *   also stores the logits z = h·Wᵀ + b as rg_flash_zs_bytes(B, A) bytes of 32-item × 32-row tiles for
 *   rg_flash_dw_adam_planes (which then skips recomputing them). */
int rg_flash_fwd_top(const void* Hk, const void* Wk, const void* Wr, const float* bias_pad, int B, int A, int HF,
                     int terms, int nsplit, float* pm, float* pl, float* pO, float* pbest, int32_t* parg, float* cmax,
                     float* zs, rg_stream_t stream);
int64_t rg_flash_zs_bytes(int B, int A);
/* rg_flash_score: evaluation scoring (evaluate / update_train_metrics, eval_protocol.py:123-359)
 *   — pass 1's S-part without the O contraction: pm / pl (-> rg_flash_lse), per-split first maximum
 *   (pbest / parg) and every 32-item chunk's row maximum cmax (ceil(A/32) x B, -> rg_flash_topk for
 *   the exact canonical top-K); no (B x A) logits.  terms 6 / 9 (636 reads as 6). */
int rg_flash_score(const void* Hk, const void* Wk, const float* bias_pad, int B, int A, int HF, int terms, int nsplit,
                   float* pm, float* pl, float* pbest, int32_t* parg, float* cmax, rg_stream_t stream);
/* rg_flash_amax_fwd: argmax only (the double-Q target, sqn_gru.py:222-226) — pass 1's S-part on the
 *   K-planes of h and W with per-split first maximum (pbest / parg as rg_flash_fwd_top), no softmax. */
int rg_flash_amax_fwd(const void* Hk, const void* Wk, const float* bias_pad, int B, int A, int HF, int terms,
                      int nsplit, float* pbest, int32_t* parg, rg_stream_t stream);
int rg_flash_argmax(const float* pbest, const int32_t* parg, int nsplit, int B, int32_t* out, float* out_max,
                    rg_stream_t stream);
/* Exact argmax by screening (the same double-Q target at half the MFMA work):
 * rg_flash_amax_screen: rg_flash_amax_fwd on terms = 3 plane products (planes 0-1 only) or 1
 *   (plane 0 only) that also writes every 32-item chunk's row maximum cmax (ceil(A/32) × B); merge
 *   pbest/parg with rg_flash_argmax.  The screened logit is within 3·2^-18 (terms 3) / 3.91e-3
 *   (terms 1) of ||h_b||_2·||W_a||_2 of the fp32 one; tol below must cover twice that.
 * rg_row_norm_max: out[0] = max_a ||W_a||_2 (A × HF rows, HF % 4 == 0).
 * rg_flash_argmax_exact: re-scores in fp32 (fmaf chain over k, + bias) every item of every chunk whose
 *   screened maximum is >= tau − (tol·||h_b||_2·wnorm[0] + 1e-6·|tau|), tau = out_val (rg_flash_argmax's
 *   screening maximum), and writes the first maximum into out_idx / out_val (in place over the
 *   screening result); a row with more than rg_flash_topk_cap() candidate chunks is scanned whole
 *   (the first maximum of every item's fp32 logit) and counted in err (optional).  lim: B floats,
 *   cand: B × rg_flash_topk_cap() int32, ncand: B int32 (work). */
int rg_flash_amax_screen(const void* Hk, const void* Wk, const float* bias_pad, int B, int A, int HF, int nsplit,
                         int terms, float* pbest, int32_t* parg, float* cmax, rg_stream_t stream);
int rg_row_norm_max(const float* W, int64_t A, int HF, float* out, rg_stream_t stream);
int rg_flash_argmax_exact(const float* cmax, int B, int A, const float* h, const float* W, const float* bias, int HF,
                          const float* wnorm, float tol, float* lim, int32_t* cand, int32_t* ncand, int32_t* out_idx,
                          float* out_val, int32_t* err, rg_stream_t stream);
int rg_flash_topk_cap(void);
int64_t rg_flash_topk_work_bytes(int B, int A, int K);
/* rg_flash_topk on the screened chunk maxima of rg_flash_amax_screen (3 plane products): candidate
 * chunks within tol·||h_b||_2·wnorm[0] + 1e-6·|tau| of tau (wnorm: rg_row_norm_max), then the same
 * exact fp32 re-scoring, including the whole-row scan past the candidate cap (err counts those rows). */
int rg_flash_topk_screened(const float* cmax, int ldc, int B, int A, int K, float tol, const float* wnorm,
                           const float* h, const float* W, const float* bias, int HF, int32_t* cand, int32_t* ncand,
                           int32_t* out_idx, float* out_val, int32_t* err, void* work, rg_stream_t stream);
int rg_flash_topk(const float* cmax, int ldc, int B, int A, int K, float tol_abs, float tol_rel, const float* h,
                  const float* W, const float* bias, int HF, int32_t* cand, int32_t* ncand, int32_t* out_idx,
                  float* out_val, int32_t* err, void* work, rg_stream_t stream);
int rg_flash_lse(const float* pm, const float* pl, int nsplit, const float* h, const float* W, const float* bias,
                 const int64_t* tgt, int64_t lo, int A, int64_t A_full, int B, int HF, float* lse, float* zt,
                 rg_stream_t stream);
int rg_flash_rows(const float* lse, const int64_t* tgt, int64_t lo, int A, int B, void* rowinfo, rg_stream_t stream);
int rg_flash_dh(const float* pm, const float* pO, const void* rowinfo, int nsplit, const float* W, float gscale,
                int B, int HF, float* dh, rg_stream_t stream);
int rg_flash_dw_adam(const void* Hk, const void* Hr, const void* Wk, const float* bias_pad, const void* rowinfo,
                     float gscale, int B, int A, int HF, int terms, float* W, float* mW, float* vW, float* bias,
                     float* mb, float* vb, const float* adam6, float* dW_out, float* db_out, rg_stream_t stream);
/* rg_flash_dw_adam (Adam mode) that also writes the updated W as the next pass 1's operand
 * planes (Wk_out / Wr_out, rg_head_planes layout; Wk_out may be Wk — a workgroup reads and
 * rewrites only its own items) and the updated bias into bias_pad_out (pad entries untouched):
 * rg_head_planes of the new W is then not needed before the next rg_flash_fwd.  Wk_out, Wr_out
 * and bias_pad_out together or all NULL; not with dW_out.  work (rg_flash_dw_work_bytes(B, A, HF)
 * bytes; optional): the item blocks past the last whole round of 256 workgroups are then split
 * over the row chunks (partial dW / db summed in order by a finishing kernel).  zs: the logits
 * pass 1 stored (rg_flash_fwd_top, same h / W / b): read instead of recomputed (no K-planes of h
 * or W are read then). */
int rg_flash_dw_adam_planes(const void* Hk, const void* Hr, const void* Wk, const float* bias_pad,
                            const void* rowinfo, float gscale, int B, int A, int HF, int terms, float* W, float* mW,
                            float* vW, float* bias, float* mb, float* vb, const float* adam6, float* dW_out,
                            float* db_out, void* Wk_out, void* Wr_out, float* bias_pad_out, void* work,
                            int64_t work_bytes, const float* zs, rg_stream_t stream);
int64_t rg_flash_dw_work_bytes(int B, int A, int HF);
/* rg_head_fwd_x from h's planes (rg_head_work_bytes layout) with the rows split
 * over workgroups: rpb rows per workgroup (multiple of 32), parg optional.
 * The sampled softmax's split forward (rg_sampled_fwd_x) runs on it with the
 * gathered negatives' rows as W (A = S). */
int rg_head_fwd_xp(const void* hplanes, const float* W, const float* bias, int B, int A, int HF, int terms, int rpb,
                   float* ZT, int64_t ldz, float* pmax, float* psum, int32_t* parg, int want_sum, rg_stream_t stream);
/* partials -> lse (B), argmax (B) (torch.argmax semantics: first maximum),
 * loss_row (B) = lse - Z[a_b, b], mx (B) = the row maximum.  Every output is
 * optional.  work: 3*min(128,nJ)*B floats. */
int rg_lse_combine(const float* pmax, const float* psum, const int32_t* parg, int B, int nJ, float* work,
                   const float* ZT, int64_t ldz, const int64_t* tgt, int A, float* lse, int32_t* amax,
                   float* loss_row, float* mx, rg_stream_t stream);
int rg_sum_scale(const float* x, int n, float scale, float* out, double* out64, rg_stream_t stream);
/* ---- item-sharded head (multi-GPU; no reference counterpart): rank r owns
 * items [lo, hi).  lse over all items = logsumexp over ranks of the per-rank
 * lse (nr x B, rank-major); zt[b] = Z[a_b, b] if a_b is local else 0 (then
 * summed over ranks); tgt_loc = a - lo; out = a - b elementwise. */
int rg_lse_merge_ranks(const float* lse_r, int nr, int B, float* lse, rg_stream_t stream);
int rg_shard_targets(const float* ZT, int64_t ldz, const int64_t* tgt, int64_t lo, int64_t hi, int B, float* zt,
                     int64_t* tgt_loc, rg_stream_t stream);
int rg_sub(const float* a, const float* b, int n, float* out, rg_stream_t stream);
/* multi-GPU double-Q (config C4, csrc/shard.hip): out[i] = idx[i] - lo if lo <= idx[i] < hi else -1
 * (exactly one of idx64/idx32); rg_q_gather / rg_q_backward skip rows with index -1. */
int rg_shard_index(const int64_t* idx64, const int32_t* idx32, int n, int64_t lo, int64_t hi, int64_t* out,
                   rg_stream_t stream);
/* global argmax per row from nr ranks' (row max, local argmax) (rank-major nr x n); ties -> lowest
 * global index (torch.argmax / sqn_gru.py get_max_action over the whole row) */
int rg_argmax_merge_ranks(const float* mx, const int32_t* am, int nr, int n, int64_t A, int32_t* out,
                          float* out_max, rg_stream_t stream);
/* global canonical top-K per row (value desc, index asc) from nr ranks' local top-K lists (nr x n x K) */
int rg_topk_merge_ranks(const float* vals, const int32_t* idx, int nr, int n, int K, int64_t A, int32_t* out_idx,
                        float* out_val, rg_stream_t stream);
/* backward of CE + Linear w.r.t. h: dh slabs (returns number of slabs > 0). */
int rg_head_dh(const float* ZT, int64_t ldz, const float* lse, const int64_t* tgt, float gscale, const float* W,
               int B, int A, int HF, int splits, float* slabs, rg_stream_t stream);
/* ---- A8 (head part): backward w.r.t. W, b fused with the Adam update of the
 * same rows (torch.optim.Adam.step, GRU4Rec/model.py:149-153).  adam6 (HOST
 * float[6]) = {1-b1, b2, 1-b2, sqrt(1-b2^t), eps, -lr/(1-b1^t)}.  With dW_out /
 * db_out non-NULL the raw gradients are written instead (test hook). */
int rg_head_dw_adam(const float* ZT, int64_t ldz, const float* lse, const int64_t* tgt, float gscale,
                    const float* h, int B, int A, int HF, float* W, float* mW, float* vW, float* bias, float* mb,
                    float* vb, const float* adam6, float* dW_out, float* db_out, rg_stream_t stream);

/* ---- A8 dense Adam sweeps (torch.optim.Adam._single_tensor_adam). */
int rg_adam_dense(float* P, float* M, float* V, float* G, int64_t n, const float* adam6, int zero_grad,
                  rg_stream_t stream);
/* row-sparse gradients (embedding, Q heads) with dense-Adam semantics:
 * untagged rows take g = 0 (moments still decay, p still moves). */
int rg_adam_rows(float* P, float* M, float* V, float* G, const int32_t* tags, int32_t tag, int64_t rows, int cols,
                 const float* adam6, rg_stream_t stream);
/* Catch-up Adam (dense semantics, bitwise): a table read a few rows at a time (the
 * embedding, the sampled head) keeps last[r] = table steps applied to row r and hist (float[8] per
 * step, step s at 8·(s − 1): adam6, RN(1 / adam6[3]), 0) = every step's scalars; a row's zero-gradient steps are replayed only
 * before it is read.  Replaces rg_adam_rows' sweep over every row (GRU4Rec/model.py:124-127,153).
 * rg_lazy_mark_rows: need[id] = stamp for the n int64 ids in [0, rows) and, with S > 0, the S
 *   negatives of draw `counter` (rg_sample_uniform's stream over [0, rows)).
 * rg_lazy_catch_up: rows with need[r] == stamp (need NULL: every row) replay steps
 *   last[r] + 1 .. n_steps with g = 0; P16 (optional) = fp16(P) of those rows; Pb / Mb / Vb
 *   (optional): a one-column companion table (a head's bias) sharing last[].
 * rg_lazy_adam_rows: table step `step` (writes hist row step − 1): rows with tags[r] == tag replay
 *   last[r] + 1 .. step − 1, then step with their gradient rows G (Gb), cleared; last[r] = step.
 *   Rows without a gradient are not touched. */
int rg_lazy_mark_rows(const int64_t* ids, int64_t n, int64_t rows, uint64_t seed, uint64_t counter, int S,
                      int32_t* need, int32_t stamp, rg_stream_t stream);
/* rg_lazy_mark_rows32: need[id − lo] = stamp for the n int32 global ids in [lo, lo + rows) (a row
 *   shard: the ids the ranks requested from it). */
int rg_lazy_mark_rows32(const int32_t* ids, int n, int64_t lo, int64_t rows, int32_t* need, int32_t stamp,
                        rg_stream_t stream);
int rg_lazy_catch_up(float* P, float* M, float* V, int cols, uint16_t* P16, float* Pb, float* Mb, float* Vb,
                     int64_t rows, int32_t* last, const int32_t* need, int32_t stamp, int32_t n_steps, float* hist,
                     rg_stream_t stream);
int rg_lazy_adam_rows(float* P, float* M, float* V, float* G, int cols, uint16_t* P16, float* Pb, float* Mb, float* Vb,
                      float* Gb, int64_t rows, int32_t* last, const int32_t* tags, int32_t tag, int32_t step,
                      float* hist, const float* adam6, rg_stream_t stream);
/* Split-bf16 trunk GEMMs (precision f32x6* / f32x9: terms 6 or 9 plane products of exact
 * 3-way bf16 splits, fp32 accumulation; GRU4Rec/model.py:49-55,76 via nn.GRU).
 * rg_gemm_x6: C = A·Bᵀ (+ bias): A (M × K, row stride lda) k-contiguous; B (N × K) k-contiguous
 *   (b_kcontig = 1) or (K × N) n-contiguous, row stride ldb; K % 32 == 0, N % 4 == 0; M read from
 *   Mptr when given (grid sized for M).  Replaces rg_gemm_f32 for Gi = X·W_ihᵀ + b, dX = dGi·W_ih.
 * rg_wgrad_x6: rg_wgrad's contract (dW, db token-split slabs) on the same arithmetic. */
int rg_gemm_x6(const float* A, int64_t lda, const float* B, int64_t ldb, int b_kcontig, float* C, int64_t ldc,
               const float* bias, int M, const int32_t* Mptr, int N, int K, int terms, rg_stream_t stream);
/* rg_gemm_x6_sk: rg_gemm_x6 with split-K (slab z of C at C + z·slab covers k in the z-th of `splits`
 *   equal 32-aligned ranges; rg_reduce_slabs sums them) and A either (M × K) k-contiguous
 *   (a_kcontig = 1) or (K × M) m-contiguous (a_kcontig = 0, lda = the stride between k rows);
 *   no bias, M from the host (the sampled head's dh = dZ·W_neg and dW_neg = dZᵀ·h). */
int rg_gemm_x6_sk(const float* A, int64_t lda, int a_kcontig, const float* B, int64_t ldb, int b_kcontig, float* C,
                  int64_t ldc, int64_t slab, int M, int N, int K, int splits, int terms, rg_stream_t stream);
int rg_wgrad_x6(const float* G, int M, const float* X, int N, int T_max, const int32_t* Tptr, int splits,
                float* dw_slabs, float* db_slabs, int terms, rg_stream_t stream);
/* split-K weight-gradient slabs summed in order, then Adam (or g_out). */
int rg_adam_slabs(float* P, float* M, float* V, const float* slabs, int nslab, int64_t n, const float* adam6,
                  float* g_out, rg_stream_t stream);

/* ---- A10/A11 Q heads: replaces q_out.gather(1, a) (SQN/sqn_gru.py:221-222,
 * :232) and gather_from_3d (recommenders/utils/tensor_operations.py:4-33).
 * W / bias: HOST arrays of nh device pointers; idx int64 or int32 (one NULL). */
int rg_q_gather(const float* h, int HF, const float* const* W, const float* const* bias, int nh,
                const int64_t* idx64, const int32_t* idx32, int B, float* q, rg_stream_t stream);
/* backward without float atomics: dh += sum_i dq_bi W_i[a_b] (heads in order); writes the
 * gradient contributions rows (nh x B x HF) = dq_bi h_b and rows_b (nh x B) = dq_bi, ids (B,
 * int32, -1 = skipped) and n_rows[0] = B for the sorted scatter rg_scatter_rows into G_i / Gb_i
 * (one sort shared by all heads: reuse_sort). */
int rg_q_backward(const float* h, int HF, const float* const* W, int nh, const int64_t* idx, int B, const float* dq,
                  float* dh, float* rows, float* rows_b, int32_t* ids, int32_t* n_rows, rg_stream_t stream);
/* SQN TD loss (SQN/sqn_gru.py:234-239), f64 like the reference. */
int rg_sqn_td(const float* q, float* qn, const double* r, const uint8_t* is_end, float gamma, int B, double scale,
              double* sq, float* dq, rg_stream_t stream);
/* SMORL weighted TD loss (SMORL/smorl_gru.py:295,317-325; weighted_q_loss
 * tensor_operations.py:36-47). */
int rg_smorl_td(const float* q, float* qn, const float* r, const uint8_t* is_end, const float* w, int nh,
                float gamma, float grad_row, int B, float* row_loss, float* dq, rg_stream_t stream);
int rg_sum64(const double* x, int n, double scale, double* out64, float* out32, rg_stream_t stream);
/* A12 diversity reward: recommenders/evaluate/diversity.py:15-73.  D has Drows
 * rows; a row whose last action or predicted id lies outside [0, Drows) (an
 * unmapped tokenizer id, where the reference's stoi raises KeyError) gets NaN
 * and no table read. */
int rg_diversity(const int64_t* s, int L, const int64_t* lens, int pad_end, const int32_t* idx, int k, int ldi,
                 const float* D, int64_t Drows, int Ed, float eps, int B, float* out, rg_stream_t stream);
/* A13 novelty reward: recommenders/evaluate/novelty.py:12-47 (U as a bitmap
 * over n_items actions); a row with an id outside [0, n_items) gets NaN and no
 * bitmap read. */
int rg_novelty(const int32_t* idx, int k, int ldi, const uint32_t* bitmap, int n_items, float reward, int B,
               float* out, rg_stream_t stream);

/* ---- A14 / A12 / A13 top-k: replaces torch.topk(preds, k) on host-copied
 * (B, A) logits (recommenders/evaluate/eval_protocol.py:75,199; diversity.py:51;
 * novelty.py:33).  Exact; ties ordered (value desc, index asc).  Uses the
 * forward kernel's block maxima pmax (nJ x B) to prune.  out_idx (B, k),
 * out_val (B, k) optional; *err |= 2 on candidate overflow (massive ties). */
int rg_topk(const float* ZT, int64_t ldz, const float* pmax, int B, int A, int k, int32_t* out_idx, float* out_val,
            int32_t* err, rg_stream_t stream);
/* repetition counts (recommenders/evaluate/repetitiveness.py:21-57): out[q] += number of
 * (b, t, j) with s[b, t] == idx[b, j] and j < ks[q] (ks: HOST int array, nk <= 16, k <= K;
 * integer counts, deterministic).  idx: (B, K) predicted ids in the input vocabulary. */
int rg_repetitions(const int64_t* s, int L, const int32_t* idx, int K, int B, const int* ks, int nk,
                   unsigned long long* out, rg_stream_t stream);
/* HR@k / NDCG@k sums (eval_protocol.py:26-100) accumulated into out
 * (2*nk doubles: hits..., ndcg...); ks: HOST int array, k <= K. */
int rg_hits_ndcg(const int32_t* idx, int K, const int64_t* tgt, int B, const int* ks, int nk, double* out,
                 rg_stream_t stream);

/* misc elementwise: y = x * mask * scale (dropout fwd/bwd, BidirGRU4Rec/model.py:60,93) */
int rg_mask_scale(const float* x, const float* mask, float scale, int64_t n, float* y, rg_stream_t stream);
/* W_comb = sum_i w_i W_i (SMORL target weights, tensor_operations.py:50-70) */
int rg_weighted_sum(const float* const* X, const float* w, int nh, int64_t n, float* out, rg_stream_t stream);
/* The SMORL target's combined Q head in one pass (csrc/misc.hip): Wc = sum_i w_i W_i (A × HF),
 * bc = sum_i w_i b_i (as rg_weighted_sum), Wc's K-planes and the -inf padded bias (as
 * rg_head_planes, ceil(A/32)·32 rows) and *wnorm = max_a ||Wc[a]||_2 (for rg_flash_argmax_exact).
 * W, b, w: HOST arrays of nh <= 4 device pointers / weights; HF in {32, 64, 128, 256}.  nplanes 3
 * writes all three K-planes, 1 only plane 0 (what rg_flash_amax_screen with terms = 1 reads). */
int rg_qcomb(const float* const* W, const float* const* b, const float* w, int nh, int A, int HF, int nplanes,
             float* Wc, float* bc, void* planes_k, float* bias_pad, float* wnorm, rg_stream_t stream);
/* replay-buffer transitions from a device session store (csrc/replay.hip; SURVEY §8f rank 2,
 * rules of preprocessing.py:5-29, 143-170, 426-464): sessions as CSR — items (int32) and rewards
 * (f64) per event, ev_sess (int32) the event's session, sess_off (int64, n_sess + 1) — and B event
 * indices ev -> the trainers' batch: s / s_next (B × L int64, pad_id padded at the end when
 * pad_end else at the beginning), a, r, true_len = clamp(n_bef, 1, L), true_next_len =
 * min(n_bef + 1, L), is_end (uint8) */
int rg_build_transitions(const int32_t* items, const double* rew, const int32_t* ev_sess, const int64_t* sess_off,
                         const int64_t* ev, int B, int L, int64_t pad_id, int pad_end, int64_t* s, int64_t* a,
                         double* r, int64_t* s_next, int64_t* len, int64_t* next_len, uint8_t* is_end,
                         rg_stream_t stream);
/* tokenizer remap of predicted ids, output -> input vocabulary (diversity.py:55-60,
 * repetitiveness.py:42-47): out[i] = lut[idx[i]]; an id outside [0, lut_n) or mapped to -1 gives -1
 * and err |= 1 (the reference raises on such an id) */
int rg_remap_ids(const int32_t* idx, int64_t n, const int32_t* lut, int64_t lut_n, int32_t* out, int32_t* err,
                 rg_stream_t stream);
/* SMORL reward matrix r (B, 3) f32 = stack([r_acc f64, r_div, r_nov]) (SMORL/smorl_gru.py:311-314, 3 rewards) */
int rg_stack_rewards(const double* r_acc, const float* r_div, const float* r_nov, int B, float* r, rg_stream_t stream);

/* Persistent wide GRU for H = 256 (config C5), whose W_hh (768 KB) fits neither one CU's VGPRs nor
 * its LDS: same contract as rg_gru_fwd / rg_gru_bwd (GRU4Rec/model.py:49-55, 76-77; one launch for
 * the whole sequence, 32 rows per workgroup, W_hh streamed from L2 as MFMA fragments every step)
 * plus wfrag, rg_gru_wide_work_bytes(H) bytes of device scratch (the fragment copy of W_hh, rebuilt
 * by each call). */
int64_t rg_gru_wide_work_bytes(int H);
int rg_gru_fwd_wide(const float* Gi, const float* Whh, const float* bhh, const int32_t* perm, const int32_t* lsort,
                    const int32_t* offs, int B, int H, float* hout, int ldh, int hoff, float* saved, int64_t plane,
                    void* wfrag, rg_stream_t stream);
int rg_gru_bwd_wide(const float* saved, int64_t plane, const float* Whh, const int32_t* perm, const int32_t* lsort,
                    const int32_t* offs, int B, int H, const float* dhout, int lddh, int dhoff, float* dGi,
                    float* dGh, void* wfrag, rg_stream_t stream);

/* ---- fp16 embedding storage (config C5: the gather reads an fp16 copy of the table, Adam keeps the
 * fp32 master and moments; fp16 = IEEE binary16 bits, round to nearest even) ---- */
int rg_gather_h(const int64_t* s, int B, int L, const int32_t* perm, const int32_t* lsort, const int32_t* offs,
                const uint16_t* emb16, int64_t n_rows, int E, int reverse, int32_t* tok_id, float* X, int32_t* err,
                rg_stream_t stream);
/* ---- A3 gather of a sampled step (north-star "embedding gather + sampled logits"): rg_gather (emb16 = 0)
 * or rg_gather_h (emb16 = 1) with the S negatives' row gather in the same launch — draw `counter` of the
 * counter-based stream (seed, S, A; rg_sample_uniform's ids) -> ids[S], bg = bias[ids], Wg (S, HF) =
 * W[ids] and Wp (S·HF·6 bytes) = the rows' bf16 planes in fragment order for rg_sampled_logits
 * (draw = 2); wfmt 1 (HF <= 128): Wp (S·HF·4 bytes) = the rows as fp32 fragments instead (draw = 3).  E, HF in {32, 64, 128, 256}, L <= 64, S % 32 == 0.  Replaces the nn.Embedding forward
 * (GRU4Rec/model.py:69,74) plus the negatives' row lookup of the build-defined sampled head. */
int rg_gather_neg(const int64_t* s, int B, int L, const int32_t* perm, const int32_t* lsort, const int32_t* offs,
                  const void* emb, int emb16, int64_t n_rows, int E, int reverse, int32_t* tok_id, float* X,
                  int32_t* err, const float* W, const float* bias, uint64_t seed, uint64_t counter, int64_t A, int S,
                  int HF, int32_t* ids, float* Wg, float* bg, void* Wp, int wfmt, rg_stream_t stream);
/* rg_adam_rows (cols % 4 == 0) that also writes P16 = fp16(P); tags == NULL: every row has a gradient */
int rg_adam_rows_h(float* P, float* M, float* V, float* G, const int32_t* tags, int32_t tag, int64_t rows, int cols,
                   const float* adam6, uint16_t* P16, rg_stream_t stream);
int rg_f32_to_f16(const float* x, int64_t n, uint16_t* out, rg_stream_t stream);

/* ---- sampled-softmax head (SURVEY §8 A7 sampled ext., config C3; build-defined,
 * no reference counterpart — replaces the full-softmax CrossEntropyLoss of
 * GRU4Rec/model.py:121,146 / BidirGRU4Rec/model.py:145,167 when the trainer is
 * built with n_negatives) ---- */
/* out[s] = uniform draw on [0, A): hi64(splitmix64(seed + phi*(counter*S + s + 1)) * A) */
int rg_sample_uniform(uint64_t seed, uint64_t counter, int S, int64_t A, int32_t* out, rg_stream_t stream);
/* number of (max, Σexp) partials per row the forward writes: terms = 0 (rg_sampled_fwd):
 * ceil(S/128); terms = 6 / 9 (rg_sampled_fwd_x, S and B multiples of 32): S/32 */
int rg_sampled_nparts(int B, int S, int terms);
/* Zᵀ[s][b] = h_b·W[neg_s] + bias[neg_s] (S × ldz) + per-(128-negative tile, row) (max, Σexp)
 * partials (rg_sampled_nparts(B, S, 0) × B); Wg/bg (optional, both or neither): the gathered rows.
 * HF ∈ {32,64,128,256}. */
int rg_sampled_fwd(const float* h, const float* W, const float* bias, const int32_t* neg, int B, int S, int HF,
                   float* ZT, int64_t ldz, float* pmax, float* psum, float* Wg, float* bg, rg_stream_t stream);
/* scratch bytes rg_sampled_fwd_x needs: (S + B)·HF·6 (the bf16 operand planes) */
int64_t rg_sampled_work_bytes(int B, int S, int HF);
/* rg_sampled_fwd computed on bf16 MFMAs from an exact three-plane bf16 split of both fp32
 * operands (csrc/common.h): terms = 9 keeps every plane product (exact products, fp32
 * accumulation), 6 drops the three below fp32's unit roundoff.  B % 32 == 0, S % 32 == 0;
 * partials as rg_sampled_nparts(B, S, terms); Wg optional, bg required.  draw = 1: neg is an output
 * filled with rg_sample_uniform(seed, counter, S, A) (the draw fused into the operand prep);
 * draw = 0: neg is an input.  work: rg_sampled_work_bytes(B, S, HF) bytes of device scratch. */
int rg_sampled_fwd_x(const float* h, const float* W, const float* bias, int32_t* neg, int draw, uint64_t seed,
                     uint64_t counter, int64_t A, int B, int S, int HF, int terms, float* ZT, int64_t ldz,
                     float* pmax, float* psum, float* Wg, float* bg, void* work, rg_stream_t stream);
/* The split-bf16 sampled forward in ONE launch for HF in {32, 64, 128, 256} (draw, the negatives' row
 * gather, both operands' bf16 split, MFMAs, logits, partials): same semantics as rg_sampled_fwd_x
 * but Z is ROW-major, Z[b·ldz + s] (ldz >= S, ldz % 4 == 0).  Wg optional, bg required.
 * h_planes (optional, HF <= 128): h's bf16 K-planes (rg_gru_fwd_dirs_planes / rg_head_planes), moved
 * to LDS by DMA instead of splitting h in the kernel.
 * draw: 0 = ids given in neg, 1 = drawn here, 2 = pre-gathered by rg_gather_neg (neg, bg, Wg already
 * hold the ids, biases and rows; w_planes = its fragment-order planes, required); 3 = the same with
 * w_planes = its fp32 fragments (wfmt 1; HF <= 128). */
int rg_sampled_logits(const float* h, const float* W, const float* bias, int32_t* neg, int draw, uint64_t seed,
                      uint64_t counter, int64_t A, int B, int S, int HF, int terms, float* Z, int64_t ldz,
                      float* pmax, float* psum, float* Wg, float* bg, const void* h_planes, const void* w_planes,
                      rg_stream_t stream);
/* in place dZ = exp(Z − lse)·g on the row-major Z of rg_sampled_logits; dbg[s] = Σ_b dZ[b][s]
 * through ceil(B/128) × S slabs (summed in order: deterministic) */
int rg_sampled_dz_rows(float* Z, int64_t ldz, const float* lse, int B, int S, float gscale, float* slabs, float* dbg,
                       rg_stream_t stream);
/* per row: z_pos = h_b·W[a_b] + bias[a_b]; lse over {z_pos} ∪ partials; loss_row = lse − z_pos;
 * ids[b] = a_b; dzpos = (exp(z_pos − lse) − 1)·g; gpos = dzpos·h_b; dhpos = dzpos·W[a_b] */
int rg_sampled_lse(const float* h, const float* W, const float* bias, const int64_t* tgt, int B, int64_t A, int HF,
                   const float* pmax, const float* psum, int nT, float gscale, float* lse, float* loss_row,
                   int32_t* ids, float* dzpos, float* gpos, float* dhpos, rg_stream_t stream);
/* in place dZᵀ = exp(Zᵀ − lse)·g; dbg[s] = Σ_b dZᵀ[s][b] */
int rg_sampled_dz(float* ZT, int64_t ldz, const float* lse, int B, int S, float gscale, float* dbg,
                  rg_stream_t stream);
/* Sampled BPR over the same logits (build-defined; north_star "sampled-softmax/BPR"; the
 * reference's trainers have CE only, GRU4Rec/model.py:121):
 * loss = mean_b (1/S) Σ_s softplus(z_b,s − z_b,pos).  Z(b, s) at Z[b·zsb + s·zss] (row-major Z of
 * rg_sampled_logits: zsb = ldz, zss = 1; Zᵀ of rg_sampled_fwd(_x): zsb = 1, zss = ldz).
 * rg_bpr_rows: per row zpos = h_b·W[a_b] + bias[a_b], loss_row (NaN for a target outside [0, A)),
 * ids, dzpos = −g·Σ_s σ(z_s − zpos)/S, gpos = dzpos·h_b, dhpos = dzpos·W[a_b].
 * rg_bpr_dz: in place dZ = g·σ(Z − zpos)/S; dbg[s] = Σ_b dZ(b, s) through ceil(B/128) × S slabs. */
int rg_bpr_rows(const float* h, const float* W, const float* bias, const int64_t* tgt, int B, int64_t A, int HF,
                const float* Z, int64_t zsb, int64_t zss, int S, float gscale, float* zpos, float* loss_row,
                int32_t* ids, float* dzpos, float* gpos, float* dhpos, rg_stream_t stream);
int rg_bpr_dz(float* Z, int64_t zsb, int64_t zss, const float* zpos, int B, int S, float gscale, float* slabs,
              float* dbg, rg_stream_t stream);

/* ---- §8e row-sharded item-embedding table (csrc/emb_shard.hip, csrc/segsum.hip): the multi-GPU
 * form of self.embedding(s) and its dense gradient + Adam (GRU4Rec/model.py:35-47, 69, 150-153).
 * Rank r holds rows [⌊r·n_rows/world⌋, ⌊(r+1)·n_rows/world⌋).  Per trunk pass each DISTINCT id of
 * the rank's batch is requested once:
 * rg_token_ids: tok_id[t] = item id of packed token t (forward time order; -1 + err if invalid).
 * rg_shard_dedup: over the T = *n_ptr tokens (n_max >= T): uids[0..U) = the distinct ids in
 *   increasing order (-1 first when a token was invalid: it goes to rank 0, whose gather returns a
 *   zero row), uslot[t] = the token's index into uids, counts[o] = distinct ids owned by rank o
 *   (world <= 256; uids is grouped by owner), *nuniq = U; ids outside [0, n_rows) count as -1.
 *   No sort: a mark per table row and one scan over the n_rows + 1 marks.  work:
 *   rg_shard_dedup_work_bytes(n_max, E, n_rows); it keeps the (u, t) pairs for
 *   rg_shard_dedup_grads of the same pass.
 * rg_shard_dedup_grads: gsend[u] = Σ_{t : uslot[t] = u} src[t] (E floats per row, summed in token
 *   order — a stable sort of the pairs by u, then segmented sums: deterministic), for the pass's
 *   last rg_shard_dedup on `work` (same n_max, n_rows).
 * rg_shard_dedup_ids: rg_token_ids + rg_shard_dedup in two launches when the host batch gives the
 *   distinct ids (uids[0..U), sorted, -1 first: dist.distinct_ids, which the host counts the
 *   exchange's splits from): the same tok_id / uslot and the (u, t) pairs in `work` for
 *   rg_shard_dedup_grads; map: n_rows + 1 int32 scratch (never cleared; one per pass in flight).
 * rg_shard_route: stable partition of the T = *ntok_ptr rows by owner rank: slot[t] (send
 *   position), send_ids[slot[t]] = tok_id[t], counts[world] (world <= 8; the sharded sampled
 *   head's per-row target exchange).
 * rg_rows_gather: owner side, rows of n received global ids from the local shard [lo, lo + n_local)
 *   (fp32, or fp16 when half = 1) and local_ids (id − lo, or -1 with a zero row).
 * rg_place_rows: X[t] = rows_in[slot[t]] widened to fp32 (slot = uslot); reverse = 1: each row's
 *   valid prefix reversed (the backward direction of BidirGRU4Rec).
 * rg_combine_dirs: dX0[t] += dX1[rev t] in place (Bidir: both directions' token gradients before
 *   rg_shard_dedup_grads).  The owner adds the received per-id sums into its rows
 *   (rg_scatter_rows with local_ids) before rg_adam_rows on its shard. */
int rg_token_ids(const int64_t* s, int B, int L, const int32_t* perm, const int32_t* lsort, const int32_t* offs,
                 int64_t n_rows, int32_t* tok_id, int32_t* err, rg_stream_t stream);
int64_t rg_shard_dedup_work_bytes(int n_max, int E, int64_t n_rows);
int rg_shard_dedup(const int32_t* tok_id, const int32_t* n_ptr, int n_max, int64_t n_rows, int world, int E,
                   int32_t* uslot, int32_t* uids, int32_t* counts, int32_t* nuniq, void* work, int64_t work_bytes,
                   rg_stream_t stream);
int rg_shard_dedup_grads(const float* src, int E, int n_max, int64_t n_rows, float* gsend, void* work,
                         int64_t work_bytes, rg_stream_t stream);
int rg_shard_dedup_ids(const int64_t* s, int B, int L, const int32_t* perm, const int32_t* lsort, const int32_t* offs,
                       const int32_t* n_ptr, int n_max, int64_t n_rows, const int32_t* uids, int U, int32_t* map,
                       int32_t* tok_id, int32_t* uslot, int32_t* err, int E, void* work, int64_t work_bytes,
                       rg_stream_t stream);
int rg_shard_route(const int32_t* tok_id, const int32_t* ntok_ptr, int64_t n_rows, int world, int32_t* slot,
                   int32_t* send_ids, int32_t* counts, rg_stream_t stream);
int rg_rows_gather(const int32_t* ids, int n, int64_t lo, int64_t n_local, const void* table, int E, int half,
                   void* rows, int32_t* local_ids, rg_stream_t stream);
int rg_place_rows(const void* rows_in, int half, const int32_t* slot, const int32_t* lsort, const int32_t* offs, int B,
                  int E, int reverse, float* X, rg_stream_t stream);
int rg_combine_dirs(float* dX0, const float* dX1, const int32_t* lsort, const int32_t* offs, int B, int E,
                    rg_stream_t stream);

/* ---- §8e item-sharded sampled head (csrc/sampled_shard.hip; the multi-GPU form of the
 * build-defined sampled softmax that replaces GRU4Rec/model.py:58-60, 80 in config C3).  Rank r
 * holds output rows [lo, hi); rows move to the data:
 * rg_neg_pick: draw `counter` of the counter-based stream (ids[S], global) and, for the negatives
 *   this rank owns, their rows Wg[S][HF] / biases bg[S] (zeros elsewhere; SUM all-reduce next);
 *   nloc[x] = id − lo or -1.
 * rg_neg_planes: fragment-order bf16 planes of Wg (rg_sampled_logits draw = 2).
 * rg_target_ids: int32 routing ids of n int64 targets (-1 outside [0, A)), *n_out = n (for
 *   rg_shard_route with n_rows = A).
 * rg_head_rows_gather: owner side, W rows and biases of n received item ids from the local shard
 *   [lo, lo + n_local): row k at rows + k·ld (ld >= HF + 1, ld % 4 == 0), its bias at + HF (zeros,
 *   local_ids -1 when not held) — rows and biases travel in ONE all-to-all.
 * rg_rows_unslot: tW[b] = row slot[b] of `rows` (stride ld), tb[b] = its bias, trow[b] = b (the CE's
 *   per-row target into tW / tb); where tid32[b] < 0 a zero row and trow[b] = -1, so
 *   rg_sampled_lse writes a NaN loss row with zero gradients, as the one-GPU head does for an
 *   invalid target.
 * rg_rows_slot: row slot[b] of gsend (stride ld) = grows[b], its bias entry = gb[b] (the targets'
 *   row and bias gradients back to their owners in one all-to-all). */
int rg_neg_pick(uint64_t seed, uint64_t counter, int64_t A, int S, int HF, int64_t lo, int64_t hi, const float* W,
                const float* bias, int32_t* ids, int32_t* nloc, float* Wg, float* bg, rg_stream_t stream);
int rg_neg_planes(const float* Wg, int S, int HF, void* Wp, rg_stream_t stream);
int rg_target_ids(const int64_t* tgt, int n, int64_t A, int32_t* out, int32_t* n_out, rg_stream_t stream);
int rg_head_rows_gather(const int32_t* ids, int n, int64_t lo, int64_t n_local, const float* W, const float* bias,
                        int HF, int ld, float* rows, int32_t* local_ids, rg_stream_t stream);
int rg_rows_unslot(const float* rows, int ld, const int32_t* slot, const int32_t* tid32, int n, int HF, float* tW,
                   float* tb, int64_t* trow, rg_stream_t stream);
int rg_rows_slot(const float* grows, const float* gb, const int32_t* slot, int n, int HF, int ld, float* gsend,
                 rg_stream_t stream);

/* ---- §8e collectives of the item-sharded step (csrc/comm.hip; RCCL over xGMI): the library's own
 * communicator, every collective enqueued on the CALLER's stream (the stream of the kernels that
 * produce and consume its buffers: no cross-stream hops).  Replaces the torch.distributed calls
 * of recommenders/hip/dist.py Comm on the nccl backend.  dtype codes: 0 u8, 1 i32, 2 f32, 3 f16,
 * 4 i64.
 * rg_comm_unique_id: rank 0's id (rg_comm_id_bytes() bytes), broadcast by the host to every rank.
 * rg_comm_init: *comm = the communicator of `rank` among `world` (collective; device made current).
 * rg_comm_alltoallv: send_counts[q] elements (consecutive, rank order) to rank q, recv_counts[q]
 *   from rank q (HOST int64 arrays of world entries); one group of sends / receives.
 * rg_comm_allreduce: SUM of n elements (in place when send == recv).
 * rg_comm_allgather: recv (world·n) <- every rank's n, rank-major.
 * rg_comm_reduce_scatter: recv (n) <- slice rank of the SUM over ranks of send (world·n). */
int rg_comm_id_bytes(void);
int rg_comm_unique_id(void* out);
int rg_comm_init(const void* id, int world, int rank, int device, void** comm);
int rg_comm_destroy(void* comm);
int rg_comm_alltoallv(void* comm, const void* send, const int64_t* send_counts, void* recv,
                      const int64_t* recv_counts, int dtype, rg_stream_t stream);
int rg_comm_allreduce(void* comm, const void* send, void* recv, int64_t n, int dtype, rg_stream_t stream);
int rg_comm_allgather(void* comm, const void* send, void* recv, int64_t n, int dtype, rg_stream_t stream);
int rg_comm_reduce_scatter(void* comm, const void* send, void* recv, int64_t n, int dtype, rg_stream_t stream);

/* ---- Gated delta rule (csrc/delta.hip): a linear-attention recurrence beside rg_gru_fwd / rg_gru_bwd.  Per value head
 * S_t = exp(g_t) S_{t-1} + beta_t k_t (v_t - exp(g_t) S_{t-1}^T k_t)^T, o_t = scale S_t^T q_t, S a Dk x Dv matrix.
 * q, k (B, T, Hk, Dk), v and d_o (B, T, Hv, Dv) of `type` (0 fp32, 1 bf16), g, beta (B, T, Hv) fp32; Hv a multiple of
 * Hk; Dk, Dv multiples of 8 up to 128; Hk Dk and Hv Dv less than 2^23 (rg_delta_step: any).  strides: HOST array of 18, the (B, T, H) strides in elements of q, k, v, g, beta,
 * d_o; rows (the last dimension) are contiguous, positions (T) at least a row and less than 2^23 elements apart, rows of
 * q, k, d_o, for rg_delta_bwd of v, and dq, dk start at multiples of 16 bytes (rg_delta_step: anywhere).  lens (B) int64,
 * optional: positions at or behind it are not read, do not change the state and get zeros.  Contiguous: o, dv
 * (B, T, Hv, Dv), dq, dk (B, T, Hk, Dk), dg, dbeta (B, T, Hv), the states (B, Hv, Dk, Dv) fp32.
 * For the backward pass the forward leaves U (B, Hv, T, Dv) and S0 (rg_delta_chunk_floats values, when T > 32); both
 * NULL otherwise.  A long T is cut into n = rg_delta_segments(..) segments; when n > 1: trans (rg_delta_trans_floats
 * values), which the backward call reads again, and local (B, Hv, n, Dk, Dv) fp32, work space of one call.  dX is of U's size, dS
 * of S0's.  state0, dstate, dstate0 optional (NULL: zero / not wanted).
 * rg_delta_step: one token, q, k (B, Hk, Dk), v (B, Hv, Dv); state updated in place, its rows state_stride apart. */
int64_t rg_delta_chunk_floats(int B, int T, int Hv, int Dk, int Dv);
int rg_delta_segments(int B, int T, int Hv, int Dk, int Dv);
int64_t rg_delta_trans_floats(int B, int T, int Hv, int Dk, int Dv);
int rg_delta_fwd(const void* q, const void* k, const void* v, const float* g, const float* beta, const int64_t* strides,
                 const int64_t* lens, const float* state0, int type, int B, int T, int Hk, int Hv, int Dk, int Dv,
                 float scale, void* o, float* state, float* U, float* S0, float* trans, float* local,
                 rg_stream_t stream);
int rg_delta_bwd(const void* q, const void* k, const void* v, const float* g, const float* beta, const void* d_o,
                 const int64_t* strides, const int64_t* lens, const float* state0, const float* dstate, const float* U,
                 const float* S0, const float* trans, int type, int B, int T, int Hk, int Hv, int Dk, int Dv,
                 float scale, float* dX, float* dS, float* local, void* dq, void* dk, void* dv, float* dg,
                 float* dbeta, float* dstate0, rg_stream_t stream);
int rg_delta_step(const void* q, const void* k, const void* v, const float* g, const float* beta,
                  const int64_t* strides, int type, int B, int Hk, int Hv, int Dk, int Dv, float scale, float* state,
                  int64_t state_stride, void* o, rg_stream_t stream);

/* ---- Linear cross entropy on half-precision activations (csrc/linear_ce.hip): output layer and loss without logits in
 * memory, beside the fp32 heads (rg_head_*, rg_flash_*).  z = h W^T + bias, loss_r = lse(z_r) - z_{r, target_r};
 * h (N, D), W (V, D) of `type` (1 bf16, 2 fp16), row strides ldh / ldw in elements, rows at multiples of 16 bytes; bias
 * (V) fp32 optional; target (N) int64, stride target_stride.  Negative targets: row ignored (loss and gradient 0);
 * targets >= V: NaN.  D a multiple of 8 up to 256, N <= 2^24.  grad = 1: also prepares the backward pass.
 * rg_linear_ce_bwd: dloss (N) fp32; dh (N, D), dW (V, D) contiguous of `type`, db (V) fp32 or NULL.  `saved`
 * (rg_linear_ce_saved_bytes) goes from the forward to the backward call; `work` (rg_linear_ce_work_floats of pass 0:
 * forward, 1: forward with grad, 2: backward) only within one. */
int64_t rg_linear_ce_work_floats(int N, int V, int D, int pass);
int64_t rg_linear_ce_saved_bytes(int N, int V, int D);
int rg_linear_ce_fwd(const void* h, int64_t ldh, const void* W, int64_t ldw, const float* bias, const int64_t* target,
                     int64_t target_stride, int type, int N, int V, int D, int grad, float* work, void* saved,
                     float* loss, rg_stream_t stream);
int rg_linear_ce_bwd(const void* W, int64_t ldw, const float* bias, const float* dloss, int64_t dloss_stride, int type,
                     int N, int V, int D, const void* saved, float* work, void* dh, void* dW, float* db,
                     rg_stream_t stream);

/* ---- Scores from a 4-bit item table (csrc/q4.hip): beside rg_head_fwd for serving.  Element types of the
 * operator entry points below: 0 fp32, 1 bf16, 2 fp16.  codes (N, K/2), two a byte, the even column in the low half;
 * scales (N, K/G) bf16; weight = scale·(code - 8).  G = 32, 64 or 128, K a multiple of G up to 1024; codes and scales
 * start at multiples of 16 bytes and are contiguous; ldw / ldx / ldy are row strides in elements (wtype, xtype 0 or 1).
 * rg_q4_pack: scale = bf16(max|w| / 7) of a group, code = clamp(round(w / scale) + 8, 0, 15).
 * rg_q4_scores: y[m, n] = sum_k x[m, k]·weight[n, k] + bias[n] (bias optional), fp32. */
int rg_q4_pack(const void* W, int wtype, int64_t ldw, int64_t N, int K, int G, uint8_t* codes, uint16_t* scales,
               rg_stream_t stream);
int rg_q4_scores(const void* x, int xtype, int64_t ldx, const uint8_t* codes, const uint16_t* scales,
                 const float* bias, int M, int64_t N, int K, int G, float* y, int64_t ldy, rg_stream_t stream);

/* items per online-softmax partial block of rg_head_fwd: pmax/psum/parg hold ceil(A/that) x B */
int rg_partial_block(void);
int rg_abi_version(void);   /* 2 (changes since 1) */
/* Kernel-exact timing (bench.py): arm two hipEvent_t (created, timing-enabled) so the next
 * gather / one-launch sampled-logits kernel stamps them at its own start / end
 * (hipExtLaunchKernelGGL) and disarms them; NULL, NULL disarms.  Returns 1 when the previous
 * arming was still pending, else 0.  Not thread-safe (one host thread drives the library). */
int rg_timing_events(void* start, void* stop);

#ifdef __cplusplus
}
#endif
#endif
