// Attention of query rows over another sequence's states with a bias learned
// by time distance, forward and backward.
//
// For sequence n and query head h (G = Hq / Hkv query heads share a key head):
//   s_ij = scale <q_i, k_j> + bias[h][bucket(q_pos_i - k_pos_j)]
//   p_ij = exp(s_ij) / sum over the live keys, o_i = sum_j p_ij v_j
// A key is live if it lies inside the sequence's length and its mask is set;
// rows without a live key, and rows past the query length, are 0. Backward,
// with D_i = <do_i, o_i>:
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (<do_i, v_j> - D_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,
//   dbias[h][b] = sum of ds_ij over the pairs in bucket b.
//
// bucket(d): n = |d| (one-sided: max(d, 0)), at most 2^32 - 1. With 2^m
// buckets an octave, n < 2^m is its own bucket and otherwise, e = floor(log2 n),
// (e - m) 2^m + (n >> (e - m)); the last bucket takes what lies beyond it, and
// negative distances of a two-sided table its second half. Integers only, so
// a distance next to a border falls on its own side.
//
// The rows of a key head's G query heads are one list of rows r = i G + g, so
// that they share each key tile and their sums into dk and dv are one loop
// over r (no atomics: every result is the same each time). Products run on
// MFMA, fp32 accumulation (fp32 inputs: v_mfma_f32_16x16x4_f32). The score
// blocks come out of the MFMA with the reduction index of the product that
// follows in a lane's own registers (key x row blocks for o and dq, row x
// key blocks for dk and dv), so p and ds go from one product to the next
// without leaving the registers; the other operand is read down the columns of
// the row-major tile in that order (16-bit types: the transposing LDS read).
//
// Which kernels run, by size (both sides of each rule, heads of 64, us: 2,000
// sequences of 32 rows x 64 keys in bf16, forward and backward, 134 in one wave
// and 274 in tiles; 500 of 32 x 200 forward 39 and 77 to 93; 24 of 512 x 600,
// which are 192 workgroups, 146 and 371, in fp32 268 and 385; half as many in
// fp32 172 by the four waves and 234. In bf16 the eight waves are ahead from
// 96 on, 135 for 196: the threshold is fp32's):
//   rows = lq G <= 32       one wave a (sequence, key head), or the keys split
//                           over workgroups and joined where sequences are few
//   rows <= 32, lk <= 64    the backward in one wave, nothing kept for it
//   more                    tiles in LDS; 8 waves a workgroup where that gives
//                           192 workgroups or more, else 4 waves along the keys
#include <climits>

#include "cross_attention.h"

namespace {

using sgl::attn::Args;

Args args_of(const sgl_attention *p) {
  Args a;
  a.p = *p;
  a.G = p->heads_q / p->heads_kv;
  a.cols = p->bias != nullptr ? p->buckets * (p->two_sided ? 2 : 1) : 0;
  a.rows = p->lq * a.G;
  return a;
}

int check_attn(const sgl_attention *p) {
  SGL_REQUIRE(p != nullptr, "cross_attention: NULL problem");
  SGL_REQUIRE(p->dtype >= 0 && p->dtype <= SGL_FP16, "cross_attention: unknown element type %d", p->dtype);
  SGL_REQUIRE(p->n >= 0 && p->lq >= 0 && p->lk >= 0 && p->n < INT_MAX && p->lq < INT_MAX && p->lk < INT_MAX,
              "cross_attention: bad sizes");
  SGL_REQUIRE(p->heads_q > 0 && p->heads_kv > 0 && p->heads_q % p->heads_kv == 0,
              "cross_attention: %d query heads over %d key heads", p->heads_q, p->heads_kv);
  const int least = p->dtype == SGL_FP32 ? 4 : 8;   // a row is read by 16-byte vectors
  SGL_REQUIRE(p->head_dim >= least && p->head_dim <= sgl::attn::kMaxDim, "cross_attention: head size %d (%d to %d)",
              p->head_dim, least, sgl::attn::kMaxDim);
  SGL_REQUIRE(p->heads_q / p->heads_kv <= 64, "cross_attention: more than 64 query heads to a key head");
  if (p->bias != nullptr) {
    SGL_REQUIRE(p->buckets > 0 && p->buckets * (p->two_sided ? 2 : 1) <= sgl::attn::kMaxCols,
                "cross_attention: a bias table of %d buckets (at most %d columns)", p->buckets, sgl::attn::kMaxCols);
    SGL_REQUIRE(p->resolution >= 0 && p->resolution <= 4, "cross_attention: bias resolution %d (0 to 4)",
                p->resolution);
    SGL_REQUIRE(p->n == 0 || ((p->lq == 0 || p->q_pos) && (p->lk == 0 || p->k_pos)),
                "cross_attention: a bias needs positions");
  }
  SGL_REQUIRE(p->n == 0 || ((p->lq == 0 || p->q) && (p->lk == 0 || (p->k && p->v))), "cross_attention: NULL array");
  const int64_t rows = p->lq * (p->heads_q / p->heads_kv);
  // a launch has fewer than 2^32 threads: one wave an item (few rows, few keys),
  // else at most a workgroup of 512 for each 64 rows or keys of one
  const int64_t items = p->n * p->heads_kv, most = std::max(rows, p->lk);
  const bool one_wave = rows <= sgl::attn::kSmallRows && p->lk <= sgl::attn::kSmallKeys;
  SGL_REQUIRE(rows < INT_MAX && items < (1 << 25) && (one_wave || items * (most / 64 + 1) < (1 << 23)),
              "cross_attention: too many rows for one call");
  return SGL_OK;
}

}  // namespace

extern "C" size_t sgl_cross_attention_workspace_bytes(const sgl_attention *p, int32_t backward) {
  if (check_attn(p) != SGL_OK || p->n == 0) return 0;
  const Args a = args_of(p);
  if (!backward) return sgl::attn::forward_bytes(a);
  return sgl::attn::is_small(a) ? sgl::attn::small_backward_bytes(a) : sgl::attn::backward_bytes(a);
}

extern "C" int32_t sgl_cross_attention_saves(const sgl_attention *p) {
  if (check_attn(p) != SGL_OK) return 0;
  const Args a = args_of(p);
  if (sgl::attn::is_small(a)) return 0;
  return 1 | (p->dtype != SGL_FP32 && p->lk > sgl::attn::kKeys ? 2 : 0);
}

extern "C" int sgl_cross_attention_forward(const sgl_attention *p, void *o, void *rest, float *lse, void *workspace,
                                           size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = check_attn(p)) return rc;
  if (p->n == 0 || p->lq == 0) return SGL_OK;
  SGL_REQUIRE(o != nullptr, "cross_attention: NULL array");
  const Args a = args_of(p);
  const size_t need = sgl::attn::forward_bytes(a);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    sgl::set_error("cross_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return SGL_ERR_WORKSPACE;
  }
  return sgl::attn::run_forward(a, o, rest, lse, workspace, stream);
}

extern "C" int sgl_cross_attention_backward(const sgl_attention *p, const void *o, const void *rest, const float *lse,
                                            const void *go, void *dq, void *dk, void *dv, float *dbias,
                                            void *workspace, size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = check_attn(p)) return rc;
  SGL_REQUIRE(dbias == nullptr || p->bias != nullptr, "cross_attention_backward: a bias gradient without a bias");
  const Args a = args_of(p);
  if (p->n == 0) {
    if (dbias != nullptr) {   // (a sum over no rows)
      sgl::sum_rows(nullptr, 0, p->heads_q * a.cols, dbias, stream);
      SGL_CHECK_LAUNCH();
    }
    return SGL_OK;
  }
  const int32_t saves = sgl_cross_attention_saves(p);
  SGL_REQUIRE((p->lq == 0 || (go && dq)) && (p->lk == 0 || (dk && dv)), "cross_attention_backward: NULL array");
  SGL_REQUIRE(p->lq == 0 || !(saves & 1) || (o && lse), "cross_attention_backward: the forward's o and lse are needed");
  SGL_REQUIRE(p->lq == 0 || !(saves & 2) || rest, "cross_attention_backward: the forward's rest is needed");
  const size_t need = sgl_cross_attention_workspace_bytes(p, 1);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    sgl::set_error("cross_attention_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return SGL_ERR_WORKSPACE;
  }
  if (sgl::attn::is_small(a)) return sgl::attn::run_small_backward(a, go, dq, dk, dv, dbias, workspace, stream);
  return sgl::attn::run_backward(a, o, rest, lse, go, dq, dk, dv, dbias, workspace, stream);
}
