// Entry points of Chord attention under a sliding window with visible first tokens, and over a 4-bit
// cache: argument checks and the choice of kernel.  A query at position p sees the keys j <= p with
// j > p - window or j < sinks; a row that sees none gives zeros.
#include <algorithm>
#include <string>

#include "capi_internal.h"
#include "chord_internal.h"
#include "common.h"

namespace motif {

namespace {

// Everything the three forward entries share: sizes, types, pointers, alignment; fills a.
struct Call {
  const char *name;
  const void *q; int64_t q_sb, q_sh, q_st;
  const float *alpha, *beta, *mu, *ssmax, *log_n; int64_t ln_sb, ln_st;
  const float *log_table; int log_table_len;
  void *out; int64_t o_sb, o_sh, o_st;
  float *lse;
  int *length_dev;
  int B, H, Hkv, L, S, D, q_start;
  float scale, eps;
  int window, sinks, dtype;
};

int fill(const Call &c, ChordArgs &a) {
  const std::string name(c.name);
  if (c.B < 0 || c.H <= 0 || c.Hkv <= 0 || c.L < 0 || c.S < 0 || c.q_start < 0 || c.H % c.Hkv)
    return set_error(MOTIF_ERR_INVALID, name + ": bad size or negative q_start");
  if (!kv4_head_dim(c.D)) return set_error(MOTIF_ERR_UNSUPPORTED, name + ": head_dim must be 16, 32, 64 or 128");
  if (c.dtype != MOTIF_BF16 && c.dtype != MOTIF_F32 && c.dtype != MOTIF_F16)
    return set_error(MOTIF_ERR_UNSUPPORTED, name + ": dtype must be bf16, fp16 or fp32");
  if (c.window < 1 || c.sinks < 0) return set_error(MOTIF_ERR_INVALID, name + ": need window >= 1 and sinks >= 0");
  if (std::max<int64_t>(c.S, static_cast<int64_t>(c.q_start) + c.L) >= kMaxWindow || c.B > 65535 || c.L > 65535 * 32)
    return set_error(MOTIF_ERR_UNSUPPORTED, name + ": sequence too long or too many batch rows");
  a = ChordArgs{};
  a.q = c.q; a.q_sb = c.q_sb; a.q_sh = c.q_sh; a.q_st = c.q_st;
  a.alpha = c.alpha; a.beta = c.beta; a.mu = c.mu; a.ssmax = c.ssmax;
  a.log_n = c.log_n; a.ln_sb = c.ln_sb; a.ln_st = c.ln_st; a.log_tab = c.log_table;
  a.out = c.out; a.o_sb = c.o_sb; a.o_sh = c.o_sh; a.o_st = c.o_st;
  a.lse = c.lse;
  a.B = c.B; a.H = c.H; a.Hkv = c.Hkv; a.L = c.L; a.S = c.S; a.q_start = c.q_start;
  a.scale = c.scale; a.eps = c.eps;
  a.splits = a.nqc = 1;
  a.len_dev = c.length_dev;
  a.window = std::min(c.window, kMaxWindow);
  a.sinks = std::min(c.sinks, kMaxWindow);
  if (c.B == 0 || c.L == 0) return MOTIF_OK;
  if (c.S == 0) return set_error(MOTIF_ERR_INVALID, name + ": empty key cache");
  if (!c.q || !c.alpha || !c.beta || !c.mu || !c.ssmax || !c.out)
    return set_error(MOTIF_ERR_INVALID, name + ": NULL pointer");
  if (c.length_dev && c.S < c.L) return set_error(MOTIF_ERR_INVALID, name + ": capacity below the query count");
  if (!c.log_n && (!c.log_table || c.log_table_len < std::max(c.S, c.q_start + c.L)))
    return set_error(MOTIF_ERR_INVALID, name + ": log_n is NULL and the log table is too short");
  const int64_t vec = c.dtype == MOTIF_F32 ? 4 : 8;
  if (((c.q_st | c.o_st | c.q_sh | c.o_sh | c.q_sb | c.o_sb) % vec) != 0 ||
      ((reinterpret_cast<uintptr_t>(c.q) | reinterpret_cast<uintptr_t>(c.out)) & 15) != 0)
    return set_error(MOTIF_ERR_UNSUPPORTED, name + ": q/out need 16-byte aligned rows");
  if (c.L == 1) a.q_st = c.D;  // (the stride of a single row is not used)
  return MOTIF_OK;
}

int fill_rows(const Call &c, ChordArgs &a, const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st, const void *v,
              int64_t v_sb, int64_t v_sh, int64_t v_st) {
  const std::string name(c.name);
  a.k = k; a.k_sb = k_sb; a.k_sh = k_sh; a.k_st = k_st;
  a.v = v; a.v_sb = v_sb; a.v_sh = v_sh; a.v_st = v_st;
  if (!k || !v) return set_error(MOTIF_ERR_INVALID, name + ": NULL pointer");
  const int64_t vec = c.dtype == MOTIF_F32 ? 4 : 8;
  if (((k_st | v_st | k_sh | v_sh | k_sb | v_sb) % vec) != 0 ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0)
    return set_error(MOTIF_ERR_UNSUPPORTED, name + ": k/v need 16-byte aligned rows");
  if (c.S == 1) a.k_st = a.v_st = c.D;
  // 32-bit offsets inside a tile of rows
  for (int64_t st : {a.q_st, a.k_st, a.v_st})
    if (st < 0 || st >= (int64_t(1) << 24)) return set_error(MOTIF_ERR_UNSUPPORTED, name + ": row stride out of range");
  return MOTIF_OK;
}

}  // namespace

}  // namespace motif

using namespace motif;

extern "C" int motif_chord_window_fwd(
    const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st,
    const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st,
    const void *v, int64_t v_sb, int64_t v_sh, int64_t v_st,
    const float *alpha, const float *beta, const float *mu, const float *ssmax,
    const float *log_n, int64_t ln_sb, int64_t ln_st, const float *log_table, int log_table_len,
    void *out, int64_t o_sb, int64_t o_sh, int64_t o_st, float *lse,
    int *length_dev, int B, int H, int Hkv, int L, int S, int D, int q_start, float scale, float eps,
    int window, int sinks, void *workspace, size_t workspace_bytes, int dtype, void *stream) {
  const Call c{"chord_window_fwd", q, q_sb, q_sh, q_st, alpha, beta, mu, ssmax, log_n, ln_sb, ln_st, log_table,
               log_table_len, out, o_sb, o_sh, o_st, lse, length_dev, B, H, Hkv, L, S, D, q_start, scale, eps,
               window, sinks, dtype};
  ChordArgs a;
  int rc = fill(c, a);
  if (rc || B == 0 || L == 0) return rc;
  if ((rc = fill_rows(c, a, k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st))) return rc;
  (void)workspace; (void)workspace_bytes;
  return launch_chord_wide_window(a, dtype, D, static_cast<hipStream_t>(stream));
}

extern "C" size_t motif_chord_window_workspace_bytes(int B, int H, int Hkv, int L, int S, int D, int window, int sinks,
                                                     int dtype) {
  (void)B; (void)H; (void)Hkv; (void)L; (void)S; (void)D; (void)window; (void)sinks; (void)dtype;
  return 0;
}

extern "C" size_t motif_chord_kv4_workspace_bytes(int B, int H, int Hkv, int L, int S, int D, int window, int sinks,
                                                  int dtype) {
  (void)B; (void)H; (void)Hkv; (void)L; (void)S; (void)D; (void)window; (void)sinks; (void)dtype;
  return 0;
}

extern "C" int motif_chord_kv4_fwd(
    const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st,
    const void *k_codes, int64_t kc_sb, int64_t kc_sh, const void *k_params, int64_t kp_sb, int64_t kp_sh,
    const void *v_codes, int64_t vc_sb, int64_t vc_sh, const void *v_params, int64_t vp_sb, int64_t vp_sh,
    const float *alpha, const float *beta, const float *mu, const float *ssmax,
    const float *log_n, int64_t ln_sb, int64_t ln_st, const float *log_table, int log_table_len,
    void *out, int64_t o_sb, int64_t o_sh, int64_t o_st,
    int *length_dev, int B, int H, int Hkv, int L, int S, int D, int q_start, float scale, float eps,
    int window, int sinks, void *workspace, size_t workspace_bytes, int dtype, void *stream) {
  const Call c{"chord_kv4_fwd", q, q_sb, q_sh, q_st, alpha, beta, mu, ssmax, log_n, ln_sb, ln_st, log_table,
               log_table_len, out, o_sb, o_sh, o_st, nullptr, length_dev, B, H, Hkv, L, S, D, q_start, scale, eps,
               window, sinks, dtype};
  ChordArgs a;
  int rc = fill(c, a);
  if (rc || B == 0 || L == 0) return rc;
  const KV4Args kv = kv4_args(k_codes, kc_sb, kc_sh, k_params, kp_sb, kp_sh, v_codes, vc_sb, vc_sh, v_params, vp_sb, vp_sh);
  if (const char *bad = kv4_check(kv, D)) return set_error(MOTIF_ERR_INVALID, std::string("chord_kv4_fwd: ") + bad);
  if (a.q_st < 0 || a.q_st >= (int64_t(1) << 24)) return set_error(MOTIF_ERR_UNSUPPORTED, "chord_kv4_fwd: row stride out of range");
  (void)workspace; (void)workspace_bytes;
  return launch_chord_wide_kv4(a, kv, dtype, D, static_cast<hipStream_t>(stream));
}
