// extern "C" entry points of the cross-attention sublayer's operators (declared
// in include/rola_b200.h): norm with the residual's addition, block-scaled e4m3
// quantisation and product, attention to another sequence's states.  Same rules
// as capi.cu: arguments are checked on the host and nothing is launched when a
// check fails.
extern "C" {

static int check_rows(const void* ptr, int fp32, int64_t ld, int64_t M, int64_t K, const char* what) {
  ROLA_CHECK(aligned16(ptr), "%s: 16-byte aligned rows required", what);
  ROLA_CHECK(M <= 1 || (ld >= K && ld % (fp32 ? 4 : 8) == 0), "%s: row stride >= K with 16-byte aligned rows required",
             what);
  return ROLA_OK;
}
static int check_norm_sizes(int64_t M, int64_t K, const char* what) {
  ROLA_CHECK(M > 0 && M < (1ll << 31), "%s: M out of range", what);
  ROLA_CHECK(K > 0 && K % 8 == 0 && K <= 16384, "%s: K must be a multiple of 8, at most 16384", what);
  return ROLA_OK;
}

static int norm_impl(AddRmsNormParams& p, const char* what, rola_stream_t stream) {
  ROLA_CHECK(p.x && (p.w || !p.norm), "%s: null pointer", what);
  ROLA_CHECK((p.res == nullptr) == (p.h == nullptr), "%s: res and h go together", what);
  ROLA_CHECK(!p.norm || aligned16(p.w), "%s: w must be 16-byte aligned", what);
  ROLA_CHECK(aligned16(p.h) && aligned16(p.y) && aligned16(p.yq), "%s: outputs must be 16-byte aligned", what);
  ROLA_TRY(check_rows(p.x, p.x_fp32, p.x_ld, p.M, p.K, what));
  if (p.res) ROLA_TRY(check_rows(p.res, p.res_fp32, p.res_ld, p.M, p.K, what));
  return cuda_status(launch_add_rms_norm(p, S(stream)), what);
}

int rola_b200_add_rms_norm(const void* x, int x_fp32, int64_t x_ld, const void* res, int res_fp32, int64_t res_ld,
                           const void* w, int w_fp32, int64_t M, int64_t K, float eps, void* h, void* y, float* rstd,
                           rola_stream_t stream) {
  ROLA_TRY(check_norm_sizes(M, K, "add_rms_norm"));
  ROLA_CHECK(y, "add_rms_norm: null pointer");
  AddRmsNormParams p{};
  p.x = x, p.x_fp32 = x_fp32 != 0, p.x_ld = x_ld;
  p.res = res, p.res_fp32 = res_fp32 != 0, p.res_ld = res_ld;
  p.w = w, p.w_fp32 = w_fp32 != 0;
  p.M = M, p.K = (int)K, p.eps = eps, p.h = h, p.y = y, p.rstd = rstd, p.norm = true;
  return norm_impl(p, "add_rms_norm", stream);
}

int rola_b200_add_rms_norm_e4m3(const void* x, int x_fp32, int64_t x_ld, const void* res, int res_fp32, int64_t res_ld,
                                const void* w, int w_fp32, int64_t M, int64_t K, float eps, void* h, void* yq,
                                float* scale, int64_t scale_sM, int64_t scale_sK, int block, rola_stream_t stream) {
  ROLA_TRY(check_norm_sizes(M, K, "add_rms_norm_e4m3"));
  ROLA_CHECK(yq && scale, "add_rms_norm_e4m3: null pointer");
  ROLA_CHECK(block == 0 || block == 128, "add_rms_norm_e4m3: block must be 128, or 0 for one scale per row");
  AddRmsNormParams p{};
  p.x = x, p.x_fp32 = x_fp32 != 0, p.x_ld = x_ld;
  p.res = res, p.res_fp32 = res_fp32 != 0, p.res_ld = res_ld;
  p.w = w, p.w_fp32 = w_fp32 != 0;
  p.M = M, p.K = (int)K, p.eps = eps, p.h = h, p.yq = yq, p.norm = true;
  p.scale = scale, p.scale_sM = scale_sM, p.scale_sK = scale_sK, p.scale_row = block == 0;
  return norm_impl(p, "add_rms_norm_e4m3", stream);
}

int rola_b200_quantize_blocks_e4m3(const void* x, int x_fp32, int64_t x_ld, int64_t M, int64_t K, void* xq,
                                   float* scale, int64_t scale_sM, int64_t scale_sK, rola_stream_t stream) {
  ROLA_TRY(check_norm_sizes(M, K, "quantize_blocks_e4m3"));
  ROLA_CHECK(xq && scale, "quantize_blocks_e4m3: null pointer");
  AddRmsNormParams p{};
  p.x = x, p.x_fp32 = x_fp32 != 0, p.x_ld = x_ld;
  p.M = M, p.K = (int)K, p.yq = xq, p.norm = false;
  p.scale = scale, p.scale_sM = scale_sM, p.scale_sK = scale_sK, p.scale_row = false;
  return norm_impl(p, "quantize_blocks_e4m3", stream);
}

size_t rola_b200_add_rms_norm_bwd_workspace(int64_t M, int64_t K) {
  if (M <= 0 || M >= (1ll << 31) || K <= 0 || K % 8 != 0 || K > 16384) return 0;
  return (size_t)add_rms_norm_bwd_parts(M, (int)K) * K * 4;
}

int rola_b200_add_rms_norm_bwd(const void* h, int h_fp32, int64_t h_ld, const void* w, int w_fp32, const float* rstd,
                               const void* dy, int64_t dy_ld, const void* dh, int dh_fp32, int64_t dh_ld, int64_t M,
                               int64_t K, void* dx, int dx_fp32, void* dres, int dres_fp32, void* dw, void* workspace,
                               size_t workspace_bytes, rola_stream_t stream) {
  const char* what = "add_rms_norm_bwd";
  ROLA_TRY(check_norm_sizes(M, K, what));
  ROLA_CHECK(h && w && rstd && dy && dx, "%s: null pointer", what);
  ROLA_CHECK(aligned16(w) && aligned16(dx) && aligned16(dres) && aligned16(dw) && aligned16(workspace),
             "%s: 16-byte aligned tensors required", what);
  ROLA_TRY(check_rows(h, h_fp32, h_ld, M, K, what));
  ROLA_TRY(check_rows(dy, 0, dy_ld, M, K, what));
  if (dh) ROLA_TRY(check_rows(dh, dh_fp32, dh_ld, M, K, what));
  ROLA_CHECK(dw == nullptr || (workspace && workspace_bytes >= rola_b200_add_rms_norm_bwd_workspace(M, K)),
             "%s: dw needs a workspace of %zu bytes", what, rola_b200_add_rms_norm_bwd_workspace(M, K));
  AddRmsNormBwdParams p{};
  p.h = h, p.h_fp32 = h_fp32 != 0, p.h_ld = h_ld;
  p.w = w, p.w_fp32 = w_fp32 != 0, p.rstd = rstd;
  p.dy = dy, p.dy_ld = dy_ld;
  p.dh = dh, p.dh_fp32 = dh_fp32 != 0, p.dh_ld = dh_ld;
  p.dx = dx, p.dx_fp32 = dx_fp32 != 0, p.dres = dres, p.dres_fp32 = dres_fp32 != 0;
  p.dw = dw, p.dw_part = dw ? static_cast<float*>(workspace) : nullptr;
  p.M = M, p.K = (int)K;
  return cuda_status(launch_add_rms_norm_bwd(p, S(stream)), what);
}

int rola_b200_quantize_tiles_e4m3(const void* w, int w_fp32, int64_t ld, int64_t N, int64_t K, void* wq, float* scale,
                                  rola_stream_t stream) {
  const char* what = "quantize_tiles_e4m3";
  ROLA_CHECK(w && wq && scale, "%s: null pointer", what);
  ROLA_CHECK(N > 0 && N <= 65536 && K > 0 && K % 8 == 0 && K <= 65536, "%s: bad sizes (K a multiple of 8)", what);
  ROLA_CHECK(aligned16(wq), "%s: wq must be 16-byte aligned", what);
  ROLA_TRY(check_rows(w, w_fp32, ld, N, K, what));
  return cuda_status(launch_quantize_tiles_e4m3(w, w_fp32 != 0, ld, (int)N, (int)K, static_cast<uint8_t*>(wq), scale,
                                                (K + 127) / 128, S(stream)),
                     what);
}

int rola_b200_gemm_fp8_block(const void* xq, const float* x_scale, int64_t xs_sM, int64_t xs_sK, const void* wq,
                             const float* w_scale, const void* bias, void* out, int64_t M, int64_t N, int64_t K,
                             rola_stream_t stream) {
  const char* what = "gemm_fp8_block";
  ROLA_CHECK(xq && x_scale && wq && w_scale && out, "%s: null pointer", what);
  ROLA_CHECK(M > 0 && M < (1ll << 27), "%s: M out of range", what);
  ROLA_CHECK(N > 0 && N % 8 == 0 && N <= 65536, "%s: N must be a multiple of 8, at most 65536", what);
  ROLA_CHECK(K > 0 && K % 16 == 0 && K <= 65536, "%s: K must be a multiple of 16, at most 65536", what);
  ROLA_CHECK(aligned16(out) && aligned16(bias), "%s: out and bias must be 16-byte aligned", what);
  CUtensorMap ta, tb;
  {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)M};
    const uint64_t strides[1] = {(uint64_t)K};
    const uint32_t box[2] = {128, 128};
    ROLA_TRY(make_map(&ta, xq, 2, dims, strides, box, "gemm_fp8_block: xq", true));
  }
  {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)N};
    const uint64_t strides[1] = {(uint64_t)K};
    const uint32_t box[2] = {128, 128};
    ROLA_TRY(make_map(&tb, wq, 2, dims, strides, box, "gemm_fp8_block: wq", true));
  }
  GemmBlockParams p{};
  p.xq = static_cast<const uint8_t*>(xq), p.wq = static_cast<const uint8_t*>(wq);
  p.xs = x_scale, p.xs_sM = xs_sM, p.xs_sK = xs_sK;
  p.ws = w_scale, p.ws_ld = (K + 127) / 128;
  p.bias = BF(bias), p.out = BFm(out);
  p.M = (int)M, p.N = (int)N, p.K = (int)K;
  return cuda_status(launch_gemm_block(ta, tb, p, S(stream)), what);
}

// ---------------------------------------------------------------------------
static int check_cross_sizes(int B, int H, int Hkv, int Lq, int Lk, const char* what) {
  ROLA_CHECK(B > 0 && H > 0 && Hkv > 0 && Lq > 0 && Lk > 0, "%s: bad sizes", what);
  ROLA_CHECK(H % Hkv == 0, "%s: the query heads must be a multiple of the key heads", what);
  ROLA_CHECK(Lq < (1 << 30) && Lk < (1 << 30), "%s: sequence too long", what);
  ROLA_CHECK((int64_t)B * H * ((Lq + 63) / 64) < (1ll << 31) && (int64_t)B * H * ((Lk + 127) / 128) * 8 < (1ll << 31),
             "%s: too many tiles", what);
  return ROLA_OK;
}
static bool head_strides_ok(int64_t sB, int64_t sH, int64_t sT) {
  return sB > 0 && sH > 0 && sT > 0 && sB % 8 == 0 && sH % 8 == 0 && sT % 8 == 0;
}

size_t rola_b200_cross_attn_workspace(int B, int H, int Hkv, int Lq, int Lk) {
  if (check_cross_sizes(B, H, Hkv, Lq, Lk, "cross_attn_workspace") != ROLA_OK) return 0;
  const CrossAttnPlan pl = cross_attn_plan(B, H, Hkv, Lq, Lk);
  return pl.nsplit > 1 ? (size_t)pl.nsplit * B * H * Lq * (128 + 1) * 4 : 0;
}

int rola_b200_cross_attn(const void* q, int64_t q_sB, int64_t q_sH, int64_t q_sT, const void* k, int64_t k_sB,
                         int64_t k_sH, int64_t k_sT, const void* v, int64_t v_sB, int64_t v_sH, int64_t v_sT,
                         const int32_t* kv_lens, int B, int H, int Hkv, int Lq, int Lk, void* out, int64_t o_sB,
                         int64_t o_sH, int64_t o_sT, float* lse, void* workspace, size_t workspace_bytes,
                         rola_stream_t stream) {
  const char* what = "cross_attn";
  ROLA_CHECK(q && k && v && out, "%s: null pointer", what);
  ROLA_TRY(check_cross_sizes(B, H, Hkv, Lq, Lk, what));
  ROLA_CHECK(head_strides_ok(q_sB, q_sH, q_sT) && head_strides_ok(k_sB, k_sH, k_sT) &&
                 head_strides_ok(v_sB, v_sH, v_sT) && head_strides_ok(o_sB, o_sH, o_sT) && aligned16(out),
             "%s: positive strides and 16-byte aligned rows required", what);
  const CrossAttnPlan pl = cross_attn_plan(B, H, Hkv, Lq, Lk);
  const size_t need = rola_b200_cross_attn_workspace(B, H, Hkv, Lq, Lk);
  ROLA_CHECK(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
             "%s: a 16-byte aligned workspace of %zu bytes is needed", what, need);
  CrossAttnParams p{};
  p.kv_lens = kv_lens;
  p.out = BFm(out), p.o_sB = o_sB, p.o_sH = o_sH, p.o_sT = o_sT;
  p.lse = lse, p.lse_ld = 128 * ((Lq + 127) / 128);
  p.B = B, p.H = H, p.Hkv = Hkv, p.G = H / Hkv, p.Lq = Lq, p.Lk = Lk;
  p.pack = pl.pack, p.nqt = pl.nqt, p.nsplit = pl.nsplit;
  p.Hgrid = pl.pack ? Hkv : H;
  p.items = (int64_t)pl.nqt * pl.nsplit * B * p.Hgrid;
  p.part_o = static_cast<float*>(workspace);
  p.part_lse = p.part_o ? p.part_o + (size_t)pl.nsplit * B * H * Lq * 128 : nullptr;
  p.q_bytes = pl.pack ? 256u * (uint32_t)(p.G * Lq) : 32768u;
  p.qk_scale = (float)(0.08838834764831845 * 1.4426950408889634);  // 128^-0.5 * log2(e)
  CUtensorMap tq, tk, tv, to;
  if (pl.pack) {  // one box holds the G heads of a key head, Lq rows each
    const uint64_t dims[4] = {128, (uint64_t)Lq, (uint64_t)H, (uint64_t)B};
    const uint32_t box[4] = {64, (uint32_t)Lq, (uint32_t)p.G, 1};
    const uint64_t qs[3] = {(uint64_t)q_sT * 2, (uint64_t)q_sH * 2, (uint64_t)q_sB * 2};
    const uint64_t os[3] = {(uint64_t)o_sT * 2, (uint64_t)o_sH * 2, (uint64_t)o_sB * 2};
    ROLA_TRY(make_map(&tq, q, 4, dims, qs, box, "cross_attn: q"));
    ROLA_TRY(make_map(&to, out, 4, dims, os, box, "cross_attn: out"));
  } else {
    ROLA_TRY(make_head_map(&tq, q, 128, q_sB, q_sH, q_sT, Lq, H, B, "cross_attn: q"));
    ROLA_TRY(make_head_map(&to, out, 128, o_sB, o_sH, o_sT, Lq, H, B, "cross_attn: out"));
  }
  ROLA_TRY(make_head_map(&tk, k, 128, k_sB, k_sH, k_sT, Lk, Hkv, B, "cross_attn: k"));
  ROLA_TRY(make_head_map(&tv, v, 128, v_sB, v_sH, v_sT, Lk, Hkv, B, "cross_attn: v"));
  return cuda_status(launch_cross_attn(tq, tk, tv, to, p, S(stream)), what);
}

struct CrossBwdLayout {
  size_t delta, part, total;
  int runs;
};
static CrossBwdLayout cross_bwd_layout(int B, int H, int Hkv, int Lq, int Lk) {
  CrossBwdLayout f{};
  f.runs = cross_bwd_runs(B, H, Hkv, Lq, Lk);
  f.part = align256((size_t)B * H * (128 * (((size_t)Lq + 127) / 128)) * 4);
  f.total = f.part + (size_t)2 * f.runs * 2 * 128 * 128 * 4;
  return f;
}

size_t rola_b200_cross_attn_bwd_workspace(int B, int H, int Hkv, int Lq, int Lk) {
  if (check_cross_sizes(B, H, Hkv, Lq, Lk, "cross_attn_bwd_workspace") != ROLA_OK) return 0;
  return cross_bwd_layout(B, H, Hkv, Lq, Lk).total;
}

int rola_b200_cross_attn_bwd(const void* q, int64_t q_sB, int64_t q_sH, int64_t q_sT, const void* k, int64_t k_sB,
                             int64_t k_sH, int64_t k_sT, const void* v, int64_t v_sB, int64_t v_sH, int64_t v_sT,
                             const void* out, int64_t o_sB, int64_t o_sH, int64_t o_sT, const void* dout, int64_t do_sB,
                             int64_t do_sH, int64_t do_sT, const int32_t* kv_lens, const float* lse, int B, int H,
                             int Hkv, int Lq, int Lk, void* dq, int64_t dq_sB, int64_t dq_sH, int64_t dq_sT, void* dk,
                             void* dv, int64_t dkv_sB, int64_t dkv_sH, int64_t dkv_sT, void* workspace,
                             size_t workspace_bytes, rola_stream_t stream) {
  const char* what = "cross_attn_bwd";
  ROLA_CHECK(q && k && v && out && dout && lse && dq && dk && dv && workspace, "%s: null pointer", what);
  ROLA_TRY(check_cross_sizes(B, H, Hkv, Lq, Lk, what));
  ROLA_CHECK(head_strides_ok(q_sB, q_sH, q_sT) && head_strides_ok(k_sB, k_sH, k_sT) &&
                 head_strides_ok(v_sB, v_sH, v_sT) && head_strides_ok(o_sB, o_sH, o_sT) &&
                 head_strides_ok(do_sB, do_sH, do_sT) && head_strides_ok(dq_sB, dq_sH, dq_sT) &&
                 head_strides_ok(dkv_sB, dkv_sH, dkv_sT),
             "%s: positive strides, multiples of 8, required", what);
  ROLA_CHECK(aligned16(out) && aligned16(dout) && aligned16(dq) && aligned16(dk) && aligned16(dv) && aligned16(lse) &&
                 aligned16(workspace),
             "%s: 16-byte aligned tensors required", what);
  const CrossBwdLayout f = cross_bwd_layout(B, H, Hkv, Lq, Lk);
  ROLA_CHECK(kv_lens == nullptr || B <= 65536, "%s: at most 65536 sequences of their own lengths", what);
  ROLA_CHECK(workspace_bytes >= f.total, "%s: workspace of %zu bytes < %zu", what, workspace_bytes, f.total);
  CUtensorMap tq, tk, tv, tdo, tdq;
  ROLA_TRY(make_head_map(&tq, q, 128, q_sB, q_sH, q_sT, Lq, H, B, "cross_attn_bwd: q", 64));
  ROLA_TRY(make_head_map(&tk, k, 128, k_sB, k_sH, k_sT, Lk, Hkv, B, "cross_attn_bwd: k", 64));
  ROLA_TRY(make_head_map(&tv, v, 128, v_sB, v_sH, v_sT, Lk, Hkv, B, "cross_attn_bwd: v", 64));
  ROLA_TRY(make_head_map(&tdo, dout, 128, do_sB, do_sH, do_sT, Lq, H, B, "cross_attn_bwd: dout", 64));
  ROLA_TRY(make_head_map(&tdq, dq, 128, dq_sB, dq_sH, dq_sT, Lq, H, B, "cross_attn_bwd: dq", 64));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  CrossBwdParams p{};
  p.kv_lens = kv_lens;
  p.lse = lse;
  p.delta = reinterpret_cast<float*>(ws + f.delta);
  p.part = reinterpret_cast<float*>(ws + f.part);
  p.dq = BFm(dq), p.dq_sB = dq_sB, p.dq_sH = dq_sH, p.dq_sT = dq_sT;
  p.dk = BFm(dk), p.dv = BFm(dv), p.dkv_sB = dkv_sB, p.dkv_sH = dkv_sH, p.dkv_sT = dkv_sT;
  p.B = B, p.H = H, p.Hkv = Hkv, p.G = H / Hkv, p.Lq = Lq, p.Lk = Lk;
  p.NQT = (Lq + 127) / 128, p.NKT = (Lk + 127) / 128, p.Lpad = 128 * p.NQT, p.runs = f.runs;
  p.qk_scale = (float)(0.08838834764831845 * 1.4426950408889634);
  p.o = BF(out), p.o_sB = o_sB, p.o_sH = o_sH, p.o_sT = o_sT;
  return cuda_status(launch_cross_attn_bwd(tq, tk, tv, tdo, tdq, p, S(stream)), what);
}

}  // extern "C"
