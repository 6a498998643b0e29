// Entry points of the passes over packed sequences: argument checks and kernel
// choice. The kernels are the pass kernels of their own files, instantiated for
// slots of packed sequences (packed.cuh).
#include <string>

#include "common.cuh"

namespace poly {
namespace {

int fail(int code, const std::string& m) {
  set_error(m);
  return code;
}

// The checks of poly_pass_fwd that apply, then those of the packed layout.
int check_packed(const PolyPassArgs& a, const int32_t* cu, int seqs, int max_len) {
  if (a.batch != 1) return fail(POLY_EINVAL, "packed passes have batch 1");
  if (a.heads > 65535) return fail(POLY_EUNSUPPORTED, "more than 65535 heads");
  if (a.heads <= 0 || a.kv_heads <= 0 || a.seq_q < 0 || a.head_dim <= 0)
    return fail(POLY_EINVAL, "heads, kv_heads and head_dim must be positive, seq_q non-negative");
  if (a.seq_q != a.seq_k) return fail(POLY_EINVAL, "packed passes have seq_q == seq_k (the rows of all sequences)");
  if (a.heads % a.kv_heads != 0) return fail(POLY_EINVAL, "heads must be divisible by kv_heads");
  if (a.dtype != POLY_F32 && a.dtype != POLY_F16 && a.dtype != POLY_BF16) return fail(POLY_EINVAL, "unknown dtype");
  if (a.head_dim > 128) return fail(POLY_EUNSUPPORTED, "head_dim > 128 is not supported");
  if (a.key_mask || a.query_mask || a.v_mul || a.causal_offset)
    return fail(POLY_EUNSUPPORTED, "packed passes take no masks, v_mul or causal_offset");
  if (seqs < 0 || max_len < 0) return fail(POLY_EINVAL, "seqs and max_len must be non-negative");
  if (a.seq_q > 0 && seqs > 0 && (!a.q || !a.k || !a.v || !a.out || !cu))
    return fail(POLY_EINVAL, "q, k, v, out and cu_seqlens are required");
  if (a.epi_out && !a.epi_mul) return fail(POLY_EINVAL, "epi_out requires epi_mul");
  if (!(a.scale == a.scale)) return fail(POLY_EINVAL, "scale is NaN");
  // 8-row slots of every head fit the grid, rows the 32-bit tile arithmetic
  if (a.seq_q > (1 << 30) || seqs > (1 << 28) || (int64_t)(a.seq_q / 8 + seqs) > 0x7fffffff / a.heads)
    return fail(POLY_EUNSUPPORTED, "too many rows or sequences for one call");
  return POLY_OK;
}

void zero_add(ZeroRest& z, void* p, int heads, int dim, int es, int64_t head_stride, int64_t row_stride) {
  if (!p) return;
  auto& t = z.t[z.n++];
  t.p = (char*)p;
  t.heads = heads;
  t.row_bytes = dim * es;
  t.head_stride = head_stride * es;
  t.row_stride = row_stride * es;
  t.wide = !(((uintptr_t)p | (uintptr_t)t.row_bytes | (uintptr_t)t.head_stride | (uintptr_t)t.row_stride) & 15);
}

int check_fwd(const PolyPackedArgs* a) {
  if (!a) return fail(POLY_EINVAL, "null args");
  return check_packed(a->pass, a->cu_seqlens, a->seqs, a->max_len);
}

enum class Kind { kSimt, kTc, kSmall, kF32 };

bool short_sequences(int max_len) { return max_len > 0 && max_len <= 128; }

// The 16-bit tensor-core kernels take the row maximum on unscaled scores: the scale
// has to be positive.
Kind choose_fwd(const PolyPackedArgs& a) {
  if (packed_f32_eligible(a)) return Kind::kF32;
  if (!packed_fwd_tc_eligible(a.pass, a.out_lo) || !(a.pass.scale > 0.f)) return Kind::kSimt;
  return short_sequences(a.max_len) ? Kind::kSmall : Kind::kTc;   // both take the same tensors
}

Kind choose_bwd(const PolyPackedBwdArgs& a) {
  if (!packed_bwd_tc_eligible(a)) return Kind::kSimt;
  return short_sequences(a.max_len) ? Kind::kSmall : Kind::kTc;
}

const char* name_of(Kind k) {
  switch (k) {
    case Kind::kTc: return "tc100";
    case Kind::kSmall: return "small";
    case Kind::kF32: return "tf32x3";
    default: return "simt";
  }
}

int check_bwd(const PolyPackedBwdArgs* a) {
  if (!a) return fail(POLY_EINVAL, "null args");
  return check_packed(a->bwd.fwd, a->cu_seqlens, a->seqs, a->max_len);
}

}  // namespace
}  // namespace poly

using namespace poly;

extern "C" {

size_t poly_sizeof_packed_args(void) { return sizeof(PolyPackedArgs); }
size_t poly_sizeof_packed_bwd_args(void) { return sizeof(PolyPackedBwdArgs); }

const char* poly_packed_pass_fwd_kernel_name(const PolyPackedArgs* a) {
  if (check_fwd(a) != POLY_OK) return "invalid";
  return name_of(choose_fwd(*a));
}

const char* poly_packed_pass_bwd_kernel_name(const PolyPackedBwdArgs* a) {
  if (check_bwd(a) != POLY_OK) return "invalid";
  return name_of(choose_bwd(*a));
}

int poly_packed_pass_fwd(const PolyPackedArgs* a, void* stream) {
  const int rc = check_fwd(a);
  if (rc) return rc;
  if (a->pass.seq_q == 0 || a->seqs == 0) return POLY_OK;
  PackedSeqs q{};
  q.cu = a->cu_seqlens;
  q.seqs = a->seqs;
  q.total = a->pass.seq_q;
  q.max_len = a->max_len;
  q.out_lo = a->out_lo;
  if (a->zero_rest) {
    const PolyPassArgs& f = a->pass;
    const int es = f.dtype == POLY_F32 ? 4 : 2;
    ZeroRest& z = q.zero;
    zero_add(z, f.out, f.heads, f.head_dim, es, f.out_stride[1], f.out_stride[2]);
    zero_add(z, f.epi_out, f.heads, f.head_dim, es, f.epi_out_stride[1], f.epi_out_stride[2]);
    zero_add(z, f.lse, f.heads, 1, 4, f.lse_stride[1], 1);
    zero_add(z, a->out_lo, f.heads, f.head_dim, es, f.out_stride[1], f.out_stride[2]);
  }
  switch (choose_fwd(*a)) {
    case Kind::kTc: return launch_packed_fwd_tc(a->pass, q, (cudaStream_t)stream);
    case Kind::kSmall: return launch_packed_fwd_small(a->pass, q, (cudaStream_t)stream);
    case Kind::kF32: return launch_packed_fwd_f32(a->pass, q, (cudaStream_t)stream);
    default: return launch_packed_fwd_simt(a->pass, q, (cudaStream_t)stream);
  }
}

size_t poly_packed_pass_bwd_workspace_size(const PolyPackedBwdArgs* a) {
  if (check_bwd(a) != POLY_OK) return 0;
  switch (choose_bwd(*a)) {
    case Kind::kTc: return packed_bwd_tc_workspace(a->bwd, a->seqs);
    case Kind::kSmall: return 0;
    default: return packed_bwd_simt_workspace(a->bwd);
  }
}

int poly_packed_pass_bwd(const PolyPackedBwdArgs* a, void* stream) {
  const int rc = check_bwd(a);
  if (rc) return rc;
  const PolyPassBwdArgs& b = a->bwd;
  if (b.fwd.seq_q == 0 || a->seqs == 0) return POLY_OK;
  if (!b.fwd.lse || !b.dout || !b.dq || !b.dk || !b.dv)
    return fail(POLY_EINVAL, "backward needs fwd.out, fwd.lse, dout, dq, dk and dv");
  if (!a->v_left != !a->v_right || !a->v_left != !a->dv_right)
    return fail(POLY_EINVAL, "v_left, v_right and dv_right come together");
  PackedSeqs q{};
  q.cu = a->cu_seqlens;
  q.seqs = a->seqs;
  q.total = b.fwd.seq_q;
  q.max_len = a->max_len;
  q.out_lo = const_cast<void*>(a->out_lo);
  q.v_left = a->v_left;
  q.v_right = a->v_right;
  q.dv_right = a->dv_right;
  for (int i = 0; i < 2; ++i) {
    q.v_left_stride[i] = a->v_left_stride[i];
    q.v_right_stride[i] = a->v_right_stride[i];
    q.dv_right_stride[i] = a->dv_right_stride[i];
  }
  const size_t need = poly_packed_pass_bwd_workspace_size(a);
  if (need && (!b.workspace || b.workspace_bytes < need))
    return fail(POLY_EINVAL, "workspace too small: need " + std::to_string(need) + " bytes");
  if ((uintptr_t)b.workspace & 15) return fail(POLY_EINVAL, "workspace must be 16-byte aligned");
  if (a->zero_rest) {
    const PolyPassArgs& f = b.fwd;
    const int es = f.dtype == POLY_F32 ? 4 : 2;
    ZeroRest& z = q.zero;
    if (!b.dq_accumulate) zero_add(z, b.dq, f.heads, f.head_dim, es, b.dq_stride[1], b.dq_stride[2]);
    zero_add(z, b.dk, f.kv_heads, f.head_dim, es, b.dk_stride[1], b.dk_stride[2]);
    zero_add(z, b.dv, f.kv_heads, f.head_dim, es, b.dv_stride[1], b.dv_stride[2]);
    zero_add(z, b.dbias, f.kv_heads, 1, 4, b.dbias_stride[1], 1);
    zero_add(z, a->dv_right, f.kv_heads, f.head_dim, es, a->dv_right_stride[0], a->dv_right_stride[1]);
  }
  switch (choose_bwd(*a)) {
    case Kind::kTc: return launch_packed_bwd_tc(b, q, (cudaStream_t)stream);
    case Kind::kSmall: return launch_packed_bwd_small(b, q, (cudaStream_t)stream);
    default: return launch_packed_bwd_simt(b, q, (cudaStream_t)stream);
  }
}

}  // extern "C"
