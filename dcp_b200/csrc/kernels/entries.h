// C entries of the kernel library that other native code calls; the kernels' sources include this too, so the compiler
// compares the two.  All return 0, or a negative code when nothing ran.
#pragma once
#include <stdint.h>

// The levels of dQ of a backward call (see attn_levels.cuh), with that call's items, rows, heads and channels.  A null
// workspace: none.
struct DcpkDqLevels {
  const void* items;
  int n_items, n_levels, q_rows, hq, channels;
  void* workspace;      // dcpk_attn_bwd_workspace() bytes
};

// An operand of an 8-bit product: `rows` x k codes with k innermost, or (rows_inner) k x rows; `pitch` bytes per row of
// memory, a multiple of 16 like the base; scales[(row >> shift) * scale_row_stride + (k / 128) * scale_k_stride], shift 0 or 7;
// code_type 0 e4m3, 1 e5m2.
struct DcpkFp8Operand {
  const void* codes;
  long pitch;
  const void* scales;
  long scale_row_stride, scale_k_stride;
  int rows, rows_inner, shift, code_type;
};

extern "C" {
int dcpk_fp8_quantize(int type, int code, int ways, const void* x, long pitch, void* codes_a, long pitch_a, void* scales_a, long scale_pitch_a,
                      void* codes_b, long pitch_b, void* scales_b, long scale_pitch_b, long n_rows, int width, void* stream);
int dcpk_fp8_norm(int type, int code, const void* x, long x_pitch, const void* residual, long residual_pitch, const void* w, void* h, void* codes,
                  long code_pitch, void* scales, long scale_pitch, float* rstd, long n_rows, int width, float eps, void* stream);
int dcpk_fp8_norm_bwd_parts(int type, long n_rows, int width, int add);
int dcpk_fp8_norm_bwd(int type, const void* h, long h_pitch, const void* w, const float* rstd, const void* dy, long dy_pitch, const void* add,
                      long add_pitch, void* dx, float* dw, float* part, long n_rows, int width, int* status, void* stream);
int dcpk_fp8_align(const void* from_a, long pitch_a, void* to_a, int rows_a, int width_a, const void* from_b, long pitch_b, void* to_b, int rows_b,
                   int width_b, void* stream);
int dcpk_fp8_gemm(const DcpkFp8Operand* q, const DcpkFp8Operand* p, int k, void* out, long out_pitch, const void* add, long add_pitch,
                  int out_type, int form, void* work, int* status, void* stream);
long dcpk_fp8_gemm_work(long q_rows, long p_rows, int q_rows_inner, int k, int form);
long dcpk_adamw_multi_work(int n_tensors);
int dcpk_adamw_multi(int n_tensors, void* const* params, const void* const* grads, void* const* masters, void* const* ms, void* const* vs,
                     void* const* m_scales, void* const* v_scales, const long* sizes, int param_type, int grad_type, int64_t* step, float lr,
                     double beta1, double beta2, float eps, float wd, float grad_scale, float clip, const float* factor, unsigned seed,
                     float* norm, const int* const* status, int n_status, double* work, void* stream);
int dcpk_attn_fwd_pair(const void* q_arena, long q_rows, const void* kv_arena, long kv_rows, int hq, int hkv, const void* tiles,
                       int n_tiles, const void* kv_entries, int n_kv_entries, const void* masks, int n_mask_rows,
                       void* const* out_ptrs, float* const* lse_ptrs, int n_dst, int lse_stride_a, int lse_stride_b, int n_dst_a,
                       int out_type, int out_channels, float scale, int channels, const void* jobs, int n_jobs,
                       void* const* job_src_ptrs, void* const* job_dst_ptrs, int job_stat_stride, int* status, void* stream);
int dcpk_attn_bwd(const void* q_arena, const void* do_arena, long q_rows, const void* kv_arena, long kv_rows, int hq, int hkv,
                  const void* ctas, int n_ctas, const void* items, int n_items_total, int max_items, const void* masks,
                  int n_mask_rows, const float* lse, const float* delta, int stat_stride, float* const* dq_ptrs,
                  float* const* dkv_ptrs, int n_dst, float scale, int channels, int n_levels, void* workspace, int level_passes,
                  const void* jobs, int n_jobs, void* const* job_src_ptrs, void* const* job_dst_ptrs, int job_stat_stride, int* status,
                  void* stream);
long dcpk_attn_bwd_workspace(int n_items_total, long q_rows, int hq, int channels, int n_levels);
int dcpk_attn_bwd_parts(int n_ctas, int hkv, int group, int max_items, int n_items_total, int any_wave);
int dcpk_attn_bwd_prep(const void* o, const void* d_o, float* delta, int n_rows, int hq, int stat_stride, float* zero0, long nz0,
                       float* zero1, long nz1, const DcpkDqLevels* levels, void* stream);
int dcpk_attn_bwd_prep_cast(int type, const void* o, const void* d_o, int d, void* d_o_rows, float* delta, int n_rows, int hq,
                            int stat_stride, float* zero0, long nz0, float* zero1, long nz1, const DcpkDqLevels* levels, void* stream);
int dcpk_pad_cast_rows(int type, const void* src0, void* dst0, long rows0, const void* src1, void* dst1, long rows1, int d,
                       void* stream);
int dcpk_cut_cast_rows(int src_f32, int type, const void* src0, void* dst0, long rows0, const void* src1, void* dst1, long rows1,
                       int d, void* stream);
int dcpk_cut_cast_gradients(int type, const DcpkDqLevels* levels, const float* dq, void* gq, const float* dkv, void* gkv, long rows1, int d,
                            void* stream);
}
