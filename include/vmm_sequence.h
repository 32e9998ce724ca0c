/* Argument structs of the sequence-encoder and training operators of vmm_kernels.h (which includes this file and says what the members mean). */
#ifndef VMM_SEQUENCE_H
#define VMM_SEQUENCE_H
#include <stdint.h>

typedef struct vmm_gated_scan_desc {
  const void* x; int64_t x_batch, x_row;
  const void* gate; int64_t gate_batch, gate_row;
  void* y; int64_t y_batch, y_row;
  const float* h0; float* h_last; const int32_t* lengths; float* states;
  const void* dy; int64_t dy_batch, dy_row;
  void* dx; int64_t dx_batch, dx_row;
  void* dgate; int64_t dgate_batch, dgate_row;
  const float* dh_last; float* dh0;
  void* workspace; int64_t workspace_bytes;
  int64_t L;
  int32_t B, D, type;
} vmm_gated_scan_desc;

typedef struct vmm_gated_ff_desc {
  const void* x; int64_t ldx;
  const void* w_gate; const void* w_up; const void* b_gate; const void* b_up;
  void* h; int64_t ldh;
  float* g_pre; float* u_pre;
  const void* dh; int64_t lddh;
  void* dx; int64_t lddx;
  void* dw_gate; void* dw_up; void* db_gate; void* db_up;
  void* workspace; int64_t workspace_bytes;
  int64_t M;
  int32_t K, F, type, act;
} vmm_gated_ff_desc;

typedef struct vmm_grad_job { void* g; int64_t n; int32_t type; int32_t reserved; } vmm_grad_job;

typedef struct vmm_clip_adam_job { float* p; const void* g; float* m; float* v; int64_t n; int32_t type; int32_t reserved; } vmm_clip_adam_job;

#endif
