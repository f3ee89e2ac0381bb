// smsgate_amd — C entries of the training operators that train_autograd.cpp calls, included by
// the kernels' sources too, so that both sides are compiled against one signature.  They
// return 0, or what was refused (1 sizes, 3 workspace) or failed (2 a launch).
#pragma once
#include <hip/hip_runtime_api.h>

extern "C" {

// embed_kernels.hip.  dtype 0 fp32, 1 bf16, 2 fp16; vec: every pointer and row is a multiple of 16 bytes
int sg_embed_fwd(const void* ids, const void* add, int is64, const void* table, void* x, int n, int V, int H,
                 float scale, int dtype, int vec, hipStream_t st);
int sg_embed_grad_ws(int n2, int V, int H);
int sg_embed_grad(const void* ids, const void* add, int is64, const void* dx, void* dt, int n, int V, int H,
                  float scale, int dtype, int vec, void* ws, int ws_units, hipStream_t st);

// attn_grad_kernels.hip.  strides: of q, k and v, in elements: batch, head, row
int sg_attn_rows(int T);
int sg_attn_split(int B, int T, int nh, int nkv);
int sg_attn_maxima(int B);
int sg_attn_fwd(const void* q, const void* k, const void* v, const void* lens, void* out, void* olo, void* lse,
                const void* strides, int B, int T, int nh, int nkv, int D, int causal, int fp16, float scale,
                hipStream_t st);
int sg_attn_bwd(const void* q, const void* k, const void* v, const void* lens, const void* out, const void* olo,
                const void* lse, const void* dout, void* dq, void* dk, void* dv, void* ws, const void* strides, int B,
                int T, int nh, int nkv, int D, int causal, int fp16, float scale, hipStream_t st);

// loss_kernels.hip.  mode 0 mean, 1 sum, 2 none
int sg_loss_plan(int N, int V, int H, void* out);
int sg_loss_fwd(const void* h, const void* table, const void* labels, int is64, int ignore, void* hc, void* ec,
                void* state, void* ws, void* loss, int N, int V, int H, int mode, int fp16, hipStream_t st);
int sg_loss_bwd(const void* hc, const void* ec, void* state, const void* g, void* ws, void* dh, void* dtable, int N,
                int V, int H, int mode, int fp16, hipStream_t st);
}
