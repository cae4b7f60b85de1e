// Differential attention on bf16 data: the kernels of diff_attn.inl.
#define UBV_ATTN_T bf16_t
#define UBV_ATTN_NAME(what) diff_attn_##what##_bf16
#include "diff_attn.inl"
