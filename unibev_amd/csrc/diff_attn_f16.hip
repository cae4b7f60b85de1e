// Differential attention on f16 data: the kernels of diff_attn.inl.
#define UBV_ATTN_T f16_t
#define UBV_ATTN_NAME(what) diff_attn_##what##_f16
#include "diff_attn.inl"
