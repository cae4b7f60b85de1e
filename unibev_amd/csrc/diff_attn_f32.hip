// Differential attention on f32 data: the kernels of diff_attn.inl.
#define UBV_ATTN_T float
#define UBV_ATTN_NAME(what) diff_attn_##what##_f32
#include "diff_attn.inl"
