// The attention kernels on the tensor cores (attention_tc.cu), as attention.cu calls them.
#pragma once
#include "attention.cuh"

bool fg_attn_tc_suits(const fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a);      // can they take this call?
int32_t fg_attn_tc_fwd(fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a);
int32_t fg_attn_tc_bwd(fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a);
// Few rows: `rows` of each sequence on average, the keys in a.splits shares.
int32_t fg_attn_few(fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a, uint32_t rows);
