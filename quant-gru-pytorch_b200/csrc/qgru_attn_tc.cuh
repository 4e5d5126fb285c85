// qgru_attn_tc.cuh - linear attention on the tensor cores (qgru_attn_tc.cu).
#pragma once
#include "qgru_attn.cuh"

namespace qgru {
namespace attn {

bool tc_takes(const qgru_attention &a);
Cut tc_cut(const qgru_attention &a, int sms);
// flag: where a kernel says that a wait of its own has run out
int tc_forward(const qgru_attention &a, const Cut &c, int *flag, cudaStream_t st);
int tc_backward(const qgru_attention &a, const Cut &c, int *flag, cudaStream_t st);

}  // namespace attn
}  // namespace qgru
