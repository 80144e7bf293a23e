// The dense operators' entry points behind one function that takes its arguments as an array of
// 64-bit words: what the Python layer calls, since converting twenty arguments one by one takes it
// longer than a small operator runs. Words stand in the order of the entry point's parameters.
#include "tcc_spmm_b200.h"

namespace {
template <typename T> T* ptr(uint64_t v) { return reinterpret_cast<T*>(static_cast<uintptr_t>(v)); }
uint32_t u32(uint64_t v) { return static_cast<uint32_t>(v); }
int i32(uint64_t v) { return static_cast<int>(v); }
} // namespace

extern "C" int tcc_dense8_call(int op, const uint64_t* v) {
    switch (op) {
    case 0:
        return tcc_quantize_blocks_fp8(ptr<void>(v[0]), i32(v[1]), v[2], ptr<void>(v[3]), i32(v[4]), v[5],
                                       ptr<uint8_t>(v[6]), u32(v[7]), u32(v[8]), u32(v[9]), ptr<CUstream_st>(v[10]));
    case 1:
        return tcc_matmul_fp8_blocks(ptr<void>(v[0]), i32(v[1]), v[2], ptr<uint8_t>(v[3]), u32(v[4]), ptr<void>(v[5]),
                                     i32(v[6]), v[7], ptr<uint8_t>(v[8]), u32(v[9]), i32(v[10]), ptr<float>(v[11]),
                                     ptr<void>(v[12]), i32(v[13]), v[14], u32(v[15]), u32(v[16]), u32(v[17]),
                                     ptr<CUstream_st>(v[18]));
    case 2:
        return tcc_activation_checkpoint_int8(ptr<void>(v[0]), v[1], ptr<void>(v[2]), v[3], i32(v[4]), ptr<int8_t>(v[5]),
                                              v[6], ptr<uint8_t>(v[7]), u32(v[8]), u32(v[9]), i32(v[10]),
                                              ptr<CUstream_st>(v[11]));
    case 3:
        return tcc_activation_backward_int8(ptr<void>(v[0]), v[1], i32(v[2]), ptr<int8_t>(v[3]), v[4], ptr<uint8_t>(v[5]),
                                            ptr<void>(v[6]), v[7], u32(v[8]), u32(v[9]), i32(v[10]),
                                            ptr<CUstream_st>(v[11]));
    case 4:
        return tcc_weight_grad_int8(ptr<void>(v[0]), i32(v[1]), v[2], ptr<int8_t>(v[3]), v[4], ptr<uint8_t>(v[5]),
                                    ptr<float>(v[6]), v[7], u32(v[8]), u32(v[9]), u32(v[10]), i32(v[11]),
                                    ptr<void>(v[12]), v[13], ptr<CUstream_st>(v[14]));
    default:
        return TCC_INVALID_ARGUMENT;
    }
}
