// What the block operators of the C++ interface answer without a GPU: their workspaces, and what they refuse.
//   test_block_ops_host workspace B T H Hkv hd window sinks   prints the bytes for both directions, and for the forward pass
//   test_block_ops_host norm rows cols                        a norm call of that shape with a gate, which aborts with a message
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "llmt/kernels/attention.h"
#include "llmt/kernels/norm_residual.h"

using namespace llmt;

namespace {

char g_data[64];

Tensor tensor(DType dtype, const Shape& shape) {
    Tensor t;
    t.data = g_data;
    t.dtype = dtype;
    t.shape = shape;
    return t;
}

}  // namespace

int main(int argc, char** argv) {
    if (argc < 2) return 2;
    long long n[8] = {};
    for (int i = 2; i < argc && i < 10; ++i) n[i - 2] = std::atoll(argv[i]);
    if (std::strcmp(argv[1], "workspace") == 0) {
        const Tensor qkv = tensor(DType::BF16, {n[0], n[1], (n[2] + 2 * n[3]) * n[4]});
        kernels::WindowSpec spec;
        spec.window = n[5];
        spec.sinks = n[6];
        std::printf("%zu %zu\n", kernels::attention_window_workspace_bytes(qkv, n[2], n[3], spec),
                    kernels::attention_window_fwd_workspace_bytes(qkv, n[2], n[3], spec));
        return 0;
    }
    if (std::strcmp(argv[1], "norm") == 0) {
        const Tensor x = tensor(DType::FP32, {n[0], n[1]}), gate = tensor(DType::FP32, {1, n[1]}), w = tensor(DType::FP32, {n[1]});
        Tensor out = x, h = x;
        kernels::NormResidual norm;
        norm.gate = &gate;
        norm.w_pre = &w;
        const RunCtx ctx{};
        kernels::norm_residual_fwd(ctx, &out, &h, x, &x, norm);
        return 0;
    }
    return 2;
}
