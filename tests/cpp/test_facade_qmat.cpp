// test_facade_qmat.cpp -- RowQuantizer and QuantizedMatrix of the C++ facade.  Built and run by tests/test_gpu_cpp_qmat.py on a GPU machine.
#include <cmath>
#include <cstdio>

#include "../../vq_b200/cpp/vq.hpp"

static int failed = 0;
#define CHECK(cond)                                                     \
    do {                                                                \
        if (!(cond)) {                                                  \
            std::printf("FAIL %s:%d  %s\n", __FILE__, __LINE__, #cond); \
            ++failed;                                                   \
        }                                                               \
    } while (0)

int main()
{
    vq::Vector<float> row({127.0f, -2.5f, 3.5f, 0.4f, -0.6f}); // scale 1: halves go to even
    const vq::RowQuantizer::Codes q = vq::RowQuantizer::fit().quantize(row);
    CHECK(q.scale == 1.0f && q.codes.data == std::vector<int8_t>({127, -2, 4, 0, -1}));
    const vq::QuantizedMatrix m = vq::QuantizedMatrix::fit({vq::Vector<float>({127.0f, 1.0f, 2.0f, 3.0f, 4.0f}), vq::Vector<float>({0.0f, 0.0f, 0.0f, 0.0f, 0.0f}),
                                                            vq::Vector<float>({1.0f, -254.0f, 4.0f, 2.0f, 254.0f})}); // scales 1, 0 and 2 (1 / 2 goes to 0)
    const std::vector<float> want = {127.0f * 127 - 2 + 8 + 0 - 4, 0.0f, 2.0f * (254 + 8 + 0 - 127)};
    CHECK(m.product(row).data == want);
    CHECK(m.product(q).data == want);
    try {
        m.product(vq::Vector<float>({1.0f}));
        CHECK(false);
    } catch (const vq::VqError &e) {
        CHECK(e.kind == vq::VqError::DimensionMismatch);
    }
    std::printf(failed ? "%d checks failed\n" : "all checks of codes and products passed\n", failed);
    return failed != 0;
}
