// Bindings of the block-128 operators: tensors cross as (pointer, pitch)
// integers, checked in Python; a refused launch raises.
#include <pybind11/pybind11.h>

#include "../kernels/block128.h"

namespace py = pybind11;
using namespace ofld::kern;

namespace {

void check(cudaError_t e, const char* what) {
    if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}
// A product kernel whose bounded wait ran out has left its result incomplete:
// the products launched after it say so, until the word is cleared.
void check_product(cudaError_t e, const char* what) {
    check(e, what);
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) return;  // nothing can have been launched
    if (const uint32_t code = block128_error(dev))
        throw std::runtime_error(std::string(what) + ": a product on this device gave up waiting (code " +
                                 std::to_string(code) +
                                 "); results since then are not complete. ops.product_error tells and clears it");
}
MatIn in(uint64_t p, int64_t ld) { return {reinterpret_cast<const void*>(p), ld}; }
MatOut out(uint64_t p, int64_t ld) { return {reinterpret_cast<void*>(p), ld}; }
Block128In qin(uint64_t q, int64_t ld, uint64_t s) {
    return {reinterpret_cast<const void*>(q), ld, reinterpret_cast<const float*>(s)};
}
Block128Out qout(uint64_t q, int64_t ld, uint64_t s) {
    return {reinterpret_cast<void*>(q), ld, reinterpret_cast<float*>(s)};
}
cudaStream_t stream(uint64_t s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace

void bind_block128(py::module_& m) {
    m.def("block128_error", &block128_error);
    m.def("block128_set_error", &block128_set_error);
    m.def("k_quantize_block128", [](uint64_t x, int64_t ldx, int type, uint64_t q, int64_t ldq, uint64_t sc,
                                    int64_t rows, int64_t cols, uint64_t s) {
        check(quantize_block128(in(x, ldx), FloatType(type), qout(q, ldq, sc), rows, cols, stream(s)),
              "quantize_block128");
    });
    m.def("k_dequantize_block128", [](uint64_t q, int64_t ldq, uint64_t sc, uint64_t x, int64_t ldx, int type,
                                      int64_t rows, int64_t cols, uint64_t s) {
        check(dequantize_block128(qin(q, ldq, sc), out(x, ldx), FloatType(type), rows, cols, stream(s)),
              "dequantize_block128");
    });
    m.def("k_swiglu_forward", [](uint64_t g, int64_t ldg, uint64_t u, int64_t ldu, int type, uint64_t h, int64_t ldh,
                                 uint64_t qg, uint64_t sg, uint64_t qu, uint64_t su, int64_t ldq, int64_t rows,
                                 int64_t cols, uint64_t s) {
        check(swiglu_forward(in(g, ldg), in(u, ldu), FloatType(type), out(h, ldh), qout(qg, ldq, sg),
                             qout(qu, ldq, su), rows, cols, stream(s)),
              "swiglu_forward");
    });
    m.def("k_swiglu_backward", [](uint64_t dh, int64_t lddh, int type, uint64_t qg, int64_t ldqg, uint64_t sg,
                                  uint64_t qu, int64_t ldqu, uint64_t su, uint64_t dg, uint64_t du, int64_t ldd,
                                  int64_t rows, int64_t cols, uint64_t s) {
        check(swiglu_backward(in(dh, lddh), FloatType(type), qin(qg, ldqg, sg), qin(qu, ldqu, su), out(dg, ldd),
                              out(du, ldd), rows, cols, stream(s)),
              "swiglu_backward");
    });
    m.def("linear_work_bytes", &linear_work_bytes);
    m.def("k_linear_block128", [](uint64_t x, int64_t ldx, int xtype, uint64_t xq, int64_t ldq, uint64_t xs,
                                  uint64_t work, uint64_t work_bytes, uint64_t wq, int64_t ldw, uint64_t ws,
                                  uint64_t bias, uint64_t y, int64_t ldy, int type, int64_t mm, int64_t n, int64_t k,
                                  uint64_t s) {
        check_product(linear_block128(in(x, ldx), FloatType(xtype), qout(xq, ldq, xs), reinterpret_cast<void*>(work),
                                      work_bytes, qin(wq, ldw, ws), reinterpret_cast<const void*>(bias), out(y, ldy),
                                      FloatType(type), mm, n, k, stream(s)),
                      "linear_block128");
    });
    m.def("grad_work_words", &grad_work_words);
    m.def("k_matmul_input_grad", [](uint64_t dy, int64_t lddy, uint64_t wq, int64_t ldw, uint64_t ws, uint64_t dx,
                                    int64_t lddx, int type, int64_t mm, int64_t n, int64_t k, uint64_t s,
                                    uint64_t work, uint32_t words) {
        check_product(matmul_input_grad(in(dy, lddy), qin(wq, ldw, ws), out(dx, lddx), FloatType(type), mm, n, k,
                                        {reinterpret_cast<uint32_t*>(work), words}, stream(s)),
                      "matmul_input_grad");
    }, py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(),
       py::arg(), py::arg(), py::arg("work") = 0, py::arg("words") = 0);
    m.def("k_matmul_weight_grad", [](uint64_t dy, int64_t lddy, uint64_t xq, int64_t ldx, uint64_t xs, uint64_t dw,
                                     int64_t lddw, int type, int64_t mm, int64_t n, int64_t k, uint64_t s,
                                     uint64_t work, uint32_t words) {
        check_product(matmul_weight_grad(in(dy, lddy), qin(xq, ldx, xs), out(dw, lddw), FloatType(type), mm, n, k,
                                         {reinterpret_cast<uint32_t*>(work), words}, stream(s)),
                      "matmul_weight_grad");
    }, py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(),
       py::arg(), py::arg(), py::arg("work") = 0, py::arg("words") = 0);
}
