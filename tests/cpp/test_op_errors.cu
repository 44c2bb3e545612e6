// CPU check of what a C entry of the training operators reports
// (alphazero_b200/csrc/ops_common.cuh): every exception becomes a code, and
// the message is of this failure, not of an earlier one.
#include "../../alphazero_b200/csrc/ops_common.cuh"

#include <cstdio>
#include <new>
#include <stdexcept>

namespace mgb {
namespace ops {
std::string& last_op_error() {
    thread_local std::string message;
    return message;
}
}  // namespace ops
}  // namespace mgb

using namespace mgb::ops;

namespace {

int failures = 0;

template <class F>
void expect(int code, const char* word, F&& body) {
    last_op_error() = "of an earlier call";
    const int got = guarded(body);
    if (got != code || last_op_error().find(word) == std::string::npos) {
        std::printf("code %d (expected %d), message \"%s\" (expected \"%s\")\n", got, code, last_op_error().c_str(), word);
        ++failures;
    }
}

}  // namespace

int main() {
    expect(MG_E_ARG, "a stride is negative", [] { need(false, "a stride is negative"); });
    expect(MG_E_DEVICE, "gave up", [] { fail(MG_E_DEVICE, "gave up"); });
    expect(MG_E_CUDA, "here: ", [] { check(cudaErrorInvalidValue, "here"); });
    expect(MG_E_STATE, "memory", [] { throw std::bad_alloc(); });
    expect(MG_E_STATE, "too long", [] { throw std::length_error("too long"); });
    expect(MG_E_STATE, "unknown", [] { throw 7; });
    expect(MG_OK, "of an earlier call", [] {});
    std::printf("%d failures\n", failures);
    return failures != 0;
}
