// What the library asks of the HIP runtime, on a host without a GPU: this program defines the runtime's calls
// itself, so that libsyntropy_hip.so's host code runs as it is built and every launch is written down in place
// of being made.  Operand addresses are only numbers: nothing reads them.
//
// Commands on stdin, a line each; answers on stdout:
//   kernels                                  every registered kernel: "kernel NAME"
//   device D                                 the current device from here on
//   i8 GATED N K ROWS XTYPE YTYPE BIAS       syn_i8_gemv, or syn_i8_gate_up_act over 2 N rows
//   i8q N K ROWS YTYPE                       syn_i8_gemv_quantized with the largest workspace it asks for
//   i8quantize K ROWS XTYPE                  syn_i8_quantize
//   i8act K ROWS XTYPE                       syn_i8_act_quantize
//   i8logits VOCAB HIDDEN ROWS               syn_i8_logits
//   logprobs XTYPE ROWS VOCAB TOP BYTES      syn_token_logprobs, tokens of BYTES bytes
//   need N K ROWS                            syn_i8_gemv_quantized_workspace_bytes: "need BYTES INVALID", the latter 1 where
//                                            the host's arithmetic raised the invalid-operation flag
// A launch: "launch DEVICE LDS LIMIT NAME", LIMIT the dynamic LDS allowed on that device for it (-1: never said).
// The end of a command: "rc CODE".
#include <cxxabi.h>

#include <cfenv>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <iostream>
#include <map>
#include <sstream>
#include <string>
#include <utility>
#include <vector>

#include "../../include/syntropy_hip.h"

namespace {
struct Dim {
    uint32_t x, y, z;
};
struct State {
    std::map<const void*, std::string> names;
    std::map<std::pair<int, const void*>, int> limits;
    Dim grid{}, block{};
    size_t lds = 0;
    void* stream = nullptr;
    int device = 0;
};
State& state() {  // (the library registers its kernels before main)
    static State s;
    return s;
}
}  // namespace

extern "C" {
void** __hipRegisterFatBinary(const void*) {
    static void* handle = nullptr;
    return &handle;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
    int rc = 0;
    char* text = abi::__cxa_demangle(name, nullptr, nullptr, &rc);
    state().names[host] = rc == 0 ? text : name;
    std::free(text);
}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
int __hipPushCallConfiguration(Dim grid, Dim block, size_t lds, void* stream) {
    State& s = state();
    s.grid = grid, s.block = block, s.lds = lds, s.stream = stream;
    return 0;
}
int __hipPopCallConfiguration(Dim* grid, Dim* block, size_t* lds, void** stream) {
    const State& s = state();
    *grid = s.grid, *block = s.block, *lds = s.lds, *stream = s.stream;
    return 0;
}
int hipGetDevice(int* device) {
    *device = state().device;
    return 0;
}
int hipGetLastError() { return 0; }
int hipFuncSetAttribute(const void* f, int, int value) {
    state().limits[{state().device, f}] = value;
    return 0;
}
int hipLaunchKernel(const void* f, Dim, Dim, void**, size_t lds, void*) {
    State& s = state();
    const auto at = s.limits.find({s.device, f});
    std::printf("launch %d %zu %d %s\n", s.device, lds, at == s.limits.end() ? -1 : at->second, s.names[f].c_str());
    return 0;
}
}

int main() {
    void* const A = reinterpret_cast<void*>(uintptr_t(1) << 40);
    const float* const scales = static_cast<const float*>(A);
    const int8_t* const w = static_cast<const int8_t*>(A);
    const uint64_t all = uint64_t(1) << 62;
    for (std::string line; std::getline(std::cin, line);) {
        std::istringstream in(line);
        std::string what;
        std::vector<uint32_t> v;
        in >> what;
        for (uint32_t n; in >> n;) v.push_back(n);
        int rc = 0;
        if (what == "kernels") {
            for (const auto& k : state().names) std::printf("kernel %s\n", k.second.c_str());
        } else if (what == "device") {
            state().device = static_cast<int>(v.at(0));
        } else if (what == "i8") {
            const uint32_t n = v.at(1), k = v.at(2), rows = v.at(3);
            const auto call = v.at(0) ? syn_i8_gate_up_act : syn_i8_gemv;
            uint64_t need = 0;
            rc = syn_i8_gemv_workspace_bytes(n, k, rows, static_cast<int>(v.at(0)), &need);
            if (rc == 0)
                rc = call(w, all, (uint64_t(k) + 15) / 16 * 16, scales, v.at(6) ? scales : nullptr, n, k, static_cast<int>(v.at(4)), A, k,
                          rows, static_cast<int>(v.at(5)), A, n, need ? A : nullptr, need, nullptr);
        } else if (what == "i8q") {
            const uint32_t n = v.at(0), k = v.at(1), rows = v.at(2);
            uint64_t need = 0;
            rc = syn_i8_gemv_quantized_workspace_bytes(n, k, rows, &need);
            if (rc == 0)
                rc = syn_i8_gemv_quantized(w, all, (uint64_t(k) + 15) / 16 * 16, scales, nullptr, n, k, rows, static_cast<int>(v.at(3)), A, n,
                                           A, need, nullptr);
        } else if (what == "i8quantize") {
            rc = syn_i8_quantize(static_cast<int>(v.at(2)), A, v.at(0), v.at(1), v.at(0), static_cast<int8_t*>(A),
                                 (uint64_t(v.at(0)) + 127) / 128 * 128, static_cast<float*>(A), nullptr);
        } else if (what == "i8act") {
            uint64_t need = 0;
            rc = syn_i8_gemv_quantized_workspace_bytes(1, v.at(0), v.at(1), &need);
            if (rc == 0) rc = syn_i8_act_quantize(static_cast<int>(v.at(2)), A, v.at(0), v.at(1), v.at(0), A, need, nullptr);
        } else if (what == "i8logits") {
            const uint32_t n = v.at(0), k = v.at(1), rows = v.at(2);
            uint64_t need = 0;
            rc = syn_i8_logits_workspace_bytes(n, k, rows, &need);
            if (rc == 0)
                rc = syn_i8_logits(w, all, (uint64_t(k) + 15) / 16 * 16, scales, n, k, scales, 1e-5f, scales, rows,
                                   static_cast<float*>(A), A, need, nullptr);
        } else if (what == "logprobs") {
            const uint32_t rows = v.at(1), vocab = v.at(2), top = v.at(3);
            uint64_t need = 0;
            rc = syn_token_logprobs_workspace_bytes(static_cast<int>(v.at(0)), rows, vocab, top, &need);
            if (rc == 0)
                rc = syn_token_logprobs(static_cast<int>(v.at(0)), A, vocab, rows, vocab, A, v.at(4), 1.0f, top,
                                        static_cast<float*>(A), static_cast<int32_t*>(A), static_cast<float*>(A),
                                        static_cast<int32_t*>(A), static_cast<float*>(A), need ? A : nullptr, need, nullptr);
        } else if (what == "need") {
            uint64_t need = 0;
            std::feclearexcept(FE_ALL_EXCEPT);
            rc = syn_i8_gemv_quantized_workspace_bytes(v.at(0), v.at(1), v.at(2), &need);
            std::printf("need %llu %d\n", static_cast<unsigned long long>(need), std::fetestexcept(FE_INVALID) != 0);
        } else {
            rc = -1;
        }
        std::printf("rc %d\n", rc);
    }
    return 0;
}
