// What the half-precision product, the norms between blocks and the sampling ask of the HIP runtime: launches.cpp's runtime
// and its form of answers, with a launch's shape checked too.
//
// Commands on stdin, a line each:
//   kernels                                  every registered kernel: "kernel NAME"
//   device D                                 the current device from here on
//   half WTYPE N K ROWS XOFF XSTRIDE YTYPE GATE RES   syn_half_gemv, x XOFF values behind a line, GATE and RES types or 9 (none)
//   halfneed N K ROWS ALIGNED                its workspace: "need BYTES INVALID"
//   norm XTYPE BTYPE YTYPE ROWS N WITH       syn_block_norm; WITH: 1 a branch, 2 post, 4 a gate of rows, 8 a gate for all, 16 g
//   sample XTYPE ROWS VOCAB TOP_K EACH       syn_sample_tokens, with settings a row where EACH
// A launch that no grid holds, or whose threads pass 32 bits in a dimension, ends the program.
#define main launches_main
#define hipLaunchKernel launches_kernel
#include "launches.cpp"
#undef main
#undef hipLaunchKernel

extern "C" int hipLaunchKernel(const void* f, Dim grid, Dim block, void** args, size_t lds, void* stream) {
    const uint64_t x = uint64_t(grid.x) * block.x;
    if (!grid.x || !grid.y || !grid.z || x >> 32 || grid.y > 65535 || grid.z > 65535 || block.x > 1024 || block.y != 1 || block.z != 1) {
        std::fprintf(stderr, "grid %u %u %u of %u threads: %s\n", grid.x, grid.y, grid.z, block.x, state().names[f].c_str());
        std::exit(3);
    }
    return launches_kernel(f, grid, block, args, lds, stream);
}

int main() {
    uint8_t* const A = reinterpret_cast<uint8_t*>(uintptr_t(1) << 40);
    const float* const f = reinterpret_cast<const float*>(A);
    const uint64_t all = uint64_t(1) << 62;
    for (std::string line; std::getline(std::cin, line);) {
        std::istringstream in(line);
        std::string what;
        std::vector<uint32_t> v;
        in >> what;
        for (uint32_t n; in >> n;) v.push_back(n);
        auto ty = [&](int i) { return static_cast<int32_t>(v.at(i)); };
        int rc = 0;
        if (what == "kernels") {
            for (const auto& k : state().names) std::printf("kernel %s\n", k.second.c_str());
        } else if (what == "device") {
            state().device = ty(0);
        } else if (what == "half") {
            const uint32_t n = v.at(1), k = v.at(2), rows = v.at(3);
            const bool on = v.at(4) % 8 == 0 && k % 128 == 0 && (rows <= 1 || v.at(5) % 8 == 0);
            uint64_t need = 0;
            rc = syn_half_gemv_workspace_bytes(n, k, rows, on, &need);
            if (rc == 0)
                rc = syn_half_gemv(ty(0), A, all, (uint64_t(k) + 127) / 128 * 128, f, n, k, A + 2 * v.at(4), v.at(5), rows, SYN_ACT_GELU, ty(7),
                                   v.at(7) == 9 ? nullptr : A, n, ty(8), v.at(8) == 9 ? nullptr : A, n, ty(6), A, n, need ? A : nullptr,
                                   need, nullptr);
        } else if (what == "halfneed") {
            uint64_t need = 0;
            std::feclearexcept(FE_ALL_EXCEPT);
            rc = syn_half_gemv_workspace_bytes(v.at(0), v.at(1), v.at(2), ty(3), &need);
            std::printf("need %llu %d\n", static_cast<unsigned long long>(need), std::fetestexcept(FE_INVALID) != 0);
        } else if (what == "norm") {
            const uint32_t rows = v.at(3), n = v.at(4), with = v.at(5);
            const bool branch = with & 1;
            rc = syn_block_norm(ty(0), A, n, ty(1), branch ? A : nullptr, n, with & 2 ? f : nullptr, with & 12 ? A : nullptr, with & 4 ? n : 0,
                                0.5f, with & 16 ? f : nullptr, 1e-5f, rows, n, A, n, ty(2), A, n, nullptr);
        } else if (what == "sample") {
            const uint32_t rows = v.at(1), vocab = v.at(2);
            const bool each = v.at(4) != 0;
            int32_t* const i = reinterpret_cast<int32_t*>(A);
            uint64_t need = 0;
            rc = syn_sample_tokens_workspace_bytes(ty(0), rows, vocab, &need);
            if (rc == 0)
                rc = syn_sample_tokens(ty(0), A, vocab, rows, vocab, f, each ? f : nullptr, each ? i : nullptr, each ? f : nullptr,
                                       each ? f : nullptr, 0.7f, ty(3), 0.9f, 0.01f, i, reinterpret_cast<float*>(A), i, need ? A : nullptr,
                                       need, nullptr);
        } else {
            rc = -1;
        }
        std::printf("rc %d\n", rc);
    }
    return 0;
}
