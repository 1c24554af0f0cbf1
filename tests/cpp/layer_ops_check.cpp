// Exercises the layer operators through the C++ mirror (include/larql_backend.hpp).
// usage: layer_ops_check <in.bin> <out.bin>
//   in : int32 rows, cols, tokens, 0; e4m3 codes [rows, cols]; f32 scales [ceil(rows / 128), ceil(cols / 128)]; f32 x [tokens, cols]
//   out: f32 [tokens, rows]
// Exit status 3 when no device / library is available.
#include <cstdio>
#include <cstring>
#include <vector>

#include "larql_backend.hpp"

int main(int argc, char** argv) {
    try {
        larql::CudaBackend be(0);
        if (argc < 3) return 0;
        FILE* f = std::fopen(argv[1], "rb");
        int32_t hdr[4];
        if (!f || std::fread(hdr, 4, 4, f) != 4) return 2;
        const size_t rows = hdr[0], cols = hdr[1], tokens = hdr[2], blocks = (rows + 127) / 128 * ((cols + 127) / 128);
        std::vector<uint8_t> codes(rows * cols), scales(blocks * 4);
        std::vector<float> x(tokens * cols);
        if (std::fread(codes.data(), 1, codes.size(), f) != codes.size() || std::fread(scales.data(), 1, scales.size(), f) != scales.size() ||
            std::fread(x.data(), 4, x.size(), f) != x.size())
            return 2;
        std::fclose(f);
        const larql::QuantMatrix w{larql::QuantFormat::FP8_B128, codes.data(), codes.size(), scales.data(), scales.size(), 1.0f,
                                   (int64_t)rows, (int64_t)cols, false};
        if (be.fp8_matmul(w, x.data(), x.size() - 1, tokens).has_value()) return 5;  // lengths: refused
        const auto out = be.fp8_matmul(w, x.data(), x.size(), tokens);
        if (!out) return 6;
        // no rows: nothing to do; an element type that does not exist is refused
        lq_block_norm_args none;
        std::memset(&none, 0, sizeof none);
        none.type = 9;
        if (be.dev_block_norm(none)) return 7;
        none.type = LQ_T_F32;
        if (!be.dev_block_norm(none) || !be.dev_fp8_quantize(nullptr, LQ_T_BF16, 0, 128, 128, nullptr, nullptr)) return 7;
        if (be.moe_create({w}, {w}, {}, x.data(), LQ_T_F32, nullptr, 1, true).has_value()) return 8;
        try {
            be.moe_create({w}, {w}, {w}, x.data(), LQ_T_F32, nullptr, 1, true);  // matrices in host memory: an argument error
            return 9;
        } catch (const larql::BackendError&) {
        }
        f = std::fopen(argv[2], "wb");
        if (!f || std::fwrite(out->data(), 4, out->size(), f) != out->size()) return 10;
        std::fclose(f);
        return 0;
    } catch (const larql::BackendError& e) {
        std::fprintf(stderr, "BackendError %d: %s\n", e.status, e.what());
        return 3;
    }
}
