// elf_string_test.cpp -- tsdf::host::elf_string_constant on a real code object, on every truncation of it and on damaged
// copies: no device.  Usage: elf_string_test <code object> <symbol>; prints the text.  Exit code 0 = pass.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <string>
#include <vector>

#include "../../tracking_sdf_amd/csrc/host_util.hpp"

int main(int argc, char** argv) {
    if (argc != 3) return 2;
    std::vector<char> img;
    FILE* f = std::fopen(argv[1], "rb");
    if (!f) return 2;
    for (int c; (c = std::fgetc(f)) != EOF;) img.push_back((char)c);
    std::fclose(f);
    std::string id, got;
    if (!tsdf::host::elf_string_constant(img.data(), img.size(), argv[2], &id)) { std::fprintf(stderr, "symbol not found\n"); return 1; }
    std::printf("%s\n", id.c_str());
    if (tsdf::host::elf_string_constant(img.data(), img.size(), "no_such_symbol", &got)) { std::fprintf(stderr, "found what is not there\n"); return 1; }
    if (tsdf::host::elf_string_constant(nullptr, 0, argv[2], &got) || tsdf::host::elf_string_constant("", 0, argv[2], &got)) return 1;
    // exact-size heap copies: a read outside the image is the address sanitizer's to catch; what is found is never another text
    for (size_t n = 0; n < img.size(); n += n < 4096 ? 7 : 997) {
        const std::vector<char> cut(img.begin(), img.begin() + (long)n);
        if (tsdf::host::elf_string_constant(cut.data(), cut.size(), argv[2], &got) && got != id) return 1;
    }
    std::mt19937 rng(11);
    const size_t head = 64, table = img.size() < 2048 ? 0 : img.size() - 2048;      // the ELF header; the section headers lie at the end
    for (int k = 0; k < 4000; ++k) {
        std::vector<char> bad(img);
        for (int b = 0; b < 1 + k % 4; ++b) bad[(k & 1 ? table + rng() % (img.size() - table) : rng() % head)] = (char)rng();
        (void)tsdf::host::elf_string_constant(bad.data(), bad.size(), argv[2], &got);
    }
    return 0;
}
