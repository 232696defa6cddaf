// The check of the paged attention's join records against its rule in 128 bits: every record that passes stays inside its tensors. Prints "ok" last.
#include <cstdint>
#include <cstdio>
#include <random>

#include "kv_join_record.h"

using augur_sm100::JoinRecord;
using Wide = unsigned __int128;

static uint64_t wrong = 0, passed = 0;

static void check(JoinRecord r, uint32_t group, uint32_t columns, uint32_t rows, uint32_t kv_heads, uint32_t spans) {
    const bool want = Wide(r.tokens) * group <= columns && Wide(r.row) + r.tokens <= rows && r.head < kv_heads && r.first <= r.last && r.last < spans;
    const bool got = augur_sm100::join_record_ok(r, group, columns, rows, kv_heads, spans);
    if (got != want) ++wrong;
    if (got) {
        ++passed;
        // what the join reads and writes: token rows [row, row + tokens), parts 2 first .. 2 last + 1, columns [0, tokens group)
        if (r.tokens && Wide(r.row) + r.tokens - 1 >= rows) ++wrong;
        if (2 * Wide(r.last) + 1 >= 2 * Wide(spans) || Wide(r.tokens) * group > columns) ++wrong;
    }
}

int main() {
    // values next to every border, and those that wrap round in 32 bits
    const uint32_t some[] = {0, 1, 7, 8, 63, 64, 65, 147, 148, 1u << 20, 0x7fffffffu, 0x80000000u, 0x80000001u, 0xaaaaaaabu, 0xfffffff8u, 0xffffffffu};
    for (const uint32_t row : some) {
        for (const uint32_t tokens : some) {
            for (const uint32_t group : {1u, 2u, 3u, 6u, 8u, 64u}) {
                for (const uint32_t last : some) check({row, tokens, 0, 0, last, {}}, group, 64, 1u << 20, 4, 148);
            }
        }
    }
    check({0xffffffffu, 1, 0, 0, 0, {}}, 6, 48, 8, 4, 148);            // row + tokens is 0 in 32 bits
    check({0, 0x80000000u, 0, 0, 0, {}}, 2, 48, 8, 4, 148);            // tokens group is 0 in 32 bits
    std::mt19937 random(1);
    auto value = [&] { return static_cast<uint32_t>(random() >> random() % 32); };
    for (int i = 0; i < 2000000; ++i) check({value(), value(), value(), value(), value(), {}}, 1 + value() % 64, 8 + value() % 57, 1 + value(), 1 + value() % 1024, 1 + value() % 256);
    if (wrong || !passed) {
        printf("%llu wrong, %llu passed\n", static_cast<unsigned long long>(wrong), static_cast<unsigned long long>(passed));
        return 1;
    }
    puts("ok");
    return 0;
}
