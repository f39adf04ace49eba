// Drives jitnn_amd/csrc/row_end.h: where the loads of a row's last pieces start, and what they leave (no GPU).  Prints what does not hold; exit status 0: all holds.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "row_end.h"

#define CHECK(e)                                                       \
    do {                                                               \
        if (!(e)) {                                                    \
            printf("%s:%d: %s does not hold\n", __FILE__, __LINE__, #e); \
            exit(1);                                                   \
        }                                                              \
    } while (0)

// A column of a row is 272 bytes at most (eight blocks of Q8_0), read in pieces of sixteen from the row's bytes on: a place of it is never further behind the end than that.
constexpr long long COLUMN = 272;

// Matrices of every size in bytes, beyond 31 and 32 bits too: in front of its last fifteen bytes a place is read where it stands, behind them from the last sixteen.
static void places() {
    for (const long long bytes : {16ll, 34ll, 3060ll, 2147483646ll, 2147483648ll, 2147483680ll, 2256076800ll, 4294967290ll, 4294967296ll, 4294967316ll, 9126805504ll, 1ll << 45}) {
        std::vector<long long> at;
        for (long long d = 0; d < 600; ++d) {
            at.push_back(d);
            at.push_back(bytes - 300 + d);
            for (int shift : {31, 32, 33}) at.push_back(bytes - (1ll << shift) - 300 + d);
            at.push_back(bytes / 3 + d);
        }
        for (const long long p : at) {
            if (p < 0 || p > bytes + COLUMN) continue;
            const int behind = jitnn::bytes_behind(p - bytes + 16);
            const long long start = p - behind;
            CHECK(behind >= 0 && start >= 0 && start + 16 <= bytes);
            CHECK(p + 16 <= bytes ? behind == 0 : start == bytes - 16);
        }
    }
}

// The bytes themselves: those of the matrix, zeros behind its end.
static void bytes_left() {
    for (int size : {16, 18, 40, 100}) {
        std::vector<uint8_t> m(size);
        for (int i = 0; i < size; ++i) m[i] = (uint8_t)(1 + 7 * i);
        for (int p = 0; p <= size + 40; ++p) {
            const int behind = jitnn::bytes_behind((long long)p - size + 16);
            jitnn::Halves v;
            memcpy(&v, m.data() + p - behind, 16);
            v = jitnn::moved_down(v, behind);
            uint8_t got[16];
            memcpy(got, &v, 16);
            for (int i = 0; i < 16; ++i) CHECK(got[i] == (p + i < size ? m[p + i] : 0));
        }
    }
}

int main() {
    places();
    bytes_left();
    return 0;
}
