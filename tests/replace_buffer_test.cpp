// Drives replace_buffer of jitnn_amd/csrc/scratch.h with an allocator that keeps books (no GPU).  Prints what does not hold; exit status 0: all holds.
#include <cstdio>
#include <cstdlib>
#include <map>

#include "scratch.h"

#define CHECK(e)                                                       \
    do {                                                               \
        if (!(e)) {                                                    \
            printf("%s:%d: %s does not hold\n", __FILE__, __LINE__, #e); \
            exit(1);                                                   \
        }                                                              \
    } while (0)

static std::map<void *, size_t> live;  // address -> bytes
static size_t room = 100;

static void *alloc(size_t bytes) {
    size_t used = 0;
    for (auto &b : live) used += b.second;
    if (used + bytes > room) return nullptr;
    static size_t next = 0x1000;
    void *p = (void *)next;
    next += bytes;
    live[p] = bytes;
    return p;
}
static void release(void *p) {
    if (!live.erase(p)) abort();  // freed twice
}

int main() {
    void *held = nullptr;
    size_t bytes = 0;
    CHECK(jitnn::replace_buffer(held, bytes, 30, false, alloc, release) && bytes == 30 && live.size() == 1 && live.count(held));
    void *const first = held;
    CHECK(!jitnn::replace_buffer(held, bytes, 80, false, alloc, release) && held == first && bytes == 30 && live.count(first));  // no room beside it: it stays
    CHECK(jitnn::replace_buffer(held, bytes, 60, false, alloc, release) && held != first && bytes == 60 && live.size() == 1);
    CHECK(jitnn::replace_buffer(held, bytes, 80, true, alloc, release) && bytes == 80 && live.size() == 1 && live.count(held));  // the old one given up first
    CHECK(!jitnn::replace_buffer(held, bytes, 101, true, alloc, release) && !held && bytes == 0 && live.empty());
    CHECK(!jitnn::replace_buffer(held, bytes, 101, false, alloc, release) && !held && bytes == 0);
    CHECK(jitnn::replace_buffer(held, bytes, 100, true, alloc, release) && bytes == 100);
    return 0;
}
