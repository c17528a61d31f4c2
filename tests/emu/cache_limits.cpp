// TEST INFRASTRUCTURE: the 4-bit cache's kernels at the largest lengths the library takes (near 2^31 slots), a workgroup at a time on the CPU execution
// model.  Arrays of 8 GB are one small piece of memory mapped over and over, between addresses that nobody may touch.
//   cache_limits weights    the last workgroup of k_cache_weights, whose batches reach past the last record
//   cache_limits select     k_cache_select over a whole sequence
//   cache_limits keep       k_cache_select with almost as many rows to keep, of few
//   cache_limits columns    k_cache_attend_rows, with waves whose columns are not there
#define EMU_DEFINE_GLOBALS
#include "hip/hip_runtime.h"

#include <initializer_list>
#include <string>

#include "homcomp_cache_kernels.cpp"

namespace {

// `bytes` of zeros that repeat every `piece` bytes; what is written to them lands in the piece.
void *repeated(size_t bytes, size_t piece = 2 << 20)
{
    const int fd = memfd_create("piece", 0);
    const size_t room = (bytes + piece - 1) / piece * piece;
    uint8_t *m = (uint8_t *)mmap(nullptr, room + 2 * piece, PROT_NONE, MAP_SHARED | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
    if (fd < 0 || ftruncate(fd, (off_t)piece) != 0 || m == MAP_FAILED) return nullptr;
    for (size_t at = 0; at < room; at += piece)
        if (mmap(m + piece + at, piece, PROT_READ | PROT_WRITE, MAP_SHARED | MAP_FIXED, fd, 0) == MAP_FAILED) return nullptr;
    return m + piece + (room - bytes);   // (they end in front of the inaccessible piece)
}
int32_t *numbers(std::initializer_list<int32_t> v)
{
    int32_t *p = (int32_t *)emu_device_alloc_named(v.size() * 4, "numbers", 4);
    std::copy(v.begin(), v.end(), p);
    return p;
}
int fail(const char *what)
{
    fprintf(stderr, "cache_limits: %s\n", what);
    return 1;
}

}  // namespace

int main(int argc, char **argv)
{
    const std::string what = argc > 1 ? argv[1] : "";
    // the library's most: table_stride * page_tokens below 2^31 - 64
    const int32_t most = INT32_MAX - 95, stride = most / 32;
    hc::CacheArgs c;
    memset(&c, 0, sizeof c);
    c.table_stride = (uint32_t)stride;
    c.page_shift = 5;
    c.kv_heads = c.n_seqs = 1;
    c.max_slots = most;
    if (what == "weights") {
        hc::AttendArgs a;
        memset(&a, 0, sizeof a);
        a.c = c;   // (no page: every record is one that the table does not name)
        a.c.table = (const int32_t *)repeated((size_t)stride * 4);
        a.c.lengths = numbers({most});
        a.starts = numbers({0, 0});
        a.group = 1;
        a.weights = (float *)repeated((size_t)most * 4);
        a.weight_stride = (uint64_t)most;
        a.weights[most - 1] = 5.0f;
        const int records = (most + 31) / 32, batches = 3;
        const unsigned groups = (records + 8 * batches - 1) / (8 * batches);
        if ((int64_t)groups * 8 * batches < (1 << 26)) return fail("the last workgroup does not reach past 2^26 records");
        if (!emu_run_grid([=]() { blockIdx.x = groups - 1; hc::k_cache_weights<2, 0>(a, records, batches); }, dim3(1), dim3(256))) return fail("weights");
        return a.weights[most - 1] == 0.0f ? 0 : fail("the last weight was not written");
    }
    if (what == "columns") {
        hc::AttendArgs a;
        memset(&a, 0, sizeof a);
        a.c = c;
        a.c.table = (const int32_t *)repeated((size_t)stride * 4);
        a.c.lengths = numbers({most});
        a.starts = numbers({0, 17});
        a.n_rows = a.max_rows = 17;
        a.group = 1;
        a.tiles = 2;
        a.splits = 1;
        a.split_records = 4;
        a.window = 40;
        a.causal = 1;
        a.wide_tiles = 1;
        a.tiles_in_wide = 16;
        a.q_row_stride = a.out_row_stride = 64;
        a.q_head_stride = a.out_head_stride = 64;
        a.scale = 1.0f;
        a.q = emu_device_alloc_named(17 * 128, "q", 16);
        a.out = emu_device_alloc_named(17 * 128, "out", 16);
        a.left_over = (uint32_t *)numbers({7});
        memset(a.out, 0x55, 17 * 128);
        if (!emu_run_grid([=]() { hc::k_cache_attend_rows<2, 0, 8, 2>(a); }, dim3(1), dim3(512))) return fail("columns");
        for (int i = 0; i < 17 * 64; ++i)
            if (((uint16_t *)a.out)[i] != 0) return fail("rows that see no page");
        return a.left_over[0] == 0 ? 0 : fail("columns left over");
    }
    hc::EvictArgs e;
    memset(&e, 0, sizeof e);
    e.c = c;
    e.to_lengths = numbers({0});
    e.weight_stride = (uint64_t)most;
    if (what == "select") {
        e.c.lengths = numbers({most});
        e.weights = (const float *)repeated((size_t)most * 4);
        e.first = 2;
        e.recent = 3;
        e.keep = 5;
        e.kept = numbers({9, 9, 9, 9, 9});
        e.to_weights = (float *)numbers({9, 9, 9, 9, 9});
        if (!emu_run_grid([=]() { hc::k_cache_select(e); }, dim3(1), dim3(hc::kSelectThreads))) return fail("select");
        const int32_t want[5] = {0, 1, most - 3, most - 2, most - 1};
        if (e.to_lengths[0] != 5 || memcmp(e.kept, want, sizeof want) != 0) return fail("other rows than the first and last ones");
        return 0;
    }
    if (what == "keep") {
        e.c.lengths = numbers({7});
        e.weights = (const float *)repeated((size_t)most * 4);
        e.keep = most;
        e.kept = (int32_t *)repeated((size_t)most * 4);
        e.to_weights = (float *)repeated((size_t)most * 4);
        e.to_weights[most - 1] = 5.0f;
        if (!emu_run_grid([=]() { hc::k_cache_select(e); }, dim3(1), dim3(hc::kSelectThreads))) return fail("keep");
        return e.to_lengths[0] == 7 && e.kept[most - 1] == -1 && e.to_weights[most - 1] == 0.0f ? 0 : fail("what lies behind the kept rows");
    }
    return fail("what?");
}
