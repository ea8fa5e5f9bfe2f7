// Host-only checks of the C++ plans of the attention step over the 4-bit cache: select and workspace_size are host functions, refused
// and empty problems return before any launch.
#include <cmath>
#include <cstdio>

#include "baracuda_kernels_kv4_plan.hpp"

using namespace baracuda;

static int failures = 0;
#define CHECK(cond)                                                          \
    do {                                                                     \
        if (!(cond)) {                                                       \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond);    \
            ++failures;                                                      \
        }                                                                    \
    } while (0)

int main() {
    PlanPreference pref, other, small;
    other.prefer_backend = BackendKind::Cublas;
    small.max_workspace_bytes = 1;
    const Kv4CacheDescriptor cache{4, 32, 2, 128};
    CHECK(cache.page_bytes() == 2u * 2u * 18u * 128u);
    alignas(16) static char bytes[4096];  // an address; nothing is launched on it
    const void* in = bytes;
    void* out = bytes;

    QkNormRopePlan rope;
    QkNormRopeDescriptor rd;
    rd.tokens = 3, rd.heads_q = 8, rd.heads_kv = 2, rd.head_dim = 128;
    CHECK(QkNormRopePlan::select(rd, pref, &rope) == Error::Ok && rope.workspace_size() == 0);
    CHECK(QkNormRopePlan::select(rd, other, &rope) == Error::Unsupported);
    QkNormRopeArgs ra;
    CHECK(rope.run(nullptr, ra) == Error::InvalidProblem);  // no keys
    ra.k = {in, 3 * 256, 256}, ra.q = {in, 3 * 1024, 1024}, ra.q_out = {out, 3 * 1024 - 1, 1024};
    CHECK(rope.run(nullptr, ra) == Error::BufferTooSmall);
    ra.q_out.len = 3 * 1024;
    CHECK(rope.run(nullptr, ra) == Error::InvalidProblem);  // no angles
    ra.cos_sin = {reinterpret_cast<const float*>(in), 127}, ra.max_pos = 1, ra.positions = {reinterpret_cast<const int32_t*>(in), 3}, ra.pos_stride = 3;
    CHECK(rope.run(nullptr, ra) == Error::BufferTooSmall);
    rd.axis_of_pair.assign(63, 0);
    CHECK(QkNormRopePlan::select(rd, pref, &rope) == Error::InvalidProblem);
    rd.axis_of_pair.assign(64, 8);
    CHECK(QkNormRopePlan::select(rd, pref, &rope) == Error::InvalidProblem);
    rd.axis_of_pair.assign(64, 2);
    rd.cache = cache;
    CHECK(QkNormRopePlan::select(rd, pref, &rope) == Error::Ok);
    rd.heads_kv = 4;
    CHECK(QkNormRopePlan::select(rd, pref, &rope) == Error::InvalidProblem);
    rd.heads_kv = 2, rd.rot_dim = 12, rd.axis_of_pair.clear();
    CHECK(QkNormRopePlan::select(rd, pref, &rope) == Error::Unsupported);

    Kv4AppendPlan append;
    Kv4ReadPlan read;
    Kv4TokensDescriptor td{2, cache};
    CHECK(Kv4AppendPlan::select(td, pref, &append) == Error::Ok && Kv4ReadPlan::select(td, pref, &read) == Error::Ok);
    const size_t need = 4 * cache.page_bytes();
    const int64_t stride = static_cast<int64_t>(cache.page_bytes());
    const int64_t* slots = reinterpret_cast<const int64_t*>(in);
    CHECK(append.run(nullptr, {in, 512, 256}, {in, 512, 256}, {out, need - 1, stride}, {slots, 2}) == Error::BufferTooSmall);
    CHECK(append.run(nullptr, {in, 512, 256}, {in, 512, 255}, {out, need, stride}, {slots, 2}) == Error::InvalidProblem);
    CHECK(append.run(nullptr, {in, 512, 256}, {in, 512, 256}, {out, need, stride - 16}, {slots, 2}) == Error::InvalidProblem);
    CHECK(append.run(nullptr, {in, 512, 256}, {in, 512, 256}, {out, need, stride}, {slots, 1}) == Error::BufferTooSmall);
    CHECK(read.run(nullptr, {in, need, stride}, {slots, 2}, {out, 511, 256}, {out, 512, 256}) == Error::BufferTooSmall);
    td.cache.page_size = 24;
    CHECK(Kv4AppendPlan::select(td, pref, &append) == Error::Unsupported && Kv4ReadPlan::select(td, pref, &read) == Error::Unsupported);
    td = {0, cache};
    CHECK(Kv4AppendPlan::select(td, pref, &append) == Error::Ok && append.run(nullptr, {}, {}, {}, {}) == Error::Ok);
    td.tokens = -1;
    CHECK(Kv4ReadPlan::select(td, pref, &read) == Error::InvalidProblem);

    Kv4AttentionPlan attention;
    Kv4AttentionDescriptor ad;
    ad.batch = 2, ad.max_q = 1, ad.max_kv = 100, ad.heads_q = 8, ad.cache = cache;
    CHECK(Kv4AttentionPlan::select(ad, pref, &attention) == Error::Ok && attention.workspace_size() == 0);
    Kv4AttentionArgs aa;
    CHECK(attention.run(nullptr, Workspace::none(), aa) == Error::Ok);  // no rows
    aa.total_q = 2, aa.q = {in, 2048, 1024}, aa.out = {out, 2048, 1024}, aa.cache = {in, need, stride};
    const int32_t* ints = reinterpret_cast<const int32_t*>(in);
    aa.cu_q = {ints, 2}, aa.kv_lens = {ints, 2}, aa.page_table = {ints, 8}, aa.ld_table = 4;
    CHECK(attention.run(nullptr, Workspace::none(), aa) == Error::BufferTooSmall);  // cu_q has batch + 1 entries
    aa.cu_q.len = 3, aa.ld_table = 3;
    CHECK(attention.run(nullptr, Workspace::none(), aa) == Error::InvalidProblem);
    ad.max_kv = 100000;
    CHECK(Kv4AttentionPlan::select(ad, small, &attention) == Error::Unsupported);
    CHECK(Kv4AttentionPlan::select(ad, pref, &attention) == Error::Ok && attention.workspace_size() > 0);
    aa.page_table = {ints, 2 * 3125}, aa.ld_table = 3125;
    CHECK(attention.run(nullptr, Workspace::none(), aa) == Error::WorkspaceTooSmall);
    ad.scale = std::nanf("");
    CHECK(Kv4AttentionPlan::select(ad, pref, &attention) == Error::InvalidProblem);
    ad.scale.reset();
    ad.heads_q = 7;
    CHECK(Kv4AttentionPlan::select(ad, pref, &attention) == Error::InvalidProblem);
    if (failures == 0) std::printf("kv4_plan_host_test ok\n");
    return failures != 0;
}
