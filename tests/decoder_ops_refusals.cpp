// The argument checks of the attention half's entry points, run without a GPU: the context's device does not exist, so that a call that every
// check lets through ends at cudaSetDevice (B200MOE_ERR_CUDA) before anything is launched, on a machine with GPUs too.  Prints one line for each
// call whose status is not the expected one; exit code: their number.
#include <cstdio>
#include <cstring>

#include "../edge0_b200/csrc/context.cuh"

using namespace b200moe;

static int bad = 0;
static ContextBase base;
static void expect(const char * what, int rc, int want) {
    if (rc != want) { ++bad; printf("%s: status %d, expected %d (%s)\n", what, rc, want, base.last_error.c_str()); }
}

int main() {
    base.device = -1;
    base.sm_count = 148;
    b200moe_ctx * ctx = reinterpret_cast<b200moe_ctx *>(&base);    // the entry points below use the base only
    enum { OK = B200MOE_OK, ARG = B200MOE_ERR_INVALID_ARG, UNSUP = B200MOE_ERR_UNSUPPORTED, PASSED = B200MOE_ERR_CUDA };
    alignas(16) static char mem[64];
    int32_t ints[4] = { 0, 0, 0, 0 };

    // ---- rope
    const b200moe_tensor x = { mem, { 128, 4, 3, 1 }, { 2, 256, 1024, 0 } };
    const b200moe_rope r = { 128, 1, { 64, 0, 0, 0 }, 0, 0, 0, 0, 1e6 };
    auto rope = [&](auto change) {
        b200moe_tensor a = x, d = x;
        b200moe_rope q = r;
        int type = B200MOE_TYPE_BF16;
        const int32_t * pos = ints;
        change(a, d, q, type, pos);
        return b200moe_op_rope(ctx, &a, type, pos, &q, &d, nullptr);
    };
#define ROPE(want, ...) expect("rope: " #__VA_ARGS__, rope([&](b200moe_tensor & a, b200moe_tensor & d, b200moe_rope & q, int & type, const int32_t *& pos) { (void) a; (void) d; (void) q; (void) type; (void) pos; __VA_ARGS__; }), want)
    ROPE(PASSED, );
    ROPE(OK, a.ne[2] = d.ne[2] = 0);
    ROPE(UNSUP, type = B200MOE_TYPE_NVFP4);
    ROPE(ARG, pos = nullptr);
    ROPE(ARG, a.data = nullptr);
    ROPE(ARG, a.nb[0] = 4);
    ROPE(ARG, a.nb[1] = 255);
    ROPE(ARG, a.nb[2] = -1024);
    ROPE(ARG, a.data = mem + 1);
    ROPE(ARG, a.ne[3] = 2);
    ROPE(ARG, a.ne[2] = 2);
    ROPE(ARG, d.nb[1] = 128);
    ROPE(ARG, d.nb[2] = 768);
    ROPE(PASSED, d.nb[1] = 768, d.nb[2] = 256);
    ROPE(PASSED, a.nb[1] = 0);
    ROPE(ARG, q.n_rot = 127);
    ROPE(ARG, q.n_rot = 0);
    ROPE(ARG, q.n_rot = 130, q.sections[0] = 65);
    ROPE(ARG, q.n_axes = 0);
    ROPE(ARG, q.n_axes = 5);
    ROPE(ARG, q.sections[0] = 63);
    ROPE(ARG, q.n_axes = 2, q.sections[0] = 65, q.sections[1] = -1);
    ROPE(PASSED, q.n_axes = 3, q.sections[0] = 24, q.sections[1] = q.sections[2] = 20, q.interleaved = 1);
    ROPE(PASSED, q.n_axes = 2, q.sections[0] = 0, q.sections[1] = 64);
    ROPE(ARG, q.n_axes = 2, q.sections[0] = 0, q.sections[1] = 64, q.interleaved = 1);
    ROPE(ARG, q.base = 0.0);
    ROPE(ARG, q.base = -1.0);
    ROPE(ARG, q.base = 1.0 / 0.0);
    ROPE(UNSUP, a.ne[2] = d.ne[2] = (int64_t) 1 << 31);
    expect("rope: null context", b200moe_op_rope(nullptr, &x, 0, ints, &r, &x, nullptr), ARG);
    expect("rope: null rope", b200moe_op_rope(ctx, &x, B200MOE_TYPE_BF16, ints, nullptr, &x, nullptr), ARG);
    expect("rope: null tensors", b200moe_op_rope(ctx, nullptr, B200MOE_TYPE_BF16, ints, &r, nullptr, nullptr), ARG);

    // ---- cache
    const b200moe_kv_cache c = { B200MOE_KV_Q8, 4, 128, 64, 10, mem, mem, mem, mem };
    int64_t nv = 0, ns = 0;
    b200moe_kv_cache sized = c;
    expect("bytes q8", b200moe_kv_cache_bytes(&sized, &nv, &ns), OK);
    expect("bytes q8: values", (int) nv, 10 * 64 * 4 * 128);
    expect("bytes q8: scales", (int) ns, 10 * 64 * 4 * 4);
    sized.type = B200MOE_KV_Q4;
    expect("bytes q4", b200moe_kv_cache_bytes(&sized, &nv, &ns), OK);
    expect("bytes q4: values", (int) nv, 10 * 64 * 4 * 64);
    expect("bytes q4: scales", (int) ns, 10 * 64 * 4 * 8);
    sized.type = B200MOE_KV_BF16;
    expect("bytes bf16", b200moe_kv_cache_bytes(&sized, &nv, &ns), OK);
    expect("bytes bf16: values", (int) nv, 10 * 64 * 4 * 256);
    expect("bytes bf16: scales", (int) ns, 0);
    sized.n_pages = (int64_t) 1 << 24;
    expect("bytes of a cache beyond 32 bits", b200moe_kv_cache_bytes(&sized, &nv, &ns), OK);
    expect("bytes of a cache beyond 32 bits: values", nv == ((int64_t) 1 << 40) ? 1 : 0, 1);
    expect("bytes: null", b200moe_kv_cache_bytes(nullptr, &nv, &ns), ARG);
    expect("bytes: null result", b200moe_kv_cache_bytes(&c, nullptr, &ns), ARG);
    auto move = [&](bool write, auto change) {
        b200moe_kv_cache q = c;
        b200moe_tensor k = x, v = x;
        int type = B200MOE_TYPE_BF16;
        const int32_t * slots = ints;
        change(q, k, v, type, slots);
        return write ? b200moe_kv_write(ctx, &q, &k, &v, type, slots, nullptr) : b200moe_kv_read(ctx, &q, slots, &k, &v, type, nullptr);
    };
#define MOVE(want, ...) for (int w = 0; w < 2; ++w) expect(w ? "write: " #__VA_ARGS__ : "read: " #__VA_ARGS__, move(w, [&](b200moe_kv_cache & q, b200moe_tensor & k, b200moe_tensor & v, int & type, const int32_t *& slots) { (void) q; (void) k; (void) v; (void) type; (void) slots; __VA_ARGS__; }), want)
    MOVE(PASSED, );
    MOVE(OK, k.ne[2] = v.ne[2] = 0);
    MOVE(ARG, k.ne[2] = 2);
    MOVE(ARG, v.ne[1] = 3);
    MOVE(ARG, k.ne[0] = v.ne[0] = 64);
    MOVE(ARG, slots = nullptr);
    MOVE(UNSUP, type = 1);
    MOVE(UNSUP, q.type = 3);
    MOVE(UNSUP, q.type = -1);
    MOVE(UNSUP, q.head_dim = 96);
    MOVE(UNSUP, q.page_size = 8);
    MOVE(UNSUP, q.page_size = 48);
    MOVE(UNSUP, q.page_size = 512);
    MOVE(ARG, q.n_pages = 0);
    MOVE(ARG, q.n_head_kv = 0);
    MOVE(UNSUP, q.n_pages = (int64_t) 1 << 26);
    MOVE(ARG, q.k = nullptr);
    MOVE(ARG, q.v_scale = nullptr);
    MOVE(PASSED, q.type = B200MOE_KV_BF16, q.k_scale = q.v_scale = nullptr);
    MOVE(ARG, q.v = mem + 8);
    MOVE(ARG, q.k_scale = mem + 4);
    expect("write: broadcast heads", move(true, [&](auto &, b200moe_tensor & k, auto &, int &, auto &) { k.nb[1] = 0; }), PASSED);
    expect("read: overlapping rows", move(false, [&](auto &, b200moe_tensor & k, auto &, int &, auto &) { k.nb[1] = 0; }), ARG);

    // ---- attention
    const b200moe_tensor q8 = { mem, { 128, 8, 3, 1 }, { 2, 256, 2048, 0 } };
    const b200moe_attn at = { 3, 1, 300, 50000, 5, 0.1f, nullptr, ints, ints, ints };
    auto attend = [&](auto change) {
        b200moe_kv_cache kv = c;
        b200moe_tensor q = q8, o = q8;
        b200moe_attn a = at;
        int type = B200MOE_TYPE_BF16;
        void * ws = mem;
        size_t room = (size_t) 1 << 40;
        change(kv, q, o, a, type, ws, room);
        return b200moe_attention(ctx, &kv, &a, &q, type, &o, nullptr, ws, room, nullptr);
    };
#define ATTEND(want, ...) expect("attend: " #__VA_ARGS__, attend([&](b200moe_kv_cache & kv, b200moe_tensor & q, b200moe_tensor & o, b200moe_attn & a, int & type, void *& ws, size_t & room) { (void) kv; (void) q; (void) o; (void) a; (void) type; (void) ws; (void) room; __VA_ARGS__; }), want)
    ATTEND(PASSED, );
    ATTEND(OK, q.ne[2] = o.ne[2] = 0);
    ATTEND(OK, a.n_seq = 0);
    ATTEND(OK, a.max_new = 0, a.q_start = ints);
    ATTEND(ARG, a.max_new = 0);
    ATTEND(ARG, a.max_new = 2);
    ATTEND(PASSED, a.max_new = 2, a.q_start = ints);
    ATTEND(ARG, a.n_seq = -1);
    ATTEND(ARG, a.max_new = -1);
    ATTEND(ARG, a.prefix_len = -1);
    ATTEND(ARG, a.max_kv_len = -1);
    ATTEND(ARG, a.max_kv_len = 321);
    ATTEND(PASSED, a.max_kv_len = 320);
    ATTEND(PASSED, a.max_kv_len = 0, a.pages_stride = 0, a.pages = nullptr);
    ATTEND(ARG, a.pages = nullptr);
    ATTEND(ARG, a.kv_len = nullptr);
    ATTEND(ARG, a.prefix_pages = nullptr);
    ATTEND(PASSED, a.prefix_len = 0, a.prefix_pages = nullptr);
    ATTEND(ARG, a.n_seq = 4);
    ATTEND(PASSED, a.n_seq = 4, a.q_start = ints);
    ATTEND(ARG, a.scale = 1.0f / 0.0f);
    ATTEND(ARG, q.ne[1] = o.ne[1] = 6);
    ATTEND(ARG, o.ne[1] = 4);
    ATTEND(ARG, kv.head_dim = 64);
    ATTEND(ARG, q.nb[0] = 4);
    ATTEND(ARG, o.nb[2] = 256);
    ATTEND(UNSUP, type = B200MOE_TYPE_Q3_K);
    ATTEND(ARG, ws = nullptr);
    ATTEND(ARG, ws = mem + 8);
    ATTEND(ARG, room = 16);
    ATTEND(UNSUP, a.prefix_len = INT32_MAX);
    ATTEND(UNSUP, q.ne[2] = o.ne[2] = (int64_t) 1 << 29, a.q_start = ints);
    ATTEND(UNSUP, kv.page_size = 20);
    ATTEND(UNSUP, a.n_seq = 65536, a.q_start = ints);
    ATTEND(ARG, kv.k = nullptr);
    size_t need = 0;
    expect("workspace", b200moe_attention_workspace(ctx, &c, &at, 8, 3, &need), OK);
    expect("workspace: some", need > 0, 1);
    ATTEND(PASSED, room = need);
    expect("workspace: null", b200moe_attention_workspace(ctx, &c, &at, 8, 3, nullptr), ARG);
    expect("workspace: null attn", b200moe_attention_workspace(ctx, &c, nullptr, 8, 3, &need), ARG);
    expect("workspace: heads", b200moe_attention_workspace(ctx, &c, &at, 9, 3, &need), ARG);
    expect("workspace: null context", b200moe_attention_workspace(nullptr, &c, &at, 8, 3, &need), ARG);
    b200moe_attn one = at;
    one.prefix_len = 0;
    one.max_kv_len = 100;
    expect("workspace: one chunk", b200moe_attention_workspace(ctx, &c, &one, 8, 3, &need), OK);
    expect("workspace: one chunk needs none", need == 0, 1);
    ATTEND(PASSED, a.prefix_len = 0, a.max_kv_len = 100, ws = nullptr, room = 0);
    return bad;
}
