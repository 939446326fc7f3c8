// Runs the row products' argument checks (hk_rows_args.h) on the host, one
// case a line, and prints "<name> <status>" for each.  Pointers are never
// followed: they are addresses made up for the checks.
#include <cstdio>

#include "../hawking_amd/csrc/hk_rows_args.h"

using namespace hk;

static void* at(uintptr_t a) { return reinterpret_cast<void*>(a); }
static const int32_t* ints(uintptr_t a) { return reinterpret_cast<const int32_t*>(a); }
static int32_t* outs(uintptr_t a) { return reinterpret_cast<int32_t*>(a); }
static void say(const char* name, const RowsCheck& c) { std::printf("%s %d\n", name, c.code); }

int main() {
    const uintptr_t X = 0x10000000, Y = 0x20000000, W = 0x30000000, O = 0x40000000;
    const hk_rows x{at(X), HK_T_BF16, 8, 256}, y{at(Y), HK_T_F32, 8, 64};
    auto product = [&](int kind, hk_rows a, hk_rows b, uintptr_t order, uint32_t per_row, uintptr_t off, uintptr_t ws, size_t bytes) {
        return check_product(kind, 64, 256, &a, ints(order), per_row, ints(off), &b, at(ws), bytes, 4096);
    };
    auto with = [](hk_rows r, int field, uint64_t v) {
        if (field == 0) r.data = at(v);
        if (field == 1) r.type = (int32_t)v;
        if (field == 2) r.n = (uint32_t)v;
        if (field == 3) r.stride = v;
        return r;
    };
    say("ok", product(HK_Q4, x, y, 0, 1, O, W, 4096));
    say("ok_order", product(HK_MIXED, with(x, 2, 2), y, O, 4, O, W, 4096));
    say("ok_no_rows", product(HK_Q8, with(x, 2, 0), with(with(y, 2, 0), 0, 0), 0, 1, O, 0, 0));
    say("ok_one_row_any_stride", product(HK_BIN, with(with(x, 2, 1), 3, 0), with(with(y, 2, 1), 3, 0), 0, 1, O, W, 4096));
    say("kind_f32", product(HK_F32, x, y, 0, 1, O, W, 4096));
    say("kind_rice", product(HK_BIN_RICE, x, y, 0, 1, O, W, 4096));
    say("type", product(HK_Q4, with(x, 1, 3), y, 0, 1, O, W, 4096));
    say("type_negative", product(HK_Q4, x, with(y, 1, (uint32_t)-1), 0, 1, O, W, 4096));
    say("null_x", product(HK_Q4, with(x, 0, 0), y, 0, 1, O, W, 4096));
    say("misaligned_y", product(HK_Q4, x, with(y, 0, Y + 2), 0, 1, O, W, 4096));
    say("misaligned_x", product(HK_Q4, with(x, 0, X + 1), y, 0, 1, O, W, 4096));
    say("x_stride", product(HK_Q4, with(x, 3, 255), y, 0, 1, O, W, 4096));
    say("y_stride", product(HK_Q4, x, with(y, 3, 63), 0, 1, O, W, 4096));
    say("stride_overflow", product(HK_Q4, x, with(y, 3, (uint64_t)1 << 60), 0, 1, O, W, 4096));
    say("too_many", product(HK_Q4, with(x, 2, 0x80000000u), y, 0, 1, O, W, 4096));
    say("few_x", product(HK_Q4, with(x, 2, 7), y, 0, 1, O, W, 4096));
    say("no_x", product(HK_Q4, with(x, 2, 0), y, O, 1, O, W, 4096));
    say("per_row", product(HK_Q4, x, y, O, 0, O, W, 4096));
    say("null_offsets", product(HK_Q4, x, y, 0, 1, 0, W, 4096));
    say("null_ws", product(HK_Q4, x, y, 0, 1, O, 0, 4096));
    say("misaligned_ws", product(HK_Q4, x, y, 0, 1, O, W + 16, 4096));
    say("short_ws", product(HK_Q4, x, y, 0, 1, O, W, 4095));
    say("overlap", product(HK_Q4, x, with(y, 0, X + 256 * 2 * 7), 0, 1, O, W, 4096));
    say("touching_is_ok", product(HK_Q4, x, with(y, 0, X + 256 * 2 * 8), 0, 1, O, W, 4096));
    say("ws_in_x", product(HK_Q4, x, y, 0, 1, O, X, 4096));
    say("ws_in_y", product(HK_Q4, x, y, 0, 1, O, Y, 4096));

    auto group = [&](uintptr_t ids, uint32_t n, uint32_t g, uintptr_t off, uintptr_t order, uintptr_t pos, uintptr_t ws,
                     size_t bytes, size_t need) {
        return check_group(ints(ids), n, g, outs(off), outs(order), outs(pos), at(ws), bytes, need);
    };
    say("g_ok", group(X, 10, 4, O, Y, W, 0, 0, 0));
    say("g_ok_empty", group(0, 0, 4, O, 0, 0, 0, 0, 0));
    say("g_no_groups", group(X, 10, 0, O, Y, W, 0, 0, 0));
    say("g_many_groups", group(X, 10, 8193, O, Y, W, 0, 0, 0));
    say("g_many_ids", group(X, 0x80000000u, 4, O, Y, W, 0, 0, 0));
    say("g_one_id_more", group(X, (1u << 24) + 1u, 4, O, 2 * X + (1u << 28), 3 * X + (1u << 29), 0, 0, 0));
    say("g_null_ids", group(0, 10, 4, O, Y, W, 0, 0, 0));
    say("g_null_pos", group(X, 10, 4, O, Y, 0, 0, 0, 0));
    say("g_null_offsets", group(X, 10, 4, 0, Y, W, 0, 0, 0));
    say("g_alias", group(X, 10, 4, O, X, W, 0, 0, 0));
    say("g_alias_offsets", group(X, 10, 4, X + 36, Y, W, 0, 0, 0));
    say("g_no_ws", group(X, 10, 4, O, Y, W, 0, 0, 64));
    say("g_short_ws", group(X, 10, 4, O, Y, W, W + 4096, 63, 64));

    const hk_rows c{at(X), HK_T_BF16, 80, 100}, o{at(Y), HK_T_F32, 8, 100}, b{at(W), HK_T_F32, 8, 100};
    auto combine = [&](hk_rows a, uintptr_t pos, uintptr_t w, uint32_t k, uint32_t cols, const hk_rows* base, hk_rows out) {
        return check_combine(&a, ints(pos), reinterpret_cast<const float*>(w), k, cols, base, &out);
    };
    const hk_rows half{at(Y + 400), HK_T_F32, 8, 100}, few{at(W), HK_T_F32, 7, 100};
    say("c_ok", combine(c, O, O, 10, 100, &b, o));
    say("c_ok_in_place", combine(c, O, O, 10, 100, &o, o));
    say("c_ok_no_x", combine(with(c, 2, 0), O, O, 10, 100, nullptr, o));
    say("c_cols", combine(c, O, O, 10, 0, nullptr, o));
    say("c_per_row", combine(c, O, O, 0, 100, nullptr, o));
    say("c_null_pos", combine(c, 0, O, 10, 100, nullptr, o));
    say("c_null_w", combine(c, O, 0, 10, 100, nullptr, o));
    say("c_stride", combine(c, O, O, 10, 101, nullptr, o));
    say("c_base_few", combine(c, O, O, 10, 100, &few, o));
    say("c_base_overlap", combine(c, O, O, 10, 100, &half, o));
    say("c_x_overlap", combine(with(c, 0, Y), O, O, 10, 100, nullptr, o));

    say("b_ok", check_bank(HK_Q8, 8, 256));
    say("b_kind", check_bank(HK_F32, 8, 64));
    say("b_slots", check_bank(HK_Q8, 0, 64));
    say("b_rank", check_bank(HK_Q8, 8, 257));
    say("a_ok", check_adapter(8, 64, 7, 64, at(X), at(Y), HK_T_BF16));
    say("a_ok_empty", check_adapter(8, 64, 7, 0, nullptr, nullptr, 0));
    say("a_slot", check_adapter(8, 64, 8, 64, at(X), at(Y), HK_T_BF16));
    say("a_rank", check_adapter(8, 64, 7, 65, at(X), at(Y), HK_T_BF16));
    say("a_type", check_adapter(8, 64, 7, 64, at(X), at(Y), HK_T_F32));
    say("a_null", check_adapter(8, 64, 7, 64, at(X), nullptr, HK_T_F16));
    say("a_misaligned", check_adapter(8, 64, 7, 64, at(X + 1), at(Y), HK_T_F16));
    return 0;
}
