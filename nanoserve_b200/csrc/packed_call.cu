// Entry points behind one that takes its arguments as an array of 64-bit words: a binding that pays for every argument it converts
// (ctypes: 0.09 us each, 3 us for the attention call) fills an array instead.
#include "common.cuh"

namespace {
struct Words {
    const int64_t* w;
    template <typename T> T* ptr(int i) const { return reinterpret_cast<T*>(static_cast<intptr_t>(w[i])); }
    int32_t i32(int i) const { return static_cast<int32_t>(w[i]); }
    double f64(int i) const {
        double d;
        memcpy(&d, w + i, sizeof d);
        return d;
    }
};
}  // namespace

extern "C" int ns_call(int32_t op, const int64_t* words, int32_t n_words) {
    static const int32_t expected[] = {8, 32, 15, 34};
    NS_REQUIRE(op >= 0 && op <= NS_OP_RAGGED_PAGED_ATTN_Q8, NS_ERR_INVALID_ARG, "ns_call: unknown operation %d", op);
    NS_REQUIRE(words && n_words == expected[op], NS_ERR_INVALID_ARG, "ns_call: operation %d takes %d words, not %d", op, expected[op], n_words);
    const Words a{words};
    const int64_t* w = words;
    switch (op) {
        case NS_OP_ROPE_TABLES:
            return ns_rope_tables(a.ptr<const int64_t>(0), a.ptr<const float>(1), a.f64(2), a.ptr<float>(3), a.ptr<float>(4), w[5], a.i32(6),
                                  a.ptr<void>(7));
        case NS_OP_ROPE_APPEND:
            return ns_rope_append(a.ptr<const void>(0), a.ptr<const void>(1), a.ptr<const void>(2), w[3], w[4], w[5], a.ptr<const float>(6),
                                  a.ptr<const float>(7), a.i32(8), a.i32(9), a.ptr<void>(10), a.ptr<void>(11), a.ptr<void>(12), a.ptr<void>(13),
                                  a.ptr<void>(14), a.ptr<float>(15), a.ptr<float>(16), a.ptr<const int64_t>(17), w[18], w[19], a.i32(20), a.i32(21),
                                  a.i32(22), a.i32(23), w[24], w[25], w[26], w[27], w[28], a.i32(29), a.i32(30), a.ptr<void>(31));
        case NS_OP_KV_VALUES:
            return ns_kv_values(a.ptr<const void>(0), a.ptr<const float>(1), a.ptr<void>(2), w[3], a.i32(4), a.i32(5), a.i32(6), w[7], w[8], w[9],
                                w[10], w[11], a.i32(12), a.i32(13), a.ptr<void>(14));
        default:
            return ns_ragged_paged_attn_q8(a.ptr<const void>(0), a.ptr<const void>(1), a.ptr<const void>(2), a.ptr<const float>(3),
                                           a.ptr<const float>(4), a.ptr<const int32_t>(5), a.ptr<const int32_t>(6), a.ptr<const int32_t>(7),
                                           a.ptr<const int32_t>(8), a.ptr<void>(9), a.i32(10), w[11], a.i32(12), a.i32(13), a.i32(14), a.i32(15),
                                           a.i32(16), a.i32(17), w[18], w[19], w[20], w[21], w[22], w[23], w[24], w[25], (float)a.f64(26), a.i32(27),
                                           a.i32(28), a.ptr<void>(29), w[30], a.i32(31), a.i32(32), a.ptr<void>(33));
    }
}
