// Which calls the matrix-unit kernel takes, how it cuts them, its launch.
#include "attend_span_mfma.hpp"

namespace vq {

static bool plain_rows_fit(const vq_kv_store &s) {
    if (s.n_tail == 0) return true;
    bool ok = (((uintptr_t)s.k_tail | (uintptr_t)s.v_tail) & 15) == 0;
    for (int d = 0; d < 3; ++d) ok = ok && s.k_strides[d] % 8 == 0 && s.v_strides[d] % 8 == 0;
    // 64 rows behind one 32-bit offset
    return ok && s.k_strides[2] >= 0 && s.v_strides[2] >= 0 && s.k_strides[2] < (1 << 24) && s.v_strides[2] < (1 << 24);
}
static bool packed_slots_fit(const vq_store_attend_args &a, const vq_kv_store &s) {
    if (s.n_packed == 0) return true;
    const uintptr_t all = (uintptr_t)s.k_packed | (uintptr_t)s.k_scale | (uintptr_t)s.k_zero | (uintptr_t)s.v_packed | (uintptr_t)s.v_scale | (uintptr_t)s.v_zero;
    return (all & 15) == 0 && s.cap_tokens % a.group == 0 && s.cap_tokens % (32 / a.pack_bits) == 0;
}

bool span_mfma_supported(const vq_store_attend_args &a) {
    if ((a.D != 64 && a.D != 128 && a.D != 256) || a.dtype == VQ_F32 || (((uintptr_t)a.q | (uintptr_t)a.out) & 15) != 0) return false;
    if (!plain_rows_fit(a.prefix) || !plain_rows_fit(a.own)) return false;
    const bool tails = a.prefix.n_tail + a.own.n_tail > 0;
    if (a.prefix.n_packed + a.own.n_packed == 0) return a.tail_dtype == a.dtype;
    return (a.pack_bits == 2 || a.pack_bits == 4) && (a.group == 32 || a.group == 64 || a.group == 128) && a.D % a.group == 0 && a.meta_dtype == VQ_F16 &&
           a.v_layout == VQ_V_TOKEN_PACKED && (!tails || a.tail_dtype == VQ_F16 || a.tail_dtype == VQ_BF16) && packed_slots_fit(a, a.prefix) &&
           packed_slots_fit(a, a.own);
}

void span_mfma_plan(SpanCall &c, int maps) {
    const vq_store_attend_args &a = c.a;
    const int64_t unit = a.D == 256 ? 32 : 64;
    auto units_of = [&](const vq_kv_store &s) { return cdiv(s.n_packed, unit) + cdiv(s.n_tail, unit); };
    const int64_t r1 = a.Hq / a.Hkv * a.Sq, all = a.B * r1, prefix = units_of(a.prefix), own = units_of(a.own);
    const int most = 32 * SP_WAVES / maps;   // rows of a block
    // the prefix in blocks of its own where a sequence's rows fill half a block or less
    c.apart = prefix > 0 && a.B > 1 && r1 <= most / 2;
    auto tiling = [&](int64_t rows, int &wt, int &tiles) {
        wt = a.D != 256 && rows <= most / 2 ? 2 : 1;
        tiles = (int)cdiv(rows, most / wt);
    };
    tiling(all, c.pwt, c.ptiles);
    tiling(r1, c.owt, c.otiles);
    // one round of blocks of equal runs, one block a CU; sequences that differ in length even out over four rounds
    const int64_t round = a.seq_lens != nullptr ? 1024 : 256;
    const int64_t walk = c.apart ? own : prefix + own;
    const int64_t work = (c.apart ? a.Hkv * c.ptiles * prefix : 0) + a.B * a.Hkv * c.otiles * walk;
    int64_t run = cdiv(work, round);
    if (run < 4) run = 4;
    c.psplits = c.apart ? (int)cdiv(prefix, run) : 0;
    c.osplits = walk > 0 ? (int)cdiv(walk, run) : 0;
    c.nparts = c.psplits + c.osplits;
}

int launch_span_mfma(const SpanCall &c, int maps) {
    const vq_store_attend_args &a = c.a;
    if (a.prefix.n_packed + a.own.n_packed > 0) return a.pack_bits == 4 ? launch_span_packed4(c, maps) : launch_span_packed2(c, maps);
    return a.dtype == VQ_F16 ? launch_span_rows_f16(c, maps) : launch_span_rows_bf16(c, maps);
}

}  // namespace vq
