// Which calls the matrix-unit kernel takes, how it cuts them, its launch.
#include "attend_span_few.hpp"

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

// a prefix in tiles and own slots of few rows in one launch (heads of 256 channels have other waves a CU for each)
static bool span_both(const SpanCall &c) { return c.apart && !c.pfew && c.ofew && c.a.D != 256; }

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
    const bool packed = a.prefix.n_packed + a.own.n_packed > 0;
    const int64_t r1 = a.Hq / a.Hkv * a.Sq, all = a.B * r1;
    const int most = 32 * SP_WAVES / maps, few = 32 / maps;   // rows of a block of the one kernel, of the other
    auto units_of = [](const vq_kv_store &s, int64_t unit) { return cdiv(s.n_packed, unit) + cdiv(s.n_tail, unit); };
    // The prefix in blocks of its own where a sequence's rows fill half a block or less; not where prefix and own slots are few enough for one
    // block a row tile and no parts (8 sequences of 33 slots on 700 packed: 11.7 us, and 13.4 apart; 32 of them 12.5 and 22.7; 12 of five rows and
    // 60 slots on 200 plain: 11.5 and 15.4).
    const bool prefix_slots = a.prefix.n_packed + a.prefix.n_tail > 0;
    const bool brief = packed ? r1 <= few && a.D != 256 && units_of(a.prefix, 32) + units_of(a.own, 32) <= 40 && a.B * a.Hkv <= 256
                              : a.D != 256 && units_of(a.prefix, 64) + units_of(a.own, 64) <= 8 && a.B * a.Hkv <= 512;
    c.apart = prefix_slots && a.B > 1 && r1 <= most / 2 && !brief;
    const int64_t p32 = units_of(a.prefix, 32), p64 = units_of(a.prefix, 64), o32 = units_of(a.own, 32), o64 = units_of(a.own, 64);
    // Few rows by the kernel for them, in so many tiles: each reads and reconstructs the slots again, as the other kernel's blocks do, but no wave
    // waits for another, and none of them idles at heads of 256 channels, where the other's waves share no rows.  A prefix: 64 rows over 16k slots
    // 27.8 us, and 33.1 by the other kernel, 126 rows of 256 channels 64 and 78; 128 rows of 128 channels 44.7 and 41.1.  Own slots, two maps and 80
    // rows over 8k 32 us and 37, but 155 and 148 for 16 sequences of 16k; next to a prefix in tiles 66 and 71 for 16 sequences of 36 rows, 46 and 41
    // for four.
    c.pfew = packed && all <= (a.D == 256 ? 8 : 3) * few;
    c.ofew = packed && (r1 <= few || (r1 <= 2 * few && 2 * a.B * a.Hkv * o32 <= 65536 && (!c.apart || c.pfew || a.B * a.Hkv >= 64)));
    // Two waves share rows where those fill half a block, and over plain rows where blocks of as many rows as fit would leave half of the chip empty
    // (two maps, 8 heads over 500 tokens: 13.8 us, and 16.4; 8 sequences of five rows and 200 slots on 2000: 16.5 and 18.0).
    auto blocks_of = [&](int64_t rows, int64_t units, int64_t times) { return times * a.Hkv * cdiv(rows, most) * cdiv(units, 6); };
    const bool roomy = !packed && (c.apart ? blocks_of(all, p64, 1) + blocks_of(r1, o64, a.B) : blocks_of(r1, p64 + o64, a.B)) <= 256;
    // One round of blocks of equal runs, two blocks a CU (one of few rows of 256 channels, or of tiles beside few rows), each side for itself
    // where they differ; own slots of sequences that differ in length even out over four rounds.  A run is four units a wave or more for few
    // rows, six units a block else, which a block costs to start and end (12 sequences of five rows on 4k plain slots: 25.8 us with four, 23.9
    // with six, 25.2 with eight).
    auto side = [&](bool by_few, int64_t rows, int64_t slots32, int64_t slots64, int64_t times, int &wt, int &tiles, int64_t &units, int64_t &least) {
        units = by_few || a.D == 256 ? slots32 : slots64;
        least = by_few ? 16 : 6;
        wt = !by_few && a.D != 256 && (rows <= most / 2 || roomy) ? 2 : 1;
        tiles = (int)cdiv(rows, by_few ? few : most / wt);
        return times * a.Hkv * tiles * units;   // units of all blocks
    };
    int64_t pu = 0, ou = 0, pleast = 1, oleast = 1, pwork = 0;
    if (c.apart) pwork = side(c.pfew, all, p32, p64, 1, c.pwt, c.ptiles, pu, pleast);
    const int64_t owork = side(c.ofew, r1, c.apart ? o32 : p32 + o32, c.apart ? o64 : p64 + o64, a.B, c.owt, c.otiles, ou, oleast);
    const bool together = c.apart && c.pfew == c.ofew;
    auto cut = [&](int64_t units, int64_t work, int64_t least, int64_t blocks) {
        int64_t run = cdiv(together ? pwork + owork : work, blocks);
        run = run < least ? least : run;
        return (int)cdiv(units, run);
    };
    auto round = [&](bool by_few) { return by_few && a.D == 256 ? 256 : 512; };   // blocks that run at once
    // (tiles beside few rows: one a CU where the few rows' work can fill the other half -- 43 us and 47 of two a CU for 21 sequences of 0.6k slots
    // on 16k, as tiles -- and two where not, 136 us and 150 for 128 of 80 slots on 32k)
    c.psplits = c.apart ? cut(pu, pwork, pleast, span_both(c) && pwork <= owork ? 256 : round(c.pfew)) : 0;
    c.osplits = cut(ou, owork, oleast, round(c.ofew) * (a.seq_lens != nullptr ? 4 : 1));
    // Parts are written and read again, at ~4 TB/s, and merged in a launch of ~6 us: rows of tiles stay whole where the units saved, ~1.4 us each, are
    // worth less (two maps, 16 heads over 1000 tokens: 24.5 us whole, and 40.7 in two parts).
    if (!c.apart && !c.ofew && c.osplits > 1) {
        const double traffic = (double)a.B * a.Hq * a.Sq * maps * a.D * 8 * c.osplits / 4e6;
        if (1.4 * (double)(ou - cdiv(ou, c.osplits)) < 6 + traffic) c.osplits = 1;
    }
    // Rows of few slots: a block of eight waves walks them without parts where four would leave five units a wave (16 us, and 17 of two
    // parts and their merge).
    c.owaves = 4;
    if (c.ofew && !c.apart && c.osplits > 1 && ou <= 40 && a.D != 256) {
        c.owaves = 8;
        c.osplits = 1;
    }
    if (brief && !packed && !c.apart) c.osplits = 1;
    c.nparts = c.psplits + c.osplits;
}

int launch_span_mfma(const SpanCall &c, int maps) {
    const vq_store_attend_args &a = c.a;
    if (a.prefix.n_packed + a.own.n_packed == 0) return a.dtype == VQ_F16 ? launch_span_rows_f16(c, maps) : launch_span_rows_bf16(c, maps);
    if (span_both(c)) return a.pack_bits == 4 ? launch_span_both4(c) : launch_span_both2(c);
    if (int rc = a.pack_bits == 4 ? launch_span_packed4(c, maps) : launch_span_packed2(c, maps)) return rc;
    return a.pack_bits == 4 ? launch_span_few4(c, maps) : launch_span_few2(c, maps);
}

}  // namespace vq
