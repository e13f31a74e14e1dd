// Launches of the decode step (decode_step_kernel, step.h): HID = false by tq4_decode.hip, HID = true,
// sequences with hidden tokens, by span_decode.hip.
#pragma once
#include "abi.h"

namespace tq4 {
namespace abi {

template <bool HID, int LAYOUT, int G, bool ROT, bool KF8 = false, bool KB3 = false, bool V3 = false>
void launch_step(const tq4::xdl::StepArgs &s, const StepPlan &p, int nvh, hipStream_t st) {
    launch_lds(&tq4::xdl::decode_step_kernel<LAYOUT, G, ROT, KF8, KB3, V3, HID>, dim3(nvh / p.vw, p.nx),
               dim3(tq4::kWave * p.vw * p.sw), tq4::xdl::step_lds<LAYOUT, G, ROT, KF8, KB3, V3>(p.vw, p.sw), st, s);
}
template <bool HID, int LAYOUT, int G>
void launch_step_format(const Stage1Args &a, const tq4::xdl::StepArgs &s, const StepPlan &p, int nvh, hipStream_t st) {
    const bool rot = s.rot_t != nullptr, v3 = a.value_bits == 3;
    if (a.key_fp8)
        launch_step<HID, LAYOUT, G, false, true>(s, p, nvh, st);
    else if (a.key_bits == 3 && v3)
        rot ? launch_step<HID, LAYOUT, G, true, false, true, true>(s, p, nvh, st)
            : launch_step<HID, LAYOUT, G, false, false, true, true>(s, p, nvh, st);
    else if (a.key_bits == 3)
        rot ? launch_step<HID, LAYOUT, G, true, false, true>(s, p, nvh, st)
            : launch_step<HID, LAYOUT, G, false, false, true>(s, p, nvh, st);
    else
        rot ? launch_step<HID, LAYOUT, G, true>(s, p, nvh, st) : launch_step<HID, LAYOUT, G, false>(s, p, nvh, st);
}

// The step's own launches by a plan, from checked arguments (check_stage1; mfma_applies): the rotation
// where the step does not do it, and decode_step_kernel, which leaves out / lse (plan.whole) or part
// rows in a.mid_o.
template <bool HID>
int launch_step_by(const Stage1Args &a, const StepIo &io, const StepPlan &plan, const tq4::xdl::Hidden &hidden,
                   hipStream_t st) {
    const int nvh = a.Hk * xdl_parts(a);
    tq4::xdl::StepArgs s{};
    s.query = io.query;
    s.q_dtype = io.query_dtype;
    if (!a.key_fp8 && io.rotated) {
        s.query = io.q_rot_ws;
    } else if (!a.key_fp8) {
        if (io.query_dtype == TQ4_F32 || !plan.rotates) {  // the in-kernel rotation takes 16-bit queries
            const int rc = rotate_query(io.query, io.query_dtype, io.rot_t, io.q_rot_ws, a.B * a.Hq, a.D, nullptr,
                                        nullptr, st);
            if (rc)
                return rc;
            s.query = io.q_rot_ws;
        } else {
            s.rot_t = io.rot_t;
        }
    }
    s.centroids = io.centroids;
    s.cache = a.cache;
    s.block_table = a.bt;
    s.seq_lens = a.seq_lens;
    s.sinks = a.sinks;
    s.parts = a.mid_o;
    s.out = io.out;
    s.lse = io.lse;
    s.block_stride = a.stride;
    s.score_scale_log2 = a.scale * tq4::kLog2e;
    s.out_dtype = io.out_dtype;
    s.batch = a.B;
    s.num_q_heads = a.Hq;
    s.num_kv_heads = a.Hk;
    s.block_size_log2 = log2_int(a.bs);
    s.max_blocks = a.max_blocks;
    s.slot_pos = a.slot_pos;
    s.slot_head = a.slot_head;
    s.num_splits = a.S;
    s.group = a.Hq / a.Hk;
    s.n_hp = xdl_parts(a);
    s.vw = plan.vw;
    s.sw = plan.sw;
    s.per_seq = plan.per_seq;
    s.whole = plan.whole;
    s.hidden = hidden;
    if (xdl_heads(a) == 4)
        a.kl == 0 ? launch_step_format<HID, 0, 4>(a, s, plan, nvh, st) : launch_step_format<HID, 1, 4>(a, s, plan, nvh, st);
    else
        a.kl == 0 ? launch_step_format<HID, 0, 8>(a, s, plan, nvh, st) : launch_step_format<HID, 1, 8>(a, s, plan, nvh, st);
    return launch_status("decode_step");
}

}  // namespace abi
}  // namespace tq4
