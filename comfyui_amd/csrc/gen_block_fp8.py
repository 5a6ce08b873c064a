#!/usr/bin/env python3
"""Writes block_fp8_asm.inc: the K loop of the block-scaled e4m3fn contraction on 256 x 256 tiles (blockscale.hip). Run by the build.

    python comfyui_amd/csrc/gen_block_fp8.py [output file]

Eight waves, two per SIMD; a wave multiplies 128 weight rows (8 MFMA tiles f) with 64 tokens (4 tiles t, each the fourth one of the block's).
A K step is one scale block of 128: 32 MFMAs (v_mfma_f32_16x16x128_f8f6f4) that start from zero, and behind each the four v_fmac of the MFMA
three places before, which bring its result into the accumulators with the factor of its tokens and weight block. A tile with fewer rows has
a text of its own for every 64 of them, with 1 to 3 token tiles a wave. Left to the compiler each MFMA waits for its own
result (11 wait states) and every fragment for its read.

Order: pairs of f, and in a pair token tile by token tile, so that every fragment is refilled in place 7 to 9 MFMAs before its next use:
weights in a ring of four, tokens after the last pair has used them. LDS holds two stages of tokens and three of weights. One barrier a
step, in front of MFMA 6 nt - 2 (of 8 nt): all of this stage has been read and all of the next one has landed. Behind it the reads turn to the next stage
and the token loads of the step after that go out into this one; the weight loads of that step have gone out before, into the stage
that the step before has left. Loads are spread over the step: a burst of them keeps both waves of a SIMD waiting at the memory queue.

Register map (per wave):
  v[128:255]  accumulators, tile (f, t) at 128 + 4 (4 f + t)
  v[96:127]   token fragments, v[64:95] weight fragments (ring of four)
  v[48:63]    results of the last four MFMAs
  v[32:47]    factors: 32 + 8 (step & 1) + 4 (w3) + t
  v[26:29]    token scales of the next step, v[30:31] its weight scales
  v[8:25]     addresses (below)
  v[0:7]      left to the compiler
"""
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
OUT = os.path.join(HERE, "block_fp8_asm.inc")
ACC, B, A, P, M, SX, SW = 128, 96, 64, 48, 32, 26, 30
TAIL, ADDR_T, ADDR_W, TOK, VA, VB = 8, 10, 12, 14, 18, 22
NF, NT = 8, 4
STAGE = 32768          # of one operand; two of tokens at 0, three of weights at 2 STAGE
BEHIND = 3             # MFMAs between one and its v_fmac


class At:
    """Places (MFMA index within a step) of a step's events, by the token tiles of a wave."""
    def __init__(self, nt):
        self.nt, self.m = nt, 8 * nt
        self.order = [(2 * p + r % 2, r // 2) for p in range(NF // 2) for r in range(2 * nt)]
        self.ready = 6 * nt - 2     # the barrier stands in front of it
        # reads, in order: (behind which MFMA, operand, index); a fragment is overwritten behind the last MFMA that uses it
        self.own = [(2 * nt - 2, "a", 4), (2 * nt - 1, "a", 5), (4 * nt - 2, "a", 6), (4 * nt - 1, "a", 7)]
        self.next = sorted([(6 * nt - 2, "a", 0), (6 * nt - 1, "a", 1), (8 * nt - 2, "a", 2), (8 * nt - 1, "a", 3)]
                           + [(6 * nt + 2 * t + 1, "b", t) for t in range(nt)], key=lambda x: x[0])
        free = list(range(self.ready + 1, self.m))
        self.load_w = [max(0, nt - 2) + nt * j for j in range(4)]                 # before the barrier
        self.load_t = [free[j * len(free) // nt] for j in range(nt)]              # behind it
        assert self.load_w[-1] < self.ready and len(set(self.load_t)) == nt


def quad(r):
    return f"v[{r}:{r + 3}]"


def oct_(r):
    return f"v[{r}:{r + 7}]"


def read_a(f, stage):
    s = A + 8 * (f % 4)
    return [f"ds_read_b128 {quad(s + 4 * h)}, v{ADDR_W + h} offset:{2048 * f}" for h in range(2)]


def read_b(t, stage):
    s = B + 8 * t
    return [f"ds_read_b128 {quad(s + 4 * h)}, v{ADDR_T + h} offset:{stage * STAGE + 8192 * t}" for h in range(2)]


def reads_at(at, q, stage):
    out = [(kind, i, read_a(i, stage)) for place, kind, i in at.own if place == q]
    return out + [(kind, i, (read_a if kind == "a" else read_b)(i, stage ^ 1)) for place, kind, i in at.next if place == q]


def fmac(at, q, parity, swiglu):
    """Of the MFMA at place q of a step with this parity of the factors."""
    f, t = at.order[q]
    m = M + 8 * parity + (4 if swiglu and f >= 4 else 0) + t
    p, a = P + 4 * (q % 4), ACC + 4 * (NT * f + t)
    return [f"v_fmac_f32 v{a + i}, v{p + i}, v{m}" for i in range(4)]


def step(stage, swiglu, at, label):
    """One K step out of `stage`; its number has the stage's parity. `label`: three free numbers from it on."""
    L = []
    # reads in flight at the start, oldest first
    flight = [(k, i) for _, k, i in at.next]
    load_at = {}
    for j in range(at.nt):
        load_at[at.load_t[j]] = (f"s_add_u32 m0, %[ldsw], {stage * STAGE + 8192 * j}", f"buffer_load_dwordx4 v{VA + j}, %[ra], %[so] offen lds")
    for j in range(4):
        rb = "%[rb1]" if swiglu and j & 1 else "%[rb0]"
        load_at[at.load_w[j]] = (f"s_add_u32 m0, s62, {8192 * j}", f"buffer_load_dwordx4 v{VB + j}, {rb}, %[so] offen lds")
    # behind the barrier: the factors of the next step, then its successor's scales into the registers they came from
    work = [f"v_mul_f32 v{M + 8 * (stage ^ 1) + 4 * w + t}, v{SX + t}, v{SW + w}" for w in range(2 if swiglu else 1) for t in range(at.nt)]
    work += [f"buffer_load_dword v{SX + t}, v{TOK + t}, %[rs], %[ss] offen" for t in range(at.nt)]
    work += [f"buffer_load_dword v{SW + w}, off, %[rw{w}], %[sw]" for w in range(2 if swiglu else 1)]
    rate = -(-len(work) // (at.m - at.ready - 1))
    for q, (f, t) in enumerate(at.order):
        need = [("a", f), ("b", t)]
        if q == 0:
            # K offsets of the step after the next; past the last one the scales are read again and the rows are none
            L += ["s_add_u32 %[so], %[so], 128", "s_sub_u32 %[left], %[left], 1", "s_cmp_gt_i32 %[left], 0", f"s_cbranch_scc1 {label}f"]
            L += [f"v_or_b32 v{r}, v{TAIL}, v{r}" for r in list(range(VA, VA + 4)) + list(range(VB, VB + 4))]
            L += [f"v_bfrev_b32 v{TAIL}, 1", f"{label}:", "s_cmp_ge_i32 %[left], 0",
                  "s_cselect_b32 s60, %[ssi], 0", "s_cselect_b32 s61, 4, 0", "s_add_u32 %[ss], %[ss], s60", "s_add_u32 %[sw], %[sw], s61"]
            # the weights' stage of that step: the one in front of this step's
            L += [f"s_add_u32 s62, %[ws], {-STAGE}", "s_cmp_eq_u32 %[ws], 0", f"s_cselect_b32 s62, {2 * STAGE}, s62", "s_add_u32 s62, s62, %[ldsw]",
                  f"s_add_u32 s62, s62, {2 * STAGE}"]
        if q == at.ready:
            L += [f"s_mov_b32 s60, {STAGE}", f"s_cmp_eq_u32 %[ws], {2 * STAGE}", f"s_cselect_b32 s60, {-2 * STAGE}, s60", "s_add_u32 %[ws], %[ws], s60"]
            L += [f"v_add_u32 v{ADDR_W + h}, s60, v{ADDR_W + h}" for h in range(2)]
            # the weights of the step after the next are on their way; a tile's first two steps have landed before it begins, and behind
            # their loads the stores of the tile before may be
            if stage == 0:
                L += ["s_cmp_eq_u32 %[n], %[steps]", f"s_cbranch_scc1 {label + 1}f"]
            L += ["s_waitcnt vmcnt(4)"] + ([f"{label + 1}:"] if stage == 0 else []) + ["s_waitcnt lgkmcnt(0)", "s_barrier"]
            flight = []
        pending = [k for k, x in enumerate(flight) if x in need]
        if pending:
            behind = len(flight) - 1 - max(pending)
            L.append(f"s_waitcnt lgkmcnt({min(2 * behind, 15)})")
            flight = flight[max(pending) + 1:]
        if q in load_at:
            L.append(load_at[q][0])
        L.append(f"v_mfma_f32_16x16x128_f8f6f4 {quad(P + 4 * (q % 4))}, {oct_(A + 8 * (f % 4))}, {oct_(B + 8 * t)}, 0")
        if q in load_at:
            L.append(load_at[q][1])
        for kind, i, text in reads_at(at, q, stage):
            L += text
            flight.append((kind, i))
        L += fmac(at, q - BEHIND, stage, swiglu) if q >= BEHIND else fmac(at, q - BEHIND + at.m, stage ^ 1, swiglu)
        if q > at.ready:
            L += work[(q - at.ready - 1) * rate:(q - at.ready) * rate]
    assert flight == [(k, i) for _, k, i in at.next]
    return L


def flush(stage, swiglu, at):
    """What the last step has left, behind the wait states between an MFMA and a read of its result."""
    L = ["s_nop 15"]
    for q in range(at.m - BEHIND, at.m):
        L += fmac(at, q, stage, swiglu)
    return L


def fill(at):
    L = []
    for _, kind, i in at.next:
        L += (read_a if kind == "a" else read_b)(i, 0)
    return L


def loop(swiglu, nt):
    at, b = At(nt), 100 * nt
    L = fill(at) + [f"{b + 11}:"] + step(0, swiglu, at, b + 20) + ["s_sub_u32 %[n], %[n], 1", "s_cmp_eq_u32 %[n], 0", f"s_cbranch_scc1 {b + 12}f"]
    L += step(1, swiglu, at, b + 30) + ["s_sub_u32 %[n], %[n], 1", "s_cmp_lg_u32 %[n], 0", f"s_cbranch_scc1 {b + 11}b"]
    return L + flush(1, swiglu, at) + ["s_branch 90f", f"{b + 12}:"] + flush(0, swiglu, at) + ["s_branch 90f"]


def tile(swiglu):
    # the results of the last step's MFMAs that the first step takes for joined, and their factors, are zero
    L = [f"v_mov_b32 v{r}, 0" for r in list(range(M + 8, M + 16)) + list(range(P, P + 16)) + list(range(ACC, 256))]
    for nt in range(1, NT):
        L += [f"s_cmp_eq_u32 %[nt], {nt}", f"s_cbranch_scc1 {100 * nt}f"]
    for nt in range(NT, 0, -1):
        L += [f"{100 * nt}:"] + loop(swiglu, nt)
    return L + ["90:", "s_waitcnt vmcnt(0) lgkmcnt(0)", "s_barrier"]


def generate():
    out = ["// Generated by gen_block_fp8.py; do not edit. See that script for the register map and the schedule.", ""]
    for name, lines in (("HDMOE_BLOCK_PLAIN", tile(False)), ("HDMOE_BLOCK_SWIGLU", tile(True))):
        out.append(f"#define {name} \\")
        out.append(" \\\n".join('  "' + ln + '\\n"' for ln in lines))
        out.append("")
    return "\n".join(out)


if __name__ == "__main__":
    path = sys.argv[1] if len(sys.argv) > 1 else OUT
    text = generate()
    if not os.path.exists(path) or open(path).read() != text:
        with open(path, "w") as f:
            f.write(text)
