"""Wait states between MFMAs and the first use of their results, over every path (CPU).

A VALU or memory instruction may read or overwrite an MFMA's result only some wait states
after it: 7 for v_mfma_f32_16x16x32_bf16, 11 for 32x32x16, 18 for v_mfma_f32_32x32x2_f32
(an MFMA that accumulates onto it needs none). The compiler inserts them, but where it sank
the reading instructions below a branch it has inserted too few on the taken path, and the
last registers of a result were read before they were written. pin_before_branch (common.h)
prevents that in the sources; this test compiles the window and 8-bit cache kernels with
the build's flags and follows every path behind every MFMA.
"""
import os
import re
import shutil
import subprocess

import pytest

FILES = ["attn_window.hip", "attn_window_bwd.hip", "kvcache8_attend.hip"]
_REG = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def _regs(text):
    out = set()
    for kind, lo, hi, one in _REG.findall(text):
        out |= {(kind, int(one))} if one else {(kind, i) for i in range(int(lo), int(hi) + 1)}
    return out


def _need(op):
    return 18 if "32x32x2_f32" in op else 7 if "16x16x32" in op else 11


def _parse(t):
    op, _, rest = t.partition(" ")
    ops = rest.split(",") if rest else []
    dst = _regs(ops[0]) if ops else set()
    src = set().union(*(_regs(o) for o in ops[1:]))
    if op.startswith(("ds_write", "global_store", "buffer_store", "flat_store", "scratch_store")):
        src, dst = src | dst, set()
    return op, dst, src, ops


def scan(text):
    """(function, MFMA, use, wait states between them) wherever there are too few."""
    bad = []
    for fn in re.split(r"\n(?=[A-Za-z_][\w.$]*:)", text):
        ins, labels = [], {}
        for line in fn.split("\n"):
            t = line.split(";")[0].strip()
            m = re.match(r"(\.?L?BB\w+):", t)
            if m:
                labels[m.group(1)] = len(ins)
            elif t and not t.startswith(".") and not t.endswith(":"):
                ins.append(t)
        parsed = [_parse(t) for t in ins]

        def after(i):
            op, target = parsed[i][0], ins[i].split()[-1]
            if op == "s_endpgm":
                return []
            if op == "s_branch":
                return [labels[target]]
            return [i + 1] + ([labels[target]] if op.startswith("s_cbranch") and target in labels else [])

        for i, (op, dst, _, _) in enumerate(parsed):
            if not op.startswith("v_mfma"):
                continue
            best, todo = {}, [(j, 0, frozenset(dst)) for j in after(i)]
            while todo:
                j, waited, live = todo.pop()
                if waited >= _need(op) or j >= len(ins) or best.get(j, 99) <= waited:
                    continue
                best[j] = waited
                o, d, s, ops = parsed[j]
                if o.startswith("v_mfma"):
                    used = _regs(ops[1]) | _regs(ops[2])  # accumulating is fine
                elif o.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")):
                    used = s | (d if o.startswith("v_") else set())
                else:
                    used = set()
                if used & live:
                    bad.append((fn.split(":")[0], ins[i], ins[j], waited))
                    continue
                live = live - d
                if live:
                    w = waited + 1 + (int(ins[j].split()[1]) if o == "s_nop" else 0)
                    todo += [(k, w, live) for k in after(j)]
    return bad


@pytest.mark.parametrize("name", FILES)
def test_results_are_waited_for_on_every_path(name, tmp_path):
    from gonn_amd import build
    if not (os.path.exists(build.HIPCC) or shutil.which(build.HIPCC)):
        pytest.skip("hipcc not available")
    out = str(tmp_path / "a.s")
    r = subprocess.run([build.HIPCC, *[f for f in build.CFLAGS if f != "-fPIC"], *build.FILE_FLAGS.get(name, []),
                        "--cuda-device-only", "-S", os.path.join(build.CSRC, name), "-o", out],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    text = open(out).read()
    assert "v_mfma_f32_32x32x16_bf16" in text
    bad = scan(text)
    assert not bad, (len(bad), bad[:3])
    if name == "attn_window_bwd.hip":  # its inline MFMAs: the rules of test_asm_hazards
        from tests.test_asm_hazards import _scan
        fns = [f for f in re.split(r"\n(?=[A-Za-z_][\w.$]*:)", text) if f.startswith("_ZN4gonn23window_dkdv_pipe_kernel")]
        assert len(fns) == 2
        for f in fns:
            broken, first = _scan(f.split(".Lfunc_end")[0].split("\n"))
            assert first is not None and not broken, (len(broken), broken[:3])


def test_the_scan_follows_branches():
    mfma = "f:\n\tv_mfma_f32_32x32x16_bf16 a[0:15], v[0:3], v[4:7], 0\n"
    read = "\tv_accvgpr_read_b32 v9, a15\n\ts_endpgm\n"
    assert len(scan(mfma + "\ts_nop 2\n" + read)) == 1
    assert not scan(mfma + "\ts_nop 7\n\ts_nop 2\n" + read)
    taken = mfma + "\ts_cbranch_vccnz .LBB0_1\n\ts_nop 7\n\ts_nop 7\n.LBB0_1:\n" + read
    assert [b[3] for b in scan(taken)] == [1]
