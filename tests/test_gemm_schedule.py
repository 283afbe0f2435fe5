"""The end of the 8-wave GEMM's main loop (csrc/kernels/gemm_pingpong.h), modelled on the CPU: its waves stage operands
straight into LDS and then turn the same LDS into scratch of the epilogue.  No wave may write there before every wave of the
workgroup has waited for its own loads.  And products whose epilogue writes LDS at once repeat bit for bit on the GPU."""
import pathlib
import re

import pytest
import torch

HEADER = pathlib.Path(__file__).parent.parent / "distributed_tensorflow_amd" / "csrc" / "kernels" / "gemm_pingpong.h"
TOKEN = re.compile(r"(if \(wr == (?P<group>[01])\) )?__builtin_amdgcn_s_barrier\(\)|(?P<drain>s_waitcnt vmcnt\(0\))")


def events(text, group):
    """Barriers ("b") and complete waits ("w") that a wave of row group `group` executes in a piece of the source."""
    out = []
    for m in TOKEN.finditer(text):
        if m["drain"]:
            out.append("w")
        elif m["group"] is None or int(m["group"]) == group:
            out.append("b")
    return out


def parts():
    text = re.sub(r"//[^\n]*", "", HEADER.read_text().split("// ---- prologue")[1])
    before, rest = text.split("for (int kt = 0;", 1)
    body, tail = rest.split("\n  }\n", 1)
    return before, body, tail.split("#undef PP_PHASE")[0]


def test_no_wave_reuses_lds_before_every_wave_has_drained_its_loads():
    before, body, tail = parts()
    loop = ["b"] * 2 * body.count("PP_PHASE")
    assert len(loop) == 16
    runs = [events(before, g) + loop + events(tail, g) for g in (0, 1)]
    assert runs[0].count("b") == runs[1].count("b")              # else the workgroup would hang or fall apart
    barriers = runs[0].count("b")                                # what a wave has passed when its epilogue starts
    for run in runs:
        assert "w" in run
        at = len(run) - 1 - run[::-1].index("w")
        assert run[:at].count("b") < barriers, "a wave may still have loads into LDS under way when another one's epilogue writes there"


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,d", [(256, 50000, 256), (1024, 12544, 512), (2048, 8192, 264)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products_with_a_shallow_k_repeat_bit_for_bit(n, v, d, dtype):
    """The fewer K-tiles a workgroup has, the closer its last loads are to the epilogue's first LDS writes."""
    from distributed_tensorflow_amd.ops import vocab_xent as vx
    g = torch.Generator(device="cuda").manual_seed(n)
    x, w = (torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((n, d), (v, d)))
    lab = torch.randint(0, v, (n,), generator=g, device="cuda")

    def step():
        r = vx.vocab_xent_fwd(x, w, lab)
        return (r.rows, *vx.vocab_xent_bwd(r, x, w, lab)[:2])
    first = [t.clone() for t in step()]
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(step(), first))
