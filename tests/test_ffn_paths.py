"""Which calls ops.ffn makes, and where, with the kernels' wrappers replaced by recorders (CPU only)."""
import pytest

torch = pytest.importorskip("torch")

from loom_skills_b200 import ops  # noqa: E402


@pytest.fixture
def block(monkeypatch):
    """Runs ffn on stand-ins; returns the recorded calls as (name, current device, keyword arguments)."""
    state = {"dev": 0, "calls": []}

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.old, state["dev"] = state["dev"], self.dev

        def __exit__(self, *a):
            state["dev"] = self.old

    def recorder(name, out):
        def call(*a, **kw):
            state["calls"].append((name, state["dev"], kw))
            return out(*a, **kw)
        monkeypatch.setattr(ops, name, call)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["dev"])
    monkeypatch.setattr(torch.cuda, "device", Device)

    def run(tokens, h, f, fmt="q4_0", dtype=torch.float32, on=0, residual=True, **kw):
        state["calls"].clear()
        monkeypatch.setattr(ops, "_device", lambda *ts: on)
        recorder("rms_norm", lambda x, *a, **k: ((x, x), x) if k.get("residual") is not None else (x, x))
        recorder("gemm_ex", lambda *a, **k: torch.zeros(tokens, 1, dtype=k["out_dtype"]))
        recorder("row_scale_f16", lambda a: (a, a))
        recorder("mv_q8_ex", lambda *a, **k: torch.zeros(1))
        x = torch.zeros(tokens, h, dtype=dtype)
        ops.ffn(fmt, x, x[0], x, x, x, h, f, residual=x if residual else None, **kw)
        return list(state["calls"])

    return run


@pytest.mark.parametrize("on", [0, 1])
@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_every_call_runs_on_the_tensors_device(block, on, prefill, residual):
    calls = block(8, 128, 64, on=on, prefill=prefill, residual=residual)
    names = ["rms_norm", "gemm_ex", "row_scale_f16", "gemm_ex"] if prefill else ["rms_norm", "mv_q8_ex", "mv_q8_ex"]
    assert [c[0] for c in calls] == names
    assert all(c[1] == on for c in calls)
    assert torch.cuda.current_device() == 0


@pytest.mark.parametrize("fmt,tokens,h,f,kw,prefill", [
    ("q4_0", 63, 128, 64, {}, False), ("q4_0", 64, 128, 64, {}, True), ("q3_k", 1, 256, 256, {}, True),
    # widths that the GEMM does not take
    ("q4_0", 64, 96, 64, {}, False), ("q8_0", 200, 128, 160, {}, False), ("q4_0", 64, 96, 256, dict(fmt_down="q4_k"), False),
    ("mxfp4", 4, 96, 64, {}, True), ("q4_0", 64, 96, 64, dict(prefill=True), True)])
def test_which_path(block, fmt, tokens, h, f, kw, prefill):
    calls = block(tokens, h, f, fmt=fmt, **kw)
    assert ("gemm_ex" in [c[0] for c in calls]) == prefill


@pytest.mark.parametrize("dtype,between", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                           (torch.float32, torch.float32)])
def test_the_type_between_the_gemms(block, dtype, between):
    calls = [c for c in block(64, 128, 64, dtype=dtype) if c[0] == "gemm_ex"]
    assert [c[2]["out_dtype"] for c in calls] == [between, dtype]
