"""Results, workspaces and copies that a call with stream= makes for itself come
from that stream's memory, and not from the current one's."""
import ctypes

import pytest

import vtx_attn as V
from test_paged_edges import FakeStreams, SideStream

torch = pytest.importorskip("torch")


class Lib:
    """Calls that succeed, and ask for a workspace."""

    def __getattr__(self, name):
        return lambda *_: 1024 if name.endswith("workspace") else 0


def z(*s, dtype=torch.float32):
    return torch.zeros(s, dtype=dtype)


def calls():
    i32 = torch.zeros(3, dtype=torch.int32)
    buf = [z(8, 2 * 64, dtype=torch.float16)] * 3
    batch = V.DecodeBatchPlan(buf, buf, i32, 4, 2, 64, V.F16, 256, 128, 8, 0.1)
    layer = V.DecodeLayerPlan(buf, buf, i32, i32, i32, 4, 2, 64, V.F16, 256, 8, 0.1)
    return {"flash_attn_ext": (lambda s: V.flash_attn_ext(z(1, 4, 3, 64), z(1, 2, 5, 64), z(1, 2, 5, 64), None, 0.1, stream=s), 2),
            "decode_batched": (lambda s: batch(z(3, 4, 64), stream=s), 1),
            "kv_append": (lambda s: V.kv_append(z(3, 2, 64), z(3, 2, 64), i32, i32, buf[0], buf[1], V.F16, q=z(3, 4, 64), stream=s), 1),
            "decode_layer": (lambda s: layer(z(3, 4, 64), z(3, 2, 64), z(3, 2, 64), stream=s), 1),
            "out_proj": (lambda s: V.out_proj(z(1, 3, 4, 64), z(32, 256, dtype=torch.float16), stream=s), 1)}


@pytest.mark.parametrize("name", ["flash_attn_ext", "decode_batched", "kv_append", "decode_layer", "out_proj"])
def test_made_on_the_writing_stream(name, monkeypatch):
    monkeypatch.setattr(V, "_lib", Lib())
    call, count = calls()[name]
    fake = FakeStreams(monkeypatch)
    side = SideStream()
    call(side)
    assert fake.made == [side] * count and fake.noted == ["main"] * count and fake.current == ["main"]


@pytest.mark.gpu
def test_results_and_workspaces_are_their_own():
    """flash_attn_ext with split keys: neither its result nor its workspace is a
    block that work on the current stream still writes."""
    torch.manual_seed(0)
    q, k, v = (torch.randn(1, h, n, 128, device="cuda", dtype=t) for h, n, t in
               ((32, 1, torch.float32), (8, 3000, torch.float16), (8, 3000, torch.float16)))
    want = V.flash_attn_ext(q, k, v, None, 0.1)
    need = V.workspace_bytes(q, k, v, 0.1)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        torch.cuda._sleep(20_000_000)
        for busy in (torch.empty_like(want), torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")):
            busy.fill_(7)
        del busy
        out = V.flash_attn_ext(q, k, v, None, 0.1, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
