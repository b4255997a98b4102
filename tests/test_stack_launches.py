"""The decode stack without a GPU: stand-ins for the library's weights and caches,
and every torch operation of a step counted, each of which is a kernel launch on
the device that a captured step repeats."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

VIEWS = ("view", "slice", "_unsafe_view", "detach", "alias")


class Weight:
    @classmethod
    def quantize(cls, w, encoding, gated=False):
        return cls()

    def forward(self, x, y, alpha=1.0, stream=None):
        return y


class Cache:
    def __init__(self, *args, **kw):
        self.calls = []

    def append(self, *args, **kw):
        self.calls.append(("append", None))

    def append_rotary(self, *args, positions=None, **kw):
        self.calls.append(("append_rotary", positions.clone()))

    def attend(self, *args, **kw):
        self.calls.append(("attend", None))


class Library:
    ENCODING_AQ4_G128 = 0
    LinearWeight, KvCache = Weight, Cache


class Count(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.ops = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        name = func.overloadpacket.__name__
        if name not in VIEWS:
            self.ops.append(name)
        return func(*args, **(kwargs or {}))


def stack_of(**over):
    import stack
    weights = [{n: torch.zeros(1, 1) for n in ("qkv", "o", "gate_up", "down")} for _ in range(2)]
    return stack.DecodeStack(Library, torch, torch.device("cpu"), batch=3, layers=2, hidden=256,
                             qkv=512, ffn=64, vocab=10,
                             weights={**dict(enumerate(weights)), "lm_head": torch.zeros(1, 1)},
                             **over)


@pytest.fixture(autouse=True)
def paths(uh, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


@pytest.mark.parametrize("bits", [4, 8])
def test_a_step_without_rotation_counts_lengths_alone(bits):
    st = stack_of(context=64, kv_bits=bits)
    with Count() as c:
        st.step()
    assert c.ops == ["add_"]
    assert st.lengths.tolist() == [1, 1, 1]
    assert [x for x, _ in st.caches[0].calls] == ["append", "attend"]


def test_a_step_with_rotation_counts_positions_too():
    st = stack_of(context=64, rope_base=10000.0)
    h = torch.zeros((6, 256), dtype=torch.bfloat16)
    st.prompt(h, [1, 2, 3])
    for cache in st.caches:
        cache.calls.clear()
    with Count() as c:
        st.step()
    assert [op for op in c.ops if op != "clone"] == ["add_", "add_", "sub"]
    assert st.lengths.tolist() == st.given.tolist() == [2, 3, 4]
    for cache in st.caches:
        assert cache.calls[0][0] == "append_rotary"
        assert cache.calls[0][1].tolist() == [1, 2, 3]


def test_a_step_without_a_cache_launches_nothing_of_its_own():
    st = stack_of()
    with Count() as c:
        st.step()
    assert c.ops == []
