"""What the Python cache refuses before the library is called, without a GPU:
a ValueError that names the argument.  Tensors here are on the CPU, so the
cache is one of the device number that torch gives them."""
import pytest
import torch


@pytest.fixture
def cache(uh, monkeypatch):
    monkeypatch.setattr(uh, "_raw_stream", lambda: 0)
    c = uh.KvCache.__new__(uh.KvCache)
    c.handle, c.kv_heads, c.head_dim, c.block_tokens, c.device = None, 2, 128, 64, -1
    return c


def _args():
    q = torch.zeros((2, 4, 128), dtype=torch.bfloat16)
    return q, torch.zeros(2, dtype=torch.int32), torch.zeros((2, 3), dtype=torch.int32)


def _calls(c):
    q, n, t = _args()
    kv = q[:, :2]
    i64 = 1 << 64
    return [
        (lambda: c.attend(q, n, t, window=-1), "window"),
        (lambda: c.attend(q, n, t, window=1 << 32), "window"),
        (lambda: c.attend(q, n, t, window=2.5), "field"),
        (lambda: c.attend(q, n, t, scale="1"), "field"),
        (lambda: c.attend(q[0], n, t), "q must be"),
        (lambda: c.attend(q[0, 0], n, t), "q must be"),
        (lambda: c.attend(q[:, :, :64], n, t), "q must be"),
        (lambda: c.attend(q.float(), n, t), "q must be"),
        (lambda: c.attend(q, n, t[0]), "tables"),
        (lambda: c.attend(q, n, t[:, :, None]), "tables"),
        (lambda: c.attend(q, n, t, out=q[:1]), "rows"),
        (lambda: c.attend(q, n, t, lse=torch.zeros(2, 3)), "lse"),
        (lambda: c.attend(q, n, t, stream=-1), "field"),
        (lambda: c.attend_plan(q, n, t, window=-1), "window"),
        (lambda: c.attend_plan(q[0], n, t), "q must be"),
        (lambda: c.append(q, q, n, t), "k must be"),
        (lambda: c.append(kv[0], kv, n, t), "k must be"),
        (lambda: c.append(kv, kv[:1], n, t), "rows"),
        (lambda: c.append(kv, kv, n, t, weights=torch.zeros(2, 3)), "weights"),
        (lambda: c.gather(n, t, -1), "rows"),
        (lambda: c.gather_weights(n, t, -1), "rows"),
        (lambda: c.gather(n, t[0], 2), "tables"),
        (lambda: c.evict(n, t, t, -1), "keep"),
        (lambda: c.evict(n, t, t, 64, sink=-1), "sink"),
        (lambda: c.evict(n, t, t, 64, recent=-1), "recent"),
        (lambda: c.evict(n, t[0], t, 64), "tables"),
        (lambda: c.evict(n, t, t, 256), "new_tables"),
        (lambda: c.evict(n, t, t, 64, sink=i64), "field")]


@pytest.mark.parametrize("i", range(28))
def test_refusals_name_the_argument(cache, i):
    call, word = _calls(cache)[i]
    with pytest.raises(ValueError, match=word):
        call()


def test_valid_arguments_reach_the_library(uh, cache):
    """The handle is all that is missing."""
    q, n, t = _args()
    kv = q[:, :2]
    assert len(_calls(cache)) == 28
    for call in (lambda: cache.attend(q, n, t, window=3), lambda: cache.append(kv, kv, n, t),
                 lambda: cache.gather(n, t, 2), lambda: cache.gather_weights(n, t, 2),
                 lambda: cache.evict(n, t, t, 64)):
        with pytest.raises(uh.HipError, match="handle is null"):
            call()


def test_tensors_of_another_device_are_refused(cache):
    """The kernels would follow their addresses."""
    q, n, t = _args()
    kv, w = q[:, :2], torch.zeros(2, 2)
    s = torch.zeros(3, dtype=torch.int32)
    lse, ws = torch.zeros(2, 4), torch.zeros(256, dtype=torch.uint8)

    class Other(torch.Tensor):
        def get_device(self):
            return 0

    def one_elsewhere(fn, names, **args):
        for name in names:
            with pytest.raises(ValueError, match="on GPU"):
                fn(**{**args, name: args[name].as_subclass(Other)})

    one_elsewhere(cache.append, ["k", "v", "lengths", "tables", "starts", "weights"],
                  k=kv, v=kv, lengths=n, tables=t, starts=s, weights=w)
    one_elsewhere(cache.attend, ["q", "lengths", "tables", "starts", "out", "lse", "workspace"],
                  q=q, lengths=n, tables=t, starts=s, out=q.clone(), lse=lse, workspace=ws)
    for fn in (cache.gather, cache.gather_weights):
        one_elsewhere(fn, ["lengths", "tables", "starts"], lengths=n, tables=t, rows=2, starts=s)
    one_elsewhere(cache.evict, ["lengths", "tables", "new_tables"], lengths=n, tables=t,
                  new_tables=t, keep=64)
