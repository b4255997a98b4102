"""The decode stack at the end of its context."""
import pytest
import torch

from test_gpu_kv_calls import small_stack

pytestmark = pytest.mark.gpu


def test_prompt_and_step_stop_at_the_context(uh, gpu):
    st = small_stack(uh, gpu, context=100, evict_to=40)          # 2 blocks of 64
    h = torch.randn((131, 512), device=gpu).bfloat16()
    with pytest.raises(ValueError, match="room for 128"):
        st.prompt(h, [129, 1, 1])
    st.prompt(h[:130], [128, 1, 1])
    assert st.lengths.tolist() == [128, 1, 1]
    with pytest.raises(ValueError, match="129 tokens"):
        st.step()
    assert st.lengths.tolist() == [128, 1, 1]                     # nothing ran
    st.evict()
    assert st.lengths.tolist() == [40, 1, 1]
    for _ in range(3):
        st.step()
    with pytest.raises(ValueError):
        st.prompt(h[:88], [86, 1, 1])
    st.prompt(h[:87], [85, 1, 1])
    assert st.lengths.tolist() == [128, 5, 5]
    st.destroy()


def test_replays_are_announced(uh, gpu):
    st = small_stack(uh, gpu, context=64)
    h = torch.randn((183, 512), device=gpu).bfloat16()
    st.prompt(h, [61, 61, 61])
    st.h0.copy_(h[:3])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        st.step()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        st.step()                                                 # not counted: it does not run
    for _ in range(2):
        st.replayed()
        g.replay()
    torch.cuda.synchronize()
    assert st.lengths.tolist() == [64, 64, 64]
    with pytest.raises(ValueError):
        st.replayed()
    with pytest.raises(ValueError):
        st.step()
    st.destroy()
