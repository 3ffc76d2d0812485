"""The pipeline in a captured graph: what a call clears before it works (keep masks, the screened search's row counter) is cleared on every replay."""
import pytest
import torch

import lbm_amd
from lbm_amd.synth import synth_epochs, synth_ica

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("kw", [dict(vq_method="screen", emit_cleaned=False), dict(fuse_post=False), dict(do_tokenize=False, emit_cleaned=False)],
                         ids=["fused post, screened search", "separate post", "features alone"])
def test_replays_of_a_captured_chunk_equal_eager_runs(shipped, kw):
    taps = lbm_amd.create_filter(500.0, 4.0, 30.0)
    A, b = lbm_amd.ica_projection(**synth_ica(30))

    def make():
        return lbm_amd.EpochPipeline(lbm_amd.PipelineConfig(**kw), taps, A, b, shipped, shipped["vq_layer.embedding.weight"])
    pipe, eager = make(), make()

    def epochs(turn):
        x = synth_epochs(12, 30, 1500, seed=60 + turn) * 2.0
        x[turn::5, 3, 700] -= 1e-2              # rejected, others each time
        return x.to(DEV)
    names = ("tokens", "psd", "bandpower", "keep")
    x = epochs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pipe.run(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pipe.run(x)
    kept = []
    for turn in range(4):
        x.copy_(epochs(turn))
        graph.replay()
        torch.cuda.synchronize()
        got = {k: out[k].clone() for k in names if k in out}
        want = eager.run(epochs(turn))
        for k, v in got.items():
            assert torch.equal(v, want[k]), (turn, k)
        kept.append(got["keep"].clone())
    assert all(not k.all() and k.any() for k in kept) and not torch.equal(kept[0], kept[1])
