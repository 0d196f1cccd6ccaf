"""A model's decode step is recorded as a graph built of nodes: no stream of the process is captured meanwhile, so that null-stream calls of
other threads go on (a captured stream has them refused, and is lost to them)."""
import os
import re
import shutil
import subprocess
import tempfile

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "nano_vllm_amd", "csrc")


def test_launches_become_nodes(tmp_path):
    rocm = "/opt/rocm/include"
    if shutil.which("g++") is None or not os.path.isdir(rocm):
        pytest.skip("no host compiler or HIP headers")
    exe = str(tmp_path / "recording_driver")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-D__HIP_PLATFORM_AMD__", "-I", rocm, "-I", CSRC, "-o", exe,
                        os.path.join(ROOT, "tests", "recording_driver.cpp"), "-lpthread"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_the_step_captures_no_stream_and_launches_nothing_past_the_recording():
    """The files that a step's launches come from: no capture in the model, no launch and no copy of the step that would run instead of
    being recorded."""
    model = open(os.path.join(CSRC, "nvk_model.hip")).read()
    assert "BeginCapture" not in model
    body = model[model.index("auto enqueue_linked"):model.index("auto enqueue_body")]
    assert not re.search(r"\bhip(Memcpy|Memset|Event|Launch)\w*\(", body)
    for name in ("nvk_model.hip", "nvk_batch.hip", "nvk_linear.hip", "nvk_paged_attn.hip"):
        text = open(os.path.join(CSRC, name)).read()
        assert "hipLaunchKernelGGL(" not in text and "<<<" not in text, name


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [1, 3])
def test_steps_are_recorded_and_replayed(seqs, capfd, monkeypatch):
    """The second step of a shape is recorded, later ones replay it: the bits of direct launches, and no refusal."""
    import nano_vllm_amd as nv
    from golden_defs import write_checkpoint

    spec = dict(dim=96, hidden_dim=256, n_layers=2, n_heads=6, n_kv_heads=6, vocab_size=200, max_seq_len=64, block_size=8, num_blocks=8 * seqs,
                weight_seed=5, weight_gain=0.35, shared=False)
    monkeypatch.setenv("NVK_GRAPH_DEBUG", "1")
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "m.bin")
        write_checkpoint(path, spec)
        got = []
        for graphs in (False, True):
            with nv.LlamaModel(path, 8, spec["num_blocks"], max_seqs=seqs) as m:
                m.use_graphs(graphs)
                for r in range(seqs):
                    m.add_request(r)
                rows = []
                for step in range(12):
                    _, logits = m.step(list(range(seqs)), [(7 * r + 3 * step) % 199 + 1 for r in range(seqs)], True)
                    rows.append(logits.copy())
                got.append(np.stack(rows))
    err = capfd.readouterr().err
    assert (got[0].view(np.uint32) == got[1].view(np.uint32)).all()
    assert f"recorded a {seqs}-request decode step" in err and "refused" not in err, err
