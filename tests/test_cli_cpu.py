"""Command line: generate from a synthetic preset on CPU, inspect / tokenize / stage a GGUF written by the library itself."""
import json
import os

import pytest
import torch

from gemm_b200.__main__ import main
from gemm_b200.models import loader
from gemm_b200.models.config import get_config
from gemm_b200.models.weights import RandomSource


def test_generate_synthetic_cpu(capsys):
    main(["generate", "--model", "synthetic:tiny-dense", "--device", "cpu", "--ids", "--prompt", "1 2 3 4 5", "--prompt", "9 8 7",
          "--max-new-tokens", "4", "--pages", "16", "--page-size", "16"])
    out = [json.loads(l) for l in capsys.readouterr().out.strip().splitlines()]
    assert len(out) == 2 and all(len(o["token_ids"]) == 4 for o in out)


def test_inspect_and_stage(tmp_path, capsys):
    cfg = get_config("tiny-dense")
    path = str(tmp_path / "m.gguf")
    loader.save_gguf(cfg, RandomSource(cfg, 1, "cpu"), path, wtype="F16")
    main(["inspect", path, "--tensors"])
    txt = capsys.readouterr().out
    assert "general.architecture" in txt and "blk.0.attn_q.weight" in txt
    out_dir = str(tmp_path / "staged")
    main(["stage", "--model", path, "--out", out_dir, "--format", "bf16", "--tp", "2"])
    assert json.loads(capsys.readouterr().out.strip().splitlines()[-1])["ranks"] == 2
    assert os.path.exists(os.path.join(out_dir, "manifest.json"))


def test_estimate_roofline():
    from gemm_b200.models.config import get_config
    from gemm_b200.utils import estimate as est
    cfg = get_config("qwen3-30b-a3b")
    assert abs(est.experts_touched(128, 8, 64) - 126.0) < 1.0
    r1 = est.estimate(cfg, 64, 2048, 1, "mxfp8")
    r8 = est.estimate(cfg, 64, 2048, 8, "mxfp8")
    assert r1["fits"] and r8["fits"]
    assert 5.0 < r1["decode_ms_per_step"] < 14.0                # measured 13.3 ms on one B200: the estimate is a ceiling
    assert r8["decode_ms_per_step"] < r1["decode_ms_per_step"]
    assert r1["decode_bound"] == "memory"
    assert est.estimate(cfg, 64, 2048, 1, "bf16")["decode_memory_ms"] > r1["decode_memory_ms"]


def test_compare_command_cpu_side(capsys):
    from gemm_b200.__main__ import main
    main(["compare", "--model", "synthetic:tiny-dense", "--steps", "3", "--prompt-len", "12", "--oracle"])
    rep = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert len(rep["cpu_tokens"]) == 3 and rep["cpu_vs_fp32_oracle_rel"] < 3e-2


def test_dump_command_writes_layer_states(tmp_path, capsys):
    import numpy as np
    from gemm_b200.__main__ import main
    main(["dump", "--model", "synthetic:tiny-dense", "--device", "cpu", "--ids", "1 2 3 4 5", "--out", str(tmp_path)])
    rep = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert rep["layers"] == 2 and rep["tokens"] == 5
    h = np.load(tmp_path / "layer_001.npy")
    lg = np.load(tmp_path / "logits.npy")
    assert h.shape == (5, 256) and lg.shape[0] == 5 and np.isfinite(h).all()


def test_context_parallel_cost_model():
    from gemm_b200.models.config import get_config
    from gemm_b200.utils import estimate as est
    cfg = get_config("qwen3-30b-a3b")
    one = est.context_parallel_decode(cfg, 1, 1 << 20, 1)
    eight = est.context_parallel_decode(cfg, 1, 1 << 20, 8)
    assert one["partial_bytes"] == 32 * 129 * 4                       # 16 512 bytes of (O, lse) for 32 heads of 128
    assert abs(eight["kv_read_us_per_layer"] * 8 - one["kv_read_us_per_layer"]) < 1e-6
    assert eight["merge_allgather_us"] < eight["merge_tree_us"] < eight["merge_ring_us"]      # one exchange beats dependent hops on a switch
    assert eight["attention_us_per_layer"] < one["attention_us_per_layer"]


def test_generate_speculative_flag_gives_the_greedy_tokens(capsys):
    base = ["generate", "--model", "synthetic:tiny-dense", "--device", "cpu", "--ids", "--prompt", "1 2 3 1 2 3 1 2", "--prompt", "7 7 7 7",
            "--max-new-tokens", "10", "--pages", "16", "--page-size", "16"]
    main(base)
    plain = [json.loads(l)["token_ids"] for l in capsys.readouterr().out.strip().splitlines()]
    main(base + ["--speculative", "3"])
    cap = capsys.readouterr()
    spec = [json.loads(l)["token_ids"] for l in cap.out.strip().splitlines()]
    assert spec == plain
    summary = json.loads(cap.err.strip().splitlines()[-1])
    assert summary["verify_steps"] <= 9 and "draft_acceptance" in summary


@pytest.mark.parametrize("model,flags,says", [
    ("tiny-dense", ["--tree", "3"], "--speculative"), ("tiny-fidolix", ["--speculative", "2", "--tree", "2"], "recurrent"), ("tiny-qwen35", ["--speculative", "2"], "recurrent"),
    ("tiny-dense", ["--speculative", "3", "--tree", "300"], "256")])
def test_generate_says_what_speculation_cannot_do(model, flags, says):
    """A message instead of a traceback, and no flag that is passed over."""
    with pytest.raises(SystemExit) as e:
        main(["generate", "--model", f"synthetic:{model}", "--device", "cpu", "--ids", "--prompt", "1 2 3 1 2", "--max-new-tokens", "3", "--pages", "16", "--page-size", "16"] + flags)
    assert isinstance(e.value.code, str) and says in e.value.code


def test_speculative_speedup_model():
    from gemm_b200.utils.estimate import speculative_speedup
    r = speculative_speedup(1.0, 4, 1.38)
    assert r["tokens_per_step"] == 5.0 and abs(r["speedup"] - 5 / 1.38) < 1e-9
    r = speculative_speedup(0.0, 4, 1.38)
    assert r["tokens_per_step"] == 1.0 and r["speedup"] < 1.0
    r = speculative_speedup(0.5, 2, 1.26)
    assert abs(r["tokens_per_step"] - 1.75) < 1e-9
