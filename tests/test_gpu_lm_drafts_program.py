"""cml_generate --drafts for models in 32 bits: the drafter is the folder's 8-bit form, which is bfloat16."""
import subprocess
from pathlib import Path

import pytest

import lm_util

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


def test_drafts_of_a_model_in_32_bits(synth, tmp_path):
    cfg, w, folder = lm_util.build(synth, tmp_path, "mixed")
    run = lambda *a: subprocess.run([str(ROOT / "bin" / "cml_generate"), "--model", str(folder), "--tokens", "5,6,7,8,9", "--max-new", "12", *a], capture_output=True, text=True, timeout=600)
    for extra in ((), ("--temperature", "0.9", "--seed", "4"), ("--drafter", str(folder))):
        r = run("--dtype", "float32", "--drafts", "3", *extra)
        assert r.returncode == 0 and len(r.stdout.split("\t")[0].split()) == 12, (extra, r.stderr[-500:])
    plain = run("--dtype", "float32")
    assert plain.returncode == 0 and run("--dtype", "float32", "--drafts", "3").stdout == plain.stdout        # greedy: what the model says without a drafter
