"""cml_generate --drafts, as far as it comes without a device."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def test_files_have_no_form_to_draft_with(tmp_path):
    """Said before the model is loaded; with a drafter of its own the same line goes on to load it."""
    f = tmp_path / "model.gguf"
    f.write_bytes(b"no model")
    run = lambda *a: subprocess.run([str(ROOT / "bin" / "cml_generate"), "--model", str(f), "--tokens", "1,2", *a], capture_output=True, text=True, timeout=600)
    r = run("--drafts", "2")
    assert r.returncode == 2 and "--drafter" in r.stderr and "cannot load" not in r.stderr
    r = run("--drafts", "2", "--drafter", str(tmp_path))
    assert r.returncode == 2 and "cannot load" in r.stderr
