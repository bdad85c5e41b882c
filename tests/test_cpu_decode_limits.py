"""What the decoding operators report and refuse, where no GPU is needed to see it."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.usefixtures("libs")


def _run(code, **env):
    """A process of its own that sees no GPU."""
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, env={**os.environ, "CUDA_VISIBLE_DEVICES": "", **env}, capture_output=True, text=True,
                          timeout=300)


@pytest.mark.parametrize("name", ["reef_page_tables__rows16_mp64_ps16_pages1024_tokens16", "reef_paged_append__tokens16_kvh12_d64_ps16_pages1024_kt1",
                                  "reef_paged_attention__tokens16_rows16_heads12_kvh12_d64_ps16_mp64_pages1024_kt0",
                                  "reef_beam_scan__requests4_beams4_vocab1000", "add"])
def test_a_device_that_cannot_be_prepared_is_reported(name):
    """A kernel whose setup has failed must not look ready: its launches would fail later, with another message."""
    r = _run(f"from reef_b200 import capi\nk = capi.Kernel({name!r})\ntry:\n    k.prepare([0] * k.num_args)\nexcept capi.ReefError as e:\n"
             "    print('status', e.status, 'no CUDA' in str(e) or 'driver' in str(e))")
    assert r.stdout.strip() == "status 1 True", r.stdout + r.stderr


def test_the_module_can_be_imported_before_the_libraries_are_built(tmp_path):
    """A clone that is not built: tests are collected, and a call says what is missing."""
    shutil.copytree(os.path.join(ROOT, "reef_b200"), tmp_path / "reef_b200", ignore=shutil.ignore_patterns("*.so", "csrc", "__pycache__"))
    r = subprocess.run([sys.executable, "-c", "import torch\nfrom reef_b200 import capi, decode\nx = torch.zeros(2, 4, dtype=torch.int32)\n"
                        "try:\n    decode.page_tables(x, x[0], x[1], pages=1, page_size=1, tokens=1)\nexcept capi.ReefError as e:\n    print(e)"],
                       cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert "is not built" in r.stdout, r.stdout + r.stderr


def test_the_libraries_are_built_without_torch():
    r = _run("import sys\nsys.modules['torch'] = None\nfrom reef_b200 import build, capi\nprint(len(build.build_all()))\ncapi.kernel_plan('add')")
    assert r.stdout.strip() == "2" and r.returncode == 0, r.stdout + r.stderr
