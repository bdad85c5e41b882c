"""What the decoding operators report and refuse, where no GPU is needed to see it."""
import os
import shutil
import subprocess
import sys

import pytest
import torch

from reef_b200 import capi, decode
from reef_b200.resources import decoding

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


# the steps of all rows together (0x70000000) bound the form that adds them up, not the one that takes a row to a block
WIDE = dict(heads=32, kv_heads=32, dim=128, page_size=64, max_pages=2048, pages=4096, cache="bfloat16")


def test_many_tokens_over_long_tables():
    for tokens, fits in ((3583, True), (8192, False)):          # 32 passes a token, 16384 steps a pass
        names = decoding.paged_attention(tokens, 4, **WIDE)
        assert len(names) == 1
        capi.kernel_plan(names[0])
        for form in ("parts", "join"):
            name = names[0].replace("attention__", f"attention_{form}__")
            if fits:
                capi.kernel_plan(name)
            else:
                with pytest.raises(capi.ReefError):
                    capi.kernel_plan(name)
    # tables so long that the division among blocks would be taken: only as far as it can count
    for tokens, forms in ((64, 2), (4096, 2), (8192, 1)):
        names = decoding.paged_attention(tokens, 4, 1, 1, 256, 1024, 512, 600, "float32")
        assert len(names) == forms
        for name in names:
            capi.kernel_plan(name)


def _big(*shape, dtype=torch.int32):
    return torch.zeros(1, dtype=dtype).expand(*shape)


def _why(fn, *args, **kw):
    with pytest.raises(capi.ReefError) as e:
        fn(*args, **kw)
    assert e.value.status == capi.OUT_OF_RANGE
    return str(e.value)


def test_sizes_beyond_the_kernels_are_named():
    f = torch.float32

    def attend(tokens=2, heads=2, rows=2, most=4, pages=8, kv=1, page=16):
        c = _big(pages, kv, page, 64, dtype=f)
        return _why(decode.paged_attention, _big(tokens, heads, 64, dtype=f), c, c, _big(rows, most), _big(tokens, 4))

    assert "not on a GPU" in attend() and "not on a GPU" in attend(tokens=65536, rows=65536, heads=1024, page=1024, most=1 << 20)
    assert "tokens: 65537, at most 65536" in attend(tokens=65537)
    assert "rows: 65537, at most 65536" in attend(rows=65537)
    assert "heads: 1025, at most 1024" in attend(heads=1025)
    assert "tokens of a page: 1025, at most 1024" in attend(page=1025)
    assert "tokens of a row: " in attend(most=(1 << 26) + 1)
    assert "keys of the cache: " in attend(pages=1 << 23, kv=16)

    def append(tokens=2, kv=1, forks=None, pages=8):
        c, k = _big(pages, kv, 16, 64, dtype=f), _big(tokens, kv, 64, dtype=f)
        return _why(decode.paged_append, k, k, _big(tokens, 4), c, c, fork=None if forks is None else _big(forks, 4))

    assert "not on a GPU" in append() and "not on a GPU" in append(tokens=1 << 20, forks=1 << 20)
    assert "tokens: 1048577, at most 1048576" in append(tokens=(1 << 20) + 1)
    assert "values of all tokens: " in append(tokens=1 << 20, kv=32)
    assert "forks: 1048577, at most 1048576" in append(forks=(1 << 20) + 1)
    assert "kv heads: 1025, at most 1024" in append(kv=1025)
    assert "tokens of the cache: " in append(pages=1 << 27)

    def tables(rows=2, most=4, page=16):
        return _why(decode.page_tables, _big(rows, most), _big(rows), _big(rows), pages=8, page_size=page, tokens=2)

    assert "not on a GPU" in tables() and "not on a GPU" in tables(rows=1024, most=1 << 20)
    assert "tokens of a row: " in tables(most=(1 << 26) + 1)
    assert "ids of the table: " in tables(rows=1024, most=(1 << 20) + 1)

    def beams(rows=2, words=100, start=None):
        return _why(decode.beam_select, _big(rows, words, dtype=f), _big(rows, dtype=f), _big(rows), beams=1, eos=0)

    assert "not on a GPU" in beams() and "not on a GPU" in beams(rows=1 << 20)
    assert "words: " in beams(words=1 << 27)
    assert "rows: 1048577" in beams(rows=(1 << 20) + 1)


def test_signatures_and_kernels_do_not_pile_up():
    """A server whose prompts have every length: what is kept of them has a bound."""
    r = _run("""
import resource, torch, weakref
from reef_b200 import capi, decode
native = decode._decode
native.count()
native = decode._decode
seen = []
def many(first, n):
    for i in range(first, first + n):
        k = capi.Kernel(f"reef_paged_append__tokens{i + 1}_kvh1_d64_ps16_pages8_kt0")
        native.define(99, (None,), None, (i,), [(k.handle, k.dims, k.dyn_smem, [0])], [], 0, [], [], [k])
        seen.append(weakref.ref(k))
many(0, 6000)
assert native.count() == 4096 and native.call(99, (None,), None, (1,)) is None
alive = [i for i, k in enumerate(seen) if k() is not None]
assert 4096 <= len(alive) <= 4097 and alive[0] >= 1903, (len(alive), alive[0])
before = resource.getrusage(resource.RUSAGE_SELF).ru_maxrss
many(6000, 60000)
assert native.count() == 4096
print("kept", resource.getrusage(resource.RUSAGE_SELF).ru_maxrss - before < 24 << 10)
native.define(99, (None,), None, (65999,), [], [], 0, [], [], [])      # one that is there is replaced
assert native.count() == 4096
""")
    assert r.stdout.strip() == "kept True", r.stdout + r.stderr


def test_inputs_that_carry_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    f = torch.float32
    c = torch.zeros(8, 1, 16, 64)
    with fw.dual_level(), torch.no_grad():
        q = fw.make_dual(torch.zeros(2, 1, 64), torch.ones(2, 1, 64))
        for call in (lambda x: decode.paged_attention(x, c, c, _big(2, 4), _big(2, 4)), lambda x: decode.paged_append(x, x, _big(2, 4), c, c.clone()),
                     lambda x: decode.beam_select(x[:, 0], x[:, 0, 0], _big(2), beams=1, eos=0)):
            assert "tangents" in _why(call, q) and "not on a GPU" in _why(call, fw.unpack_dual(q).primal)


def test_views_that_stand_for_their_negative_are_refused():
    """The imaginary part of a conjugate holds the values of the other sign."""
    c, q = torch.zeros(8, 1, 16, 64), torch.zeros(2, 1, 64)
    score = torch.zeros(1, dtype=torch.complex64).conj().imag
    assert score.is_neg() and score.is_contiguous()
    neg = torch._neg_view
    assert "negative" in _why(decode.paged_attention, q, neg(c), c, _big(2, 4), _big(2, 4))
    assert "negative" in _why(decode.paged_append, q, q, _big(2, 4), neg(c), c)
    assert "negative" in _why(decode.page_tables, neg(_big(2, 4).clone()), _big(2), _big(2), pages=8, page_size=16, tokens=2)
    assert "negative" in _why(decode.beam_select, neg(torch.zeros(1, 9)), torch.zeros(1), _big(1), beams=1, eos=0)
