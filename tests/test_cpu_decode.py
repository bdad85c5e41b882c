"""Refusals of the decoding operators that need no GPU: kernel names, argument checks, sizes that a schedule must bring."""
import numpy as np
import pytest
import torch

from reef_b200 import capi, decode
from reef_b200.resources import decoding
from reef_b200.resources.graph import Graph

pytestmark = pytest.mark.usefixtures("libs")


def _names():
    return [decoding.page_tables(16, 64, 16, 1024, 16, False), decoding.page_tables(16, 64, 16, 1024, 16, True),
            decoding.paged_append(16, 12, 64, 16, 1024, "bfloat16"), decoding.paged_append(16, 12, 64, 16, 1024, "float32", 16),
            *decoding.paged_attention(16, 16, 12, 12, 64, 16, 4, 1024, "float16"),
            *decoding.paged_attention(16, 16, 32, 4, 128, 16, 640, 1024, "bfloat16"),
            *decoding.beam_select(4, 4, 30522, 2), *decoding.beam_select(4, 4, 30522, 2, tokens=16)]


@pytest.mark.parametrize("name", _names())
def test_names_are_planned(name):
    dims, smem, nargs = capi.kernel_plan(name)
    assert dims[3:] == [256, 1, 1] and dims[0] >= 1 and smem <= 227 * 1024
    k = capi.Kernel(name)
    assert k.num_args == nargs and all(b > 0 for b in k.arg_bytes)
    assert capi.kernel_cost(name)[1] > 0


TABLES = "reef_page_tables__rows16_mp64_ps16_pages1024_tokens16"
APPEND = "reef_paged_append__tokens16_kvh12_d64_ps16_pages1024_kt1"
ATTEND = "reef_paged_attention__tokens16_rows16_heads12_kvh12_d64_ps16_mp64_pages1024_kt0"
SCAN, PICK = "reef_beam_scan__requests4_beams4_vocab1000", "reef_beam_pick__requests4_beams4_vocab1000_eos2"


@pytest.mark.parametrize("name,old,new", [
    (TABLES, "rows16", "rows0"), (TABLES, "rows16", "rows1025"), (TABLES, "mp64", "mp0"), (TABLES, "ps16", "ps0"), (TABLES, "ps16", "ps1025"),
    (TABLES, "pages1024", "pages0"), (TABLES, "pages1024", "pages524289"), (TABLES, "tokens16", "tokens0"), (TABLES, "tokens16", "tokens1048577"),
    (TABLES, "_tokens16", ""), (TABLES, "mp64", "mp67108865"), (TABLES, "ps16", "ps4294967312"),
    (APPEND, "d64", "d96"), (APPEND, "d64", "d32"), (APPEND, "kvh12", "kvh0"), (APPEND, "kt1", "kt3"), (APPEND, "kt1", "kt1_ks770"),
    (APPEND, "kt1", "kt1_ks764"), (APPEND, "kt1", "kt1_vo2"), (APPEND, "pages1024", "pages134217728"), (APPEND, "kt1", "kt1_forks1048577"),
    (APPEND, "kt1", "kt1_ks4294967296"), (APPEND, "tokens16", "tokens1048577"), (ATTEND, "heads12", "heads13"), (ATTEND, "heads12", "heads0"), (ATTEND, "rows16", "rows65537"), (ATTEND, "tokens16", "tokens65537"),
    (ATTEND, "kt0", "kt0_qs764"), (ATTEND, "d64", "d512"), (ATTEND, "mp64", "mp67108865"),
    (SCAN, "beams4", "beams17"), (SCAN, "beams4", "beams0"), (SCAN, "vocab1000", "vocab0"), (SCAN, "vocab1000", "vocab1000_tokens0"),
    (PICK, "eos2", "eos1000"), (PICK, "_eos2", ""),
])
def test_names_out_of_range_are_unknown(name, old, new):
    capi.kernel_plan(name)
    assert old in name
    with pytest.raises(capi.ReefError) as e:
        capi.kernel_plan(name.replace(old, new))
    assert e.value.status == capi.NOT_FOUND


def test_a_schedule_with_a_small_cache_is_refused(tmp_path):
    def write(short):
        g = Graph("m")
        args = [g.input("k", 4 * 64), g.input("v", 4 * 64), g.input("tok", 16, "int32"),
                g.add_storage("k_cache", 8 * 16 * 64 * 2, "byte"), g.add_storage("output", 8 * 16 * 64 * 2 - short, "byte")]
        g.kernel(decoding.paged_append(4, 1, 64, 16, 8, "bfloat16"), args)
        return g.write(str(tmp_path / str(short)), capi.plan_fn)

    import ctypes as C
    lib = capi.host_lib()
    for short, ok in ((0, True), (1, False)):
        assert (lib.reef_model_check(C.c_char_p((write(short) + ".json").encode()), None, C.c_size_t(0)) == 0) == ok


def _cpu(*shape, dtype=torch.int32):
    return torch.zeros(shape, dtype=dtype)


def _refused(fn, *args, **kw):
    with pytest.raises(capi.ReefError) as e:
        fn(*args, **kw)
    assert e.value.status == capi.OUT_OF_RANGE
    return str(e.value)


def test_tensors_off_the_gpu_are_refused():
    f = torch.float32
    assert "not on a GPU" in _refused(decode.page_tables, _cpu(2, 4), _cpu(2), _cpu(2), pages=8, page_size=16, tokens=2)
    assert "not on a GPU" in _refused(decode.paged_append, _cpu(2, 1, 64, dtype=f), _cpu(2, 1, 64, dtype=f), _cpu(2, 4), _cpu(8, 1, 16, 64, dtype=f),
                                      _cpu(8, 1, 16, 64, dtype=f))
    assert "not on a GPU" in _refused(decode.paged_attention, _cpu(2, 1, 64, dtype=f), _cpu(8, 1, 16, 64, dtype=f), _cpu(8, 1, 16, 64, dtype=f),
                                      _cpu(2, 4), _cpu(2, 4))
    assert "not on a GPU" in _refused(decode.beam_select, _cpu(4, 100, dtype=f), _cpu(4, dtype=f), _cpu(4), beams=2, eos=1)


def test_values_that_are_no_sizes_are_refused():
    t, r = _cpu(2, 4), _cpu(2)
    for kw in (dict(pages=0, page_size=16, tokens=2), dict(pages=8, page_size=0, tokens=2), dict(pages=8, page_size=16, tokens=0),
               dict(pages=8.0, page_size=16, tokens=2), dict(pages=8, page_size=1025, tokens=2), dict(pages=(1 << 19) + 1, page_size=1, tokens=2)):
        _refused(decode.page_tables, t, r, r, **kw)
    _refused(decode.page_tables, None, r, r, pages=8, page_size=16, tokens=2)
    _refused(decode.page_tables, _cpu(1025, 4), _cpu(1025), _cpu(1025), pages=8, page_size=16, tokens=2)
    s = _cpu(4, dtype=torch.float32)
    for kw in (dict(beams=0, eos=1), dict(beams=17, eos=1), dict(beams=3, eos=1), dict(beams=2, eos=100), dict(beams=2, eos=-1)):
        _refused(decode.beam_select, _cpu(4, 100, dtype=torch.float32), s, _cpu(4), **kw)


def test_inputs_that_want_gradients_are_refused():
    q = torch.zeros(2, 1, 64, requires_grad=True)
    c = torch.zeros(8, 1, 16, 64)
    assert "gradients" in _refused(decode.paged_attention, q, c, c, _cpu(2, 4), _cpu(2, 4))
    with torch.no_grad():
        assert "gradients" not in _refused(decode.paged_attention, q, c, c, _cpu(2, 4), _cpu(2, 4))


def test_a_kernel_wants_its_arguments():
    k = capi.Kernel(SCAN)
    with pytest.raises(capi.ReefError):
        k.launch([0, 0])
    with pytest.raises(capi.ReefError):
        capi.Kernel("reef_beam_scan")
