"""The paged cache's entry points without a GPU: argument checks come before any device call, NULL handles fail
cleanly, and the Python mirror refuses bad tensors before the library is reached."""
import ctypes as C

import numpy as np
import pytest

from picolm_qwen_amd import PagedAttention, PagedBatch, PQAError, _lib

torch = pytest.importorskip("torch")


def create(*shape, memory=(None, None, None, None), bounds=0):
    h = C.c_void_p()
    rc = _lib.lib().pqa_paged_create(C.byref(h), *shape, bounds, *memory)
    assert not h.value
    return rc, _lib.lib().pqa_paged_last_error(None).decode()


@pytest.mark.parametrize("shape,code,what", [
    ((0, 4, 16, 8, 2, 128, 0), _lib.PQA_ERR_ARG, "positive"), ((1, -4, 16, 8, 2, 128, 0), _lib.PQA_ERR_ARG, "positive"),
    ((1, 4, 16, 8, 3, 128, 0), _lib.PQA_ERR_ARG, "multiple"), ((1, 4, 8, 8, 2, 128, 0), _lib.PQA_ERR_UNSUPPORTED, "page_size"),
    ((1, 4, 48, 8, 2, 128, 0), _lib.PQA_ERR_UNSUPPORTED, "page_size"), ((1, 4, 512, 8, 2, 128, 0), _lib.PQA_ERR_UNSUPPORTED, "page_size"),
    ((1, 4, 16, 8, 2, 80, 0), _lib.PQA_ERR_UNSUPPORTED, "head_dim"), ((1, 4, 16, 8, 2, 320, 0), _lib.PQA_ERR_UNSUPPORTED, "head_dim"),
    ((1, 4, 16, 8, 2, 128, 3), _lib.PQA_ERR_ARG, "type"), ((1, 4, 16, 8, 2, 128, -1), _lib.PQA_ERR_ARG, "type"),
    ((1, 1 << 24, 128, 8, 8, 128, 0), _lib.PQA_ERR_UNSUPPORTED, "2^31")])
def test_create_rejects_bad_shapes_before_any_device_call(shape, code, what):
    rc, message = create(*shape)
    assert rc == code and what in message


def test_create_rejects_half_given_and_misaligned_memory():
    good = (1, 4, 16, 8, 2, 128, 0)
    assert create(*good, memory=(4096, None, None, None))[0] == _lib.PQA_ERR_ARG
    assert create(*good, memory=(4096, 8192, 64, 64))[0] == _lib.PQA_ERR_ARG            # bounds' memory without bounds
    assert create(*good, memory=(4096, 8192, None, None), bounds=1)[0] == _lib.PQA_ERR_ARG
    assert create(*good, memory=(4096 + 8, 8192, None, None))[0] == _lib.PQA_ERR_ARG
    assert create(*good, memory=(4096, 8192, 64, 66), bounds=1)[0] == _lib.PQA_ERR_ARG


def test_null_handles_fail_cleanly():
    L = _lib.lib()
    assert L.pqa_paged_create(None, 1, 4, 16, 8, 2, 128, 0, 0, None, None, None, None) == _lib.PQA_ERR_ARG
    assert L.pqa_paged_memory(None, None, None, None, None) == _lib.PQA_ERR_ARG
    assert L.pqa_paged_set_rope(None, 0, 64, 4, None, None) == _lib.PQA_ERR_ARG
    assert L.pqa_paged_set_qk_norm(None, 0, None, None) == _lib.PQA_ERR_ARG
    assert L.pqa_batch_create(None, None, 1, 1, 1) == _lib.PQA_ERR_ARG
    assert L.pqa_batch_set(None, 0, None, None, None, 0, None) == _lib.PQA_ERR_ARG
    assert L.pqa_paged_append(None, None, 0, *[None, 0] * 4, None) == _lib.PQA_ERR_ARG
    assert L.pqa_paged_attend(None, None, 0, *[None, 0] * 2, None) == _lib.PQA_ERR_ARG
    assert L.pqa_paged_forward(None, None, 0, *[None, 0] * 4, None) == _lib.PQA_ERR_ARG
    assert L.pqa_paged_attend_sparse(None, None, 0, None, 0, 4, 1, 2, None, None, 0, None) == _lib.PQA_ERR_ARG
    assert b"NULL" in L.pqa_paged_last_error(None)
    L.pqa_paged_destroy(None)
    L.pqa_batch_destroy(None)


def detached(kind="bf16"):
    """A PagedAttention whose checks run but which holds no cache: a call that got past them would raise RuntimeError."""
    a = PagedAttention.__new__(PagedAttention)
    a._h, a._index, a._device = None, -1, None
    a.n_heads, a.n_kv_heads, a.head_dim, a.q_dim, a.kv_dim = 8, 2, 64, 512, 128
    a.io_type = {"bf16": torch.bfloat16, "f32": torch.float32}[kind]
    a._calls, a._empty_like, a._zeros_like, a._raw_stream = _lib.lib(), torch.empty_like, torch.zeros_like, None
    b = PagedBatch.__new__(PagedBatch)
    b.att, b._h, b.n_tokens = a, None, 3
    return a, b


def rows(n, dim, dtype=torch.bfloat16):
    return torch.zeros((n, dim), dtype=dtype)


@pytest.mark.parametrize("call", [
    lambda a, b: a.attend(0, b, rows(2, 512)),                              # fewer rows than tokens
    lambda a, b: a.attend(0, b, rows(3, 511)),
    lambda a, b: a.attend(0, b, rows(3, 512, torch.float32)),
    lambda a, b: a.attend(0, b, rows(512, 3).t()),                          # elements of a row apart
    lambda a, b: a.attend(0, b, rows(3, 512), out=rows(1, 512).expand(3, 512)),  # rows on top of each other
    lambda a, b: a.attend(0, b, rows(3, 512)[:, :256].repeat(1, 2).view(-1)),
    lambda a, b: a.append(0, b, rows(3, 512), rows(3, 64), rows(3, 128)),
    lambda a, b: a.append(0, b, rows(3, 512), rows(3, 128), rows(2, 128)),
    lambda a, b: a.forward(0, b, rows(3, 512), rows(3, 128), rows(3, 128), out=rows(3, 512, torch.float16)),
    lambda a, b: a.attend_sparse(0, b, rows(3, 512), 0),
    lambda a, b: a.attend_sparse(0, b, rows(3, 512), 4, chosen=torch.zeros((3, 2, 5), dtype=torch.int32)),
    lambda a, b: a.attend_sparse(0, b, rows(3, 512), 4, chosen=torch.zeros((3, 2, 4), dtype=torch.int64))])
def test_bad_rows_raise_before_the_library(call):
    with pytest.raises(ValueError):
        call(*detached())


def test_good_rows_reach_the_absent_cache():
    a, b = detached()
    for call in (lambda: a.attend(0, b, rows(3, 512)), lambda: a.attend(0, b, rows(4, 700)[:, 100:612]),
                 lambda: a.append(0, b, rows(3, 512), rows(3, 128), rows(3, 128)), lambda: b.set([1], [1], [[0]])):
        with pytest.raises(RuntimeError, match="destroyed"):
            call()


def test_python_mirror_checks_its_memory_and_raises_without_a_gpu():
    with pytest.raises(ValueError, match="dtype"):
        PagedAttention(1, 4, 16, 8, 2, 64, dtype="int8")
    k = torch.zeros((1, 4, 2, 16, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="together"):
        PagedAttention(1, 4, 16, 8, 2, 64, key_pages=k)
    with pytest.raises(ValueError, match="together"):
        PagedAttention(1, 4, 16, 8, 2, 64, key_pages=k, val_pages=k, key_scales=torch.zeros(4, 2))
    with pytest.raises(ValueError, match="shape"):
        PagedAttention(1, 4, 16, 8, 2, 64, key_pages=k[:, :3], val_pages=k)
    with pytest.raises(ValueError, match="GPU"):
        PagedAttention(1, 4, 16, 8, 2, 64, key_pages=k, val_pages=k)
    with pytest.raises(ValueError, match="float16"):
        PagedAttention(1, 4, 16, 8, 2, 64, key_pages=k.float(), val_pages=k)
    if not torch.cuda.is_available():
        with pytest.raises(PQAError):
            PagedAttention(1, 4, 16, 8, 2, 64)


def test_batch_arrays_are_checked():
    from picolm_qwen_amd.paged import _int_array
    for bad in ([1.5], np.array([1.0]), [2**31], [-2**31 - 1], ["a"]):
        with pytest.raises(ValueError):
            _int_array(bad, "n_new")
    assert _int_array([], "n_new").dtype == np.int32 and _int_array(np.array([3], np.uint8), "n_new").tolist() == [3]
