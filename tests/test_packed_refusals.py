"""What the operators of a cache held in 4 bits refuse, without a GPU: the checks of the arguments alone."""

import pytest

from packed_plain import refusals


def test_refused_before_anything_is_launched(monkeypatch):
    from yalis_b200.ops import packed
    from yalis_b200.ops._lib import KernelError

    def launched():
        raise AssertionError("an argument that should have been refused reached the library")

    monkeypatch.setattr(packed, "_need_here", lambda *a: "cpu")
    monkeypatch.setattr(packed, "lib", launched)
    for what, call in refusals("cpu"):
        with pytest.raises(KernelError):
            call()
            pytest.fail(what)


def test_tensors_on_the_cpu_are_refused():
    import torch
    from packed_plain import Cache
    from yalis_b200.ops._lib import KernelError
    from yalis_b200.ops.packed import evict_tokens, packed_kv_write
    c = Cache([40], 2, 64, 16)
    pages, table = c.to("cpu")
    x, at = torch.zeros(1, 128), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(KernelError, match="GPU"):
        packed_kv_write(x, x, pages, at, at, table)
    with pytest.raises(KernelError, match="GPU"):
        evict_tokens(pages.pools(), c.sums, at, table, 4)


def test_argument_types_are_those_of_the_library():
    """The types that the wrappers set are those of the C entries' parameters, in order."""
    import glob
    import os
    import re

    from yalis_b200.ops import packed
    root = os.path.dirname(os.path.dirname(packed.__file__))
    entries = {}
    for path in glob.glob(os.path.join(root, "csrc", "*.cu")):
        for name, parameters in re.findall(r"YALIS_API [\w ]+?(\w+)\(([^)]*)\)", open(path).read()):
            kinds = ["p" if "*" in x or "cudaStream_t" in x else {"long": "l", "int64_t": "l", "float": "f"}.get(x.split()[0], "i") for x in parameters.split(",") if x.strip()]
            entries[name] = "".join(kinds)
    used = re.findall(r'_entry\("(\w+)", ((?:"[plif]*"(?: \+ )?)+)', open(packed.__file__).read())
    assert len(used) >= 6
    for name, signature in used:
        assert "".join(re.findall(r'"([plif]*)"', signature)) == entries[name], name


def test_options_of_a_packed_cache():
    from yalis_b200 import InferenceConfig
    from yalis_b200.cache.storage import group_page_bytes
    from yalis_b200.config.engine_config import EngineConfig
    from yalis_b200.parts.base import PagedKV
    for bad in (8, 2, True, "4"):
        with pytest.raises(ValueError, match="cache_bits"):
            EngineConfig(cache_bits=bad)
    assert InferenceConfig(cache_bits=4).engine_config("bf16").cache_bits == 4 and EngineConfig().cache_bits is None
    request = PagedKV(8, 128, packable=True)
    assert group_page_bytes([request], [None], 64, 2, 4) == {"kv_all": 8 * 64 * (128 + 4)}
    assert group_page_bytes([request], [None], 64, 2) == {"kv_all": 8 * 64 * 512}


def test_rotate_heads_refuses_cpu_tensors():
    import torch
    from yalis_b200.ops._lib import KernelError
    from yalis_b200.ops.elementwise import rotate_heads
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(KernelError):
        rotate_heads(torch.zeros(2, 64), i, i, None, 2, 16)
