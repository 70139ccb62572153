"""Arguments that the operators of tree verification and block-sparse decode refuse before any CUDA call, and the host part."""
import ctypes

import numpy as np
import pytest
import torch

NULL, ONE, F = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_float(0.0625)


@pytest.fixture(scope="module")
def lib(q27):
    lib = ctypes.CDLL(q27.LIB_PATH)
    lib.q27b_last_error.restype = ctypes.c_char_p
    return lib


# per entry point: pointer arguments ("p": required, "?": optional; the output of attention is o or (xq, xd)), then its numbers
CALLS = {
    "attn_decode_tree": (["qn", "qg", "kc", "vc", "o", "xq?", "xd?", "pos0", "mask"],
                         dict(T=8, scale=F, nqh=24, nkvh=4, n_ctx=1000, q8=1)),
    "attn_decode_tree_paged": (["qn", "qg", "kp", "vp", "table", "lens", "mask", "o", "xq?", "xd?"],
                               dict(B=3, T=8, scale=F, nqh=24, nkvh=4, n_pages=10, max_pages=4, max_seq_len=1000)),
    "kv_commit": (["kc", "vc", "pos0", "path", "count"], dict(T=8, nkvh=4, n_ctx=1000, q8=1)),
    "kv_commit_paged": (["kp", "vp", "table", "lens", "path", "count"], dict(B=3, T=8, nkvh=4, n_pages=10, max_pages=4)),
    "kv_bounds": (["kc", "bounds", "pos0"], dict(T=8, nkvh=4, n_ctx=1000, q8=1)),
    "kv_bounds_paged": (["kp", "bounds", "table", "lens"], dict(B=3, T=8, nkvh=4, n_pages=10, max_pages=4)),
    "select_blocks": (["qn", "bounds", "sel", "pos0"], dict(T=4, k=8, n_sink=1, n_recent=2, nqh=24, nkvh=4, n_ctx=1000)),
    "select_blocks_paged": (["qn", "bounds", "sel", "table", "lens"],
                            dict(B=3, T=4, k=8, n_sink=1, n_recent=2, nqh=24, nkvh=4, n_pages=10, max_pages=4, max_seq_len=1000)),
    "attn_decode_blocks": (["qn", "qg", "kc", "vc", "o", "xq?", "xd?", "pos0", "sel"],
                           dict(T=4, k=8, scale=F, nqh=24, nkvh=4, n_ctx=1000, q8=1)),
    "attn_decode_blocks_paged": (["qn", "qg", "kp", "vp", "table", "lens", "sel", "o", "xq?", "xd?"],
                                 dict(B=3, T=4, k=8, scale=F, nqh=24, nkvh=4, n_pages=10, max_pages=4)),
}
BAD = {
    "T": (0, -1, 65, 5), "B": (0, -1, 65536), "nkvh": (0, -1, 2 ** 20), "nqh": (0, 23, 25), "n_ctx": (0, -5, 2 ** 31 - 1),
    "n_pages": (0, -1, 2 ** 24), "max_pages": (0, -1, 2 ** 23), "max_seq_len": (0, 3, 4 * 256 + 1), "k": (0, -1, 16385, 2),
    "n_sink": (-1, 7, 9), "n_recent": (0, -1, 8, 2 ** 31 - 1),
}


def call(lib, name, pointers=None, **changed):
    ptrs, nums = CALLS[name]
    nums = dict(nums, **changed)
    args = [(pointers or {}).get(p.rstrip("?"), NULL if p.endswith("?") else ONE) for p in ptrs]
    return getattr(lib, "q27b_" + name)(*args, *nums.values(), NULL)


@pytest.mark.parametrize("name", CALLS)
def test_bad_shapes_are_refused(q27, lib, name):
    _, nums = CALLS[name]
    for key, values in BAD.items():
        if key not in nums:
            continue
        for v in values:
            if key == "T" and ("bounds" in name and v > 0 or v == 5 and nums["T"] == 8):
                continue  # bounds take any number of rows that the cache has, trees up to 64
            if key == "k" and v == 2 and "select" not in name:
                continue  # (less than n_sink + n_recent)
            assert call(lib, name, **{key: v}) == q27.BAD_SHAPE, (key, v)
            assert ("%s: bad shape" % name).encode() in lib.q27b_last_error()


def test_more_rows_than_the_cache_has(q27, lib):
    assert call(lib, "kv_bounds", T=1001) == q27.BAD_SHAPE
    assert call(lib, "kv_bounds_paged", T=1025) == q27.BAD_SHAPE
    assert call(lib, "attn_decode_tree", T=8, n_ctx=7) == q27.BAD_SHAPE
    assert call(lib, "attn_decode_tree_paged", B=8192, T=8) == q27.BAD_SHAPE
    assert call(lib, "select_blocks", n_ctx=2 ** 20 + 1) == q27.UNSUPPORTED
    assert call(lib, "select_blocks_paged", max_pages=4097, n_pages=5000, max_seq_len=2 ** 20 + 1) == q27.UNSUPPORTED
    assert b"1048576 positions" in lib.q27b_last_error()


@pytest.mark.parametrize("name", CALLS)
def test_null_pointers_are_refused(q27, lib, name):
    for p in CALLS[name][0]:
        if not p.endswith("?"):
            assert call(lib, name, {p: NULL}) == q27.BAD_SHAPE, p
            assert ("%s: null pointer" % name).encode() in lib.q27b_last_error()
    if "xq?" in CALLS[name][0]:
        assert call(lib, name, {"xq": ONE}) == q27.BAD_SHAPE  # without xd


@pytest.mark.parametrize("name", CALLS)
def test_addresses_between_boundaries_are_refused(q27, lib, name):
    """The kernels load and store 16 bytes at a time."""
    wide = [p.rstrip("?") for p in CALLS[name][0] if p.rstrip("?") in ("qn", "qg", "kc", "vc", "kp", "vp", "o", "xq", "bounds")]
    if name.startswith("select"):
        wide.remove("qn")  # read value by value
    assert wide
    for p in wide:
        for off in (4, 8, 12):
            ptrs = {p: ctypes.c_void_p(16 + off)}
            if p == "xq":
                ptrs["xd"] = ONE
            assert call(lib, name, ptrs) == q27.BAD_SHAPE, p
            assert ("%s: pointers must be 16-byte aligned" % name).encode() in lib.q27b_last_error()


def test_sizes_of_the_bounds(q27):
    assert q27.kv_bounds_bytes(4, 1000) == 4 * 16 * 1024
    assert q27.kv_bounds_bytes(2, 64) == 2 * 1024 and q27.kv_bounds_bytes(2, 65) == 4 * 1024
    assert q27.kv_bounds_bytes(1, 2 ** 31 - 1) == 2 ** 25 * 1024
    assert q27.kv_bounds_pool_bytes(4, 10) == 10 * 4 * 4 * 1024
    assert q27.kv_bounds_bytes(0, 100) == q27.kv_bounds_bytes(4, -1) == q27.kv_bounds_pool_bytes(-1, 4) == 0


def test_tree_plan(q27):
    mask, depth = q27.tree_plan([-1, 0, 0, 1, -1, 4, 3])
    assert mask.dtype == np.int64 and depth.dtype == np.int32
    assert mask.tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000, 0b110000, 0b1001011]
    assert depth.tolist() == [0, 1, 1, 2, 0, 1, 3]
    mask, depth = q27.tree_plan(list(range(-1, 63)))
    assert depth.tolist() == list(range(64)) and mask[63] == -1 and mask[62] == 2 ** 63 - 1
    for bad in ([], [0], [-1, 1], [-2], [-1, 0, 5], [-1] * 65):
        with pytest.raises(q27.Q27Error, match="tree_plan") as e:
            q27.tree_plan(bad)
        assert e.value.code == q27.BAD_SHAPE


@pytest.mark.parametrize("name", CALLS)
def test_python_layer_refuses_other_tensors(q27, name):
    """Tensors that are not on the GPU, None where a tensor is needed, a wrong number of arguments, numbers that are none."""
    ptrs, nums = CALLS[name]
    plain = [None if p.endswith("?") else 16 for p in ptrs]
    numbers = [0.0625 if n == "scale" else v for n, v in nums.items()]
    fn = getattr(q27, name)
    for i, p in enumerate(ptrs):
        args = list(plain)
        args[i] = torch.zeros(4)
        with pytest.raises(q27.Q27Error, match="contiguous CUDA tensors") as e:
            fn(*args, *numbers)
        assert e.value.code == q27.BAD_SHAPE
        if not p.endswith("?") and p != "o":
            args[i] = None
            with pytest.raises(q27.Q27Error, match="null tensor"):
                fn(*args, *numbers)
    with pytest.raises(TypeError):
        fn(*plain)
    for i in range(len(numbers)):
        if list(nums)[i] != "q8":
            with pytest.raises((TypeError, ValueError)):
                fn(*plain, *(numbers[:i] + ["x"] + numbers[i + 1:]))
