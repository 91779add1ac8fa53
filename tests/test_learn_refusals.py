"""What the calls that learn from clicks refuse. Every argument is checked before the context is looked at, so the
refusals show without a GPU: a call whose other arguments are in order is refused for its null context alone."""
import pytest

from search_engine_amd import abi

P = 1 << 20  # stands for a device address; no call here gets as far as a device
F32, BF16, BIN1 = abi.VS_F32, abi.VS_BF16, abi.VS_BIN1

LOOKUP = dict(d_rows=P, dtype=F32, n_rows=10, row_stride=8, dim=8, d_ids=P, n_ids=4, d_offsets=P, n_bags=2, d_weights=P,
              scale=1.0, d_out=P, out_dtype=F32, out_stride=8, stream=None)
GRAD = dict(d_grad_out=P, dtype=F32, grad_out_stride=8, dim=8, d_ids=P, n_ids=4, d_offsets=P, n_bags=2, d_weights=P, scale=1.0,
            n_rows=10, d_workspace=P, workspace_bytes=1 << 30, d_grad_rows=P, grad_rows_dtype=F32, grad_rows_stride=8,
            d_unique_ids=P, d_n_unique=P, stream=None)
WEIGHTS = dict(d_rows=P, dtype=F32, n_rows=10, row_stride=8, dim=8, d_ids=P, n_ids=4, d_offsets=P, n_bags=2, scale=1.0,
               d_grad_out=P, grad_dtype=F32, grad_out_stride=8, d_grad_weights=P, stream=None)
XENT = dict(d_queries=P, n_q=3, query_stride=8, d_rows=P, n_rows=10, row_stride=8, dtype=F32, dim=8, d_targets=P, d_mask_words=P,
            scale=1.0, d_workspace=P, workspace_bytes=1 << 33, d_loss=P, d_lse=P, stream=None)
XENT_GRAD = dict(d_queries=P, n_q=3, query_stride=8, d_rows=P, n_rows=10, row_stride=8, dtype=F32, dim=8, d_targets=P,
                 d_mask_words=P, scale=1.0, d_loss=P, d_lse=P, d_grad_loss=P, d_workspace=P, workspace_bytes=1 << 33,
                 d_grad_queries=P, d_grad_rows=P, stream=None)
CALLS = {"vs_lookup_device": LOOKUP, "vs_lookup_grad_device": GRAD, "vs_lookup_grad_weights_device": WEIGHTS,
         "vs_xent_device": XENT, "vs_xent_grad_device": XENT_GRAD}


def refusal(name, **change):
    args = dict(CALLS[name], **change)
    code = getattr(abi.lib, name)(None, *args.values())
    with pytest.raises(abi.VsError) as e:
        abi._check(code)
    return e.value


@pytest.mark.parametrize("name", CALLS)
def test_arguments_in_order_reach_the_context(name):
    assert "null context" in refusal(name).message


NULLABLE = {"d_offsets", "d_weights", "d_mask_words", "d_grad_loss", "stream"}


@pytest.mark.parametrize("name,arg", [(n, a) for n, c in CALLS.items() for a, v in c.items() if v is P])
def test_null_buffers(name, arg):
    e = refusal(name, **{arg: None})
    if arg in NULLABLE or (name == "vs_xent_grad_device" and arg in ("d_grad_queries", "d_grad_rows")):
        assert "null context" in e.message
    else:
        assert e.code == abi.VS_E_INVALID_ARG and "null context" not in e.message, e.message


BAD = [("dim", 0), ("dim", abi.VS_LEARN_MAX_DIM + 1), ("dtype", BIN1), ("dtype", -1), ("out_dtype", BIN1), ("grad_dtype", 7),
       ("grad_rows_dtype", BIN1), ("row_stride", 7), ("out_stride", 7), ("grad_out_stride", 7), ("grad_rows_stride", 0),
       ("query_stride", 7), ("row_stride", 1 << 62), ("n_rows", 0), ("n_rows", 0xFFFFFFFF), ("n_rows", 1 << 40),
       ("n_ids", abi.VS_LOOKUP_MAX_IDS + 1), ("n_bags", abi.VS_LOOKUP_MAX_IDS + 1), ("n_q", abi.VS_XENT_MAX_QUERIES + 1),
       ("d_rows", P + 2), ("d_out", P + 1), ("d_grad_out", P + 3), ("d_queries", P + 2), ("d_grad_rows", P + 1),
       ("d_grad_queries", P + 2)]


@pytest.mark.parametrize("name,arg,value", [(n, a, v) for n, c in CALLS.items() for a, v in BAD if a in c])
def test_values_out_of_range(name, arg, value):
    e = refusal(name, **{arg: value})
    assert e.code == abi.VS_E_INVALID_ARG and "null context" not in e.message, e.message


@pytest.mark.parametrize("name", ["vs_lookup_grad_device", "vs_xent_device", "vs_xent_grad_device"])
def test_workspace_too_small(name):
    e = refusal(name, workspace_bytes=64)
    assert e.code == abi.VS_E_CAPACITY and "workspace" in e.message


def test_unique_ids_and_their_number_come_together():
    assert "null context" not in refusal("vs_lookup_grad_device", d_unique_ids=None).message
    assert "null context" not in refusal("vs_lookup_grad_device", d_n_unique=None).message
    assert "null context" in refusal("vs_lookup_grad_device", d_unique_ids=None, d_n_unique=None).message


def test_workspace_questions():
    import ctypes
    n = ctypes.c_uint64(0)
    for args, part in (((None, 1, 0, 8, F32), "rows"), ((None, 1, 10, 0, F32), "dimension"), ((None, 1, 10, 8, BIN1), "type"),
                       ((None, abi.VS_XENT_MAX_QUERIES + 1, 10, 8, F32), "n_q"), ((None, 1, 10, 8, F32), "null context")):
        code = abi.lib.vs_xent_workspace_bytes(*args, ctypes.byref(n))
        with pytest.raises(abi.VsError) as e:
            abi._check(code)
        assert part in e.value.message
    for args, part in (((None, 1, 0, 8), "rows"), ((None, 1, 10, 0), "dimension"),
                       ((None, abi.VS_LOOKUP_MAX_IDS + 1, 10, 8), "ids"), ((None, 1, 10, 8), "null context")):
        code = abi.lib.vs_lookup_grad_workspace_bytes(*args, ctypes.byref(n))
        with pytest.raises(abi.VsError) as e:
            abi._check(code)
        assert part in e.value.message


def test_store_calls_refuse_a_null_store():
    for name, n in (("vs_store_lookup_device", 10), ("vs_store_xent_device", 11), ("vs_store_xent_grad_device", 13)):
        f = getattr(abi.lib, name)
        args = [0 if t not in (abi._vp,) else None for t in f.argtypes]
        assert f(*args) == abi.VS_E_INVALID_ARG
