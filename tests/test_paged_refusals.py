"""What the operators of a serving loop over the paged cache refuse, checked on the host before anything is launched (no GPU
needed: the handles describe host memory as device memory, and every call here ends at a check)."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def call(pkg):
    def run(name, args, order, *numbers):
        d = pkg.diopi
        held = []
        for key in order:
            if args[key] is None:
                held.append((None, ctypes.c_void_p(None)))
                continue
            h = d.Handle(args[key])
            h.desc.device = d.DIOPI_DEVICE
            held.append((h, h.ptr))
        with d.Context(0) as ctx:
            d.call(name, ctx, *[p for _, p in held], *numbers)
    return run


CHUNK = ("diopiPagedContextAttentionInference", ("out", "q", "k", "v", "b_loc", "start", "new", "lens"))
WINDOW = ("diopiTokenDecodeAttentionWindowInference", ("out", "q", "k", "v", "b_loc", "start", "lens"))
APPEND = ("diopiRotaryDestIndexCopyKVPair", ("out_q", "q", "out_k", "k", "out_v", "v", "cos", "sin", "pos", "dest"))


def chunk(**changes):
    two = torch.ones(2, dtype=torch.int32)
    args = dict(q=torch.zeros(3, 4, 64), out=torch.zeros(3, 4, 64), k=torch.zeros(6, 2, 64), v=torch.zeros(6, 2, 64), b_loc=torch.zeros(2, 5, dtype=torch.int32), start=two, new=two, lens=two)
    return dict(args, **changes)


@pytest.mark.parametrize("changes,says", [
    (dict(q=None), "q must be"), (dict(k=None), "k and v must be"), (dict(v=None), "k and v must be"), (dict(out=None), "out must have"), (dict(b_loc=None), "b_loc must be"),
    (dict(start=None), "b_start_loc is null"), (dict(new=None), "b_new_len is null"), (dict(lens=None), "b_seq_len is null"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float64)), "unsupported dtype"), (dict(q=torch.zeros(3, 256)), "q must be"),
    (dict(out=torch.zeros(3, 64, 4)), "out must have"), (dict(out=torch.zeros(3, 4, 64).half()), "out must have"),
    (dict(k=torch.zeros(6, 2, 64).half()), "k and v are"), (dict(v=torch.zeros(5, 2, 64)), "differ at dim 0"), (dict(v=torch.zeros(6, 1, 64)), "differ at dim 1"),
    (dict(k=torch.zeros(6, 3, 64), v=torch.zeros(6, 3, 64)), "multiple"), (dict(k=torch.zeros(6, 2, 32), v=torch.zeros(6, 2, 32)), "mismatch"),
    (dict(k=torch.zeros(0, 2, 64), v=torch.zeros(0, 2, 64)), "no slots"), (dict(k=torch.zeros(6, 0, 64), v=torch.zeros(6, 0, 64)), "multiple"),
    (dict(k=torch.zeros(6, 64, 2).transpose(1, 2)), "contiguous"), (dict(out=torch.zeros(3, 4, 128)[..., ::2]), "contiguous"),
    (dict(b_loc=torch.zeros(2, 4, dtype=torch.int32)), "columns"), (dict(b_loc=torch.zeros(2, 5)), "int32 or int64"), (dict(b_loc=torch.zeros(5, 2, dtype=torch.int32).t()), "contiguous last dim"),
    (dict(b_loc=torch.zeros(10, dtype=torch.int32)), "b_loc must be"), (dict(lens=torch.zeros(3, dtype=torch.int32)), "2 entries"), (dict(new=torch.zeros(2)), "int32 or int64"),
    (dict(start=torch.zeros(4, dtype=torch.int32)[::2]), "dense"),
    (dict(q=torch.zeros(3, 4, 1040), out=torch.zeros(3, 4, 1040), k=torch.zeros(6, 2, 1040), v=torch.zeros(6, 2, 1040)), "exceeds 1024"),
])
def test_new_tokens(pkg, call, changes, says):
    with pytest.raises(pkg.diopi.DiopiError, match=says):
        call(CHUNK[0], chunk(**changes), CHUNK[1], 2, 5, 0, 0)


@pytest.mark.parametrize("numbers,says", [((-1, 5, 0, 0), "max_new_len is -1"), ((2, -1, 0, 0), "max_input_len -1"), ((2, 5, -1, 0), "window of -1"), ((2, 5, 3, -4), "-4 first ones")])
def test_numbers_of_new_tokens(pkg, call, numbers, says):
    with pytest.raises(pkg.diopi.DiopiError, match=says):
        call(CHUNK[0], chunk(), CHUNK[1], *numbers)


def test_longer_sequences_than_32_bits_hold(pkg, call):
    wide = torch.empty(1, 2 ** 30 + 1, dtype=torch.int32).expand(2, -1)         # (never touched)
    for name, order, numbers in ((*CHUNK, (2, 2 ** 30 + 1, 0, 0)), (*WINDOW, (2 ** 30 + 1, 3, 0))):
        args = chunk(b_loc=wide)
        if name == WINDOW[0]:
            args = dict(args, q=torch.zeros(2, 4, 64), out=torch.zeros(2, 4, 64))
        with pytest.raises(pkg.diopi.DiopiError, match="exceed 2"):
            call(name, args, order, *numbers)


@pytest.mark.parametrize("changes,says", [
    (dict(q=None), "q must be"), (dict(k=None), "k/v must be"), (dict(v=None), "bad v"), (dict(out=None), "out must be"), (dict(b_loc=None), "b_loc is null"),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.float64)), "dtype"), (dict(out=torch.zeros(2, 64, 4)), "shaped like q"), (dict(out=torch.zeros(2, 4, 128)[..., :64]), "dense"),
    (dict(k=torch.zeros(6, 3, 64), v=torch.zeros(6, 3, 64)), "multiple"), (dict(k=torch.zeros(0, 2, 64), v=torch.zeros(0, 2, 64)), "no slots"),
    (dict(b_loc=torch.zeros(2, 4, dtype=torch.int32)), "columns"), (dict(lens=torch.zeros(3, dtype=torch.int32)), "entries"),
    (dict(q=torch.zeros(2, 4, 1040), out=torch.zeros(2, 4, 1040), k=torch.zeros(6, 2, 1040), v=torch.zeros(6, 2, 1040)), "exceeds 1024"),
])
def test_single_tokens(pkg, call, changes, says):
    args = chunk(q=torch.zeros(2, 4, 64), out=torch.zeros(2, 4, 64))
    with pytest.raises(pkg.diopi.DiopiError, match=says):
        call(WINDOW[0], dict(args, **changes), WINDOW[1], 5, 3, 0)
    for numbers, says in (((-1, 3, 0), "columns"), ((5, -3, 0), "window of -3"), ((5, 3, -1), "-1 first ones")):
        with pytest.raises(pkg.diopi.DiopiError, match=says):
            call(WINDOW[0], args, WINDOW[1], *numbers)


@pytest.mark.parametrize("changes,says", [
    (dict(k=None), "null tensor"), (dict(out_v=None), "null tensor"), (dict(cos=None), "null tensor"), (dict(dest=None), "null tensor"), (dict(out_q=None), "both"), (dict(q=None), "both"),
    (dict(k=torch.zeros(3, 128)), "three dims"), (dict(v=torch.zeros(3, 2, 64).half()), "v is float16"), (dict(q=torch.zeros(3, 4, 32), out_q=torch.zeros(3, 4, 32)), "head_dim of 32"),
    (dict(out_k=torch.zeros(6, 2, 128)[..., ::2]), "contiguous"), (dict(q=torch.zeros(3, 64, 4).transpose(1, 2)), "contiguous"), (dict(v=torch.zeros(2, 2, 64)), "differ at dim 0"),
    (dict(out_v=torch.zeros(7, 2, 64)), "differ at dim 0"), (dict(out_q=torch.zeros(3, 5, 64)), "differ at dim 1"), (dict(out_k=torch.zeros(6, 4, 64), out_v=torch.zeros(6, 4, 64)), "the pools 4"),
    (dict(q=torch.zeros(4, 4, 64), out_q=torch.zeros(4, 4, 64)), "q has 4 tokens"), (dict(dest=torch.zeros(3)), "int32 or int64"), (dict(dest=torch.zeros(4, dtype=torch.int32)), "3 tokens"),
    (dict(dest=torch.zeros(3, 1, dtype=torch.int32)), "one dim"), (dict(pos=torch.zeros(2, dtype=torch.int32)), "positions"), (dict(pos=torch.zeros(3)), "positions"),
    (dict(sin=torch.zeros(3, 64)), "alike"), (dict(cos=torch.zeros(3, 1, 32), sin=torch.zeros(3, 1, 32)), "alike"), (dict(cos=torch.zeros(3, 32).half(), sin=torch.zeros(3, 32).half()), "cos is float16"),
    (dict(cos=torch.zeros(3, 31), sin=torch.zeros(3, 31)), "neither"), (dict(cos=torch.zeros(2, 32), sin=torch.zeros(2, 32)), "divide"), (dict(cos=torch.zeros(0, 32), sin=torch.zeros(0, 32)), "divide"),
    (dict(out_k=torch.zeros(0, 2, 64), out_v=torch.zeros(0, 2, 64)), "no slots"),
])
def test_append(pkg, call, changes, says):
    args = dict(q=torch.zeros(3, 4, 64), out_q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), out_k=torch.zeros(6, 2, 64), out_v=torch.zeros(6, 2, 64),
                cos=torch.zeros(3, 32), sin=torch.zeros(3, 32), pos=None, dest=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(pkg.diopi.DiopiError, match=says):
        call(APPEND[0], dict(args, **changes), APPEND[1], True)


def test_head_sizes_and_types_of_the_append(pkg, call):
    def rows(d, dtype=torch.float32):
        z = torch.zeros(3, 2, d, dtype=dtype)
        return dict(q=z, out_q=z.clone(), k=z, v=z, out_k=z.clone(), out_v=z.clone(), cos=torch.zeros(3, d // 2), sin=torch.zeros(3, d // 2), pos=None, dest=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(pkg.diopi.DiopiError, match="odd"):
        call(APPEND[0], rows(63), APPEND[1], True)
    with pytest.raises(pkg.diopi.DiopiError, match="unsupported dtype float64"):
        call(APPEND[0], rows(64, torch.float64), APPEND[1], True)
