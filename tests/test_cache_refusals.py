"""What the operators around the paged cache refuse, checked on the host before anything is launched (no GPU needed: the
handles describe host memory as device memory, and every call here ends at a check)."""
import ctypes

import pytest
import torch


class Args(dict):
    def but(self, **changes):
        return Args(self, **changes)


@pytest.fixture(scope="module")
def call(pkg):
    def run(name, args, order, *numbers):
        d = pkg.diopi
        held = []
        for key in order:
            t = args[key]
            if t is None:
                held.append((None, ctypes.c_void_p(None)))
                continue
            h = d.Handle(t)
            h.desc.device = d.DIOPI_DEVICE
            held.append((h, h.ptr))
        with d.Context(0) as ctx:
            d.call(name, ctx, *[p for _, p in held], *numbers)
    return run


def pools(slots=6, heads=2, d=64):
    return dict(kp=torch.zeros(slots, heads, d, dtype=torch.int8), ks=torch.zeros(slots, heads), vp=torch.zeros(slots, heads, d, dtype=torch.int8), vs=torch.zeros(slots, heads))


WRITE = ("diopiDestIndexCopyKVPairInt8", ("kp", "ks", "k", "vp", "vs", "v", "loc"))
READ = ("diopiIndexSelectKVPairInt8", ("k", "v", "kp", "ks", "vp", "vs", "loc"))
INT8 = ("diopiTokenDecodeAttentionInt8Inference", ("out", "q", "kp", "ks", "vp", "vs", "b_loc", "start", "lens"))
PREFIX = ("diopiTokenDecodeAttentionSharedPrefixInference", ("out", "q", "k", "v", "prefix", "b_loc", "start", "lens"))


@pytest.mark.parametrize("name,order", [WRITE, READ])
@pytest.mark.parametrize("changes,says", [
    (dict(k=None), "null"), (dict(ks=None), "null"), (dict(loc=None), "one dim"),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.float64), v=torch.zeros(3, 2, 64, dtype=torch.float64)), "float64"),
    (dict(v=torch.zeros(3, 2, 64).bfloat16()), "v rows are|v rows bfloat16"),
    (dict(v=torch.zeros(2, 2, 64)), "differ|slots for"),
    (dict(kp=torch.zeros(6, 2, 64)), "int8"), (dict(ks=torch.zeros(6, 2).half()), "float32"),
    (dict(ks=torch.zeros(6, 2, 1)), "scales"), (dict(vs=torch.zeros(5, 2)), "scales"),
    (dict(k=torch.zeros(3, 4, 64), v=torch.zeros(3, 4, 64)), "those of the pool"),
    (dict(k=torch.zeros(3, 128)), "kv_heads, head_dim"),
    (dict(vp=torch.zeros(7, 2, 64, dtype=torch.int8), vs=torch.zeros(7, 2)), "differ"),
    (dict(k=torch.zeros(3, 2, 128)[..., ::2]), "contiguous"), (dict(vp=torch.zeros(6, 64, 2, dtype=torch.int8).transpose(1, 2)), "contiguous"),
    (dict(loc=torch.zeros(3, dtype=torch.int16)), "int32 or int64"), (dict(loc=torch.zeros(4, dtype=torch.int32)), "slots for"),
    (dict(loc=torch.zeros(3, 1, dtype=torch.int32)), "one dim"),
    (pools(0), "no slots"),
])
def test_cache_rows(pkg, call, name, order, changes, says):
    args = Args(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), loc=torch.zeros(3, dtype=torch.int32), **pools())
    with pytest.raises(pkg.diopi.DiopiError, match=says):
        call(name, args.but(**changes), order)


@pytest.mark.parametrize("changes,says", [
    (dict(q=None), "q must be"), (dict(kp=None), "k must be"), (dict(vs=None), "v must be"), (dict(out=None), "out must be"), (dict(b_loc=None), "b_loc is null"),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.float64)), "unsupported dtype"),
    (dict(out=torch.zeros(2, 4, 64).half()), "out must be"), (dict(out=torch.zeros(2, 64, 4)), "shaped like q"),
    (dict(out=torch.zeros(2, 4, 128)[..., :64]), "dense"),
    (dict(kp=torch.zeros(6, 2, 64).half()), "int8"), (dict(vs=torch.zeros(6, 2).bfloat16()), "float32"), (dict(ks=torch.zeros(6, 1)), "scales of k"),
    (dict(kp=torch.zeros(6, 3, 64, dtype=torch.int8), ks=torch.zeros(6, 3)), "multiple"),
    (dict(kp=torch.zeros(6, 2, 32, dtype=torch.int8)), "mismatch"),
    (dict(vp=torch.zeros(5, 2, 64, dtype=torch.int8), vs=torch.zeros(5, 2)), "differ"),
    (dict(kp=torch.zeros(6, 64, 2, dtype=torch.int8).transpose(1, 2)), "contiguous"),
    (pools(0), "no slots"),
    (dict(b_loc=torch.zeros(2, 4, dtype=torch.int32)), "columns"), (dict(b_loc=torch.zeros(3, 5, dtype=torch.int32)), "b_loc must be"),
    (dict(b_loc=torch.zeros(2, 5)), "int32/int64"), (dict(lens=torch.zeros(3, dtype=torch.int32)), "entries"),
    (dict(q=torch.zeros(2, 4, 1040), out=torch.zeros(2, 4, 1040), **pools(6, 2, 1040)), "exceeds 1024"),
])
def test_int8_attention(pkg, call, changes, says):
    two = torch.ones(2, dtype=torch.int32)
    args = Args(q=torch.zeros(2, 4, 64), out=torch.zeros(2, 4, 64), b_loc=torch.zeros(2, 5, dtype=torch.int32), start=two, lens=two, **pools())
    with pytest.raises(pkg.diopi.DiopiError, match=says):
        call(INT8[0], args.but(**changes), INT8[1], 5)
    with pytest.raises(pkg.diopi.DiopiError, match="columns"):
        call(INT8[0], args, INT8[1], -1)


@pytest.mark.parametrize("changes,says", [
    (dict(q=None), "q must be"), (dict(k=None), "k/v must be"), (dict(v=None), "bad v"), (dict(prefix=None), "prefix_loc"), (dict(out=None), "out must be"),
    (dict(prefix=torch.zeros(3)), "int32 or int64"), (dict(prefix=torch.zeros(3, 1, dtype=torch.int32)), "one dim"),
    (dict(k=torch.zeros(6, 2, 64).half()), "differs from q"), (dict(v=torch.zeros(6, 2, 64).half()), "bad v"), (dict(v=torch.zeros(5, 2, 64)), "differ"),
    (dict(out=torch.zeros(2, 64, 4)), "shaped like q"), (dict(out=torch.zeros(2, 4, 64).half()), "out must be"),
    (dict(k=torch.zeros(6, 3, 64), v=torch.zeros(6, 3, 64)), "multiple"),
    (dict(k=torch.zeros(0, 2, 64), v=torch.zeros(0, 2, 64)), "no slots"),
    (dict(b_loc=torch.zeros(2, 4, dtype=torch.int32)), "columns"), (dict(lens=torch.zeros(1, dtype=torch.int32)), "entries"),
    (dict(prefix=torch.zeros(1, dtype=torch.int32).expand(2 ** 31)), "exceed 2"), (dict(prefix=torch.zeros(1, dtype=torch.int32).expand(2 ** 30 - 4)), "exceed 2"),
    (dict(q=torch.zeros(2, 4, 1040), out=torch.zeros(2, 4, 1040), k=torch.zeros(6, 2, 1040), v=torch.zeros(6, 2, 1040)), "exceeds 1024"),
])
def test_shared_prefix(pkg, call, changes, says):
    two = torch.ones(2, dtype=torch.int32)
    args = Args(q=torch.zeros(2, 4, 64), out=torch.zeros(2, 4, 64), k=torch.zeros(6, 2, 64), v=torch.zeros(6, 2, 64), prefix=torch.zeros(3, dtype=torch.int32),
                b_loc=torch.zeros(2, 5, dtype=torch.int32), start=two, lens=two)
    with pytest.raises(pkg.diopi.DiopiError, match=says):
        call(PREFIX[0], args.but(**changes), PREFIX[1], 5)


@pytest.mark.parametrize("name,order", [WRITE, READ])
def test_pools_of_too_many_slots(pkg, call, name, order):
    many = {key: t[:1].expand(2 ** 31, *t.shape[1:]) for key, t in pools().items()}
    args = Args(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), loc=torch.zeros(3, dtype=torch.int32), **many)
    with pytest.raises(pkg.diopi.DiopiError, match="2147483648 slots exceed"):
        call(name, args, order)


@pytest.mark.parametrize("name,order", [WRITE, READ])
def test_more_rows_than_a_launch_holds(pkg, call, name, order):
    rows = torch.zeros(1, 128, 1).expand(2 ** 24, 128, 1)
    with pytest.raises(pkg.diopi.DiopiError, match="16777216 rows of 128 heads exceed"):
        call(name, Args(k=rows, v=rows, loc=torch.zeros(1, dtype=torch.int32).expand(2 ** 24), **pools(6, 128, 1)), order)


def test_more_heads_than_a_launch_holds(pkg, call):
    one, batch = torch.ones(65535, dtype=torch.int32), 65535
    table = dict(b_loc=torch.zeros(batch, 1, dtype=torch.int32), start=one, lens=one)
    q = torch.zeros(1, 1, 16).bfloat16()
    args = Args(q=q.expand(batch, 1024, 16), out=torch.empty(batch, 1024, 16, dtype=torch.bfloat16), **table, **pools(6, 1024, 16))
    with pytest.raises(pkg.diopi.DiopiError, match="workgroups exceed"):
        call(INT8[0], args, INT8[1], 1)
    k = torch.zeros(6, 1, 16).bfloat16()
    args = Args(q=q.expand(batch, 300, 16), out=torch.empty(batch, 300, 16, dtype=torch.bfloat16), k=k, v=k, prefix=torch.zeros(3, dtype=torch.int32), **table)
    with pytest.raises(pkg.diopi.DiopiError, match="65535 sequences of 300 heads exceed"):
        call(PREFIX[0], args, PREFIX[1], 1)


def test_a_closed_context_and_host_tensors(pkg):
    d = pkg.diopi
    z = torch.zeros(3, 2, 64)
    ctx = d.Context(0)
    ctx.close()
    with pytest.raises(d.DiopiError, match="null diopiContext"):
        d.fn(WRITE[0])(None, *[ctypes.c_void_p(None)] * 7)
        d.raise_failure(WRITE[0], 1)
    with d.Context(0) as ctx, pytest.raises(d.DiopiError, match="lives on the host"):
        d.call(WRITE[0], ctx, *[d.Handle(z).ptr] * 7)
