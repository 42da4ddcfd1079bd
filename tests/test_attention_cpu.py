"""What the attention launchers refuse, checked before anything is launched, so that no GPU is
needed: the pointers below are never followed."""
import pytest

from futhark_amd import FutharkError, Kernels, heads

FA_EINVAL, FA_ENOTSUP, FA_ESCRATCH, FA_EALIGN = -1, -2, -3, -4
PTR = 1 << 20  # aligned, never followed


@pytest.fixture(scope="module")
def K():
    return Kernels()


def H(n, dim, data=PTR, row=None, head=None):
    return heads(data, n * dim if row is None else row, dim if head is None else head)


def attention_args(**w):
    a = dict(t="bf16", n=10, kn=10, h=4, hk=2, dim=64, m=2, scale=0.125, causal=1, seg=PTR, kseg=PTR, lse=PTR,
             q=None, k=None, v=None, out=None)
    a.update(w)
    q, k, v, out = (a[x] if a[x] is not None else H(a["h"] if x in ("q", "out") else a["hk"], a["dim"])
                    for x in ("q", "k", "v", "out"))
    return a, [None, a["t"], q, a["n"], k, v, a["kn"], a["h"], a["hk"], a["dim"], a["seg"], a["seg"],
               a["kseg"], a["kseg"], a["m"], a["scale"], a["causal"], out, a["lse"]]


def grad_args(ws=PTR, wb=1 << 30, grads=None, dout=None, **w):
    a, args = attention_args(**w)
    dq, dk, dv = grads or (H(a["h"], a["dim"]), H(a["hk"], a["dim"]), H(a["hk"], a["dim"]))
    return args + [dout or H(a["h"], a["dim"]), dq, dk, dv, ws, wb, None, 0]


def paged_args(**w):
    a = dict(t="f16", n=10, h=4, hk=2, dim=64, m=2, seg=PTR, past=PTR, scale=0.125, kp=PTR, vp=PTR, pages=8, page=16,
             table=PTR, cols=4, lse=None, ws=PTR, wb=1 << 40, q=None, out=None)
    a.update(w)
    q, out = (a[x] or H(a["h"], a["dim"]) for x in ("q", "out"))
    return [None, a["t"], q, a["n"], a["h"], a["hk"], a["dim"], a["seg"], a["seg"], a["m"], a["past"], a["scale"],
            a["kp"], a["vp"], a["pages"], a["page"], a["table"], a["cols"], out, a["lse"], a["ws"], a["wb"], None, 0]


def append_args(**w):
    a = dict(t="f16", n=10, h=4, hk=2, dim=64, m=2, seg=PTR, past=PTR, freqs=PTR, rot=64, kp=PTR, vp=PTR, pages=8,
             page=16, table=PTR, cols=4, q=None, qo=None, k=None, v=None)
    a.update(w)
    q, qo = (a[x] or H(a["h"], a["dim"]) for x in ("q", "qo"))
    k, v = (a[x] or H(a["hk"], a["dim"]) for x in ("k", "v"))
    return [None, a["t"], q, qo, k, v, a["n"], a["h"], a["hk"], a["dim"], a["seg"], a["seg"], a["m"], a["past"],
            a["freqs"], a["rot"], 0, a["kp"], a["vp"], a["pages"], a["page"], a["table"], a["cols"], None, 0]


def refused(call, args, code):
    with pytest.raises(FutharkError) as e:
        call(*args)
    assert e.value.code == code


SHAPES = [(dict(t="f32"), FA_ENOTSUP), (dict(t="i32"), FA_ENOTSUP), (dict(dim=0), FA_EINVAL),
          (dict(dim=-8), FA_EINVAL), (dict(dim=60), FA_ENOTSUP), (dict(dim=136), FA_ENOTSUP),
          (dict(h=0), FA_EINVAL), (dict(hk=0), FA_EINVAL), (dict(h=5, hk=2), FA_EINVAL),
          (dict(h=129, hk=1), FA_ENOTSUP), (dict(h=65536, hk=65536), FA_ENOTSUP), (dict(n=-1), FA_EINVAL),
          (dict(m=-1), FA_EINVAL), (dict(n=1 << 31), FA_ENOTSUP), (dict(m=1 << 31), FA_ENOTSUP),
          (dict(seg=None), FA_EINVAL), (dict(seg=PTR + 4), FA_EALIGN)]
STRIDES = [(dict(data=None), FA_EINVAL), (dict(data=PTR + 8), FA_EALIGN), (dict(row=-256), FA_EINVAL),
           (dict(head=-64), FA_EINVAL), (dict(row=260), FA_EALIGN), (dict(head=68), FA_EALIGN),
           (dict(row=1 << 61), FA_EINVAL)]
OVERLAP = [(dict(row=0), FA_EINVAL), (dict(head=0), FA_EINVAL), (dict(row=248), FA_EINVAL),
           (dict(head=56), FA_EINVAL), (dict(row=64, head=632), FA_EINVAL)]
SCALES = [(dict(scale=x), FA_EINVAL) for x in (0.0, -1.0, float("nan"), float("inf"))]
CACHE = [(dict(page=0), FA_EINVAL), (dict(page=-16), FA_EINVAL), (dict(page=24), FA_ENOTSUP),
         (dict(cols=-1), FA_EINVAL), (dict(cols=1 << 28), FA_ENOTSUP), (dict(pages=-1), FA_EINVAL),
         (dict(pages=1 << 31), FA_ENOTSUP), (dict(past=None), FA_EINVAL), (dict(table=None), FA_EINVAL),
         (dict(kp=None), FA_EINVAL), (dict(vp=None), FA_EINVAL), (dict(kp=PTR + 8), FA_EALIGN),
         (dict(vp=PTR + 2), FA_EALIGN), (dict(past=PTR + 4), FA_EALIGN), (dict(table=PTR + 2), FA_EALIGN)]


@pytest.mark.parametrize("w,code", SHAPES + SCALES + [(dict(kn=-1), FA_EINVAL), (dict(kn=1 << 31), FA_ENOTSUP),
                                                      (dict(kseg=None), FA_EINVAL), (dict(kseg=PTR + 4), FA_EALIGN),
                                                      (dict(lse=PTR + 2), FA_EALIGN)])
def test_attention_refuses(K, w, code):
    refused(K.attention, attention_args(**w)[1] + [None, 0], code)
    refused(K.attention_grad, grad_args(**w), code)


@pytest.mark.parametrize("which", ["q", "k", "v", "out"])
@pytest.mark.parametrize("w,code", STRIDES)
def test_attention_refuses_arrays(K, which, w, code):
    x = H(4, 64, **w)
    refused(K.attention, attention_args(hk=4, **{which: x})[1] + [None, 0], code)
    refused(K.attention_grad, grad_args(hk=4, **{which: x}), code)


@pytest.mark.parametrize("w,code", OVERLAP)
def test_written_arrays_do_not_overlap_themselves(K, w, code):
    x = H(4, 64, **w)
    refused(K.attention, attention_args(out=x)[1] + [None, 0], code)
    refused(K.attention_paged, paged_args(out=x), code)
    refused(K.kv_append, append_args(qo=x), code)
    ok = H(4, 64)
    for i in range(3):
        grads = [ok, ok, ok]
        grads[i] = x
        refused(K.attention_grad, grad_args(hk=4, grads=grads), code)


@pytest.mark.parametrize("scale,ok", [(2.358e38, True), (2.36e38, False), (3.4028234e38, False), (1e-45, True)])
def test_scales_whose_product_with_log2_e_is_not_finite(K, scale, ok):
    """A score of zero times an infinite factor would be NaN.  (What is taken is refused for its
    missing workspace, or has nothing to do.)"""
    if not ok:
        refused(K.attention, attention_args(scale=scale)[1] + [None, 0], FA_EINVAL)
        refused(K.attention, attention_args(n=0, kn=0, scale=scale)[1] + [None, 0], FA_EINVAL)
    else:
        K.attention(*attention_args(n=0, kn=0, scale=scale)[1], None, 0)
    refused(K.attention_grad, grad_args(ws=None, scale=scale), FA_ESCRATCH if ok else FA_EINVAL)
    refused(K.attention_paged, paged_args(n=1000, h=8, hk=8, m=1000, ws=None, scale=scale), FA_ESCRATCH if ok else FA_EINVAL)


def test_gradient_refuses_what_it_needs(K):
    refused(K.attention_grad, grad_args(lse=None), FA_EINVAL)
    refused(K.attention_grad, grad_args(dout=H(4, 64, data=None)), FA_EINVAL)
    need = K.attention_grad_workspace_bytes(10, 10, 4, 2, 64, 2)
    assert need > 0
    refused(K.attention_grad, grad_args(wb=need - 1), FA_ESCRATCH)
    refused(K.attention_grad, grad_args(ws=None), FA_ESCRATCH)
    refused(K.attention_grad, grad_args(ws=PTR + 8), FA_EALIGN)


@pytest.mark.parametrize("w,code", SHAPES + CACHE)
def test_cache_operators_refuse(K, w, code):
    refused(K.attention_paged, paged_args(**w), code)
    refused(K.kv_append, append_args(**w), code)


@pytest.mark.parametrize("w,code", SCALES + [(dict(lse=PTR + 2), FA_EALIGN)])
def test_paged_attention_refuses(K, w, code):
    refused(K.attention_paged, paged_args(**w), code)


@pytest.mark.parametrize("w,code", STRIDES)
def test_cache_operators_refuse_arrays(K, w, code):
    x = H(4, 64, **w)
    refused(K.attention_paged, paged_args(q=x), code)
    refused(K.attention_paged, paged_args(out=x), code)
    for which in ("q", "qo", "k", "v"):
        refused(K.kv_append, append_args(hk=4, **{which: x}), code)


@pytest.mark.parametrize("w,code", [(dict(rot=-2), FA_EINVAL), (dict(rot=3), FA_EINVAL), (dict(rot=66), FA_EINVAL),
                                    (dict(freqs=None), FA_EINVAL), (dict(freqs=PTR + 2), FA_EALIGN)])
def test_append_refuses(K, w, code):
    refused(K.kv_append, append_args(**w), code)


def test_paged_workspace(K):
    """A long cache and few rows need one; too small a one is refused."""
    sizes = (1, 8, 1, 128, 1, 16, 1 << 16)
    need = K.attention_paged_workspace_bytes(*sizes)
    if need:
        w = dict(n=1, h=8, hk=1, dim=128, m=1, page=16, cols=1 << 16)
        refused(K.attention_paged, paged_args(wb=need - 1, **w), FA_ESCRATCH)
        refused(K.attention_paged, paged_args(ws=None, **w), FA_ESCRATCH)
        refused(K.attention_paged, paged_args(ws=PTR + 8, **w), FA_EALIGN)
    assert K.attention_paged_workspace_bytes(0, 8, 1, 128, 0, 16, 4) == 0


def test_nothing_to_do_is_no_error(K):
    K.attention(*attention_args(n=0, kn=0)[1], None, 0)
    K.attention(*attention_args(m=0, seg=None, kseg=None)[1], None, 0)
    K.attention_grad(*grad_args(n=0, kn=0))
    K.attention_grad(*grad_args(m=0, seg=None, kseg=None))
    K.attention_paged(*paged_args(n=0))
    K.attention_paged(*paged_args(m=0, seg=None))
    K.kv_append(*append_args(n=0))
    K.kv_append(*append_args(m=0, seg=None))


def test_a_table_without_columns_needs_the_same_workspace(K):
    """Sequences that hold nothing make the launcher's choice between its ways no other: 1000 of them
    go the way that writes a workspace."""
    need = K.attention_paged_workspace_bytes(1000, 8, 8, 64, 1000, 16, 0)
    assert need == K.attention_paged_workspace_bytes(1000, 8, 8, 64, 1000, 16, 4) > 0
    refused(K.attention_paged, paged_args(n=1000, h=8, hk=8, m=1000, cols=0, table=None, ws=None, wb=0), FA_ESCRATCH)


def test_limits_of_strides_and_launches(K):
    """A row stride of 2^27 elements, more heads than a launch numbers, more blocks than it has."""
    for row, code in ((1 << 27, FA_ENOTSUP), ((1 << 27) + 4, FA_EALIGN)):
        x = H(4, 64, row=row)
        for which in ("q", "k", "v", "out"):
            refused(K.attention, attention_args(hk=4, **{which: x})[1] + [None, 0], code)
            refused(K.attention_grad, grad_args(hk=4, **{which: x}), code)
        for which in ("q", "out"):
            refused(K.attention_paged, paged_args(**{which: x}), code)
        for which in ("q", "qo", "k", "v"):
            refused(K.kv_append, append_args(hk=4, **{which: x}), code)
    most = (1 << 31) - 4096
    many = dict(n=most, kn=most, h=64, hk=64)
    refused(K.attention, attention_args(**many)[1] + [None, 0], FA_ENOTSUP)
    refused(K.attention_grad, grad_args(wb=1 << 62, **many), FA_ENOTSUP)
    many.pop("kn")
    refused(K.attention_paged, paged_args(wb=1 << 62, **many), FA_ENOTSUP)       # many rows a sequence
    refused(K.attention_paged, paged_args(wb=1 << 62, m=most, **many), FA_ENOTSUP)  # one row a sequence
    refused(K.kv_append, append_args(n=1 << 24), FA_ENOTSUP)


def test_version_tells_of_these_launchers(K):
    assert K.lib.fa_version() >= 1003


@pytest.mark.parametrize("h,hk,dim,keys", [(16, 4, 64, 1536), (32, 8, 128, 1024), (128, 2, 128, 16)])
def test_what_takes_one_launch_needs_no_workspace(K, h, hk, dim, keys):
    """Four short sequences of a token each: a block a unit, whose parts meet in LDS.  With one more
    column the keys are cut over all waves, and parts go through the workspace."""
    assert K.attention_paged_workspace_bytes(4, h, hk, dim, 4, 16, keys // 16) == 0
    need = K.attention_paged_workspace_bytes(4, h, hk, dim, 4, 16, 1537 // 16 + 1)
    assert need > 0
    refused(K.attention_paged, paged_args(n=4, h=h, hk=hk, dim=dim, m=4, cols=97, wb=need - 1), FA_ESCRATCH)
    refused(K.attention_paged, paged_args(n=4, h=h, hk=hk, dim=dim, m=4, cols=97, ws=None, wb=0), FA_ESCRATCH)


def test_long_table_needs_a_workspace(K):
    assert K.attention_paged_workspace_bytes(1, 8, 1, 128, 1, 16, 1 << 16) > 0
