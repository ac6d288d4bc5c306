"""GPU: rotary positions, the paged 4-bit cache and the attention over it
against float64 numpy (tests/kv4_oracle.py).

Tolerances, with u = 2^-24 (half a step of fp32) and h = half a step of the
output type (relative to the value):
 * rope, in fp32 from 64-bit angles: the cosine and sine are rounded once, then
   a product and a fused or separate sum: |error| <= 3.1 u m (|x1| + |x2|) before
   the output's rounding, h |y|, and the smallest subnormal's half.
 * append: codes and scales are those of the exact value, so rows read back
   in fp32 are equal to the oracle's.
 * attention: a score is a sum of head_dim products of fp32 operands (q held to
   at least 22 bits, codes exact, bf16 scales exact), scaled twice: off by at
   most e = (hd + 8) 2^-22 scale sum_c |q_c| |k|_max(c), k bounded by 15 scales
   because the stored codes carry a bias of 8. exp2 and its argument add
   2^-20 (|arguments that matter| <= 32). Weights held in fp16 (16-bit types)
   are off by 2^-11, in two fp16 terms by 2^-21, and multiply codes of at most
   15 with their bias taken off again (8): at most 23 scales. In all
   |out error| <= sum_j w_j (2 e + 2^-20 + r) 23 s_j + h |out|,
   r = 2^-11 or 2^-21, s_j the value group's scale.
"""
from __future__ import annotations

import numpy as np
import pytest

import kv4_oracle as ko

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def torch():
    import torch

    torch.zeros(1, device="cuda")
    return torch


def types(torch, rc, name):
    return {"f32": (torch.float32, rc.F32), "f16": (torch.float16, rc.F16),
            "bf16": (torch.bfloat16, rc.BF16)}[name]


def f64(t):
    return t.double().cpu().numpy()


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------- rope --
ROPES = [
    # dtype, tokens, heads, head_dim, rot, layout, far, row gap, element offset, in place
    ("f32", 1, 16, 128, 128, "interleaved", 255, 0, 0, False),
    ("f32", 5, 3, 128, 64, "half", 1 << 20, 0, 0, False),
    ("bf16", 257, 40, 128, 64, "half", 131072, 0, 0, False),
    ("f16", 33, 8, 80, 32, "half", 65536, 0, 0, False),
    ("bf16", 7, 5, 80, 40, "half", 5000, 0, 0, True),       # pairs 20 apart: no whole vectors
    ("f16", 9, 2, 96, 48, "interleaved", 5000, 0, 0, True),
    ("f32", 3, 1, 2, 2, "interleaved", 2 ** 31 - 1, 0, 0, False),
    ("f32", 4, 2, 6, 2, "half", 2 ** 31 - 1, 0, 0, False),
    ("bf16", 11, 3, 256, 256, "half", 1000, 24, 0, True),   # a row of a fused projection
    ("f16", 6, 4, 64, 64, "half", 1000, 5, 3, False),       # odd stride, odd address
    ("f32", 130, 2, 512, 512, "interleaved", 9000, 0, 1, False),
    ("f32", 2, 3, 1024, 512, "half", 9000, 4, 0, False),
    ("bf16", 1000, 1, 64, 64, "interleaved", 40000, 0, 0, True),
    ("bf16", 2, 3, 66, 66, "interleaved", 40000, 0, 0, False),
    ("f16", 19001, 1, 512, 512, "half", 100000, 0, 0, True),  # many tokens a CTA, the largest table
    ("f32", 5000, 2, 64, 32, "interleaved", 9000, 0, 0, False),
]


@pytest.mark.parametrize("dtype,T,heads,hd,rot,layout,far,gap,off,inplace", ROPES)
def test_rope(torch, rc, dtype, T, heads, hd, rot, layout, far, gap, off, inplace):
    dt, code = types(torch, rc, dtype)
    g = torch.Generator("cuda").manual_seed(T * 31 + hd)
    stride = heads * hd + gap
    buf = torch.randn(T * stride + off + 8, generator=g, device="cuda").to(dt)
    x = buf[off:off + T * stride].view(T, stride)
    src = f64(x)
    ybuf = buf if inplace else torch.full_like(buf, 7.0)
    y = ybuf[off:off + T * stride].view(T, stride)
    pos = torch.randint(0, far, (T,), generator=g, device="cuda").int()
    pos[0] = far
    rope = rc.Rope(hd, rot_dim=rot, layout=rc.ROPE_HALF if layout == "half" else rc.ROPE_INTERLEAVED,
                   magnitude=1.25)
    rope.apply_dev(code, x.data_ptr(), y.data_ptr(), pos.data_ptr(), T, heads, x_stride=stride,
                   y_stride=stride, stream=stream(torch))
    xs = src[:, :heads * hd].reshape(T, heads, hd)
    want = ko.rotate(xs, pos.cpu().numpy(), ko.freqs(rot), layout, 1.25)
    got = f64(y)
    gap_want = src[:, heads * hd:] if inplace else np.full((T, gap), 7.0)
    np.testing.assert_array_equal(got[:, heads * hd:], gap_want)  # between the rows: untouched
    np.testing.assert_array_equal(f64(ybuf[off + T * stride:]),
                                  f64(buf[off + T * stride:]) if inplace else 7.0)
    got = got[:, :heads * hd].reshape(T, heads, hd)
    np.testing.assert_array_equal(got[..., rot:], xs[..., rot:])
    a, b = ko.pair_channels(rot, layout)
    size = np.zeros_like(want)
    size[..., a] = size[..., b] = np.abs(xs[..., a]) + np.abs(xs[..., b])
    # 2^-50 of an angle below 2^31: the 64-bit angle of positions that far
    angle = 2.0 ** -50 * far
    bar = (3.1 * U + angle) * 1.25 * size + 1.01 * ko.HALF_STEP[dtype] * np.abs(want) + 2.0 ** -25
    assert (np.abs(got - want) <= bar).all()


def test_rope_scaled_negative_positions_and_nan(torch, rc):
    """Positions below zero turn the other way; a NaN stays in its pair."""
    T, hd = 3, 64
    rope = rc.Rope(hd, scaling=rc.ROPE_SCALE_YARN, factor=8.0, original_ctx=4096)
    x = torch.randn(T, 1, hd, device="cuda")
    x[1, 0, 10] = float("nan")
    y = torch.empty_like(x)
    pos = torch.tensor([-5, 5, 100000], dtype=torch.int32, device="cuda")
    rope.apply_dev(rc.F32, x.data_ptr(), y.data_ptr(), pos.data_ptr(), T, 1, stream=stream(torch))
    f = ko.freqs(hd, scaling="yarn", factor=8.0, low=1.0, high=32.0, ctx=4096)
    want = ko.rotate(f64(x), pos.cpu().numpy(), f, "interleaved", 1 + 0.1 * np.log(8.0))
    got = f64(y)
    bad = np.zeros_like(want, bool)
    bad[1, 0, 10:12] = True
    np.testing.assert_array_equal(np.isnan(got), bad)
    assert np.abs(got - want)[~bad].max() <= 2 * 3.1 * U * 1.25 * np.nanmax(np.abs(f64(x))) + 2.0 ** -24 * 8


# ----------------------------------------------------------------- append --
APPENDS = [
    # dtype, tokens, kv heads, head_dim, page, rope (rot, layout) or None, gap, offset
    ("f32", 1, 16, 128, 16, (128, "interleaved"), 0, 0),
    ("bf16", 64, 8, 128, 64, (128, "half"), 0, 0),
    ("f16", 77, 3, 80, 32, (32, "half"), 0, 0),
    ("bf16", 19, 2, 80, 16, (40, "half"), 0, 0),       # pairs 20 apart
    ("f32", 33, 1, 8, 16, (6, "interleaved"), 0, 0),   # the smallest head, a rotation that ends inside it
    ("f16", 50, 5, 256, 48, (256, "half"), 16, 0),     # rows of a fused projection
    ("bf16", 40, 2, 96, 128, (90, "half"), 3, 1),      # odd stride and address
    ("f32", 16, 4, 40, 16, None, 0, 0),
    ("bf16", 300, 1, 64, 1024, None, 0, 0),
    ("f16", 200, 7, 32, 16, (16, "interleaved"), 0, 0),
    ("f32", 70, 2, 160, 32, (160, "half"), 0, 0),
]


def filled(torch, rc, kv, rows, dtype="f32", layer=0):
    """Fill slots 0.. of `kv` with rows (k, v) [n, heads, hd]."""
    dt, code = types(torch, rc, dtype)
    k, v = (r.to(dt).contiguous() for r in rows)
    slots = torch.arange(k.shape[0], device="cuda")
    kv.append_dev(layer, code, k.data_ptr(), v.data_ptr(), slots.data_ptr(), k.shape[0],
                  stream=stream(torch))
    torch.cuda.synchronize()


def read(torch, rc, kv, slots, layer=0, dtype="f32", fill=0.0):
    dt, code = types(torch, rc, dtype)
    s = torch.as_tensor(slots, dtype=torch.int64, device="cuda")
    k, v = (torch.full((len(s), kv.n_kv_heads, kv.head_dim), fill, dtype=dt, device="cuda")
            for _ in "kv")
    kv.read_dev(layer, code, s.data_ptr(), len(s), k.data_ptr(), v.data_ptr(), stream=stream(torch))
    return f64(k), f64(v)


@pytest.mark.parametrize("dtype,T,nkv,hd,page,rp,gap,off", APPENDS)
def test_append(torch, rc, dtype, T, nkv, hd, page, rp, gap, off):
    dt, code = types(torch, rc, dtype)
    g = torch.Generator("cuda").manual_seed(T + hd)
    n_pages = -(-T // page) + 2
    kv = rc.Kv4(n_layers=2, n_kv_heads=nkv, head_dim=hd, page_size=page, n_pages=n_pages)
    assert kv.nbytes == 2 * n_pages * nkv * page * -(-hd // 32) * 36
    old = [torch.randn(n_pages * page, nkv, hd, generator=g, device="cuda") for _ in "kv"]
    for layer in range(2):
        filled(torch, rc, kv, old, layer=layer)
    stride = nkv * hd + gap
    bufs = [(torch.randn(T * stride + off, generator=g, device="cuda") * 3).to(dt) for _ in "kv"]
    k, v = (b[off:].view(T, stride)[:, :nkv * hd].unflatten(1, (nkv, hd)) for b in bufs)
    k[0, 0, :8] = 0  # zeros beside others
    v[T - 1, nkv - 1, :] = 0  # groups of zeros
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:T]
    slots[T // 2:T // 2 + T // 8] = -1
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device="cuda").int()
    rope = rp and rc.Rope(hd, rot_dim=rp[0], layout=rc.ROPE_HALF if rp[1] == "half" else rc.ROPE_INTERLEAVED,
                          magnitude=1.125)
    kv.append_dev(1, code, k.data_ptr(), v.data_ptr(), slots.data_ptr(), T, rope=rope,
                  d_positions=pos.data_ptr(), k_stride=stride, v_stride=stride, stream=stream(torch))
    kv.check(stream(torch))
    kx = f64(k)
    if rp:
        kx = ko.rotate(kx, pos.cpu().numpy(), ko.freqs(rp[0]), rp[1], 1.125)
    want = [ko.hold(f64(o).astype(np.float32).astype(np.float64))[0] for o in old]
    keep = slots.cpu().numpy() >= 0
    for w, new in zip(want, (kx, f64(v))):
        w[slots.cpu().numpy()[keep]] = ko.hold(new)[0][keep]
    every = np.arange(n_pages * page)
    for got, w in zip(read(torch, rc, kv, every, layer=1), want):
        np.testing.assert_array_equal(got, w)
    for got, o in zip(read(torch, rc, kv, every, layer=0), old):  # the other layer: untouched
        np.testing.assert_array_equal(got, ko.hold(f64(o))[0])


def test_append_extremes_and_read_types(torch, rc):
    """The largest and smallest magnitudes, halves exactly between codes, and
    infinities and NaN, which stay in their group; rows read back in 16 bits
    are the rounded ones; rows of skipped slots stay."""
    hd = 64
    kv = rc.Kv4(n_layers=1, n_kv_heads=1, head_dim=hd, page_size=16, n_pages=2)
    x = torch.zeros(12, 1, hd)
    x[0, 0, :32] = torch.linspace(-3.4e38, 3.4e38, 32)
    x[1, 0, :32] = torch.linspace(-1e-40, 1e-40, 32)          # below the smallest normal
    x[2, 0, :32] = torch.linspace(-7, 7, 32)
    x[3, 0, :29] = torch.arange(-7, 7.5, 0.5)                 # scale 1: every half is a tie
    x[4, 0, 5] = float("inf")
    x[5, 0, 40] = float("nan")
    x[6, 0, 1] = float("-inf")
    x[7, 0, 0] = 1e-45
    x[8] = torch.randn(1, hd) * 1e-38
    x[9] = torch.randn(1, hd) * 1e37
    x[10, 0, 31], x[10, 0, 32] = 1.0, -1e-30
    x[11] = -0.0
    x = x.cuda()
    filled(torch, rc, kv, (x, x))
    want = ko.hold(f64(x))[0]
    for got in read(torch, rc, kv, range(12)):
        np.testing.assert_array_equal(got, want)
    for dtype in ("f16", "bf16"):
        dt = types(torch, rc, dtype)[0]
        for got in read(torch, rc, kv, [2, -1, 3, 10], dtype=dtype, fill=5.0):
            w = f64(torch.from_numpy(want[[2, 2, 3, 10]]).float().to(dt))
            w[1] = 5.0
            np.testing.assert_array_equal(got, w)


def test_slots_out_of_range_are_reported_and_skipped(torch, rc):
    kv = rc.Kv4(n_layers=1, n_kv_heads=2, head_dim=32, page_size=16, n_pages=2)
    x = torch.randn(3, 2, 32, device="cuda")
    slots = torch.tensor([31, 32, 1 << 40], device="cuda")
    kv.append_dev(0, rc.F32, x.data_ptr(), x.data_ptr(), slots.data_ptr(), 3, stream=stream(torch))
    with pytest.raises(rc.RabbitCudaError, match="slot") as e:
        kv.check(stream(torch))
    assert e.value.status == rc.ERR_ARGS
    kv.check(stream(torch))  # reported once
    k, _ = read(torch, rc, kv, [31, 32, 30], fill=9.0)
    with pytest.raises(rc.RabbitCudaError, match="slot"):
        kv.check(stream(torch))
    np.testing.assert_array_equal(k[0], ko.hold(f64(x))[0][0])
    assert (k[1] == 9.0).all() and (k[2] == 0).all()


def test_wrong_rope_layer_and_pointers_are_refused(torch, rc):
    kv = rc.Kv4(n_layers=1, n_kv_heads=1, head_dim=64, page_size=16, n_pages=1)
    x = torch.zeros(1, 1, 64, device="cuda")
    s = torch.zeros(1, dtype=torch.int64, device="cuda")
    p, sp = x.data_ptr(), s.data_ptr()
    ws = rc.Kv4Scratch(kv)
    b = rc.Kv4Batch(n_seqs=1, max_pages=1, d_kv_len=sp, d_page_table=sp)
    bad = [lambda: kv.append_dev(0, rc.F32, p, p, sp, 1, rope=rc.Rope(32), d_positions=sp),
           lambda: kv.append_dev(0, rc.F32, p, p, sp, 1, rope=rc.Rope(64)),
           lambda: kv.append_dev(1, rc.F32, p, p, sp, 1), lambda: kv.append_dev(-1, rc.F32, p, p, sp, 1),
           lambda: kv.append_dev(0, 7, p, p, sp, 1), lambda: kv.append_dev(0, rc.F32, 0, p, sp, 1),
           lambda: kv.append_dev(0, rc.F32, p, 0, sp, 1), lambda: kv.append_dev(0, rc.F32, p, p, 0, 1),
           lambda: kv.append_dev(0, rc.F32, p + 2, p, sp, 1),
           lambda: kv.append_dev(0, rc.F32, p, p, sp, 1, k_stride=32),
           lambda: kv.append_dev(0, rc.F32, p, p, sp + 4, 1), lambda: kv.append_dev(0, rc.F32, p, p, sp, -1),
           lambda: kv.read_dev(0, rc.F32, 0, 1, p, p), lambda: kv.read_dev(2, rc.F32, sp, 1, p, p),
           lambda: kv.read_dev(0, rc.F16, sp, 1, p + 1, p),
           lambda: kv.attention_dev(0, ws, rc.F32, p, p, 1, 1, b, window=-1),
           lambda: kv.attention_dev(0, ws, rc.F32, p, p, 1, 1, b, scale=float("nan")),
           lambda: kv.attention_dev(0, ws, 9, p, p, 1, 1, b), lambda: kv.attention_dev(3, ws, rc.F32, p, p, 1, 1, b),
           lambda: kv.attention_dev(0, ws, rc.F32, 0, p, 1, 1, b),
           lambda: kv.attention_dev(0, ws, rc.F32, p, p, 1, 0, b),
           lambda: kv.attention_dev(0, ws, rc.F32, p, p, 1, 1, b, q_stride=128),
           lambda: kv.attention_dev(0, ws, rc.F32, p, p, -1, 1, b),
           lambda: kv.attention_dev(0, ws, rc.F32, p, p, 1 << 16, 1 << 15, b),
           lambda: kv.attention_dev(0, ws, rc.F32, p, p, 1, 1, rc.Kv4Batch(n_seqs=1, d_kv_len=sp + 2)),
           lambda: kv.attention_dev(0, ws, rc.F32, p, p, 1, 1, rc.Kv4Batch(n_seqs=1, max_pages=1)),
           lambda: kv.attention_dev(0, ws, rc.F32, p, p, 1, 1, rc.Kv4Batch(n_seqs=-1, d_kv_len=sp))]
    for call in bad:
        with pytest.raises(rc.RabbitCudaError) as e:
            call()
        assert e.value.status == rc.ERR_ARGS
    two = rc.Kv4(n_layers=1, n_kv_heads=2, head_dim=32, page_size=16, n_pages=1)
    with pytest.raises(rc.RabbitCudaError):  # 3 query heads over 2
        two.attention_dev(0, rc.Kv4Scratch(two), rc.F32, p, p, 1, 3, b)
    kv.append_dev(0, rc.F32, 0, 0, 0, 0)  # nothing to do
    kv.attention_dev(0, ws, rc.F32, 0, 0, 0, 1, b)
    kv.check(stream(torch))


# -------------------------------------------------------------- attention --
class Case:
    """A filled cache with a shuffled page table, and the oracle over it. Slots
    behind each sequence's end, and pages of no sequence, hold NaN and
    infinities."""

    def __init__(self, torch, rc, *, dtype, nh, nkv, hd, page, lens, qs=None, window=0, scale=0.0,
                 pad=0, gap=0, off=0, seed=0, q_gain=1.0, max_pages=None, poison=True):
        self.torch, self.rc, self.dtype = torch, rc, dtype
        self.nh, self.nkv, self.hd, self.page, self.window = nh, nkv, hd, page, window
        self.lens, self.qs = lens, qs or [1] * len(lens)
        self.scale = scale
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + 2
        order = rng.permutation(n_pages)
        self.wide = max_pages or max(1, max(need))
        table = np.full((len(lens), self.wide), -1, np.int32)  # unused entries: no page
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        g = torch.Generator("cuda").manual_seed(seed + 1)
        k, v = (torch.randn(n_pages * page, nkv, hd, generator=g, device="cuda") * 2 for _ in "kv")
        k *= 1 + 3 * torch.rand(nkv, hd, generator=g, device="cuda").pow(8)
        v *= torch.randn(n_pages * page, 1, 1, generator=g, device="cuda").exp()
        used = np.zeros(n_pages * page, bool)
        self.slots = []
        for i, n in enumerate(lens):
            p = np.arange(n)
            s = table[i, p // page].astype(np.int64) * page + p % page if n else np.zeros(0, np.int64)
            used[s] = True
            self.slots.append(s)
        if poison:
            gone = torch.from_numpy(~used).cuda()
            k[gone], v[gone] = float("nan"), float("inf")
        self.kv = rc.Kv4(n_layers=1, n_kv_heads=nkv, head_dim=hd, page_size=page, n_pages=n_pages)
        filled(torch, rc, self.kv, (k, v))
        self.k, _ = ko.hold(f64(k))
        self.v, self.vs = ko.hold(f64(v))
        _, self.ks = ko.hold(f64(k))
        dt, self.code = types(torch, rc, dtype)
        self.rows = sum(self.qs)
        self.stride = nh * hd + gap
        self.qbuf = (torch.randn((self.rows + pad) * self.stride + off, generator=g, device="cuda") *
                     q_gain).to(dt)
        self.off, self.pad = off, pad
        self.table = torch.from_numpy(table).cuda()
        self.len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.start = torch.tensor(np.concatenate([[0], np.cumsum(self.qs)]), dtype=torch.int32,
                                  device="cuda")
        self.ws = rc.Kv4Scratch(self.kv)
        self.out = torch.full_like(self.qbuf, 7.0)

    def batch(self, one_each=False):
        return self.rc.Kv4Batch(n_seqs=len(self.lens), max_pages=self.wide, max_q_len=max(self.qs),
                                d_q_start=None if one_each else self.start.data_ptr(),
                                d_kv_len=self.len.data_ptr(), d_page_table=self.table.data_ptr())

    def call(self, out=None, ws=None, one_each=False, strm=None):
        size = self.qbuf.element_size()
        o = self.out if out is None else out
        self.kv.attention_dev(0, ws or self.ws, self.code, self.qbuf.data_ptr() + self.off * size,
                              o.data_ptr() + self.off * size, self.rows + self.pad, self.nh,
                              self.batch(one_each), scale=self.scale, window=self.window,
                              q_stride=self.stride, out_stride=self.stride,
                              stream=stream(self.torch) if strm is None else strm)

    def rows_of(self, buf):
        n = (self.rows + self.pad) * self.stride
        return f64(buf[self.off:self.off + n].view(-1, self.stride))

    def oracle(self, q):
        """(out [rows, nh, hd], the largest error allowed)"""
        scale = self.scale or self.hd ** -0.5
        out = np.zeros((self.rows, self.nh, self.hd))
        bar = np.zeros_like(out)
        r, row, G = 2.0 ** -21 if self.dtype == "f32" else 2.0 ** -11, 0, self.nh // self.nkv
        for n, nq, s in zip(self.lens, self.qs, self.slots):
            for h in range(self.nh):
                k, v = self.k[s, h // G], self.v[s, h // G]
                qq = q[row:row + nq, h]
                o, w = ko.attend(qq, k, v, range(n - nq, n), self.window, scale)
                if n:
                    e = (self.hd + 8) * 2.0 ** -22 * scale * (np.abs(qq) @ (15 * self.ks[s, h // G]).T)
                    e = (e * (w > 0)).max(1)[:, None]
                    bar[row:row + nq, h] = (2 * e + 2.0 ** -20 + r) * (w @ (23 * self.vs[s, h // G]))
                out[row:row + nq, h] = o
            row += nq
        return out, bar + 1.01 * ko.HALF_STEP[self.dtype] * (np.abs(out) + bar) + 1e-30

    def check(self, buf=None, q=None):
        buf = self.out if buf is None else buf
        q = self.rows_of(self.qbuf) if q is None else q
        want, bar = self.oracle(q[:self.rows, :self.nh * self.hd].reshape(self.rows, self.nh, self.hd))
        got = self.rows_of(buf)[:self.rows, :self.nh * self.hd].reshape(want.shape)
        assert np.isfinite(got).all()
        worst = (np.abs(got - want) / bar).max()
        assert worst <= 1, worst
        self.kv.check(stream(self.torch))


ATTN = [
    # one token a sequence: lengths from nothing to several tiles, ragged
    dict(dtype="f32", nh=16, nkv=16, hd=128, page=16, lens=[255]),
    dict(dtype="f32", nh=8, nkv=2, hd=128, page=16, lens=[0, 1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 300]),
    dict(dtype="bf16", nh=32, nkv=8, hd=128, page=64, lens=[700, 0, 63, 64, 65, 1, 1500], pad=3),
    dict(dtype="f16", nh=6, nkv=2, hd=64, page=32, lens=[1, 999, 32]),
    dict(dtype="bf16", nh=7, nkv=1, hd=80, page=16, lens=[5, 130, 77]),
    dict(dtype="f16", nh=3, nkv=3, hd=96, page=48, lens=[49, 47, 48, 200]),
    dict(dtype="f32", nh=9, nkv=1, hd=64, page=16, lens=[50, 80]),       # more heads than 8 a group
    dict(dtype="bf16", nh=32, nkv=2, hd=128, page=16, lens=[100, 37]),   # 16 a group
    dict(dtype="f16", nh=20, nkv=1, hd=32, page=16, lens=[70, 1]),       # 20 a group
    dict(dtype="f32", nh=40, nkv=2, hd=256, page=16, lens=[40, 90]),
    dict(dtype="bf16", nh=4, nkv=2, hd=256, page=128, lens=[500, 129]),
    dict(dtype="f16", nh=2, nkv=1, hd=160, page=16, lens=[33]),
    dict(dtype="f32", nh=2, nkv=2, hd=8, page=16, lens=[20, 3]),
    dict(dtype="bf16", nh=2, nkv=1, hd=40, page=16, lens=[64]),
    dict(dtype="f32", nh=5, nkv=5, hd=224, page=16, lens=[18, 16]),
    # windows
    dict(dtype="bf16", nh=8, nkv=2, hd=128, page=32, lens=[500, 10, 0, 100], window=100),
    dict(dtype="f32", nh=4, nkv=4, hd=64, page=16, lens=[300, 17], window=1),
    # scale given, large scores, strided rows, odd addresses
    dict(dtype="f32", nh=4, nkv=2, hd=64, page=16, lens=[90], scale=0.3, gap=8),
    dict(dtype="f32", nh=4, nkv=2, hd=128, page=16, lens=[400], q_gain=20.0),
    dict(dtype="bf16", nh=4, nkv=2, hd=64, page=16, lens=[90, 33], gap=3, off=1),
    dict(dtype="f16", nh=4, nkv=1, hd=128, page=16, lens=[90, 33], q_gain=1e-3),
    dict(dtype="bf16", nh=4, nkv=1, hd=128, page=16, lens=[90, 33], scale=1e-3, q_gain=1e4),
    # several query rows a sequence, also more than are cached
    dict(dtype="f32", nh=6, nkv=1, hd=64, page=16, lens=[100, 7, 40], qs=[4, 4, 1]),
    dict(dtype="bf16", nh=8, nkv=2, hd=128, page=32, lens=[200, 64, 3, 0], qs=[5, 64, 7, 2], pad=1),
    dict(dtype="f16", nh=4, nkv=4, hd=80, page=16, lens=[130, 33], qs=[130, 17]),
    dict(dtype="f32", nh=12, nkv=2, hd=128, page=16, lens=[90, 300], qs=[33, 20], window=40),
    dict(dtype="bf16", nh=4, nkv=1, hd=256, page=16, lens=[150], qs=[150], gap=8),
    dict(dtype="bf16", nh=16, nkv=2, hd=64, page=64, lens=[257, 65], qs=[65, 65], window=64),
    dict(dtype="f32", nh=16, nkv=1, hd=32, page=16, lens=[70], qs=[70]),
    dict(dtype="f16", nh=32, nkv=8, hd=128, page=64, lens=[600], qs=[256]),
    # chunks on many SMs: 64 query rows a CTA, tiles of 64 positions
    dict(dtype="bf16", nh=16, nkv=8, hd=64, page=16, lens=[300, 90, 70], qs=[90, 90, 70], pad=2),
    dict(dtype="f16", nh=8, nkv=8, hd=80, page=32, lens=[257, 200, 64, 65], qs=[129, 1, 64, 100]),
    dict(dtype="bf16", nh=10, nkv=10, hd=96, page=48, lens=[511, 130], qs=[130, 130], window=100),
    dict(dtype="f16", nh=40, nkv=20, hd=32, page=16, lens=[100, 0, 20], qs=[64, 3, 33], window=1, gap=3, off=1),
    dict(dtype="bf16", nh=48, nkv=8, hd=128, page=64, lens=[333, 77], qs=[77, 77], gap=8, scale=0.2),
    dict(dtype="f16", nh=8, nkv=8, hd=40, page=16, lens=[700], qs=[320], q_gain=30.0),
    dict(dtype="bf16", nh=16, nkv=16, hd=8, page=16, lens=[150], qs=[150], q_gain=1e-3),
    # few chunks among many sequences of one row
    dict(dtype="bf16", nh=8, nkv=8, hd=64, page=16, lens=[200] + [30 + i for i in range(20)], qs=[150] + [1] * 20),
    dict(dtype="f16", nh=8, nkv=4, hd=128, page=16, lens=[300, 200, 9, 40], qs=[150, 150, 1, 1], window=130),
    # more sequences than a CTA has threads, among them many that have not begun
    dict(dtype="bf16", nh=2, nkv=1, hd=32, page=16, lens=[(7 * i) % 61 * (i % 5 > 0) for i in range(700)], pad=1),
    dict(dtype="f32", nh=1, nkv=1, hd=160, page=16, lens=[(11 * i) % 37 for i in range(300)]),
    dict(dtype="f16", nh=4, nkv=2, hd=64, page=16, lens=[5 + i % 90 for i in range(600)],
         qs=[1 + i % 3 for i in range(600)]),
    # a long sequence beside short ones: split over many SMs
    dict(dtype="bf16", nh=8, nkv=2, hd=128, page=64, lens=[9000, 1, 0, 200], poison=False),
    dict(dtype="f32", nh=4, nkv=1, hd=64, page=16, lens=[6000], poison=False),
]


@pytest.mark.parametrize("i", range(len(ATTN)))
def test_attention(torch, rc, i):
    c = Case(torch, rc, seed=i, **ATTN[i])
    c.call()
    c.check()
    got = c.rows_of(c.out)
    assert (got[c.rows:] == 7.0).all()                      # rows behind the last sequence
    assert (got[:, c.nh * c.hd:] == 7.0).all()              # between the rows
    assert (f64(c.out[:c.off]) == 7.0).all()
    again = c.torch.full_like(c.out, 3.0)
    c.call(out=again)                                       # same call, same bits
    c.torch.cuda.synchronize()
    np.testing.assert_array_equal(c.rows_of(again)[:c.rows, :c.nh * c.hd], got[:c.rows, :c.nh * c.hd])


def test_attention_one_row_a_sequence_without_q_start_and_in_place(torch, rc):
    c = Case(torch, rc, dtype="bf16", nh=8, nkv=2, hd=64, page=16, lens=[40, 0, 500], seed=3)
    q = c.rows_of(c.qbuf)
    c.call(one_each=True)
    c.check()
    c.call(out=c.qbuf, one_each=True)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(c.rows_of(c.qbuf), c.rows_of(c.out))
    c.check(buf=c.qbuf, q=q)


def test_attention_of_values_that_are_not_finite(torch, rc):
    """A visible group that holds an infinity or NaN makes the channels it
    feeds NaN: a key's all of the row, a value's its own 32."""
    c = Case(torch, rc, dtype="f32", nh=2, nkv=1, hd=64, page=16, lens=[40, 40], seed=5)
    x = torch.randn(1, 1, 64, device="cuda")
    bad_v, bad_k = x.clone(), x.clone()
    bad_v[0, 0, 40], bad_k[0, 0, 3] = float("inf"), float("nan")
    for i, (k, v) in enumerate([(x, bad_v), (bad_k, x)]):
        s = torch.tensor([c.slots[i][17]], device="cuda")
        c.kv.append_dev(0, rc.F32, k.data_ptr(), v.data_ptr(), s.data_ptr(), 1, stream=stream(torch))
    c.call()
    nan = np.isnan(c.rows_of(c.out).reshape(2, 2, 64))
    assert nan[0, :, 32:].all() and not nan[0, :, :32].any()
    assert nan[1].all()


@pytest.mark.parametrize("dtype,nq", [("bf16", 20), ("f16", 200), ("f32", 200)])
def test_values_that_are_not_finite_in_a_chunk(torch, rc, dtype, nq):
    """Within a chunk only the rows behind a position see it: a NaN key there
    makes them NaN, a NaN value their channels of its group, and the rows
    before it stay as they are."""
    c = Case(torch, rc, dtype=dtype, nh=16, nkv=8, hd=64, page=16, lens=[nq + 50], qs=[nq], seed=6)
    bad_k, bad_v = nq + 50 - 7, nq + 50 - 12  # positions near the chunk's end
    x = torch.randn(2, 8, 64, device="cuda")
    k, v = x.clone(), x.clone()
    k[0, 3, 5] = float("nan")
    v[1, 2, 40] = float("-inf")
    s = torch.from_numpy(c.slots[0][[bad_k, bad_v]]).cuda()
    c.kv.append_dev(0, rc.F32, k.data_ptr(), v.data_ptr(), s.data_ptr(), 2, stream=stream(torch))
    c.call()
    nan = np.isnan(c.rows_of(c.out).reshape(nq, 16, 64))
    want = np.zeros_like(nan)
    want[nq - 7:, 6:8] = True
    want[nq - 12:, 4:6, 32:] = True
    np.testing.assert_array_equal(nan, want)


def test_attention_reports_what_is_out_of_range(torch, rc):
    """Lengths past the table, pages past the cache, q_start out of order:
    reported once each, nothing read there, the other sequences unharmed."""
    def fresh():
        return Case(torch, rc, dtype="f32", nh=4, nkv=2, hd=64, page=16, lens=[40, 33, 20], seed=9)

    def good(c, which):
        want, bar = c.oracle(c.rows_of(c.qbuf).reshape(c.rows, c.nh, c.hd))
        got = c.rows_of(c.out).reshape(want.shape)
        assert (np.abs(got - want) <= bar)[which].all()

    for what, harm in [("kv_len", lambda c: c.len.__setitem__(1, 16 * c.wide + 1)),
                       ("kv_len", lambda c: c.len.__setitem__(1, -3)),
                       ("page", lambda c: c.table.__setitem__((1, 0), 1000)),
                       ("page", lambda c: c.table.__setitem__((1, 1), -7)),
                       ("q_start", lambda c: c.start.copy_(torch.tensor([0, 1, 0, 1], dtype=torch.int32))),
                       ("q_start", lambda c: c.start.copy_(torch.tensor([0, 1, 5, 6], dtype=torch.int32))),
                       ("q_start", lambda c: c.start.copy_(torch.tensor([-1, 0, 1, 2], dtype=torch.int32)))]:
        c = fresh()
        harm(c)
        c.call()
        with pytest.raises(rc.RabbitCudaError, match=what) as e:
            c.kv.check(stream(torch))
        assert e.value.status == rc.ERR_ARGS
        if what != "q_start":
            good(c, [0, 2])
        c.kv.check(stream(torch))
        assert np.isfinite(c.rows_of(c.out)).all()
    # the same in a chunk: a page of the second sequence
    c = Case(torch, rc, dtype="bf16", nh=16, nkv=8, hd=64, page=16, lens=[200, 150, 90],
             qs=[100, 100, 90], seed=10)
    c.table[1, 2] = 12345
    c.call()
    with pytest.raises(rc.RabbitCudaError, match="page"):
        c.kv.check(stream(torch))
    want, bar = c.oracle(c.rows_of(c.qbuf).reshape(c.rows, c.nh, c.hd))
    got = c.rows_of(c.out).reshape(want.shape)
    assert (np.abs(got - want) <= bar)[:100].all() and (np.abs(got - want) <= bar)[200:].all()
    assert np.isfinite(got).all()


def test_attention_in_a_graph_and_on_two_streams(torch, rc):
    """A captured call reads lengths, table and queries at replay; two graphs
    with a scratch each, replayed together on two streams, keep their results."""
    cases = [Case(torch, rc, dtype="bf16", nh=8, nkv=2, hd=128, page=16, lens=[3000, 5, 900], seed=s,
                  poison=False) for s in (21, 22)]
    graphs, streams = [], [torch.cuda.Stream() for _ in cases]
    for c, s in zip(cases, streams):
        c.call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.call(strm=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for round_ in range(3):
        for c in cases:
            c.lens = [3000 - 700 * round_, 5 + round_, 900]
            c.slots = [sl[:n] if n <= len(sl) else None for sl, n in zip(c.slots, c.lens)]
            if c.slots[1] is None:  # one more position of the page already held
                first = int(c.table[1, 0]) * c.page
                c.slots[1] = np.arange(first, first + c.lens[1])
            c.len.copy_(torch.tensor(c.lens, dtype=torch.int32))
            c.qbuf.normal_()
            c.out.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for c in cases:
            c.check()


def test_a_decode_step_of_the_three_together(torch, rc):
    """Rotate q, append the rotated k and v, attend: five steps of three
    sequences, against the oracle over everything appended so far."""
    nh, nkv, hd, page, steps = 8, 2, 64, 16, 40
    rng = np.random.default_rng(4)
    kv = rc.Kv4(n_layers=2, n_kv_heads=nkv, head_dim=hd, page_size=page, n_pages=12)
    ws = rc.Kv4Scratch(kv)
    rope = rc.Rope(hd, layout=rc.ROPE_HALF, scaling=rc.ROPE_SCALE_LINEAR, factor=2.0)
    f = ko.freqs(hd, scaling="linear", factor=2.0)
    table = rng.permutation(12).reshape(3, 4).astype(np.int32)
    d_table = torch.from_numpy(table).cuda()
    held = [([], []) for _ in range(3)]
    for t in range(steps):
        lens = np.array([t + 1, t // 2 + 1, max(0, t - 3)])  # the last one starts later
        active = lens > 0
        qkv = torch.randn(3, (nh + 2 * nkv) * hd, device="cuda")
        src = f64(qkv)
        pos = torch.from_numpy((lens - 1).clip(0).astype(np.int32)).cuda()
        new = np.array([t == 0 or lens[i] != len(held[i][0]) for i in range(3)]) & active
        slots = np.where(new, table[np.arange(3), (lens - 1).clip(0) // page] * page + (lens - 1) % page, -1)
        d_slots = torch.from_numpy(slots.astype(np.int64)).cuda()
        d_len = torch.from_numpy(lens.astype(np.int32)).cuda()
        out = torch.empty(3, nh, hd, device="cuda")
        st, p, row = stream(torch), qkv.data_ptr(), qkv.shape[1]
        rope.apply_dev(rc.F32, p, p, pos.data_ptr(), 3, nh, x_stride=row, y_stride=row, stream=st)
        kv.append_dev(1, rc.F32, p + 4 * nh * hd, p + 4 * (nh + nkv) * hd, d_slots.data_ptr(), 3,
                      rope=rope, d_positions=pos.data_ptr(), k_stride=row, v_stride=row, stream=st)
        b = rc.Kv4Batch(n_seqs=3, max_pages=4, max_q_len=1, d_kv_len=d_len.data_ptr(),
                        d_page_table=d_table.data_ptr())
        kv.attention_dev(1, ws, rc.F32, p, out.data_ptr(), 3, nh, b, q_stride=row, stream=st)
        kv.check(st)
        x = src.reshape(3, nh + 2 * nkv, hd)
        q = ko.rotate(x[:, :nh], pos.cpu().numpy(), f, "half")
        k = ko.hold(ko.rotate(x[:, nh:nh + nkv], pos.cpu().numpy(), f, "half"))[0]
        v = ko.hold(x[:, nh + nkv:])[0]
        got = f64(out)
        for i in range(3):
            if new[i]:
                held[i][0].append(k[i])
                held[i][1].append(v[i])
            if not active[i]:
                assert (got[i] == 0).all()
                continue
            ks, vs = (np.stack(h) for h in held[i])
            for h in range(nh):
                want, w = ko.attend(q[i, h:h + 1], ks[:, h // 4], vs[:, h // 4], [lens[i] - 1], 0, hd ** -0.5)
                # as above with |q| <= 5, |k| <= 15/7 * 5: e <= 72 2^-22 8^-1 64 25 15/7 < 2^-9.2 in
                # the worst case; the bar below is 2^-14 of the largest value, 16 times what
                # such sums of random signs (sqrt(64) instead of 64 terms) come to
                assert np.abs(got[i, h] - want[0]).max() <= 2.0 ** -14 * 5


@pytest.mark.parametrize("page", [48, 64])
def test_a_cache_past_32_bits_of_bytes(torch, rc, page):
    """The last pages of a layer of more than 2^32 bytes hold what a small cache's do."""
    nkv, hd, n = 8, 128, 3 * page - 5
    big = 2 ** 32 // (page // 16 * nkv * 2304) + 100
    g = torch.Generator("cuda").manual_seed(5)
    k, v = (torch.randn(n, nkv, hd, generator=g, device="cuda") for _ in "kv")
    outs = []
    for n_pages in (3, big):
        kv = rc.Kv4(n_layers=1, n_kv_heads=nkv, head_dim=hd, page_size=page, n_pages=n_pages)
        ws, st = rc.Kv4Scratch(kv), stream(torch)
        slots = torch.arange(n, device="cuda") + (n_pages - 3) * page
        kv.append_dev(0, rc.F32, k.data_ptr(), v.data_ptr(), slots.data_ptr(), n, stream=st)
        read = torch.zeros(2, n, nkv, hd, device="cuda")
        kv.read_dev(0, rc.F32, slots.data_ptr(), n, read[0].data_ptr(), read[1].data_ptr(), stream=st)
        got = [read]
        table = torch.arange(n_pages - 3, n_pages, dtype=torch.int32, device="cuda")
        length = torch.tensor([n], dtype=torch.int32, device="cuda")
        for rows, heads in ((1, 16), (n, 40)):  # a decoding token, a chunk
            start = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
            q = torch.randn(rows, heads, hd, generator=torch.Generator("cuda").manual_seed(6),
                            device="cuda").half()
            out = torch.empty_like(q)
            b = rc.Kv4Batch(n_seqs=1, max_pages=3, max_q_len=rows, d_q_start=start.data_ptr(),
                            d_kv_len=length.data_ptr(), d_page_table=table.data_ptr())
            kv.attention_dev(0, ws, rc.F16, q.data_ptr(), out.data_ptr(), rows, heads, b, stream=st)
            got.append(out)
        kv.check(st)
        outs.append(got)
    assert np.array_equal(f64(outs[0][0][0]), ko.hold(f64(k))[0])
    for small, large in zip(*outs):
        assert torch.equal(small, large)
