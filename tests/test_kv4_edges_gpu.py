"""GPU: the paged 4-bit cache and its attention at their edges: many items a CTA,
waits that run out, numbers of very different size, against float64 numpy (tests/kv4_oracle.py)."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_oracle as ko
import kv4_signs as ks
import test_rope_kv4_gpu as base

pytestmark = pytest.mark.gpu

torch = base.torch  # the module's fixture


@pytest.mark.parametrize("dtype,nh", [("bf16", 4), ("f32", 10)])
def test_many_items_of_all_lengths_in_a_cta(torch, rc, dtype, nh):
    """Some thirty items to a CTA, each merged by one warp while it makes the
    operands of those behind: short ones that a warp takes alone, longer ones
    that all share, ones that a run's border cuts. Twenty runs, the same bits."""
    lens = [1 + (37 * i) % 230 for i in range(1100)]
    c = base.Case(torch, rc, dtype=dtype, nh=nh, nkv=2, hd=32, page=16, lens=lens, seed=40)
    c.call()
    c.check()
    first = c.out.clone()
    for _ in range(20):
        c.out.fill_(7.0)
        c.call()
        assert torch.equal(c.out, first)
    c.kv.check(base.stream(torch))


@pytest.mark.parametrize("kw", [
    dict(dtype="bf16", nh=8, nkv=2, hd=128, page=16, lens=[9000, 40, 700], poison=False),
    dict(dtype="f32", nh=4, nkv=4, hd=64, page=16, lens=[255]),
    dict(dtype="f32", nh=2, nkv=1, hd=256, page=16, lens=[40] * 300),          # short items first
    dict(dtype="bf16", nh=8, nkv=2, hd=128, page=32, lens=[400, 90], qs=[5, 7]),
    dict(dtype="f16", nh=8, nkv=8, hd=64, page=16, lens=[1500], qs=[640]),     # chunks: more tiles than stages
    dict(dtype="bf16", nh=16, nkv=16, hd=128, page=16, lens=[150], qs=[300]),  # and fewer
])
def test_a_wait_that_runs_out_is_a_status(torch, rc, kw):
    """One arrival is withheld, so waits of a CTA run out: the launch ends, the check
    says so once, and the next call, with a new scratch, is right."""
    c = base.Case(torch, rc, seed=41, **kw)
    spoiled = rc.Kv4Scratch(c.kv)
    try:
        rc.check(rc.lib().rabbit_cuda_set_wait_limit_us(20000))
        rc.check(rc.lib().rabbit_cuda_kv4_debug_withhold(c.kv.handle))
        c.call(ws=spoiled)
        with pytest.raises(rc.RabbitCudaError) as e:
            c.kv.check(base.stream(torch))
        assert e.value.status == rc.ERR_TIMEOUT
    finally:
        rc.check(rc.lib().rabbit_cuda_set_wait_limit_ms(2000))
    c.kv.check(base.stream(torch))  # said once
    c.call()
    c.check()


@pytest.mark.parametrize("order", ["page first", "slot behind"])
def test_a_timeout_is_not_hidden_by_what_is_out_of_range(torch, rc, order):
    """A scratch is spoiled after a timeout, so its status comes before the others'."""
    c = base.Case(torch, rc, dtype="bf16", nh=8, nkv=2, hd=64, page=16, lens=[3000, 40], seed=42)
    st = base.stream(torch)
    if order == "page first":
        bad = c.table.clone()
        c.table[1, 0] = 100000
        c.call()
        c.table.copy_(bad)
    try:
        rc.check(rc.lib().rabbit_cuda_set_wait_limit_us(20000))
        rc.check(rc.lib().rabbit_cuda_kv4_debug_withhold(c.kv.handle))
        c.call(ws=rc.Kv4Scratch(c.kv))
    finally:
        rc.check(rc.lib().rabbit_cuda_set_wait_limit_ms(2000))
    if order == "slot behind":
        x = torch.zeros(1, 2, 64, device="cuda")
        s = torch.tensor([1 << 40], device="cuda")
        c.kv.append_dev(0, rc.F32, x.data_ptr(), x.data_ptr(), s.data_ptr(), 1, stream=st)
    with pytest.raises(rc.RabbitCudaError, match=order.split()[0]) as e:
        c.kv.check(st)
    assert e.value.status == rc.ERR_TIMEOUT
    c.kv.check(st)
    c.call()
    c.check()


def rewrite(torch, rc, c, slots, k, v):
    """Rows (fp32) into slots of a Case's cache, and of its oracle."""
    s = torch.as_tensor(np.asarray(slots), dtype=torch.int64, device="cuda")
    c.kv.append_dev(0, rc.F32, k.data_ptr(), v.data_ptr(), s.data_ptr(), len(s),
                    stream=base.stream(torch))
    (c.k[slots], c.ks[slots]), (c.v[slots], c.vs[slots]) = ko.hold(base.f64(k)), ko.hold(base.f64(v))


# many query rows a sequence, and few
CHUNKS = [dict(dtype="bf16", nh=16, nkv=8, hd=64, page=48, lens=[300, 90, 73], qs=[90, 90, 70]),
          dict(dtype="f16", nh=8, nkv=8, hd=128, page=16, lens=[700], qs=[600])]
DECODES = [dict(dtype="bf16", nh=8, nkv=2, hd=128, page=48, lens=[300, 90, 73]),
           dict(dtype="f32", nh=8, nkv=2, hd=64, page=16, lens=[700, 33], qs=[9, 2])]


@pytest.mark.parametrize("big", [2.0 ** 20, 2.0 ** 30, 1e30])
@pytest.mark.parametrize("kw", CHUNKS + DECODES)
def test_finite_rows_that_no_query_row_sees(torch, rc, kw, big):
    """Rows of any size behind a sequence's end, as an earlier user of the page leaves
    them, and before a window have no part in the result."""
    for window in (0, 20):
        c = base.Case(torch, rc, seed=43, poison=False, window=window, **kw)
        used = np.concatenate(c.slots)
        hidden = [np.setdiff1d(np.arange(c.kv.n_pages * c.page), used)]
        if window:
            hidden += [s[:max(0, n - q - window + 1)] for s, n, q in zip(c.slots, c.lens, c.qs)]
        hidden = np.concatenate(hidden)
        k, v = (torch.randn(len(hidden), c.nkv, c.hd, device="cuda") * big for _ in "kv")
        rewrite(torch, rc, c, hidden, k, v)
        c.call()
        c.check()


@pytest.mark.parametrize("dtype,big", [("f16", 1000.0), ("bf16", 2.0 ** 30), ("bf16", 1e30)])
@pytest.mark.parametrize("kw", CHUNKS + DECODES[1:])
def test_a_large_value_seen_by_some_rows_of_a_chunk(torch, rc, kw, dtype, big):
    """The rows before its position do not see it, those behind do: each is right."""
    c = base.Case(torch, rc, seed=44, poison=False, **{**kw, "dtype": dtype})
    at = [(s, n - q // 2) for s, n, q in zip(c.slots, c.lens, c.qs)]
    k, v = (torch.randn(len(at), c.nkv, c.hd, device="cuda") for _ in "kv")
    rewrite(torch, rc, c, [s[p - 1] for s, p in at], k, v * big)
    c.call()
    c.check()


@pytest.mark.parametrize("ratio", [2.0 ** 16, 2.0 ** 22, 2.0 ** 26])
@pytest.mark.parametrize("kw", CHUNKS)
def test_channel_groups_of_very_different_size_in_a_chunk(torch, rc, kw, ratio):
    """32 channels of keys and values that are much larger than the others, and that
    the queries do not look at: the scores, and the others' outputs, keep their
    accuracy."""
    c = base.Case(torch, rc, seed=45, poison=False, **{**kw, "dtype": "bf16"})
    every = np.arange(c.kv.n_pages * c.page)
    g = torch.Generator("cuda").manual_seed(46)
    k, v = (torch.randn(len(every), c.nkv, c.hd, generator=g, device="cuda") for _ in "kv")
    k[..., :32] *= ratio
    v[..., :32] *= ratio
    rewrite(torch, rc, c, every, k, v)
    c.qbuf.view(c.rows, c.nh, c.hd)[..., :32] = 0
    c.call()
    c.check()


@pytest.mark.parametrize("dtype,nq,n", [("bf16", 64, 80000), ("bf16", 1, 480000), ("f32", 1, 480000)])
def test_a_value_behind_many_that_are_zero(torch, rc, dtype, nq, n):
    """The weights of zero values are as large as those of others in the sum that
    divides, however many they are. The first positions' scores are lower, so that
    those behind weigh 2^7.5 times as much; the last value is the only one."""
    hd, page, sms = 32, 64, torch.cuda.get_device_properties(0).multi_processor_count
    seqs = 80 if nq > 1 else sms  # all over the same pages; a CTA each
    kv = rc.Kv4(n_layers=1, n_kv_heads=1, head_dim=hd, page_size=page, n_pages=n // page)
    k, v = torch.zeros(2, n, 1, hd, device="cuda")
    k[nq + 512:, 0, 0] = 7
    v[-nq] = 7  # the chunk's first row's own position; the rows behind it see zeros again
    base.filled(torch, rc, kv, (k, v))
    dt, code = base.types(torch, rc, dtype)
    q = torch.zeros(seqs * nq, 1, hd, dtype=dt, device="cuda")
    q[..., 0] = 1
    out = torch.empty_like(q)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(n // page, **i32).repeat(seqs, 1)
    lens, start = torch.full((seqs,), n, **i32), torch.arange(seqs + 1, **i32) * nq
    b = rc.Kv4Batch(n_seqs=seqs, max_pages=n // page, max_q_len=nq, d_q_start=start.data_ptr(),
                    d_kv_len=lens.data_ptr(), d_page_table=table.data_ptr())
    st = base.stream(torch)
    kv.attention_dev(0, rc.Kv4Scratch(kv), code, q.data_ptr(), out.data_ptr(), seqs * nq, 1, b,
                     scale=7.5 * np.log(2) / 7, stream=st)
    kv.check(st)
    w = 2.0 ** 7.5
    seen = n - nq + 1 + np.arange(nq)                # positions a row sees
    want = 7 * w / ((nq + 512) + (seen - nq - 512) * w)
    got = base.f64(out).reshape(seqs, nq, hd)
    # exp2 and its argument 2^-20, the weight in fp16 2^-11, the division and the sum 2^-20
    bar = 2.0 ** -11 + 2.0 ** -19 + 1.01 * ko.HALF_STEP[dtype]
    assert np.abs(got / want[None, :, None] - 1).max() <= bar


def hold(x):
    """The oracle's groups, their codes within -7..7: a scale among bf16's smallest
    numbers may have been rounded down by up to a half."""
    y, s = ko.hold(x)
    return np.clip(y, -7 * s, 7 * s)


@pytest.mark.parametrize("turn", [False, True])
def test_codes_of_the_smallest_groups_stay_in_range(torch, rc, turn):
    """Largest magnitudes from bf16's smallest scale to where its scales have all
    their bits, of both signs, as keys, rotated keys and values."""
    tops = np.concatenate([[9e-40, 1.5e-39, 2.2e-39, 3.3e-40, 4e-39], np.geomspace(2e-40, 2e-38, 91)])
    T, hd = len(tops), 64
    rng = np.random.default_rng(47)
    x = rng.uniform(-1, 1, (T, 2, hd))
    x[:, 0, 3], x[:, 1, 35] = 1, -1
    x = torch.from_numpy((x * tops[:, None, None]).astype(np.float32)).cuda()
    kv = rc.Kv4(n_layers=1, n_kv_heads=2, head_dim=hd, page_size=16, n_pages=-(-T // 16))
    slots, pos = torch.arange(T, device="cuda"), torch.arange(T, device="cuda").int() * 1001
    kv.append_dev(0, rc.F32, x.data_ptr(), x.data_ptr(), slots.data_ptr(), T,
                  rope=rc.Rope(hd) if turn else None, d_positions=pos.data_ptr(),
                  stream=base.stream(torch))
    kx = ko.rotate(base.f64(x), pos.cpu().numpy(), ko.freqs(hd), "interleaved") if turn else base.f64(x)
    k, v = base.read(torch, rc, kv, range(T))
    np.testing.assert_array_equal(v, hold(base.f64(x)))
    np.testing.assert_array_equal(k, hold(kx))


@pytest.mark.parametrize("steps", [1, 5, 6, 100])
def test_rotated_keys_among_the_smallest_numbers(torch, rc, steps):
    """Where fp32 has steps of 2^-149 an error bound relative to the value is none:
    scales and codes are still those of the exactly rotated key. Largest magnitudes
    within a step or two of those at which the scale's rounding turns: a seventh of them
    is `steps` and a half steps of bf16's subnormal numbers, and half a step of fp32's."""
    T, nkv, hd = 8192, 2, 128
    x = np.random.default_rng(48).uniform(-1, 1, (T, nkv, hd))
    pos, f = np.arange(T), ko.freqs(hd)
    top = np.abs(ko.rotate(x, pos, f, "interleaved")).reshape(T, nkv, 4, 32).max(-1)
    x = x * np.repeat(7 * ((steps + 0.5) * 2.0 ** -133 + 0.5 * 2.0 ** -149 * (-1) ** steps) / top, 32, -1)
    x = torch.from_numpy(x.astype(np.float32)).cuda()
    kv = rc.Kv4(n_layers=1, n_kv_heads=nkv, head_dim=hd, page_size=64, n_pages=T // 64)
    slots, d_pos = torch.arange(T, device="cuda"), torch.from_numpy(pos).int().cuda()
    kv.append_dev(0, rc.F32, x.data_ptr(), x.data_ptr(), slots.data_ptr(), T, rope=rc.Rope(hd),
                  d_positions=d_pos.data_ptr(), stream=base.stream(torch))
    want = hold(ko.rotate(base.f64(x), pos, f, "interleaved"))
    k, _ = base.read(torch, rc, kv, range(T))
    np.testing.assert_array_equal(k, want)


@pytest.mark.parametrize("big", [1e4, 1e8, 1e18, 1e30])
@pytest.mark.parametrize("kw", CHUNKS + DECODES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_scores_past_the_whole_numbers_of_fp32(torch, rc, kw, dtype, big):
    """Scores whose steps in fp32 are large beside the exponents of the weights: equal
    ones share, a larger one has all, whatever the values' size."""
    value = 1e3 if dtype == "f16" else 1e-20 if big < 1e9 else 1e30
    c = base.Case(torch, rc, seed=49, poison=False, **{**kw, "dtype": dtype})
    n = c.kv.n_pages * c.page
    g = torch.Generator("cuda").manual_seed(50)
    v = torch.randn(n, c.nkv, c.hd, generator=g, device="cuda") * value
    v[::3] /= 1000
    k = torch.zeros_like(v)
    pick = torch.randint(1, 4, (n, c.nkv), generator=g, device="cuda") * 7.0  # scales 1, 2, 3
    q = torch.zeros(c.rows, c.nh, c.hd, device="cuda")
    q[..., 0] = torch.where(torch.rand(c.rows, c.nh, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    if dtype == "f16":  # the queries' type holds up to 65504
        k[..., 0], c.scale = pick * min(big, 1e30), 1.0
    else:
        k[..., 0], c.scale = pick, 1.0
        q *= big
    c.qbuf.copy_(q.to(c.qbuf.dtype).flatten())
    rewrite(torch, rc, c, np.arange(n), k, v)
    c.call()
    c.kv.check(base.stream(torch))
    got = c.rows_of(c.out).reshape(c.rows, c.nh, c.hd)
    q, row, G = c.rows_of(c.qbuf).reshape(got.shape), 0, c.nh // c.nkv
    for length, nq, s in zip(c.lens, c.qs, c.slots):
        for h in range(c.nh):
            at = range(length - nq, length)
            want, w = ko.attend(q[row:row + nq, h], c.k[s, h // G], c.v[s, h // G], at, c.window, 1.0)
            size = ko.attend(q[row:row + nq, h], c.k[s, h // G], np.abs(c.v[s, h // G]), at, c.window, 1.0)[0]
            # equal weights and weights of zero: a common factor is off, 2^-20, and each fp16
            # weight by 2^-11, once more in its product with the value's scale
            bar = (2.0 ** -10 + 2.0 ** -19) * size + 1.01 * ko.HALF_STEP[dtype] * np.abs(want) + 1e-30
            assert (np.abs(got[row:row + nq, h] - want) <= bar).all()
        row += nq


def test_a_check_loses_nothing_that_another_stream_found(torch, rc):
    """One thread makes and checks bad slots on its stream, another bad lengths on its own:
    each length is reported by one check or the other."""
    import threading
    import time

    kv = rc.Kv4(n_layers=1, n_kv_heads=1, head_dim=32, page_size=16, n_pages=2)
    ws, a, b = rc.Kv4Scratch(kv), torch.cuda.Stream(), torch.cuda.Stream()
    x = torch.zeros(1, 1, 32, device="cuda")
    out, slot = torch.empty_like(x), torch.tensor([99], device="cuda")
    length, table = torch.tensor([17], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = rc.Kv4Batch(n_seqs=1, max_pages=1, d_kv_len=length.data_ptr(), d_page_table=table.data_ptr())
    torch.cuda.synchronize()
    said, rounds, stop = [], [0], threading.Event()

    def look(s):
        try:
            kv.check(s.cuda_stream)
        except rc.RabbitCudaError as e:
            assert e.status == rc.ERR_ARGS
            said.append(str(e))

    def slots():
        while not stop.is_set():
            kv.append_dev(0, rc.F32, x.data_ptr(), x.data_ptr(), slot.data_ptr(), 1, stream=a.cuda_stream)
            look(a)
            rounds[0] += 1

    t = threading.Thread(target=slots)
    t.start()
    try:
        for _ in range(400):
            before = len(said)
            kv.attention_dev(0, ws, rc.F32, x.data_ptr(), out.data_ptr(), 1, 1, batch, stream=b.cuda_stream)
            look(b)
            done = rounds[0] + 2  # a check of the other thread that was under way is over
            while rounds[0] < done and t.is_alive():
                time.sleep(1e-5)
            assert any("kv_len" in m for m in said[before:])
    finally:
        stop.set()
        t.join()
    assert any("slot" in m for m in said)


# ---------------------------------------------------------------- each token, in place --
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("i", range(len(ks.CASES)))
def test_every_token_has_its_part(torch, rc, i, dtype):
    """Random signs whose result tells each token from the others (tests/kv4_signs.py;
    that every one lost, doubled or misplaced passes the bar is shown there)."""
    kw = ks.CASES[i]
    c = base.Case(torch, rc, dtype=dtype, seed=i, poison=False, scale=ks.SCALE, **kw)
    q, seqs = ks.inputs(i, nh=c.nh, nkv=c.nkv, hd=c.hd, lens=c.lens, qs=c.qs)
    for s, (k, v) in zip(c.slots, seqs):
        if len(s):
            kx = np.zeros(v.shape, np.float32)
            kx[..., ks.PICK] = 7 * k
            rewrite(torch, rc, c, s, torch.from_numpy(kx).cuda(), 7 * torch.from_numpy(v).float().cuda())
    qx = torch.zeros(c.rows, c.nh, c.hd)
    qx[..., ks.PICK] = torch.from_numpy(q).float()
    c.qbuf.copy_(qx.to(c.qbuf.dtype).flatten())
    c.call()
    c.kv.check(base.stream(torch))
    got, row, G = c.rows_of(c.out).reshape(c.rows, c.nh, c.hd), 0, c.nh // c.nkv
    for (k, v), n, nq in zip(seqs, c.lens, c.qs):
        for r in range(nq):
            for h in range(c.nh):
                want = ks.attend(q[row + r, h], k[:, h // G], v[:, h // G], n - nq + r, c.window)[0]
                assert (np.abs(got[row + r, h] - want) <= ks.bar(want, ko.HALF_STEP[dtype])).all(), (n, r, h)
        row += nq


class Close(base.Case):
    """The same cases with bars from the keys and values at hand instead of bounds on
    them. With T_j = |scale| sum_c |q_c| |k_jc|, where the 16-bit decode kernel's codes have
    a bias of 8 scales on top:
     * a matrix instruction adds 16 products to a sum, each cut off at 2^-23 of the largest:
       17 2^-23 of it. A group of 32 channels takes 2 (fp32 queries: 4), whose sums are at most
       T_j's part, in a chunk 2 in a row over all groups: e_j = (17 m + 6) 2^-23 T_j with
       m = 2, 4 or 2 groups; the 6 are the groups' sum, the unit and the query's two terms.
     * a weight is off by e_j, by 2^-19 (exp2 and its argument), by its rounding, r = 2^-11 or
       2^-21, or, where that is more, by 7 2^-31 of the largest weight times scale.
     * a granule's product is added with 17 2^-23 of the sum; a warp of a long sequence that
       many SMs share has at most 64 of them.
    """

    def oracle(self, q):
        scale = self.scale or self.hd ** -0.5
        out = np.zeros((self.rows, self.nh, self.hd))
        bar = np.zeros_like(out)
        split, row, G = self.dtype == "f32", 0, self.nh // self.nkv
        r, m = 2.0 ** -21 if split else 2.0 ** -11, max(4, 2 * -(-self.hd // 32))
        for n, nq, s in zip(self.lens, self.qs, self.slots):
            for h in range(self.nh):
                k, v = self.k[s, h // G], self.v[s, h // G]
                qq = q[row:row + nq, h]
                o, w = ko.attend(qq, k, v, range(n - nq, n), self.window, scale)
                if n:
                    big = np.abs(k) if split else np.abs(k) + 8 * self.ks[s, h // G]
                    e = (17 * m + 6) * 2.0 ** -23 * abs(scale) * (np.abs(qq) @ big.T) + 2.0 ** -19
                    a = np.abs(v)
                    bar[row:row + nq, h] = (
                        (w * (e + r + min(n / 16, 64) * 17 * 2.0 ** -23)) @ a + np.abs(o) * (w * e).sum(1)[:, None] +
                        n * 7 * 2.0 ** -31 * (w[:, :, None] * self.vs[s, h // G]).max(1))
                out[row:row + nq, h] = o
            row += nq
        # half a step of the output's type: of its value, of its smallest for subnormal fp16
        least = 2.0 ** -25 if self.dtype == "f16" else 1e-30
        return out, bar + 1.01 * ko.HALF_STEP[self.dtype] * (np.abs(out) + bar) + least


@pytest.mark.parametrize("i", range(len(base.ATTN)))
def test_attention_within_close_bars(torch, rc, i):
    c = Close(torch, rc, seed=100 + i, **base.ATTN[i])
    c.call()
    c.check()


# ------------------------------------------------------------------ ways of calling --
def test_one_scratch_for_calls_of_all_kinds_in_turn(torch, rc):
    """On one stream, without a wait between them: other types, head counts, layers, kernels
    and numbers of sequences. Each gives what it gives with a scratch of its own."""
    kv = rc.Kv4(n_layers=2, n_kv_heads=4, head_dim=64, page_size=16, n_pages=400)
    for layer in range(2):
        g = torch.Generator("cuda").manual_seed(layer)
        base.filled(torch, rc, kv, torch.randn(2, 6400, 4, 64, generator=g, device="cuda"), layer=layer)
    ws, st, i32 = rc.Kv4Scratch(kv), base.stream(torch), dict(dtype=torch.int32, device="cuda")
    table = torch.randperm(400, generator=torch.Generator().manual_seed(9)).int().cuda()
    calls = []
    for dtype, layer, nh, nq, lens in [("bf16", 0, 16, 1, [6400]), ("f32", 1, 4, 1, [700, 30, 5000]),
                                       ("f16", 0, 32, 300, [2000]), ("f32", 0, 24, 4, [3000] * 3),
                                       ("bf16", 1, 4, 1, [9] * 40), ("bf16", 1, 40, 90, [100, 90, 91]),
                                       ("f16", 1, 8, 2, [6400, 0, 1])]:
        dt, code = base.types(torch, rc, dtype)
        rows = nq * len(lens)
        q = torch.randn(rows, nh, 64, generator=torch.Generator("cuda").manual_seed(nh), device="cuda").to(dt)
        keep = (torch.tensor(lens, **i32), torch.arange(len(lens) + 1, **i32) * nq, table.repeat(len(lens), 1))
        b = rc.Kv4Batch(n_seqs=len(lens), max_pages=400, max_q_len=nq, d_q_start=keep[1].data_ptr(),
                        d_kv_len=keep[0].data_ptr(), d_page_table=keep[2].data_ptr())
        calls.append((layer, code, q, rows, nh, b, keep))

    def run(own):
        outs = []
        for layer, code, q, rows, nh, b, _ in calls:
            outs.append(torch.zeros_like(q))
            w = rc.Kv4Scratch(kv) if own else ws
            kv.attention_dev(layer, w, code, q.data_ptr(), outs[-1].data_ptr(), rows, nh, b, stream=st)
            if own:
                torch.cuda.synchronize()
        kv.check(st)
        return outs

    want = run(True)
    for _ in range(10):
        for got, w in zip(run(False), want):
            assert torch.equal(got, w)


@pytest.mark.parametrize("dtype,nq", [("f32", 1), ("bf16", 1), ("bf16", 100)])
def test_sequences_that_share_pages(torch, rc, dtype, nq):
    """A common beginning of some pages, and the very same sequence twice."""
    c = base.Case(torch, rc, dtype=dtype, nh=32, nkv=8, hd=64, page=32, lens=[300, 270, 300], qs=[nq] * 3,
                  seed=51, poison=False)
    c.table[1, :5] = c.table[0, :5]
    c.table[2] = c.table[0]
    c.slots[1] = np.concatenate([c.slots[0][:160], c.slots[1][160:]])
    c.slots[2] = c.slots[0]
    c.qbuf.view(3 * nq, -1)[2 * nq:] = c.qbuf.view(3 * nq, -1)[:nq]
    c.call()
    c.check()


def test_a_cache_on_another_device_than_the_current_one(torch, rc):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    kv = rc.Kv4(n_layers=1, n_kv_heads=2, head_dim=64, page_size=16, n_pages=4, device=1)
    ws = rc.Kv4Scratch(kv)
    assert torch.cuda.current_device() == 0
    with torch.cuda.device(1):
        st = torch.cuda.current_stream().cuda_stream
        x = torch.randn(2, 40, 2, 64, device="cuda:1")
        q, out = torch.randn(1, 4, 64, device="cuda:1"), torch.empty(1, 4, 64, device="cuda:1")
        slots, table = torch.arange(40, device="cuda:1"), torch.arange(4, dtype=torch.int32, device="cuda:1")
        n = torch.tensor([40], dtype=torch.int32, device="cuda:1")
        torch.cuda.synchronize()
    b = rc.Kv4Batch(n_seqs=1, max_pages=4, d_kv_len=n.data_ptr(), d_page_table=table.data_ptr())
    kv.append_dev(0, rc.F32, x[0].data_ptr(), x[1].data_ptr(), slots.data_ptr(), 40, stream=st)
    kv.attention_dev(0, ws, rc.F32, q.data_ptr(), out.data_ptr(), 1, 4, b, stream=st)
    kv.check(st)
    assert torch.cuda.current_device() == 0
    k, v = (ko.hold(base.f64(y))[0] for y in x)
    for h in range(4):
        want, w = ko.attend(base.f64(q)[:, h], k[:, h // 2], v[:, h // 2], [39], 0, 0.125)
        assert np.abs(base.f64(out)[0, h] - want[0]).max() <= 2.0 ** -14 * np.abs(v).max()


@pytest.mark.parametrize("kw", CHUNKS + DECODES)
def test_a_scale_below_zero_and_the_widest_window(torch, rc, kw):
    c = Close(torch, rc, seed=52, **{**kw, "scale": -0.2, "window": 2 ** 31 - 1})
    c.call()
    c.check()


@pytest.mark.parametrize("kw", CHUNKS + DECODES)
def test_a_query_that_is_not_finite_stays_in_its_row(torch, rc, kw):
    """Its own head's row is NaN, every other row has the same bits as without it."""
    c = base.Case(torch, rc, seed=53, **kw)
    c.call()
    want = c.rows_of(c.out).reshape(c.rows, c.nh, c.hd)
    q = c.qbuf.view(c.rows, c.nh, c.hd)
    q[0, 1, 3], q[c.rows - 1, 0, c.hd - 1], q[c.rows - 1, c.nh - 1, :] = float("nan"), float("inf"), float("-inf")
    again = torch.zeros_like(c.out)
    c.call(out=again)
    c.kv.check(base.stream(torch))
    got = c.rows_of(again).reshape(want.shape)
    odd = np.zeros(want.shape[:2], bool)
    odd[0, 1] = odd[-1, 0] = odd[-1, -1] = True
    assert np.isnan(got[odd]).all()
    np.testing.assert_array_equal(got[~odd], want[~odd])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kw", CHUNKS + DECODES)
def test_keys_of_the_largest_numbers(torch, rc, kw, dtype):
    """Keys up to 3e38 under queries that bring the scores back to a few units."""
    c = Close(torch, rc, seed=54, poison=False, scale=2.0 ** -115, **{**kw, "dtype": dtype})
    g = torch.Generator("cuda").manual_seed(55)
    n = c.kv.n_pages * c.page
    k, v = (torch.rand(n, c.nkv, c.hd, generator=g, device="cuda") * 2 - 1 for _ in "kv")
    rewrite(torch, rc, c, np.arange(n), k * 3e38, v)
    q = torch.randn(c.rows, c.nh, c.hd, generator=g, device="cuda") * 2.0 ** -13
    c.qbuf.copy_(q.to(c.qbuf.dtype).flatten())
    c.call()
    c.check()
