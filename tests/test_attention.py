"""The attention sublayer (moe_qk_norm_rope, moe_kv_append, moe_kv_read,
moe_kv_attention, moe_attention) against the plain 64-bit oracle.

Tolerances. u = 2^-24 is a rounding to f32; a rounding to a row's type is at
most half a step, eps / 2 relative.

Norm and rotation in f32 of a head of D values: sum of squares (D/32 + 5 chained
roundings, halved by the root), root, quotient, two products: under 12 u; the
angle, reduced in f64, is rounded once (pi u) and its sine and cosine are good to
2 ulp, two products and a sum follow: under 12 u of |a| + |b|. In all 24 u (|a| + |b|).

Attention: a logit is a sum of D products of exact 8-bit values with queries of
22 bits (F32 rows) or exact ones (16-bit rows, scaled by a power of two), scaled
in f32: its error is at most A (2^-22 + (D + 8) u) with A = scale * max sum
|q_d k_d|. A weight is then off by twice that (the maximum is off too) and the
exponential's 2^-21, relative; weights enter the product with 22 bits, or 11
with 16-bit rows; sums over L tokens add (L + 64) u in numerator and in
denominator. Each part moves the output by at most that share of max|v|, twice
(numerator and denominator)."""
import ctypes as C

import numpy as np
import pytest

import attn_oracle as ao
import jeromoe as jm

U = 2.0 ** -24
ACTS = {"f32": jm.F32, "f16": jm.F16, "bf16": jm.BF16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


# ------------------------------------------------------------------ refusals


def _args(**over):
    """A moe_attention call that is taken; pointers are only checked, never read."""
    P = 1 << 20
    a = {"max_tokens": 64, "out": P, "out_stride": 32 * 128,
         "cache": dict(head_dim=128, kv_heads=4, page_tokens=64, n_pages=10, n_slots=4, table_stride=4, page_table=P, k=P,
                       v=P, k_scale=P, v_scale=P, open_k=P, open_v=P),
         "batch": dict(n_seqs=4, n_tokens=4, past=P),
         "rope": dict(rope_dim=128, theta=1e6, eps=1e-6, q_norm=P, k_norm=P),
         "opts": dict(),
         "rows": dict(act=jm.F32, q_heads=32, kv_heads=4, head_dim=128, q=P, k=P, v=P, q_stride=4096, k_stride=512,
                      v_stride=512)}
    for key, v in over.items():
        part, _, name = key.partition("__")
        if name:
            a[part] = {**a[part], name: v}
        else:
            a[part] = v
    return a


def _check(a):
    jm.attention_check(a["max_tokens"], jm.KvCache(**a["cache"]), jm.KvBatch(**a["batch"]), jm.Rope(**a["rope"]),
                       jm.AttnOpts(**a["opts"]), jm.QkvRows(**a["rows"]), a["out"], a["out_stride"])


def test_check_takes_good_arguments():
    _check(_args())
    _check(_args(rows__act=jm.BF16, cache__page_tokens=16, opts__window=100, rope__rope_dim=0))
    _check(_args(batch=dict(n_seqs=2, n_tokens=7, past=1 << 20, row_start=1 << 20, slot=1 << 20)))
    _check(_args(batch=dict(n_seqs=0, n_tokens=0)))
    _check(_args(cache__table_stride=1 << 23))
    _check(_args(max_tokens=1 << 30, batch__n_tokens=1 << 27, batch__row_start=1 << 20, rope__q_norm=(1 << 20) + 4))


@pytest.mark.parametrize("over,error", [
    (dict(cache__head_dim=96), jm.CapabilityMismatch),
    (dict(cache__head_dim=256, rows__head_dim=256), jm.CapabilityMismatch),
    (dict(cache__page_tokens=24), jm.CapabilityMismatch),
    (dict(cache__page_tokens=512), jm.CapabilityMismatch),
    (dict(cache__page_tokens=0), jm.CapabilityMismatch),
    (dict(cache__kv_heads=0), jm.CapabilityMismatch),
    (dict(cache__n_pages=-1), jm.InvalidArguments),
    (dict(cache__n_slots=3), jm.TensorBoundsError),
    (dict(cache__k=0), jm.InvalidArguments),
    (dict(cache__v=(1 << 20) + 8), jm.InvalidArguments),
    (dict(cache__open_k=0), jm.InvalidArguments),
    (dict(cache__page_table=0), jm.InvalidArguments),
    (dict(batch__n_tokens=5), jm.InvalidArguments),
    (dict(batch__n_seqs=-1), jm.InvalidArguments),
    (dict(batch__max_new=-1), jm.InvalidArguments),
    (dict(batch__past=0), jm.InvalidArguments),
    (dict(max_tokens=3), jm.ContextLengthExceeded),
    (dict(rope__rope_dim=3), jm.InvalidArguments),
    (dict(rope__rope_dim=130), jm.InvalidArguments),
    (dict(rope__rope_dim=-2), jm.InvalidArguments),
    (dict(rope__theta=0.0), jm.InvalidArguments),
    (dict(rope__theta=float("nan")), jm.InvalidArguments),
    (dict(rope__eps=-1.0), jm.InvalidArguments),
    (dict(rope__eps=float("inf")), jm.InvalidArguments),
    (dict(rope__mscale=float("nan")), jm.InvalidArguments),
    (dict(rope__inv_freq=[float("inf")] * 64), jm.InvalidArguments),
    (dict(rope__inv_freq=[1.0] * 63), jm.InvalidArguments),
    (dict(opts__window=-1), jm.InvalidArguments),
    (dict(opts__scale=float("inf")), jm.InvalidArguments),
    (dict(rows__act=8), jm.CapabilityMismatch),
    (dict(rows__q_heads=30), jm.InvalidArguments),
    (dict(rows__q_heads=0), jm.CapabilityMismatch),
    (dict(rows__kv_heads=2), jm.InvalidArguments),
    (dict(rows__head_dim=64), jm.InvalidArguments),
    (dict(rows__q=0), jm.InvalidArguments),
    (dict(rows__v=0), jm.InvalidArguments),
    (dict(rows__q=(1 << 20) + 4), jm.InvalidArguments),
    (dict(rows__q_stride=4095), jm.TensorBoundsError),
    (dict(rows__k_stride=514), jm.InvalidArguments),
    (dict(out=0), jm.InvalidArguments),
    (dict(out=(1 << 20) + 4), jm.InvalidArguments),
    (dict(out_stride=4095), jm.InvalidArguments),
    (dict(out_stride=2048), jm.TensorBoundsError),
    (dict(cache__page_table=(1 << 20) + 2), jm.InvalidArguments),
    (dict(cache__v_scale=(1 << 20) + 1), jm.InvalidArguments),
    (dict(cache__table_stride=(1 << 23) + 1), jm.CapabilityMismatch),
    (dict(cache__table_stride=1 << 22, cache__kv_heads=512, rows__kv_heads=512, rows__q_heads=512, rows__q_stride=1 << 16,
          rows__k_stride=1 << 16, rows__v_stride=1 << 16, out_stride=1 << 16), jm.CapabilityMismatch),
    (dict(batch__past=(1 << 20) + 2), jm.InvalidArguments),
    (dict(batch__slot=(1 << 20) + 1), jm.InvalidArguments),
    (dict(batch__row_start=(1 << 20) + 3), jm.InvalidArguments),
    (dict(rope__q_norm=(1 << 20) + 2), jm.InvalidArguments),
    (dict(rope__k_norm=(1 << 20) + 1), jm.InvalidArguments),
    (dict(max_tokens=1 << 30, batch__n_tokens=(1 << 27) + 1, batch__row_start=1 << 20), jm.CapabilityMismatch),
])
def test_check_refuses(over, error):
    with pytest.raises(error):
        _check(_args(**over))


def test_struct_sizes_match_the_header():
    assert [C.sizeof(t) for t in (jm.KvCache, jm.KvBatch, jm.Rope, jm.QkvRows, jm.AttnOpts)] == [80, 40, 56, 64, 8]


def test_quantiser_of_the_oracle():
    x = np.zeros((16, 64), np.float32)
    x[0, :4] = [127.0, 0.5, 1.5, -2.5]     # scale 1: ties go to even
    q, s = ao.quantise(x)
    assert s == 1.0 and q[0, :4].tolist() == [127, 0, 2, -2]
    x[1, :3] = [np.nan, np.inf, -np.inf]
    q, s = ao.quantise(x)
    assert s == 1.0 and q[1, :3].tolist() == [0, 127, -127]
    assert ao.quantise(np.full((16, 64), 1e-21, np.float32))[1] == 0.0


# ----------------------------------------------------------------- GPU set-up


class Setup:
    """A context, a cache and a batch on the GPU with the oracle's view of the same."""

    def __init__(self, act="f32", D=128, q_heads=8, kv_heads=2, page=32, n_slots=4, pages_per_slot=6, seed=0, poison=True):
        import torch
        self.t = torch
        self.act, self.D, self.hq, self.hk, self.page = act, D, q_heads, kv_heads, page
        self.dtype = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[act]
        self.rng = np.random.default_rng(seed)
        self.n_slots, self.stride = n_slots, pages_per_slot
        self.n_pages = n_slots * pages_per_slot + 3
        pb = page // 16
        dev = "cuda"
        # pages hold what earlier users left: any bytes, and scales that must not leak
        self.k = torch.full((self.n_pages, kv_heads, pb, D // 64, 16, 64), 99, dtype=torch.int8, device=dev)
        self.v = torch.full((self.n_pages, kv_heads, pb, D, 16), -77, dtype=torch.int8, device=dev)
        bad = float("nan") if poison else 0.0
        self.k_scale = torch.full((self.n_pages, kv_heads, pb), bad, device=dev)
        self.v_scale = torch.full((self.n_pages, kv_heads, pb), bad, device=dev)
        self.open_k = torch.full((n_slots, kv_heads, 16, D), float("nan"), device=dev)
        self.open_v = torch.full((n_slots, kv_heads, 16, D), float("nan"), device=dev)
        self.table_np = self.rng.permutation(self.n_pages)[: n_slots * pages_per_slot].reshape(n_slots, pages_per_slot)
        self.table = torch.tensor(self.table_np, dtype=torch.int32, device=dev)
        self.ctx = jm.Context(0, max_tokens=4096)
        self.ctx.set_stream(jm.STREAM_LEGACY)
        self.cache = jm.KvCache(head_dim=D, kv_heads=kv_heads, page_tokens=page, n_pages=self.n_pages, n_slots=n_slots,
                                table_stride=pages_per_slot, page_table=self.table.data_ptr(), k=self.k.data_ptr(),
                                v=self.v.data_ptr(), k_scale=self.k_scale.data_ptr(), v_scale=self.v_scale.data_ptr(),
                                open_k=self.open_k.data_ptr(), open_v=self.open_v.data_ptr())
        self.ref = ao.Cache()
        self.lens = [0] * n_slots
        self.keep = []

    def close(self):
        self.t.cuda.synchronize()
        self.ctx.close()

    def ints(self, v):
        x = self.t.tensor(v, dtype=self.t.int32, device="cuda")
        self.keep.append(x)
        return x.data_ptr()

    def batch(self, past, new, slots, behind=0, max_new=0):
        rs = np.concatenate(([0], np.cumsum(new)))
        return jm.KvBatch(n_seqs=len(past), n_tokens=int(rs[-1]) + behind, past=self.ints(list(past)),
                          row_start=self.ints(rs.tolist()), slot=self.ints(list(slots)), max_new=max_new)

    def rows(self, T, scale=1.0, pad=0):
        """Random rows of a fused projection (with `pad` 16-byte units between rows) and their f64 values."""
        t = self.t
        width = (self.hq + 2 * self.hk) * self.D + pad * (4 if self.act == "f32" else 8)
        x = t.tensor(self.rng.standard_normal((max(T, 1), width)) * scale, dtype=self.dtype, device="cuda")
        self.keep.append(x)
        a, b = self.hq * self.D, (self.hq + self.hk) * self.D
        size = x.element_size()
        r = jm.QkvRows(act=ACTS[self.act], q_heads=self.hq, kv_heads=self.hk, head_dim=self.D, q=x.data_ptr(),
                       k=x.data_ptr() + a * size, v=x.data_ptr() + b * size, q_stride=width, k_stride=width, v_stride=width)
        f = x.double().cpu().numpy()
        return r, x, f[:, :a].reshape(-1, self.hq, self.D), f[:, a:b].reshape(-1, self.hk, self.D), \
            f[:, b:b + self.hk * self.D].reshape(-1, self.hk, self.D)

    def out(self, T, heads, fill=123.0):
        x = self.t.full((max(T, 1), heads, self.D), fill, dtype=self.dtype, device="cuda")
        self.keep.append(x)
        return x

    def into(self, q=None, k=None, v=None):
        return jm.QkvRows(act=ACTS[self.act], q_heads=self.hq, kv_heads=self.hk, head_dim=self.D,
                          q=q.data_ptr() if q is not None else 0, k=k.data_ptr() if k is not None else 0,
                          v=v.data_ptr() if v is not None else 0, q_stride=self.hq * self.D, k_stride=self.hk * self.D,
                          v_stride=self.hk * self.D)

    def rope(self, rope_dim=None, interleaved=False, norm=True, **kw):
        R = self.D if rope_dim is None else rope_dim
        w = {n: (1.0 + 0.3 * self.rng.standard_normal(self.D)).astype(np.float32) for n in ("q", "k")} if norm else {}
        dev = {n: self.t.tensor(x, device="cuda") for n, x in w.items()}
        self.keep.append(dev)
        kw = {"theta": 1e6, "eps": 1e-6, **kw}
        r = jm.Rope(rope_dim=R, interleaved=interleaved, q_norm=dev["q"].data_ptr() if norm else 0,
                    k_norm=dev["k"].data_ptr() if norm else 0, **kw)

        def plain(x, which, pos):
            return ao.norm_rope(x, w.get(which), pos, R, interleaved, theta=kw["theta"], eps=kw["eps"],
                                mscale=kw.get("mscale", 1.0), inv_freq=kw.get("inv_freq"))
        return r, plain

    def append(self, past, new, slots, rope=None, plain=None, rows=None, behind=0):
        """Appends random rows on both sides; the oracle takes keys rounded to f32 as the library does."""
        T = int(np.sum(new))
        r, x, q, k, v = rows or self.rows(T + behind)
        b = self.batch(past, new, slots, behind)
        self.ctx.kv_append(self.cache, b, rope, r)
        at = 0
        for p, n, s in zip(past, new, slots):
            if n:
                kk = k[at:at + n] if plain is None else plain(k[at:at + n], "k", p + np.arange(n))
                self.ref.append(s, p, kk, v[at:at + n])
                self.lens[s] = p + n
            at += n
        return b, r, q

    def device_blocks(self, slot):
        """(kq, ks, vq, vs) of a slot as the oracle's blocks() lays them out."""
        n = self.lens[slot]
        nb = -(-n // 16)
        pb = self.page // 16
        blocks = np.arange(nb)
        pages = self.t.tensor(self.table_np[slot][blocks // pb], device="cuda")
        at = self.t.tensor(blocks % pb, device="cuda")
        kq = self.k[pages, :, at].permute(1, 0, 3, 2, 4).reshape(self.hk, nb, 16, self.D).cpu().numpy()
        vq = self.v[pages, :, at].permute(1, 0, 3, 2).cpu().numpy()
        ks, vs = (s[pages, :, at].t().cpu().numpy() for s in (self.k_scale, self.v_scale))
        return kq, ks, vq, vs

    def check_blocks(self, slot, exact_keys=False):
        kq, ks, vq, vs = self.device_blocks(slot)
        rq, rs = self.ref.blocks(slot, "v")
        np.testing.assert_array_equal(vq, rq)
        np.testing.assert_array_equal(vs, rs)
        rq, rs = self.ref.blocks(slot, "k")
        if exact_keys:
            np.testing.assert_array_equal(kq, rq)
            np.testing.assert_array_equal(ks, rs)
            return
        # numpy's and the device's f64 functions may differ in the last place, which
        # the rounding to f32 shows once in some 10^8 values: scales within one ulp of
        # f32 (and its rounding), values within one step and all but never off
        assert np.all(np.abs(ks.astype(np.float64) - rs) <= 4 * U * rs)
        d = np.abs(kq.astype(int) - rq.astype(int))
        assert d.max(initial=0) <= 1 and np.count_nonzero(d) <= 1 + kq.size // 100000

    def check_attention(self, got, q, past, new, slots, scale=None, window=0, q_err=0.0, bad=()):
        """got [T, hq, D] f64 against the oracle over the device's own cache bits."""
        scale = scale or 1.0 / np.sqrt(self.D)
        at = 0
        for p, n, s in zip(past, new, slots):
            if not n:
                continue
            kq, ks, vq, vs = self.device_blocks(s)
            o, A, vmax = ao.attend(q[at:at + n], kq, ks, vq, vs, p, scale, window, bad)
            L = p + n
            logit = A * (2.0 ** -22 + (self.D + 8) * U + q_err)
            part = 2 * logit + 2.0 ** -21 + (2.0 ** -22 if self.act == "f32" else 2.0 ** -11) + (L + 64) * U
            tol = 2 * part * vmax + HALF_STEP[self.act] * np.abs(o)
            err = np.abs(got[at:at + n] - o)
            assert np.all(err <= tol), (s, float((err - tol).max()), float(err.max()), float(np.min(tol)))
            at += n

    def attend(self, past, new, slots, q=None, rows=None, opts=None, behind=0, max_new=0, scale=None, window=0, bad=()):
        T = int(np.sum(new))
        if rows is None:
            rows, _, q, _, _ = self.rows(T + behind)
        out = self.out(T + behind, self.hq)
        opts = opts or jm.AttnOpts(window=window, scale=scale or 0.0)
        self.ctx.kv_attention(self.cache, self.batch(past, new, slots, behind, max_new), opts, rows, out.data_ptr(),
                              self.hq * self.D)
        got = out.double().cpu().numpy()
        self.check_attention(got[:T], q, past, new, slots, scale, window, bad=bad)
        assert np.all(got[T:T + behind] == 123.0), "rows behind the last sequence were written"
        return got


@pytest.fixture
def make():
    made = []

    def f(*a, **kw):
        made.append(Setup(*a, **kw))
        return made[-1]
    yield f
    for s in made:
        s.close()


# ----------------------------------------------------------- norm and rotation


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,R,interleaved,norm", [(128, 128, False, True), (64, 64, True, True), (128, 64, True, False),
                                                  (128, 2, False, True), (64, 0, False, True), (128, 0, False, False),
                                                  (64, 34, False, True)])
def test_norm_rope(make, act, D, R, interleaved, norm):
    s = make(act, D=D, q_heads=6, kv_heads=3)
    rope, plain = s.rope(R, interleaved, norm, mscale=1.25)
    past, new = [0, 5, 1 << 20, 130], [1, 0, 7, 3]
    r, x, q, k, _ = s.rows(13, pad=1)
    oq, ok = s.out(13, s.hq), s.out(13, s.hk)
    s.ctx.qk_norm_rope(s.batch(past, new, range(4), behind=2), rope, r, s.into(oq, ok))
    pos = np.concatenate([p + np.arange(n) for p, n in zip(past, new)])
    for got, x, which in ((oq, q, "q"), (ok, k, "k")):
        ref = plain(x[:11], which, pos)
        got = got.double().cpu().numpy()
        size = 2 * np.max(np.abs(ref), axis=-1, keepdims=True) * np.sqrt(2.0)   # at least |a| + |b| of any pair
        assert np.all(np.abs(got[:11] - ref) <= 24 * U * size + HALF_STEP[act] * np.abs(ref) * (1 + 2 ** -7))
        assert np.all(got[11:] == 123.0)


@pytest.mark.gpu
def test_norm_rope_in_place_and_one_tensor(make):
    s = make("f32")
    rope, plain = s.rope()
    r, x, q, k, _ = s.rows(5)
    b = jm.KvBatch(n_seqs=5, n_tokens=5, past=s.ints([3, 1, 4, 1, 5]))
    before = x.clone()
    only_k = jm.QkvRows(**{f: getattr(r, f) for f, _ in r._fields_})
    only_k.q = None
    s.ctx.qk_norm_rope(b, rope, only_k, only_k)
    ref = plain(k, "k", [3, 1, 4, 1, 5])
    a, e = s.hq * s.D, (s.hq + s.hk) * s.D
    got = x[:, a:e].double().cpu().numpy().reshape(ref.shape)
    assert np.all(np.abs(got - ref) <= 24 * U * 4 * np.max(np.abs(ref), axis=-1, keepdims=True))
    assert s.t.equal(x[:, :a], before[:, :a]) and s.t.equal(x[:, e:], before[:, e:])


@pytest.mark.gpu
def test_norm_rope_given_frequencies_far_positions(make):
    """Angles of far positions: a frequency of 1 at position 2^30 turns by 2^30 radians."""
    s = make("f32", D=64)
    f = 1.0 / (1.0 + np.arange(32))
    rope, plain = s.rope(64, False, False, inv_freq=f)
    pos = [1 << 30, (1 << 30) + 1, 7]
    r, x, q, k, _ = s.rows(3)
    oq, ok = s.out(3, s.hq), s.out(3, s.hk)
    s.ctx.qk_norm_rope(jm.KvBatch(n_seqs=3, n_tokens=3, past=s.ints(pos)), rope, r, s.into(oq, ok))
    ref = plain(q, "q", pos)
    # numpy reduces 2^30 radians exactly; the angle itself is a product in f64: 2^30 * 2^-53 = 2^-23
    size = np.max(np.abs(q), axis=-1, keepdims=True) * 2
    assert np.all(np.abs(oq.double().cpu().numpy() - ref) <= (24 * U + 2.0 ** -22) * size)


# ------------------------------------------------------------------ the cache


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,page", [(128, 32), (64, 16), (128, 256)])
def test_append_blocks_are_the_tokens_own(make, act, D, page):
    """Histories built by different splits hold the same bits, the oracle's, open blocks among them."""
    n = 83
    splits = [[n], [1] * n, [16, 16, 51], [5, 11, 1, 15, 33, 18]]
    s = make(act, D=D, page=page, pages_per_slot=-(-96 // page) + 1)
    rope, plain = s.rope(D // 2, True)
    r, x, q, k, v = s.rows(n)
    size = x.element_size()
    for slot, parts in enumerate(splits):
        past = 0
        for m in parts:
            rr = jm.QkvRows(**{f: getattr(r, f) for f, _ in r._fields_})
            for name in ("q", "k", "v"):
                setattr(rr, name, getattr(r, name) + past * r.q_stride * size)
            s.append([past], [m], [slot], rope, plain, rows=(rr, x, q[past:], k[past:], v[past:]))
            past += m
    first = s.device_blocks(0)
    s.check_blocks(0)
    for slot in range(1, 4):
        for a, b in zip(first, s.device_blocks(slot)):
            np.testing.assert_array_equal(a, b)
    want_k, want_v = (np.asarray(x[0][80:83]) for x in ([s.ref.k[0]], [s.ref.v[0]]))
    for slot in range(4):
        got_k, got_v = (o[slot, :, :3].transpose(0, 1).cpu().numpy() for o in (s.open_k, s.open_v))
        np.testing.assert_allclose(got_k, want_k, rtol=4 * U, atol=0)
        np.testing.assert_array_equal(got_v, want_v)
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
def test_append_ragged_batch_strided_rows(make):
    s = make("bf16", q_heads=3, kv_heads=3, D=64, page=16, n_slots=6, pages_per_slot=20)
    rope, plain = s.rope()
    lens = {4: 0, 1: 0, 5: 0, 0: 0, 2: 0}
    for step in range(4):
        slots = [4, 1, 5, 0, 2]
        new = s.rng.integers(0, 60, 5).tolist() if step else [0, 16, 1, 17, 100]
        r = s.rows(sum(new) + 3, pad=step)
        s.append([lens[i] for i in slots], new, slots, rope, plain, rows=r, behind=3)
        for i, n in zip(slots, new):
            lens[i] += n
    untouched = s.k_scale.clone()
    for i, n in lens.items():
        if n:
            s.check_blocks(i)
    assert np.isnan(untouched[s.table[3].long()].cpu().numpy()).all(), "an unused slot's pages were written"
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
def test_append_odd_values(make):
    """NaN, infinities, zeros, tiny blocks and ties of the rounding, without norm or rotation."""
    s = make("f32", D=64, q_heads=2, kv_heads=2)
    r, x, q, k, v = s.rows(40)
    a, b = s.hq * s.D, (s.hq + s.hk) * s.D
    x[16:32] = 0.0
    x[32:, a:b] *= 1e-22
    x[0, a] = float("nan")
    x[1, a + 1] = float("inf")
    x[2, b] = -float("inf")
    x[3, b + 1] = float("nan")
    x[:16, b + 64:] = s.t.tensor(np.resize(np.arange(-127, 128) / 2.0, (16, 64)), device="cuda", dtype=s.dtype)
    x[0, b + 64] = 127.0
    f = x.double().cpu().numpy()
    k, v = f[:, a:b].reshape(-1, 2, 64), f[:, b:].reshape(-1, 2, 64)
    s.append([0], [40], [2], rows=(r, x, q, k, v))
    s.check_blocks(2, exact_keys=True)
    kq, ks, vq, vs = s.device_blocks(2)
    assert ks[:, 1].tolist() == [0, 0] and ks[:, 2].tolist() == [0, 0] and vs[1, 0] == 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_read_rounds_once(make, act):
    s = make(act, D=128, page=64)
    s.append([0, 0], [70, 33], [3, 1], rows=s.rows(103))
    ok, ov = s.out(50, s.hk), s.out(50, s.hk)
    s.ctx.kv_read(s.cache, s.batch([21, 3], [30, 18], [3, 1], behind=2), s.into(k=ok, v=ov))
    at = 0
    for slot, lo, n in ((3, 21, 30), (1, 3, 18)):
        kq, ks, vq, vs = s.device_blocks(slot)
        for got, qv, sc in ((ok, kq, ks), (ov, vq, vs)):
            val = (qv.astype(np.float32) * sc[..., None, None]).reshape(s.hk, -1, s.D)[:, lo:lo + n].transpose(1, 0, 2)
            want = s.t.tensor(val).to(s.dtype)
            assert s.t.equal(got[at:at + n].cpu(), want)
        at += n
    assert np.all(ok[48:].double().cpu().numpy() == 123.0)
    alone = s.out(1, s.hk)
    s.ctx.kv_read(s.cache, s.batch([21], [1], [3]), s.into(v=alone))
    assert s.t.equal(alone[0], ov[0])


# ------------------------------------------------------------------ attention


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,hq,hk,page", [(128, 8, 1, 64), (64, 14, 2, 16), (128, 2, 2, 32), (64, 16, 1, 128),
                                          (128, 15, 3, 16), (128, 33, 1, 64)])
def test_attention_lengths(make, act, D, hq, hk, page):
    """Single tokens, drafts and prompts over histories around block, page and tile ends."""
    s = make(act, D=D, q_heads=hq, kv_heads=hk, page=page, n_slots=8, pages_per_slot=-(-448 // page))
    total = [1, 2, 15, 16, 17, 64, 129, 300]
    s.append([0] * 8, total, range(8), rows=s.rows(sum(total)))
    for new in ([1] * 8, [1, 2, 3, 5, 8, 9, 17, 33], [1, 0, 15, 16, 1, 64, 129, 300]):
        slots = s.rng.permutation(8)
        n = [new[i] for i in slots]
        s.attend([total[i] - new[i] for i in slots], n, slots, behind=2, max_new=max(n))
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 2, 16, 63, 100, 10000])
def test_attention_window(make, act, window):
    s = make(act, D=64, q_heads=4, kv_heads=2, page=16, n_slots=3, pages_per_slot=20)
    total = [300, 77, 16]
    s.append([0] * 3, total, range(3), rows=s.rows(sum(total)))
    # blocks that no row sees hold poison
    for i, t in enumerate(total):
        for b in range(max(0, t - 30 - window + 1) // 16):
            s.k_scale[int(s.table_np[i][b]), :, 0] = float("nan")
            s.v_scale[int(s.table_np[i][b]), :, 0] = float("inf")
    blocks = s.device_blocks

    def clean(slot):
        return tuple(np.nan_to_num(x, nan=0.0, posinf=0.0) for x in blocks(slot))
    s.device_blocks = clean
    for new in ([1, 1, 1], [30, 9, 16]):
        s.attend([t - n for t, n in zip(total, new)], new, range(3), window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_attention_long_history_and_extreme_scales(make, act):
    """Work split over a long history; heads whose value blocks differ by orders of magnitude."""
    s = make(act, D=128, q_heads=8, kv_heads=2, page=64, n_slots=2, pages_per_slot=70)
    n = 4000
    r, x, q, k, v = s.rows(n)
    b = (s.hq + s.hk) * s.D
    gain = np.ones((n, 1), np.float32)
    gain[::3] = 1e-3
    gain[512:1024] = 1e-4 if act == "f16" else 1e-7
    gain[2000:2500] = 30.0 if act == "f16" else 1e6
    gain[3000:3100] = 0.0
    x[:, b:b + s.D] *= s.t.tensor(gain, device="cuda", dtype=s.dtype)
    f = x.double().cpu().numpy()
    v = f[:, b:].reshape(-1, 2, 128)
    s.append([0], [n], [1], rows=(r, x, q, k, v))
    s.check_blocks(1, exact_keys=True)
    s.attend([n - 1], [1], [1])
    s.attend([n - 6], [6], [1])
    s.attend([700], [1], [1])
    s.attend([n - 1], [1], [1], scale=3.0)


@pytest.mark.gpu
def test_attention_extreme_queries(make):
    """Queries beyond half precision's range and a head of zeros."""
    s = make("f32", D=64, q_heads=4, kv_heads=2, n_slots=1, pages_per_slot=8)
    s.append([0], [200], [0], rows=s.rows(200))
    r, x, q, _, _ = s.rows(3)
    x[0, :64] *= 1e7
    x[1, 64:128] = 0.0
    x[2, 128:192] *= 1e-9
    q = x[:, : 4 * 64].double().cpu().numpy().reshape(3, 4, 64)
    s.attend([197], [3], [0], q=q, rows=r, scale=1e-6)
    s.attend([197], [3], [0], q=q, rows=r, scale=1e-2)


@pytest.mark.gpu
def test_attention_bad_entries_are_skipped_and_reported(make):
    s = make("f32", D=64, q_heads=4, kv_heads=2, page=16, n_slots=4, pages_per_slot=8)
    total = [100, 60, 30, 20]
    s.append([0] * 4, total, range(4), rows=s.rows(sum(total)))
    assert s.ctx.device_status() == 0

    def status():
        with pytest.raises(jm.TensorBoundsError):
            s.ctx.device_status()
        assert s.ctx.device_status() == 0

    # page ids out of range: those blocks count as absent; a row that sees no other gets zeros
    good = s.table.clone()
    s.table[0, 2] = -1
    s.table[0, 4] = s.n_pages
    s.attend([99], [1], [0], bad=(2, 4))
    status()
    s.attend([40], [60], [0], bad=(2, 4), max_new=60)
    status()
    s.table[3, :2] = 1 << 30
    r, _, q, _, _ = s.rows(2)
    out = s.out(2, s.hq)
    s.ctx.kv_attention(s.cache, s.batch([19, 59], [1, 1], [3, 1]), None, r, out.data_ptr(), s.hq * s.D)
    got = out.double().cpu().numpy()
    assert np.all(got[0] == 0.0)
    s.check_attention(got[1:], q[1:], [59], [1], [1])
    status()
    s.table.copy_(good)
    # sequences out of range are passed over, the others computed
    for past, new, slots in (([99, 59, 29], [1, 1, 1], [0, 4, 2]), ([99, 59, 29], [1, 1, 1], [0, -1, 2]),
                             ([99, -1, 29], [1, 1, 1], [0, 1, 2]), ([99, 8 * 16, 29], [1, 1, 1], [0, 1, 2]),
                             ([99, 2147483647, 29], [1, 1, 1], [0, 1, 2])):
        r, _, q, _, _ = s.rows(3)
        out = s.out(3, s.hq)
        s.ctx.kv_attention(s.cache, s.batch(past, new, slots), None, r, out.data_ptr(), s.hq * s.D)
        got = out.double().cpu().numpy()
        assert np.all(got[1] == 123.0)
        s.check_attention(got[:1], q[:1], [99], [1], [0])
        s.check_attention(got[2:], q[2:], [29], [1], [2])
        status()
    # more rows than max_new, rows past the end, rows that go back
    r, _, q, _, _ = s.rows(4)
    out = s.out(4, s.hq)
    for rs, n in (([0, 3, 4], 2), ([0, 5, 4], 4), ([-1, 3, 4], 4)):
        b = jm.KvBatch(n_seqs=2, n_tokens=4, past=s.ints([0, 59]), row_start=s.ints(rs), slot=s.ints([2, 1]), max_new=n)
        out.fill_(123.0)
        s.ctx.kv_attention(s.cache, b, None, r, out.data_ptr(), s.hq * s.D)
        got = out.double().cpu().numpy()
        assert np.all(got[:3] == 123.0)
        status()


@pytest.mark.gpu
def test_append_and_read_bad_entries(make):
    s = make("f32", D=64, q_heads=2, kv_heads=2, page=16, n_slots=4, pages_per_slot=4)
    s.append([0], [20], [0], rows=s.rows(20))

    def status():
        with pytest.raises(jm.TensorBoundsError):
            s.ctx.device_status()
        assert s.ctx.device_status() == 0

    state = [t.clone() for t in (s.k, s.v, s.k_scale, s.open_k)]
    for past, new, slots in (([20], [1], [4]), ([20], [1], [-1]), ([60], [5], [0]), ([-3], [1], [0])):
        r = s.rows(sum(new))[0]
        s.ctx.kv_append(s.cache, s.batch(past, new, slots), None, r)
        status()
        for a, b in zip(state, (s.k, s.v, s.k_scale, s.open_k)):
            assert s.t.equal(a.nan_to_num(-5.0), b.nan_to_num(-5.0))
        ok = s.out(sum(new), 2)
        s.ctx.kv_read(s.cache, s.batch(past, new, slots), s.into(k=ok))
        status()
        assert np.all(ok.double().cpu().numpy() == 123.0)
    # a slot twice: the first is appended, the second passed over
    r, x, q, k, v = s.rows(4)
    s.ctx.kv_append(s.cache, s.batch([20, 0, 22], [2, 1, 1], [0, 1, 0]), None, r)
    status()
    s.ref.append(0, 20, k[:2], v[:2])
    s.ref.append(1, 0, k[2:3], v[2:3])
    s.lens[0], s.lens[1] = 22, 1
    s.check_blocks(0, exact_keys=True)
    s.check_blocks(1, exact_keys=True)
    # a page out of range: its tokens are not held, the others are
    s.table[2, 1] = 99
    r, x, q, k, v = s.rows(40)
    s.ctx.kv_append(s.cache, s.batch([0], [40], [2]), None, r)
    status()
    ok = s.out(40, 2)
    s.ctx.kv_read(s.cache, s.batch([0], [40], [2]), s.into(k=ok))
    status()
    got = ok.double().cpu().numpy()
    assert np.all(got[16:32] == 0.0) and np.all(np.abs(got[:16] - k[:16]) < 0.05) and np.all(np.abs(got[32:] - k[32:]) < 0.05)


# ------------------------------------------------------------ the whole step


@pytest.mark.gpu
@pytest.mark.parametrize("act,D,hq,hk,page", [("f32", 128, 8, 2, 64), ("bf16", 64, 14, 2, 16), ("f16", 128, 4, 4, 32)])
def test_attention_step_prompts_then_decode(make, act, D, hq, hk, page):
    """Ragged prompts, then single tokens and drafts, through moe_attention."""
    s = make(act, D=D, q_heads=hq, kv_heads=hk, page=page, n_slots=4, pages_per_slot=-(-256 // page))
    rope, plain = s.rope(D, D == 64)
    lens = [0, 0, 0, 0]
    for step, new in enumerate(([37, 150, 1, 0], [1, 1, 1, 20], [4, 1, 0, 1]) + tuple([1, 1, 1, 1] for _ in range(6))):
        T = sum(new)
        r, x, q, k, v = s.rows(T, pad=step % 2)
        out = s.out(T, hq)
        s.ctx.attention(s.cache, s.batch(lens, new, range(4)), rope, None, r, out.data_ptr(), hq * D)
        got = out.double().cpu().numpy()
        at, qr = 0, []
        for i, n in enumerate(new):
            if n:
                pos = lens[i] + np.arange(n)
                s.ref.append(i, lens[i], plain(k[at:at + n], "k", pos), v[at:at + n])
                qr.append(plain(q[at:at + n], "q", pos))
                s.lens[i] = lens[i] + n
                s.check_blocks(i)
            at += n
        qr = np.concatenate(qr)
        s.check_attention(got, qr, lens, new, range(4), q_err=48 * U)
        lens = [a + b for a, b in zip(lens, new)]
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
def test_decoder_layers_attention_then_ffn():
    """Attention and the FFN sublayer in turn on one context, as a decoder layer runs them:
    the FFN's results are those of a context of its own."""
    import torch
    import synth
    cfg = synth.CONFIGS[2].scaled(E=16, I=256, H=512)
    w = synth.build_weights(cfg)
    s = Setup("f32", D=64, q_heads=8, kv_heads=2, n_slots=3)
    d, keep = synth.desc_for(cfg, w)
    alone = jm.Context(0, 8, 1)
    for c in (s.ctx, alone):
        c.upload(0, d)
        c.set_ffn_norm(0, None, 1e-6)
    rope, plain = s.rope()
    past = [0, 0, 0]
    hidden = torch.from_numpy(synth.gen_x(cfg, 3)).cuda()
    for step in range(5):
        r, x, q, k, v = s.rows(3)
        out = s.out(3, 8)
        b = s.batch(past, [1, 1, 1], range(3))
        s.ctx.attention(s.cache, b, rope, None, r, out.data_ptr(), 512)
        after = hidden + 0.1 * out.view(3, 512)
        torch.cuda.synchronize()
        got = torch.empty_like(after)
        s.ctx.forward_block_ptrs(0, 3, after.data_ptr(), got.data_ptr())
        torch.cuda.synchronize()
        ref, _, _ = alone.forward_block(0, after.cpu().numpy())
        np.testing.assert_array_equal(got.cpu().numpy(), ref)
        pos = np.array(past)
        for i in range(3):
            s.ref.append(i, past[i], plain(k[i:i + 1], "k", pos[i:i + 1]), v[i:i + 1])
            s.lens[i] = past[i] + 1
        s.check_attention(out.double().cpu().numpy(), plain(q, "q", pos), past, [1] * 3, range(3), q_err=48 * U)
        past = [p + 1 for p in past]
        hidden = got
    assert s.ctx.device_status() == 0
    alone.close()
    s.close()


@pytest.mark.gpu
def test_captured_step_replays_over_growing_histories(make):
    """One graph of the step, replayed while the batch's past counts, rows and page table move on."""
    import torch
    s = make("f32", D=128, q_heads=8, kv_heads=2, page=16, n_slots=3, pages_per_slot=10)
    rope, plain = s.rope()
    stream = torch.cuda.Stream()
    past = torch.tensor([0, 40, 70], dtype=torch.int32, device="cuda")
    s.append([0, 0], [40, 70], [1, 2], rope, plain)
    r, x, _, _, _ = s.rows(3)
    out = s.out(3, 8)
    batch = jm.KvBatch(n_seqs=3, n_tokens=3, past=past.data_ptr())
    torch.cuda.synchronize()
    s.ctx.set_stream(stream.cuda_stream)
    fresh = jm.Context(0, max_tokens=8)
    fresh.set_stream(stream.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        with pytest.raises(jm.InvalidArguments):      # a context's first call allocates: refused while capturing
            fresh.attention(s.cache, batch, rope, None, r, out.data_ptr(), 1024)
        s.ctx.attention(s.cache, batch, rope, None, r, out.data_ptr(), 1024)
    fresh.close()
    for step in range(20):
        x.copy_(torch.tensor(s.rng.standard_normal(tuple(x.shape)), dtype=s.dtype))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        f = x.double().cpu().numpy()
        q, k, v = (f[:, a * 128:b * 128].reshape(3, -1, 128) for a, b in ((0, 8), (8, 10), (10, 12)))
        pos = past.cpu().numpy()
        for i in range(3):
            s.ref.append(i, int(pos[i]), plain(k[i:i + 1], "k", pos[i:i + 1]), v[i:i + 1])
            s.lens[i] = int(pos[i]) + 1
            s.check_blocks(i)
        s.check_attention(out.double().cpu().numpy(), plain(q, "q", pos), pos.tolist(), [1] * 3, range(3), q_err=48 * U)
        past += 1
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
def test_results_do_not_change_between_runs(make):
    s = make("bf16", D=128, q_heads=32, kv_heads=4, page=64, n_slots=5, pages_per_slot=40)
    total = [2500, 3, 700, 64, 1999]
    s.append([0] * 3, total[:3], range(3), rows=s.rows(sum(total[:3])))
    s.append([0] * 2, total[3:], [3, 4], rows=s.rows(sum(total[3:])))
    for new in ([1] * 5, [70, 3, 5, 1, 200]):
        r = s.rows(sum(new))[0]
        b = s.batch([t - n for t, n in zip(total, new)], new, range(5))
        first = None
        for _ in range(4):
            out = s.out(sum(new), 32)
            s.ctx.kv_attention(s.cache, b, None, r, out.data_ptr(), 32 * 128)
            first = out if first is None else first
            assert s.t.equal(first, out)


@pytest.mark.gpu
def test_two_contexts_on_two_streams(make):
    """Contexts have workspaces of their own: calls at once on two streams give what they give alone."""
    import torch
    s = make("f32", D=128, q_heads=8, kv_heads=2, page=64, n_slots=2, pages_per_slot=60)
    s.append([0], [3500], [0], rows=s.rows(3500))
    s.append([0], [3000], [1], rows=s.rows(3000))
    other = jm.Context(0, max_tokens=64)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    work = []
    for i, ctx in enumerate((s.ctx, other)):
        r, _, q, _, _ = s.rows(1)
        work.append((ctx, s.batch([s.lens[i] - 1], [1], [i]), r, s.out(1, 8), q))
    torch.cuda.synchronize()
    for (ctx, b, r, out, q), st in zip(work, streams):
        ctx.set_stream(st.cuda_stream)
    for _ in range(20):
        for ctx, b, r, out, q in work:
            ctx.kv_attention(s.cache, b, None, r, out.data_ptr(), 1024)
    torch.cuda.synchronize()
    for i, (ctx, b, r, out, q) in enumerate(work):
        s.check_attention(out.double().cpu().numpy(), q, [s.lens[i] - 1], [1], [i])
    other.close()


# ------------------------------------------------------- batches at the edges


@pytest.mark.gpu
@pytest.mark.parametrize("act,hq", [("f32", 8), ("bf16", 16), ("f16", 64)])
def test_attention_of_more_sequences_than_lanes(make, act, hq):
    """70 sequences (a plan of several passes) of 8 key heads, more segments than CTAs: runs cross segments."""
    s = make(act, D=64, q_heads=hq, kv_heads=8, page=16, n_slots=70, pages_per_slot=12)
    total = [1 + (37 * i) % 190 for i in range(70)]
    s.append([0] * 30, total[:30], range(30), rows=s.rows(sum(total[:30])))
    s.append([0] * 40, total[30:], range(30, 70), rows=s.rows(sum(total[30:])))
    order = s.rng.permutation(70).tolist()
    past = [total[i] - 1 for i in order]
    s.attend(past, [1] * 70, order, max_new=1)
    new = [min(total[i], (i * 5) % 4) for i in order]
    s.attend([total[i] - n for i, n in zip(order, new)], new, order, behind=2)
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_attention_single_tokens_and_prompts_in_one_call(make, act):
    s = make(act, D=128, q_heads=8, kv_heads=2, page=32, n_slots=6, pages_per_slot=16)
    total = [400, 130, 77, 1, 500, 300]
    s.append([0] * 6, total, range(6), rows=s.rows(sum(total)))
    new = [1, 100, 0, 1, 5, 300]
    for scale in (None, -0.05):
        s.attend([t - n for t, n in zip(total, new)], new, range(6), behind=3, scale=scale)
    s.attend([t - n for t, n in zip(total, new)], new, range(6), window=50, max_new=300)
    s.attend([t - 1 for t in total], [1] * 6, range(6), scale=-0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_attention_prompts_past_the_workspace(make, act):
    """More query rows than the workspace takes at once: several passes over the list."""
    n = 24 if act == "f32" else 46
    s = make(act, D=128, q_heads=32, kv_heads=32, page=16, n_slots=n, pages_per_slot=6)
    new = [65 + i % 7 for i in range(n)]
    s.append([0] * n, new, range(n), rows=s.rows(sum(new)))
    s.attend([0] * n, new, range(n))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("D,R,interleaved", [(128, 34, False), (64, 2, False), (128, 6, True), (64, 50, False)])
def test_step_with_odd_rotations(make, act, D, R, interleaved):
    """Pairs that do not lie lane by lane, through the append, few rows and many."""
    s = make(act, D=D, q_heads=6, kv_heads=2, page=16, n_slots=2, pages_per_slot=16)
    rope, plain = s.rope(rope_dim=R, interleaved=interleaved, mscale=1.25)
    past = [0, 0]
    for new in ([70, 3], [1, 1], [90, 30], [2, 1]):
        r, x, q, k, v = s.rows(sum(new))
        out = s.out(sum(new), 6)
        s.ctx.attention(s.cache, s.batch(past, new, [1, 0]), rope, None, r, out.data_ptr(), 6 * D)
        at, want = 0, np.empty(q.shape)
        for i, slot in enumerate((1, 0)):
            pos = past[i] + np.arange(new[i])
            rows = slice(at, at + new[i])
            s.ref.append(slot, past[i], plain(k[rows], "k", pos), v[rows])
            want[rows] = plain(q[rows], "q", pos)
            at += new[i]
            past[i] += new[i]
            s.lens[slot] = past[i]
            s.check_blocks(slot)
        # a query value is off by 24 u (|a| + |b|) <= 34 u of its turned pair's length; over a logit's products with
        # a key's pairs that is at most 48 u |q| |k|, and the largest sum |q_d k_d| of these normal rows is near
        # 2 / pi |q| |k|: more than an eighth of it
        s.check_attention(out.double().cpu().numpy(), want, [p - n for p, n in zip(past, new)], new, [1, 0], q_err=8 * 48 * U)
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
def test_append_infinite_keys_turn(make):
    """A pair with an infinite value turns into infinite values: bytes of +-127, the rest of the block untouched by them."""
    s = make("f32", D=64, q_heads=2, kv_heads=1, page=16, n_slots=1, pages_per_slot=4)
    rope, plain = s.rope(norm=False, theta=100.0)
    r, x, q, k, v = s.rows(20)
    x[5, 2 * 64 + 3] = float("inf")
    x[17, 2 * 64 + 60] = float("-inf")
    k = x.double().cpu().numpy()[:, 128:192].reshape(20, 1, 64)
    s.append([0], [20], [0], rope, plain, rows=(r, x, q, k, v))
    assert np.count_nonzero(np.isinf(s.ref.k[0])) == 4
    s.check_blocks(0)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_window_over_freed_pages(make, act):
    """Pages before every row's window may have left the page table."""
    s = make(act, D=64, q_heads=8, kv_heads=2, page=32, n_slots=2, pages_per_slot=20)
    total = [600, 333]
    s.append([0, 0], total, [0, 1], rows=s.rows(sum(total)))
    for new, window in (([1, 1], 64), ([4, 2], 100), ([40, 90], 33)):
        for i, (t, n) in enumerate(zip(total, new)):
            s.table[i, : max(0, t - n - window + 1) // 32] = -1
        s.attend([t - n for t, n in zip(total, new)], new, [0, 1], window=window)
        s.table.copy_(s.t.tensor(s.table_np, dtype=s.t.int32))
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_row_starts_out_of_order(make, act):
    """Reported, and nothing outside the batch's rows is written; the call after it is right."""
    s = make(act, D=64, q_heads=2, kv_heads=2, page=32, n_slots=10, pages_per_slot=20)
    s.append([0], [600], [6], rows=s.rows(600))
    r, _, _, _, _ = s.rows(600)
    for starts in ([-9000] * 6 + [300, 600, -9000, 0, 0], [0, 600, 0, 600, 0, 600, 0, 600, 0, 600, 0],
                   [600, 500, 400, 300, 200, 100, 0, 600, 7, 5, 600], [2 ** 31 - 1, -2 ** 31] * 5 + [600]):
        b = jm.KvBatch(n_seqs=10, n_tokens=600, past=s.ints([0] * 10), row_start=s.ints(starts))
        out = s.out(3 * 9100, 2)
        before = [x.clone() for x in (s.k, s.k_scale)]
        s.ctx.kv_attention(s.cache, b, None, r, out[9100:].data_ptr(), 128)
        with pytest.raises(jm.TensorBoundsError):
            s.ctx.device_status()
        assert bool((out[:9100] == 123.0).all()) and bool((out[9700:] == 123.0).all())
        q2, k2 = s.out(9100 * 3, 2), s.out(9100 * 3, 2)
        rope, _ = s.rope()
        s.ctx.qk_norm_rope(b, rope, r, s.into(q2[9100:], k2[9100:]))
        with pytest.raises(jm.TensorBoundsError):
            s.ctx.device_status()
        s.ctx.kv_read(s.cache, b, s.into(k=k2[9100:]))
        with pytest.raises(jm.TensorBoundsError):
            s.ctx.device_status()
        for x in (q2, k2):
            assert bool((x[:9100] == 123.0).all()) and bool((x[9700:] == 123.0).all())
        assert all(s.t.equal(a.view(s.t.uint8), b.view(s.t.uint8)) for a, b in zip(before, (s.k, s.k_scale)))
    other = s.table[6].clone()
    s.table[6] = min(set(range(s.n_pages)) - set(s.table_np.flat))   # the appends below fill a page that nothing else has
    for starts in ([-9000] * 6 + [300, 600, -9000, 0, 0], [600, 500, 400, 300, 200, 100, 0, 600, 7, 5, 600]):
        b = jm.KvBatch(n_seqs=10, n_tokens=600, past=s.ints([0] * 10), row_start=s.ints(starts))
        s.ctx.kv_append(s.cache, b, None, r)
        with pytest.raises(jm.TensorBoundsError):
            s.ctx.device_status()
    s.table[6] = other
    s.attend([500], [100], [6])
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
def test_two_graphs_share_a_context(make):
    """Graphs of single tokens and of prompts, captured from one context, replayed in turn many times."""
    import torch
    s = make("bf16", D=128, q_heads=16, kv_heads=4, page=64, n_slots=4, pages_per_slot=40)
    total = [2400, 900, 64, 2000]
    s.append([0, 0], total[:2], [0, 1], rows=s.rows(3300))
    s.append([0, 0], total[2:], [2, 3], rows=s.rows(2064))
    work = []
    for new in ([1] * 4, [200, 100, 0, 3]):
        T = sum(new)
        r, _, q, _, _ = s.rows(T)
        past = [t - n for t, n in zip(total, new)]
        work.append((s.batch(past, new, range(4), max_new=max(new)), r, s.out(T, 16), q, past, new))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    s.ctx.set_stream(stream.cuda_stream)
    graphs = []
    for b, r, out, _, _, _ in work:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            s.ctx.kv_attention(s.cache, b, None, r, out.data_ptr(), 16 * 128)
        graphs.append(g)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(20):
            for g in graphs:
                g.replay()
    torch.cuda.synchronize()
    for _, _, out, q, past, new in work:
        s.check_attention(out.double().cpu().numpy(), q, past, new, range(4))
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,hq,hk,page,window", [(128, 4, 4, 32, 0), (64, 3, 1, 16, 0), (128, 7, 1, 64, 100), (64, 16, 2, 128, 33),
                                                 (128, 2, 1, 256, 1)])
def test_attention_of_long_prompts(make, act, D, hq, hk, page, window):
    """More rows than the runs over the cache take: 256 rows at a time, whole and ragged ones, with and without a history."""
    g = hq // hk
    s = make(act, D=D, q_heads=hq, kv_heads=hk, page=page, n_slots=3, pages_per_slot=-(-1400 // page))
    new = [520 // g + 1, 768 // g + 2, 1025 // g + 1]
    past = [0, 130, 77]
    s.append([0] * 3, [p + n for p, n in zip(past, new)], range(3), rows=s.rows(sum(past) + sum(new)))
    if window:
        for i, p in enumerate(past):
            s.table[i, : max(0, p - window + 1) // page] = -1
    s.attend(past, new, range(3), window=window, behind=1, max_new=max(new))
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act,max_new", [("f32", 1), ("bf16", 2), ("f16", 17), ("f32", 18)])
def test_append_with_a_bound_on_rows(make, act, max_new):
    """The bound chooses how blocks are found: first blocks, last blocks and both at once, and sequences without rows."""
    s = make(act, D=64, q_heads=2, kv_heads=2, page=16, n_slots=12, pages_per_slot=12)
    rope, plain = s.rope()
    past = [(7 * i) % 40 for i in range(12)]
    s.append([0] * 12, past, range(12), rope, plain)
    for step in range(4):
        new = [(max_new + i * 5 + step) % (max_new + 1) for i in range(12)]
        new[step] = max_new
        new[5] = 0
        slots = s.rng.permutation(12).tolist()
        rows = s.rows(sum(new))
        r, _, _, k, v = rows
        at = [past[j] for j in slots]
        s.ctx.kv_append(s.cache, s.batch(at, new, slots, max_new=max_new), rope, r)
        row = 0
        for j, n in zip(slots, new):
            if n:
                s.ref.append(j, past[j], plain(k[row:row + n], "k", past[j] + np.arange(n)), v[row:row + n])
                past[j] += n
                s.lens[j] = past[j]
            row += n
        for j in range(12):
            if past[j]:
                s.check_blocks(j)
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act,hk", [("f32", 1), ("bf16", 3)])
def test_attention_of_many_short_sequences(make, act, hk):
    """300 sequences: several rounds of the plan; histories of a tile, longer ones among them."""
    n = 300
    s = make(act, D=64, q_heads=2 * hk, kv_heads=hk, page=32, n_slots=n, pages_per_slot=12)
    total = [1 + (i * 53) % 60 for i in range(n)]
    total[17], total[200], total[299] = 380, 300, 1
    for a in range(0, n, 60):
        s.append([0] * 60, total[a:a + 60], range(a, a + 60), rows=s.rows(sum(total[a:a + 60])))
    order = s.rng.permutation(n).tolist()
    s.attend([total[i] - 1 for i in order], [1] * n, order, max_new=1)
    b = jm.KvBatch(n_seqs=n, n_tokens=n, past=s.ints([t - 1 for t in total]))       # a row each, slot b
    r, _, q, _, _ = s.rows(n)
    out = s.out(n, 2 * hk)
    s.ctx.kv_attention(s.cache, b, None, r, out.data_ptr(), 2 * hk * 64)
    s.check_attention(out.double().cpu().numpy(), q, [t - 1 for t in total], [1] * n, range(n))
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_long_prompts_give_the_same_bits_every_time(make, act):
    """Several chunks a CTA, staged one behind another: right, and the same run after run."""
    s = make(act, D=64, q_heads=32, kv_heads=4, page=32, n_slots=3, pages_per_slot=34)
    past, new = [300, 200, 250], [700, 390, 512]
    for i in range(3):
        s.append([0], [past[i] + new[i]], [i], rows=s.rows(past[i] + new[i]))
    r, _, q, _, _ = s.rows(sum(new))
    b = s.batch(past, new, range(3), max_new=700)
    first = None
    for _ in range(40):
        out = s.out(sum(new), 32)
        s.ctx.kv_attention(s.cache, b, None, r, out.data_ptr(), 32 * 64)
        first = out if first is None else first
        assert s.t.equal(first, out)
    s.check_attention(first.double().cpu().numpy(), q, past, new, range(3))
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_few_rows_give_the_same_bits_every_time(make, act):
    """A warp's slots refilled several times a segment, and segments one behind another in a CTA: right,
    and the same run after run."""
    s = make(act, D=128, q_heads=16, kv_heads=4, page=64, n_slots=34, pages_per_slot=40)
    total = [2500, 1999] + [300 + 7 * (i % 9) for i in range(32)]
    s.append([0], total[:1], [0], rows=s.rows(total[0]))
    s.append([0], total[1:2], [1], rows=s.rows(total[1]))
    for a in (2, 12, 23):
        b = min(34, a + 11)
        s.append([0] * (b - a), total[a:b], range(a, b), rows=s.rows(sum(total[a:b])))
    for new in ([1] * 34, [2, 3] + [1 + i % 3 for i in range(32)], [1]):
        n = len(new)
        r, _, q, _, _ = s.rows(sum(new))
        past = [t - m for t, m in zip(total, new)]
        b = s.batch(past, new, range(n), max_new=max(new))
        first = None
        for _ in range(40):
            out = s.out(sum(new), 16)
            s.ctx.kv_attention(s.cache, b, None, r, out.data_ptr(), 16 * 128)
            first = out if first is None else first
            assert s.t.equal(first, out)
        s.check_attention(first.double().cpu().numpy(), q, past, new, range(n))
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
def test_prompts_of_more_key_heads_than_the_workspace_takes(make):
    """640 key heads with F32 rows of 128: not one chunk of rows of all heads fits the prompts' workspace."""
    s = make("f32", D=128, q_heads=640, kv_heads=640, page=16, n_slots=2, pages_per_slot=3)
    past, new = [3, 20], [20, 17]
    s.append([0, 0], [p + n for p, n in zip(past, new)], [1, 0], rows=s.rows(sum(past) + sum(new)))
    s.attend(past, new, [1, 0], behind=1, max_new=20)
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
def test_a_timeout_outlasts_a_bad_entry(make):
    """A wait that ran out is reported as such whatever is found after it, and the call after the report is right."""
    s = make("f32", D=128, q_heads=8, kv_heads=2, page=64, n_slots=2, pages_per_slot=48)
    s.append([0], [3000], [0], rows=s.rows(3000))
    s.attend([2999], [1], [0])
    s.ctx.debug_timeout(attention=True)
    r, _, _, _, _ = s.rows(1)
    out = s.out(1, 8)
    s.ctx.kv_attention(s.cache, s.batch([10], [1], [5]), None, r, out.data_ptr(), 1024)
    with pytest.raises(jm.DeviceTimeout):
        s.ctx.device_status()
    assert s.ctx.device_status() == 0
    s.attend([2999], [1], [0])
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
def test_status_of_forwards_and_attention_at_once():
    """moe_device_status reports a forward's wait that ran out although an attention call met a bad entry too."""
    import synth
    cfg = synth.CONFIGS[2].scaled(E=16, I=256, H=512)
    s = Setup("f32", D=64, q_heads=4, kv_heads=2)
    d, keep = synth.desc_for(cfg, synth.build_weights(cfg))
    s.ctx.upload(0, d)

    def bad_entry():
        s.ctx.kv_attention(s.cache, s.batch([0], [1], [99]), None, s.rows(1)[0], s.out(1, 4).data_ptr(), 256)

    bad_entry()
    with pytest.raises(jm.TensorBoundsError):
        s.ctx.device_status()
    for forward, attention in ((True, False), (True, True), (False, True)):
        bad_entry()
        s.ctx.debug_timeout(forward=forward, attention=attention)
        with pytest.raises(jm.DeviceTimeout) as e:
            s.ctx.device_status()
        assert ("attention" in str(e.value)) and ("forward" in str(e.value)) == forward
        assert s.ctx.device_status() == 0
    s.ctx.debug_timeout(forward=True)
    with pytest.raises(jm.DeviceTimeout):
        s.ctx.device_status()
    assert s.ctx.device_status() == 0
    s.close()


@pytest.mark.gpu
def test_prefill_leaves_the_attentions_status(make):
    """A host-pointer prefill reports its own waits only: a bad entry of an attention call before it stays for the
    next check."""
    import synth
    cfg = synth.CONFIGS[2].scaled(E=16, I=256, H=512)
    s = make("f32", D=64, q_heads=4, kv_heads=2)
    d, keep = synth.desc_for(cfg, synth.build_weights(cfg))
    s.ctx.upload(0, d)
    s.ctx.set_ffn_norm(0, None, 1e-6)
    hidden = synth.gen_x(cfg, 9)
    want = s.ctx.prefill_ffn_layers(0, 1, hidden.copy())
    s.ctx.kv_attention(s.cache, s.batch([0], [1], [99]), None, s.rows(1)[0], s.out(1, 4).data_ptr(), 256)
    np.testing.assert_array_equal(s.ctx.prefill_ffn_layers(0, 1, hidden.copy()), want)
    with pytest.raises(jm.TensorBoundsError):
        s.ctx.device_status()
    assert s.ctx.device_status() == 0


# -------------------------------------------------------- rotation frequencies


def test_check_takes_frequencies_up_to_the_limit():
    _check(_args(rope__inv_freq=[jm.ROPE_MAX_FREQ] * 64))
    _check(_args(rope__inv_freq=[-jm.ROPE_MAX_FREQ] + [0.0] * 63))
    _check(_args(rope__theta=1e-4))


@pytest.mark.parametrize("rope", [dict(inv_freq=[1e20] * 64), dict(inv_freq=[1.0] * 63 + [-65537.0]), dict(theta=1e-20),
                                  dict(theta=5e-324), dict(inv_freq=[float("nan")] * 64)])
def test_check_refuses_frequencies_past_the_limit(rope):
    with pytest.raises(jm.InvalidArguments):
        _check(_args(rope={"rope_dim": 128, **rope}))


def test_quarter_turns_hold_up_to_the_limit_and_not_far_past_it():
    """The device's reduction in exact arithmetic: up to the largest angle that the checks let through the rest stays in
    [-pi/4, pi/4], and 2 % for the rounding of 2/pi (2^47 2/pi 2^-53 quarter turns)."""
    from fractions import Fraction as F

    def rest(angle):
        t = float(F(angle) * F(0.6366197723675814) + F(6755399441055744.0))     # an fma rounds once, as float() does
        n = F(t - 6755399441055744.0)
        return abs(float(F(float(F(angle) - n * F(1.5707963267948966))) - n * F(6.123233995736766e-17)))

    rng = np.random.default_rng(3)
    for scale in (1.0, 2.0 ** 20, 2.0 ** 40, jm.ROPE_MAX_FREQ * (2.0 ** 31 - 1)):
        assert max(rest(float(a)) for a in scale * rng.uniform(-1, 1, 200)) <= 1.02 * np.pi / 4
    assert rest(1e20) > 100.0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_norm_rope_of_the_largest_angles(make, act):
    s = make(act, D=64)
    f = jm.ROPE_MAX_FREQ / (1.0 + np.arange(32)) * np.where(np.arange(32) % 3 == 0, -1.0, 1.0)
    rope, plain = s.rope(64, False, False, inv_freq=f)
    pos = [(1 << 31) - 5000, (1 << 30) + 1, 7, 0]
    r, x, q, k, _ = s.rows(4)
    oq, ok = s.out(4, s.hq), s.out(4, s.hk)
    s.ctx.qk_norm_rope(jm.KvBatch(n_seqs=4, n_tokens=4, past=s.ints(pos)), rope, r, s.into(oq, ok))
    for got, y, which in ((oq, q, "q"), (ok, k, "k")):
        ref = plain(y, which, pos)      # the angle is the same product in f64, numpy reduces it exactly
        size = np.max(np.abs(y), axis=-1, keepdims=True) * 2
        # at 1.02 pi / 4 the series' next terms, x^11 / 11! and x^12 / 12!, are below 3e-9 < u / 16
        assert np.all(np.abs(got.double().cpu().numpy() - ref) <= 25 * U * size + HALF_STEP[act] * np.abs(ref) * (1 + 2 ** -7))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("D,eps", [(128, 0.0), (64, 1e-6)])
def test_norm_of_rows_whose_squares_leave_f32(make, act, D, eps):
    """Rows whose sum of squares overflows or underflows 32 bits have a norm like any other."""
    s = make(act, D=D, q_heads=6, kv_heads=3)
    rope, plain = s.rope(eps=eps)
    r, x, _, _, _ = s.rows(8)
    gain = [1e19, 1.0, 1e30, 1e36, 1e-19, 1e-25, 1e-30, 3e18]
    x *= s.t.tensor(gain, dtype=s.dtype, device="cuda")[:, None]
    f = x.double().cpu().numpy()
    a, b = s.hq * D, (s.hq + s.hk) * D
    oq, ok = s.out(8, s.hq), s.out(8, s.hk)
    pos = [0, 5, 1 << 20, 130, 7, 9, 1000, 3]
    s.ctx.qk_norm_rope(jm.KvBatch(n_seqs=8, n_tokens=8, past=s.ints(pos)), rope, r, s.into(oq, ok))
    for got, y, which in ((oq, f[:, :a].reshape(8, -1, D), "q"), (ok, f[:, a:b].reshape(8, -1, D), "k")):
        ref = plain(y, which, pos)
        size = 2 * np.max(np.abs(ref), axis=-1, keepdims=True) * np.sqrt(2.0)
        # (bf16 holds values below its normal range, 2^-126, to 2^-134 only; f32 to 2^-150)
        tiny = 2.0 ** -134 if act == "bf16" else 2.0 ** -150
        err = np.abs(got.double().cpu().numpy() - ref)
        assert np.all(err <= 24 * U * size + HALF_STEP[act] * np.abs(ref) * (1 + 2 ** -7) + tiny), (which, err.max(axis=(1, 2)))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("scale,eps", [(1e30, 1e-6), (1e-25, 0.0)])
def test_step_of_rows_whose_squares_leave_f32(make, act, scale, eps):
    """The same for the queries of the whole step, of few rows and of many."""
    s = make(act, D=64, q_heads=8, kv_heads=2, page=16, n_slots=2, pages_per_slot=16)
    rope, plain = s.rope(eps=eps)
    past = [0, 0]
    for new in ([150, 3], [1, 1]):
        r, x, _, _, v = s.rows(sum(new))
        x[:, : 10 * 64] *= scale
        f = x.double().cpu().numpy()
        q, k = f[:, :512].reshape(-1, 8, 64), f[:, 512:640].reshape(-1, 2, 64)
        out = s.out(sum(new), 8)
        s.ctx.attention(s.cache, s.batch(past, new, range(2)), rope, None, r, out.data_ptr(), 8 * 64)
        at, want = 0, np.empty(q.shape)
        for i in range(2):
            pos = past[i] + np.arange(new[i])
            rows = slice(at, at + new[i])
            s.ref.append(i, past[i], plain(k[rows], "k", pos), v[rows])
            want[rows] = plain(q[rows], "q", pos)
            at += new[i]
            past[i] += new[i]
            s.lens[i] = past[i]
            s.check_blocks(i)
        s.check_attention(out.double().cpu().numpy(), want, [p - n for p, n in zip(past, new)], new, range(2), q_err=48 * U)
    assert s.ctx.device_status() == 0


# ------------------------------------------------- value scales far apart


def check_rows(s, got, q, past, new, slots, scale=None, window=0, q_err=0.0):
    """Every output against a bound of its own. With the notation of the head of this file: a weight is off by
    part = 2 A (2^-22 + (D + 8) u + q_err) + 2^-21 + its rounding (2^-22, or with 16-bit rows 2^-11, the cubic's
    7.5e-5 in it) + (L + 64) u, relative, and where it is below f16's normal range by half a step of 2^-24 of the
    row's largest: 2^-25. Its exponent is logit log2 e + log2 s - m, formed in two sums of at most
    E = 1.45 A + 2 S, S the largest |log2 s|, so off by 2 u E, and log2 s by 2^-22 S. An output below the normal
    range of its type is rounded to a fixed step, at most half of it off: 2^-25 (f16), 2^-134 (bf16), 2^-150 (f32).
    Returns, for each head, how often the largest output holds the bound."""
    scale = scale or 1.0 / np.sqrt(s.D)
    at, big = 0, np.zeros(s.hq)
    for p, n, slot in zip(past, new, slots):
        if not n:
            continue
        o, tol = ao.attend_bound(
            q[at:at + n], *s.device_blocks(slot), p, scale, window,
            lambda A, S: 2 * A * (2.0 ** -22 + (s.D + 8) * U + q_err) + 2.0 ** -21 + 2 * U * (1.45 * A + 2 * S)
            + 2.0 ** -22 * S + (2.0 ** -22 if s.act == "f32" else 2.0 ** -11) + (p + n + 64) * U, 2.0 ** -25)
        tol += HALF_STEP[s.act] * np.abs(o) + {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -150}[s.act]
        err = np.abs(got[at:at + n] - o)
        assert np.all(err <= tol), (slot, float((err / tol).max()), np.argwhere(err > tol)[:5].tolist())
        big = np.maximum(big, (np.abs(o) / tol).max(axis=(0, 2)))
        at += n
    return big


def _gains(act, rng, n):
    """Per token: blocks of 16 whose values differ by many orders of magnitude, zeros among them."""
    pick = [0.0, 1e-7, 1e-3, 1.0, 3e4] if act == "f16" else [0.0, 1e-18, 1e-3, 1.0, 1e10, 1e20, 1e30]
    block = rng.choice(len(pick), -(-n // 16))
    return np.repeat(np.array(pick)[block], 16)[:n]


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,n", [(64, 230), (128, 520)])
def test_value_scales_far_apart(make, act, D, n):
    """Weights count in the denominator whatever the scale of their block's values is: many rows and few, blocks of
    zeros, and a head whose first blocks are far below its last ones."""
    s = make(act, D=D, q_heads=8, kv_heads=2, page=16, n_slots=2, pages_per_slot=-(-n // 16))
    r, x, q, k, v = s.rows(n)
    b = 10 * D
    gain = np.stack([_gains(act, s.rng, n), np.where(np.arange(n) < n // 2, 0.0, 3e4 if act == "f16" else 1e30)], axis=1)
    gain[n // 4: n // 3, 1] = 1e-6 if act == "f16" else 1e-15
    x[:, b:] *= s.t.tensor(np.repeat(gain, D, axis=1), device="cuda").to(s.dtype)
    v = x.double().cpu().numpy()[:, b:].reshape(n, 2, D)
    s.append([0], [n], [1], rows=(r, x, q, k, v))
    s.check_blocks(1, exact_keys=True)
    for new, scale, window in ((n, None, 0), (n - 31, 2.0, 0), (n - 40, None, 70), (1, None, 0), (3, 2.0, 0), (5, None, 40)):
        r, _, q, _, _ = s.rows(new)
        out = s.out(new, 8)
        s.ctx.kv_attention(s.cache, s.batch([n - new], [new], [1], max_new=new), jm.AttnOpts(scale=scale or 0.0, window=window), r,
                           out.data_ptr(), 8 * D)
        big = check_rows(s, out.double().cpu().numpy(), q, [n - new], [new], [1], scale, window)
        assert np.all(big > 20), big      # zeros would not pass
    assert s.ctx.device_status() == 0


# --------------------------------------------------- the bits of F32 rows


def _rms(x):
    return float(np.sqrt(np.mean(np.square(x))))


def error_share(got, o):
    """The root mean square of each head's error, as a share of its outputs': the largest head's."""
    return max(_rms(got[:, h] - o[:, h]) / _rms(o[:, h]) for h in range(o.shape[1]))


# What F32 rows may be off by in the root mean square, as a share of the outputs', with normal queries, keys and
# values of D values and logits within +-8. The errors of a token's weight that differ from token to token:
#   queries and weights rounded to 22 bits      2^-23 each, a logit sum |q k| / |q| |k| of them: below 2^-22
#   logits summed in f32                        8 steps of 2^-25 of |logit| <= 8: below 2^-20 worst, a third of it rms
#   their exponent, in two sums of at most 32   2 * 32 u ln 2 / sqrt 3 = 2^-19.6
#   log2 of the block's scale, 2^-22 of 6       2^-19.9 with ln 2
#   the exponential 2^-22; sums over tiles in f32, L / 64 chained roundings that are random: below 2^-21
# in all 2^-18.5 = 2.7e-6 of sqrt(sum p^2 v^2), which for values of mean zero is the outputs' own root mean square.
F32_SHARE = 3e-6


def _emulated(q, kq, ks, vq, vs, past, scale, drop):
    """attend with queries and weights in two f16 halves, `drop` of them ("q", "p" or neither) with the upper only."""
    def halves(x, low):
        up = 2.0 ** (14 - np.floor(np.log2(np.max(np.abs(x), axis=-1, keepdims=True))))
        hi = (x * up).astype(np.float16).astype(np.float64)
        lo = (x * up - hi).astype(np.float16).astype(np.float64)
        return (hi + (lo if low else 0.0)) / up
    n, hq, D = q.shape
    hk = kq.shape[0]
    k = (kq.astype(np.float64) * ks.astype(np.float64)[..., None, None]).reshape(hk, -1, D)
    sv = np.repeat(vs.astype(np.float64), 16, axis=1)
    out = np.zeros((n, hq, D))
    for i in range(n):
        for h in range(hq):
            kv, L = h // (hq // hk), past + i + 1
            e = k[kv, :L] @ halves(q[i, h], drop != "q") * scale + np.log(sv[kv, :L])
            w = np.exp(e - e.max())
            out[i, h] = halves(w, drop != "p") @ vq[kv].reshape(-1, D)[:L].astype(np.float64) / (w / sv[kv, :L]).sum()
    return out


@pytest.mark.parametrize("D,L", [(128, 300), (64, 300), (128, 17), (128, 2500)])
def test_a_dropped_half_is_seen(D, L):
    """The measure above rejects products of 11 bits, of the queries or of the weights, and takes those of 22."""
    rng = np.random.default_rng(D + L)
    cache = ao.Cache()
    cache.append(0, 0, rng.standard_normal((L, 2, D)), rng.standard_normal((L, 2, D)))
    blocks = *cache.blocks(0, "k"), *cache.blocks(0, "v")
    q = rng.standard_normal((3, 4, D)).astype(np.float32).astype(np.float64)
    o, _, _ = ao.attend(q, *blocks, L - 3, 1 / np.sqrt(D), 0)
    for drop, seen in (("", False), ("q", True), ("p", True)):
        share = error_share(_emulated(q, *blocks, L - 3, 1 / np.sqrt(D), drop), o)
        assert (share > 10 * F32_SHARE) == seen and (share < F32_SHARE / 10) == (not seen), (drop, share)


@pytest.mark.gpu
@pytest.mark.parametrize("D,hq,hk", [(128, 8, 2), (64, 6, 2)])
def test_f32_rows_keep_22_bits(make, D, hq, hk):
    """Single tokens, drafts, and prompts of several tiles, with and without a history."""
    s = make("f32", D=D, q_heads=hq, kv_heads=hk, page=64, n_slots=3, pages_per_slot=42)
    for slot, n in enumerate((2600, 333, 1100)):
        s.append([0], [n], [slot], rows=s.rows(n))
    for past, new in (([2599, 332, 1099], [1] * 3), ([2597, 330, 1094], [3, 3, 6]), ([2300, 0, 900], [300, 333, 200])):
        r, _, q, _, _ = s.rows(sum(new))
        out = s.out(sum(new), hq)
        s.ctx.kv_attention(s.cache, s.batch(past, new, range(3), max_new=max(new)), None, r, out.data_ptr(), hq * D)
        got, at = out.double().cpu().numpy(), 0
        for slot, (p, n) in enumerate(zip(past, new)):
            o, _, _ = ao.attend(q[at:at + n], *s.device_blocks(slot), p, 1 / np.sqrt(D), 0)
            share = error_share(got[at:at + n], o)
            assert share < F32_SHARE, (slot, p, n, share)
            at += n
    assert s.ctx.device_status() == 0


# And 16-bit rows: a rounding is off evenly up to half a step, h / 2^f of a value 2^(e + f), and f is spread evenly over
# [0, 1): h / sqrt 3 * sqrt(3 / (8 ln 2)) = 0.425 h in the root mean square. The output's, h = 2^-11 or 2^-8, and the
# weights' to f16, 2^-11: sqrt 2 * 2.07e-4 = 2.93e-4 for f16 rows, 1.66e-3 and 2.07e-4 = 1.67e-3 for bf16 rows; the
# cubic of a quarter of the weights (7.5e-5 at most) adds less than 3e-6 to either.
# Of outputs o the square's weighted mean sum (o d)^2 / sum o^2 scatters: d^2 by 9 / 5 E(2^-4f) / E(2^-2f)^2 - 1 = 1.08
# of its square, so the mean by sqrt(1.08 sum o^4) / sum o^2 and its root by half of that. Four times that for the
# largest of some heads.
def check_share(act, got, o, what):
    for h in range(o.shape[1]):
        scatter = 0.52 * np.sqrt(np.sum(o[:, h] ** 4)) / np.sum(o[:, h] ** 2)
        share = _rms(got[:, h] - o[:, h]) / _rms(o[:, h])
        assert share < {"f16": 2.96e-4, "bf16": 1.677e-3}[act] * (1 + 4 * scatter), (what, h, share, scatter)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("D,hq,hk", [(128, 8, 2), (64, 6, 2)])
def test_16_bit_rows_lose_their_rounding_only(make, act, D, hq, hk):
    s = make(act, D=D, q_heads=hq, kv_heads=hk, page=64, n_slots=3, pages_per_slot=42)
    for slot, n in enumerate((2600, 333, 1100)):
        s.append([0], [n], [slot], rows=s.rows(n))
    for past, new in (([2599, 332, 1099], [1] * 3), ([2595, 330, 1091], [5, 3, 9]), ([2300, 0, 900], [300, 333, 200])):
        r, _, q, _, _ = s.rows(sum(new))
        out = s.out(sum(new), hq)
        s.ctx.kv_attention(s.cache, s.batch(past, new, range(3), max_new=max(new)), None, r, out.data_ptr(), hq * D)
        got, at = out.double().cpu().numpy(), 0
        for slot, (p, n) in enumerate(zip(past, new)):
            o, _, _ = ao.attend(q[at:at + n], *s.device_blocks(slot), p, 1 / np.sqrt(D), 0)
            check_share(act, got[at:at + n], o, (slot, p, n))
            at += n


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,hq,hk,page,window", [(128, 16, 2, 64, 0), (64, 14, 2, 16, 0), (128, 5, 1, 32, 50)])
def test_every_output_within_a_bound_of_its_own(make, act, D, hq, hk, page, window):
    """Lengths around block, page and tile ends, single tokens to prompts, each output against what its row can be off by."""
    s = make(act, D=D, q_heads=hq, kv_heads=hk, page=page, n_slots=8, pages_per_slot=-(-448 // page))
    total = [1, 2, 15, 16, 17, 64, 129, 440]
    s.append([0] * 8, total, range(8), rows=s.rows(sum(total)))
    for new in ([1] * 8, [1, 2, 3, 5, 8, 9, 17, 33], [1, 0, 15, 16, 1, 64, 129, 440]):
        slots = s.rng.permutation(8)
        n = [new[i] for i in slots]
        past = [total[i] - new[i] for i in slots]
        r, _, q, _, _ = s.rows(sum(n))
        out = s.out(sum(n), hq)
        s.ctx.kv_attention(s.cache, s.batch(past, n, slots, max_new=max(n)), jm.AttnOpts(window=window), r, out.data_ptr(), hq * D)
        big = check_rows(s, out.double().cpu().numpy(), q, past, n, slots, window=window)
        assert np.all(big > 50), big
    assert s.ctx.device_status() == 0


# -------------------------------------------------------------- its workspace


def test_admission_leaves_room_for_the_workspace():
    """A caller sets the workspace aside as part of the reserve; without it the admission is what it was."""
    import synth
    from test_host import _fake_desc
    d = [_fake_desc(synth.CONFIGS[2], np.zeros(16, dtype=np.uint8))]
    need = jm.admission_check(0, 64, d, free_bytes=1 << 40).total_required_bytes
    room = jm.ATTENTION_WORKSPACE_BYTES
    jm.admission_check(0, 64, d, free_bytes=need)
    fp = jm.admission_check(0, 64, d, free_bytes=need + room, reserve_bytes=room)
    assert fp.total_required_bytes == need and fp.budget_bytes == need
    with pytest.raises(jm.InsufficientLockableMemory):
        jm.admission_check(0, 64, d, free_bytes=need + room - 1, reserve_bytes=room)


@pytest.mark.gpu
def test_residency_counts_the_workspace(make):
    s = make("f32", D=64, q_heads=2, kv_heads=2)
    assert s.ctx.residency().scratch_bytes == 0
    s.append([0], [20], [0], rows=s.rows(20))
    assert 80 << 20 <= s.ctx.residency().scratch_bytes <= jm.ATTENTION_WORKSPACE_BYTES


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("D,hq,hk", [(128, 8, 2), (64, 21, 3)])
def test_step_of_16_bit_rows_loses_their_rounding_only(make, act, D, hq, hk):
    """The same through the whole step: queries are normed and turned in f32 as they are read (24 u of a pair, far below
    the weights' rounding), and no second rounding to their type may be seen."""
    s = make(act, D=D, q_heads=hq, kv_heads=hk, page=64, n_slots=2, pages_per_slot=16)
    rope, plain = s.rope()
    past = [0, 0]
    for new in ([600, 301], [1, 1], [8, 3], [40, 5], [2, 16], [100, 90]):
        r, x, q, k, v = s.rows(sum(new))
        out = s.out(sum(new), hq)
        s.ctx.attention(s.cache, s.batch(past, new, range(2), max_new=max(new)), rope, None, r, out.data_ptr(), hq * D)
        got, at = out.double().cpu().numpy(), 0
        for i in range(2):
            pos, rows = past[i] + np.arange(new[i]), slice(at, at + new[i])
            s.lens[i] = past[i] + new[i]
            o, _, _ = ao.attend(plain(q[rows], "q", pos), *s.device_blocks(i), past[i], 1 / np.sqrt(D), 0)
            check_share(act, got[rows], o, (i, new))
            at += new[i]
            past[i] += new[i]
    assert s.ctx.device_status() == 0


# ------------------------------------------------------- sizes past the usual


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_cache_past_32_bits(make, act):
    """Bytes beyond 2^32: 4.9 GiB each of keys and values, the sequences' pages spread over them."""
    s = make(act, D=128, q_heads=16, kv_heads=8, page=256, n_slots=2, pages_per_slot=10000)
    assert s.k.numel() > 1 << 32
    s.table_np[0, :3] = s.n_pages - 1, 0, s.n_pages - 2     # and the very ends of them
    s.table_np[1, :2] = s.n_pages - 3, s.n_pages // 2
    used = set(s.table_np[0, :3]) | set(s.table_np[1, :2])
    for i in range(2):
        free = [p for p in s.table_np[i, 5:] if p not in used][:7]
        s.table_np[i, 3 - i: 8] = free[: 5 + i]
        used |= set(free)
    s.table.copy_(s.t.tensor(s.table_np, dtype=s.t.int32))
    total = [1500, 700]
    s.append([0, 0], total, [0, 1], rows=s.rows(2200))
    for i in range(2):
        s.check_blocks(i, exact_keys=True)
    for new in ([1, 1], [5, 300]):
        s.attend([t - n for t, n in zip(total, new)], new, [0, 1], max_new=max(new))
    ok, ov = s.out(700, 8), s.out(700, 8)
    s.ctx.kv_read(s.cache, s.batch([0], [700], [1]), s.into(k=ok, v=ov))
    kq, ks, vq, vs = s.device_blocks(1)
    for got, q, sc in ((ok, kq, ks), (ov, vq, vs)):
        val = (q.astype(np.float32) * sc[..., None, None]).reshape(8, -1, 128)[:, :700].transpose(1, 0, 2)
        assert s.t.equal(got.cpu(), s.t.tensor(val).to(s.dtype))
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_attention_of_a_list_too_long_to_sort(make, act):
    """1200 sequences, prompts among single tokens: more chunks of rows than a launch puts in order."""
    n = 1200
    s = make(act, D=64, q_heads=3, kv_heads=1, page=16, n_slots=n, pages_per_slot=5)
    new = [(7 * i) % 50 + 20 if i % 40 == 0 else i % 2 for i in range(n)]
    total = [m + (11 * i) % 9 if m else 0 for i, m in enumerate(new)]
    for a in range(0, n, 300):
        s.append([0] * 300, total[a:a + 300], range(a, a + 300), rows=s.rows(max(1, sum(total[a:a + 300]))))
    order = s.rng.permutation(n).tolist()
    s.attend([total[i] - new[i] for i in order], [new[i] for i in order], order, behind=1, max_new=max(new))
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("hq,new", [(1024, [1, 3]), (512, [1, 1]), (509, [2, 0])])
def test_many_query_heads_a_key_head(make, act, hq, new):
    s = make(act, D=64, q_heads=hq, kv_heads=1, page=32, n_slots=2, pages_per_slot=8)
    total = [200, 77]
    s.append([0, 0], total, [0, 1], rows=s.rows(277))
    s.attend([t - n for t, n in zip(total, new)], new, [0, 1], max_new=max(new))
    rope, plain = s.rope()
    past = [t for t in total]
    r, x, q, k, v = s.rows(sum(new))
    out = s.out(sum(new), hq)
    s.ctx.attention(s.cache, s.batch(past, new, [0, 1], max_new=max(new)), rope, None, r, out.data_ptr(), hq * 64)
    want, at = np.empty(q.shape), 0
    for i in range(2):
        pos = past[i] + np.arange(new[i])
        if new[i]:
            s.ref.append(i, past[i], plain(k[at:at + new[i]], "k", pos), v[at:at + new[i]])
            want[at:at + new[i]] = plain(q[at:at + new[i]], "q", pos)
        s.lens[i] = past[i] + new[i]
        at += new[i]
    s.check_attention(out.double().cpu().numpy(), want, past, new, [0, 1], q_err=48 * U)
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,hq,hk,R,interleaved", [(64, 7, 3, 64, False), (128, 5, 2, 64, True), (64, 1, 1, 34, False)])
def test_norm_rope_of_many_tokens(make, act, D, hq, hk, R, interleaved):
    """A warp a token for all its heads: head counts that do not fill its last load, queries or keys alone, no norm on one."""
    s = make(act, D=D, q_heads=hq, kv_heads=hk)
    rope, plain = s.rope(R, interleaved)
    T = 4000
    past, new = [0, 1 << 20, 9, 77], [1500, 0, 2499, 1]
    r, x, q, k, _ = s.rows(T + 3)
    b = s.batch(past, new, range(4), behind=3)
    pos = np.concatenate([p + np.arange(n) for p, n in zip(past, new)])
    for which in ("qk", "q", "k"):
        oq, ok = s.out(T + 3, hq), s.out(T + 3, hk)
        part = jm.QkvRows(**{f: getattr(r, f) for f, _ in r._fields_})
        part.q, part.k = (r.q if "q" in which else None), (r.k if "k" in which else None)
        s.ctx.qk_norm_rope(b, rope, part, s.into(oq, ok))
        for got, y, name in ((oq, q, "q"), (ok, k, "k")):
            got = got.double().cpu().numpy()
            if name not in which:
                assert np.all(got == 123.0)
                continue
            ref = plain(y[:T], name, pos)
            size = 2 * np.max(np.abs(ref), axis=-1, keepdims=True) * np.sqrt(2.0)
            assert np.all(np.abs(got[:T] - ref) <= 24 * U * size + HALF_STEP[act] * np.abs(ref) * (1 + 2 ** -7))
            assert np.all(got[T:] == 123.0)
    assert s.ctx.device_status() == 0


@pytest.mark.gpu
def test_step_with_a_slot_twice(make):
    """The whole step refuses a slot's second appearance: the first and the other sequences are right, and so is the
    call after it."""
    s = make("f32", D=64, q_heads=4, kv_heads=2, page=16, n_slots=3, pages_per_slot=8)
    s.append([0] * 3, [40, 30, 20], range(3), rows=s.rows(90))
    for new in ([1, 1, 1], [20, 1, 30]):
        r, x, q, k, v = s.rows(sum(new))
        out = s.out(sum(new), 4)
        past = [s.lens[0], s.lens[2], s.lens[0]]
        s.ctx.attention(s.cache, s.batch(past, new, [0, 2, 0]), None, None, r, out.data_ptr(), 256)
        with pytest.raises(jm.TensorBoundsError):
            s.ctx.device_status()
        at = 0
        for slot, n in ((0, new[0]), (2, new[1])):
            s.ref.append(slot, s.lens[slot], k[at:at + n], v[at:at + n])
            s.lens[slot] += n
            s.check_blocks(slot, exact_keys=True)
            at += n
        s.check_attention(out.double().cpu().numpy()[:at], q[:at], past[:2], new[:2], [0, 2])
    s.attend([s.lens[0] - 1], [1], [0])
    assert s.ctx.device_status() == 0
