"""The paged serving operators on the GPU against their 64-bit definitions
(paged_ref.py, with the error bounds derived there)."""
import numpy as np
import pytest
import torch

import paged_ref as R
from vibethinker_webgpu_lora_b200 import kernels as K

pytestmark = pytest.mark.gpu
HD, PAGE = R.HD, R.PAGE
KV = {"f16": torch.float16, "f32": torch.float32}


def tables(n):
    inv = 1e6 ** (-np.arange(0, HD, 2) / HD)
    a = np.arange(n)[:, None] * inv
    a = np.concatenate([a, a], 1)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def i32(x, cuda):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=cuda)


# ---------------------------------------------------------------- append
class Append:
    """Ragged tokens of `runs` = [(first row, count)] in shuffled order, pages shuffled over the pool."""

    def __init__(self, cuda, runs, nh, nkv, kv, prefix=0, extra=0, seed=0, pad=()):
        rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.kv, self.prefix = nh, nkv, kv, prefix
        need = [-(-(f + n) // PAGE) for f, n in runs]
        total = sum(need) + 2
        perm = rng.permutation(total)
        self.pages = np.full((len(runs), max(need) + 1), 0xFFFFFF, np.int64)  # entries past a sequence's end: no page
        at = 0
        for i, n in enumerate(need):
            self.pages[i, :n] = perm[at:at + n]
            at += n
        tok = [(i, f + j) for i, (f, n) in enumerate(runs) for j in range(n)]
        rng.shuffle(tok)
        self.slot = np.array([t[0] for t in tok])
        self.pos = np.array([t[1] for t in tok]) + prefix
        for i in pad:
            self.pos[i] = -1
        self.width = (nh + 2 * nkv) * HD
        self.qkv = rng.standard_normal((len(tok), self.width + extra)).astype(np.float32)
        self.cos, self.sin = tables(self.pos.max() + 1)
        dt = np.float16 if kv == "f16" else np.float32
        self.kc = rng.standard_normal((total, PAGE, nkv, HD)).astype(dt)
        self.vc = rng.standard_normal((total, PAGE, nkv, HD)).astype(dt)
        d = lambda x: torch.from_numpy(x).to(cuda)  # noqa: E731
        self.d = dict(qkv=d(self.qkv)[:, :self.width], pos=i32(self.pos, cuda), slot=i32(self.slot, cuda),
                      pages=i32(self.pages, cuda), k_cache=d(self.kc), v_cache=d(self.vc), cos_t=d(self.cos),
                      sin_t=d(self.sin), nh=nh, q_out=torch.full((len(tok), nh * HD + extra), 7.0, device=cuda)[:, :nh * HD],
                      prefix_len=prefix, err=torch.zeros(1, dtype=torch.int32, device=cuda))

    def check(self, skip=()):
        """Everything written is the definition's; everything else is as it was."""
        live = np.array([t for t in range(len(self.pos)) if self.pos[t] >= 0 and t not in set(skip)], np.int64)
        x = self.qkv[live, :self.width].reshape(len(live), -1, HD)
        c, s = self.cos[self.pos[live]][:, None], self.sin[self.pos[live]][:, None]
        y, mag = R.rotate(x[:, :self.nh + self.nkv], c, s)
        rel = self.pos[live] - self.prefix
        row = self.pages[self.slot[live], rel // PAGE] * PAGE + rel % PAGE
        f16 = self.kv == "f16"
        q = np.full((len(self.pos), self.nh, HD), 7.0)
        qb = np.zeros_like(q)
        q[live], qb[live] = y[:, :self.nh], R.rotate_bound(y[:, :self.nh], mag[:, :self.nh], False)
        k, kb = self.kc.astype(np.float64).reshape(-1, self.nkv, HD), np.zeros((self.kc.size // HD // self.nkv, self.nkv, HD))
        k[row], kb[row] = y[:, self.nh:], R.rotate_bound(y[:, self.nh:], mag[:, self.nh:], f16)
        v = self.vc.copy().reshape(-1, self.nkv, HD)
        v[row] = x[:, self.nh + self.nkv:].astype(v.dtype)
        torch.cuda.synchronize()
        if self.d["q_out"] is not None:
            got = self.d["q_out"].cpu().numpy().astype(np.float64).reshape(q.shape)
            assert (abs(got - q) <= qb).all(), abs(got - q).max()
        got = self.d["k_cache"].cpu().numpy().astype(np.float64).reshape(k.shape)
        assert (abs(got - k) <= kb).all(), abs(got - k).max()
        assert np.array_equal(self.d["v_cache"].cpu().numpy().reshape(v.shape), v)


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("nh,nkv", [(16, 2), (28, 4), (4, 4), (8, 1), (32, 8), (0, 2)])
@pytest.mark.parametrize("runs,prefix", [([(0, 1)], 0), ([(15, 1), (16, 1), (0, 17)], 5), ([(3, 130), (40, 1), (0, 64)], 0)])
def test_append(cuda, kv, nh, nkv, runs, prefix):
    a = Append(cuda, runs, nh, nkv, kv, prefix)
    K.kv_append_paged(**a.d)
    a.check()
    assert a.d["err"].item() == 0


def test_append_strided_rows_no_q_and_padding(cuda):
    a = Append(cuda, [(0, 20), (7, 9)], 16, 2, "f16", extra=12, pad=(0, 5, 28))
    K.kv_append_paged(**a.d)
    a.check()
    b = Append(cuda, [(0, 20), (7, 9)], 16, 2, "f32", extra=4)
    b.d["q_out"] = None
    K.kv_append_paged(**b.d)
    b.check()


def test_append_of_a_row_that_is_a_view_of_one(cuda):
    a = Append(cuda, [(4, 1)], 16, 2, "f16", extra=8)
    K.kv_append_paged(**a.d)
    a.check()


def test_append_out_of_range_rows_are_left_out_and_flagged(cuda):
    for what in ("slot", "below", "page list", "page", "table", "negative slot"):
        a = Append(cuda, [(0, 20), (7, 9)], 16, 2, "f16", prefix=3)
        if what == "slot":
            a.d["slot"][4] = 2
        elif what == "negative slot":
            a.d["slot"][4] = -1
        elif what == "below":
            a.d["pos"][4] = 2  # inside the prefix
        elif what == "page list":
            a.d["pages"] = a.d["pages"][:, :2].contiguous()
            bad = [t for t in range(29) if a.pos[t] - 3 >= 32]
            a.d["pos"][4] = 3 + 32
            a.cos, a.sin = tables(64)
            a.d["cos_t"], a.d["sin_t"] = torch.from_numpy(a.cos).to(cuda), torch.from_numpy(a.sin).to(cuda)
            assert not bad
        elif what == "page":
            a.d["pages"][a.slot[4], (a.pos[4] - 3) // PAGE] = a.kc.shape[0]
        else:
            a.d["cos_t"], a.d["sin_t"] = a.d["cos_t"][:10].contiguous(), a.d["sin_t"][:10].contiguous()
        skip = [4]
        if what == "page":
            skip = [t for t in range(29) if a.slot[t] == a.slot[4] and (a.pos[t] - 3) // PAGE == (a.pos[4] - 3) // PAGE]
        elif what == "table":
            skip = [t for t in range(29) if a.pos[t] >= 10]
        K.kv_append_paged(**a.d)
        a.check(skip)
        assert a.d["err"].item() == 1, what


def test_append_far_rows(cuda):
    """Rows past 2^31 elements of a pool, and a far position of the table."""
    n_pages = (1 << 31) // (PAGE * 2 * HD) + 64
    kc = torch.empty(n_pages, PAGE, 2, HD, dtype=torch.float16, device=cuda)
    vc = torch.empty_like(kc)
    a = Append(cuda, [(0, 40)], 16, 2, "f16")
    a.d["k_cache"], a.d["v_cache"] = kc, vc
    a.d["pages"] = i32([[n_pages - 1, n_pages - 40, n_pages - 2]], cuda)
    K.kv_append_paged(**a.d)
    assert a.d["err"].item() == 0
    near = Append(cuda, [(0, 40)], 16, 2, "f16")
    K.kv_append_paged(**near.d)
    for i, p in enumerate([n_pages - 1, n_pages - 40, n_pages - 2]):
        n = min(PAGE, 40 - i * PAGE)
        for far, c in ((kc, "k_cache"), (vc, "v_cache")):
            assert torch.equal(far[p, :n], near.d[c][int(near.pages[0, i]), :n])


def test_append_turns_q_in_place(cuda):
    """q_out may be qkv's own q heads, as attn_prefill turns them."""
    for runs in ([(0, 20), (7, 9)], [(0, 7000)]):
        a = Append(cuda, runs, 16, 2, "f16")
        a.d["q_out"] = a.d["qkv"][:, :16 * HD]
        K.kv_append_paged(**a.d)
        a.check()


def test_append_many_tokens(cuda):
    """More heads than the small form takes."""
    a = Append(cuda, [(5, 5003), (0, 1800)], 16, 2, "f16", prefix=3, pad=(17, 6802))
    K.kv_append_paged(**a.d)
    a.check()
    b = Append(cuda, [(0, 3700)], 28, 4, "f32")
    b.d["q_out"] = None
    K.kv_append_paged(**b.d)
    b.check()


# ---------------------------------------------------------------- attention over a shared prefix
class Shared:
    def __init__(self, cuda, prefix, lens, nh, nkv, kv, seed=0, max_len=None, extra=0, spike=0.0, fill=np.nan):
        rng = np.random.default_rng(seed)
        n = len(lens)
        self.cuda, self.prefix, self.lens, self.nh, self.nkv, self.kv = cuda, prefix, list(lens), nh, nkv, kv
        self.max_len = max(max(lens), 0) if max_len is None else max_len
        np_, ns = -(-prefix // PAGE), -(-self.max_len // PAGE)
        total = np_ + n * ns + 1
        perm = rng.permutation(total)
        self.ppages, self.pages = perm[:np_], perm[np_:np_ + n * ns].reshape(n, ns)
        dt = np.float16 if kv == "f16" else np.float32
        # rows that no sequence holds (page tails, spare pages) carry NaN
        self.kc, self.vc = (np.full((total * PAGE, nkv, HD), fill, dt) for _ in range(2))
        for pages, m in [(self.ppages, prefix)] + [(p, max(ln, 0)) for p, ln in zip(self.pages, lens)]:
            rows = R.rows_of(pages, m)
            self.kc[rows] = rng.standard_normal((m, nkv, HD)).astype(dt)
            self.vc[rows] = rng.standard_normal((m, nkv, HD)).astype(dt)
        self.q = rng.standard_normal((n, nh * HD + extra)).astype(np.float32) * 1.5
        if spike and prefix:  # one key that takes nearly all the weight
            k = self.kc[R.rows_of(self.ppages, prefix)[prefix // 2]]
            k[:] = np.sign(k) * 1.0
            self.q[:, :nh * HD] = (self.q[:, :nh * HD].reshape(n, nkv, -1, HD) * 0.2 +
                                   spike * k.astype(np.float32)[None, :, None] * HD ** 0.5 / HD).reshape(n, -1)
        d = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(cuda)  # noqa: E731
        shape = (total, PAGE, nkv, HD)
        ws = K.attn_shared_prefix_bytes(n, nh, nkv, prefix, self.max_len)
        self.d = dict(q=d(self.q)[:, :nh * HD], k_cache=d(self.kc.reshape(shape)), v_cache=d(self.vc.reshape(shape)),
                      prefix_pages=i32(self.ppages, cuda), prefix_len=prefix, pages=i32(self.pages, cuda),
                      lens=i32(lens, cuda), max_len=self.max_len,
                      out=torch.full((n, nh * HD + extra), 5.0, device=cuda)[:, :nh * HD],
                      ws=torch.full((ws,), 0xFF, dtype=torch.uint8, device=cuda),
                      err=torch.zeros(1, dtype=torch.int32, device=cuda))

    def want(self, b):
        rows = np.concatenate([R.rows_of(self.ppages, self.prefix), R.rows_of(self.pages[b], self.lens[b])]).astype(np.int64)
        return R.attention(self.q[b, :self.nh * HD].reshape(self.nh, HD), self.kc[rows], self.vc[rows])

    def check(self, seqs=None):
        torch.cuda.synchronize()
        got = self.d["out"].cpu().numpy().astype(np.float64).reshape(len(self.lens), self.nh, HD)
        worst = 0.0
        for b in range(len(self.lens)) if seqs is None else seqs:
            if self.lens[b] < 0:
                assert (got[b] == 5.0).all()
                continue
            o, bound = self.want(b)
            err = abs(got[b] - o)
            assert (err <= bound).all(), (b, err.max(), (err / bound).max())
            worst = max(worst, (err / np.maximum(bound, 1e-30)).max())
        return worst


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 130, 700])
@pytest.mark.parametrize("lens", [[1], [0], [5, 0, -1, 33], [16, 17, 15, 129, 128, 300]])
def test_shared_prefix(cuda, kv, prefix, lens):
    s = Shared(cuda, prefix, lens, 16, 2, kv, seed=prefix + len(lens))
    K.attn_shared_prefix(**s.d)
    print("worst error / bound:", s.check())
    assert s.d["err"].item() == 0


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("nh,nkv,n", [(28, 4, 33), (4, 4, 9), (8, 1, 40), (32, 8, 7), (20, 1, 5), (12, 4, 150), (64, 4, 3)])
def test_shared_prefix_heads(cuda, kv, nh, nkv, n):
    lens = [(i * 37) % 90 for i in range(n)]
    s = Shared(cuda, 203, lens, nh, nkv, kv, seed=nh, extra=4)
    K.attn_shared_prefix(**s.d)
    s.check()


@pytest.mark.parametrize("kv,n,prefix", [("f16", 64, 2051), ("f16", 130, 1000), ("f16", 3, 9001), ("f32", 20, 2051), ("f16", 17, 4096)])
def test_shared_prefix_long(cuda, kv, n, prefix):
    s = Shared(cuda, prefix, [(i * 53) % 200 for i in range(n)], 16, 2, kv, seed=9)
    K.attn_shared_prefix(**s.d)
    s.check(range(0, n, max(1, n // 12)))


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("n", [2, 40])
def test_shared_prefix_one_key_takes_the_weight(cuda, kv, n):
    """One score 20 above the rest: what the others add (each 2e-9 of it, below
    the f16 range) is not lost, nor is it when the key comes late."""
    s = Shared(cuda, 3000, [100 + i for i in range(n)], 16, 2, kv, spike=2.2, seed=4)
    K.attn_shared_prefix(**s.d)
    s.check(range(0, n, max(1, n // 6)))


def test_shared_prefix_bounds_read_on_the_device(cuda):
    """A length above max_len counts as max_len, a page outside the pool as no
    rows; both are flagged, and other sequences are not touched by it."""
    s = Shared(cuda, 40, [50, 50, 50], 16, 2, "f16")
    s.d["lens"][1] = 1 << 30
    K.attn_shared_prefix(**s.d)
    s.check()
    assert s.d["err"].item() == 1
    for bad in (-1, 1 << 20):
        s = Shared(cuda, 40, [50, 50, 50], 16, 2, "f16")
        s.d["pages"][1, 3] = bad
        K.attn_shared_prefix(**s.d)
        s.check([0, 2])
        s.lens[1] = 48  # the rows of the fourth page are gone
        s.check([1])
        assert s.d["err"].item() == 1
        s = Shared(cuda, 40, [50, 50, 50] * 8, 16, 2, "f16")
        s.d["prefix_pages"][2] = bad
        K.attn_shared_prefix(**s.d)
        s.prefix = 32
        s.check()
        assert s.d["err"].item() == 1


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("nh,nkv,n", [(8, 1, 3), (12, 1, 2), (2, 2, 5), (40, 8, 6)])
@pytest.mark.parametrize("prefix,longest", [(0, 1), (0, 128), (129, 0), (0, 1000), (512, 512), (515, 513), (640, 130), (1024, 100), (2048, 640), (30, 2048), (2000, 1900), (896, 0), (600, 100), (700, 128)])
def test_shared_prefix_of_few_splits(cuda, kv, nh, nkv, n, prefix, longest):
    """1 to 9 splits: joined within a cluster up to 8, by a launch of their own from 9 on."""
    lens = [longest, -1, 0, longest // 2, longest, min(3, longest)][:n]
    s = Shared(cuda, prefix, lens, nh, nkv, kv, seed=nh + prefix, max_len=longest, extra=8)
    K.attn_shared_prefix(**s.d)
    s.check()
    assert s.d["err"].item() == 0


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("nh,nkv,lens,prefix", [(16, 2, [700], 9000), (4, 4, [0, 5000, -1], 4100), (28, 4, [130, 4000], 0),
                                                (16, 2, [1, 300, 2600], 2300), (8, 1, [0], 20000)])
def test_shared_prefix_of_many_splits(cuda, kv, nh, nkv, lens, prefix):
    """17 to 70 splits of few rows: the combine's lanes, of which some have no split."""
    s = Shared(cuda, prefix, lens, nh, nkv, kv, seed=prefix, extra=4)
    K.attn_shared_prefix(**s.d)
    s.check()
    assert s.d["err"].item() == 0


def test_shared_prefix_few_splits_of_both_streams_and_no_keys(cuda):
    """Sequences that hold nothing get zeros; replays beside an eager call agree."""
    s = Shared(cuda, 0, [0, 0, 40], 16, 2, "f16", max_len=300)
    K.attn_shared_prefix(**s.d)
    torch.cuda.synchronize()
    assert (s.d["out"][:2] == 0).all()
    s.check()
    g = torch.cuda.CUDAGraph()
    first = s.d["out"].clone()
    with torch.cuda.graph(g):
        K.attn_shared_prefix(**s.d)
    side = torch.cuda.Stream()
    b = Shared(cuda, 300, [17] * 9, 16, 2, "f32", seed=3)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        K.attn_shared_prefix(**b.d)
    for _ in range(5):
        s.d["out"].fill_(1)
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, s.d["out"])
    b.check()


def test_shared_prefix_nan_and_inf_stay_in_their_row(cuda):
    s = Shared(cuda, 100, [20] * 12, 16, 2, "f16")
    s.d["q"][3, 5] = float("nan")
    s.d["q"][7, 130] = float("inf")
    K.attn_shared_prefix(**s.d)
    s.check([b for b in range(12) if b not in (3, 7)])
    assert torch.isnan(s.d["out"][3, :HD]).all() and not torch.isnan(s.d["out"][3, HD:]).any()
    assert torch.isnan(s.d["out"][7, HD:2 * HD]).any() and not torch.isnan(s.d["out"][7, 2 * HD:]).any()


def test_shared_prefix_far_pages(cuda):
    """Pages past 2^31 elements of a pool."""
    s = Shared(cuda, 100, [40, 7], 16, 2, "f16")
    n_pages = (1 << 31) // (PAGE * 2 * HD) + 64
    off = n_pages - s.d["k_cache"].shape[0]
    for c in ("k_cache", "v_cache"):
        far = torch.empty(n_pages, PAGE, 2, HD, dtype=torch.float16, device=cuda)
        far[off:] = s.d[c]
        s.d[c] = far
    s.d["prefix_pages"] += off
    s.d["pages"] += off
    K.attn_shared_prefix(**s.d)
    s.check()


def test_shared_prefix_same_bits_every_time(cuda):
    for n, kv in ((5, "f16"), (70, "f16"), (9, "f32")):
        s = Shared(cuda, 900, [i * 7 for i in range(n)], 16, 2, kv)
        K.attn_shared_prefix(**s.d)
        first = s.d["out"].clone()
        for _ in range(3):
            s.d["out"].fill_(0)
            K.attn_shared_prefix(**s.d)
            assert torch.equal(first, s.d["out"])


def test_shared_prefix_two_streams_two_workspaces(cuda):
    a = Shared(cuda, 1500, [100] * 20, 16, 2, "f16", seed=1)
    b = Shared(cuda, 700, [300] * 11, 16, 2, "f16", seed=2)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        K.attn_shared_prefix(**a.d, stream=sa)
        K.attn_shared_prefix(**b.d, stream=sb)
    a.check(range(0, 20, 5))
    b.check(range(0, 11, 5))


def relative(s, seqs):
    torch.cuda.synchronize()
    got = s.d["out"].cpu().numpy().astype(np.float64).reshape(len(s.lens), s.nh, HD)
    want = np.stack([s.want(b)[0] for b in seqs])
    return np.linalg.norm(got[list(seqs)] - want) / np.linalg.norm(want)


def test_shared_prefix_long_suffixes_of_many(cuda):
    """A few long sequences among many: the parts stay short (a running sum on
    the tensor cores loses 2^-24.5 a step; 1024 keys over 4 warps are 32 steps,
    a score 16: together below 8e-6 of the output, where one part of 32768 keys
    would lose 2e-5)."""
    n, longest = 300, 32768
    lens = [longest if i in (17, 170) else i % 40 for i in range(n)]
    s = Shared(cuda, 20, lens[:2] + [longest], 16, 2, "f16", seed=5)  # one long run of pages, used by both
    pages = np.tile(s.pages[2], (n, 1))
    s.pages, s.lens = pages, lens
    rng = np.random.default_rng(6)
    s.q = rng.standard_normal((n, 16 * HD)).astype(np.float32)
    s.d.update(q=torch.from_numpy(s.q).to(cuda), pages=i32(pages, cuda), lens=i32(lens, cuda),
               out=torch.zeros(n, 16 * HD, device=cuda),
               ws=torch.empty(K.attn_shared_prefix_bytes(n, 16, 2, 20, longest), dtype=torch.uint8, device=cuda))
    K.attn_shared_prefix(**s.d)
    err = relative(s, [17, 170])
    print("relative error", err)
    assert err < 8e-6
    s.check([0, 16, 17, 18, 299])


@pytest.mark.parametrize("size", [1e-4, 30.0])
@pytest.mark.parametrize("n", [2, 40])
def test_shared_prefix_keys_of_any_size(cuda, n, size):
    """Keys of an f32 cache far below 1 under queries as far above it, and the other way round."""
    s = Shared(cuda, 800, [60] * n, 16, 2, "f32", seed=17)
    s.kc *= np.float32(size)
    s.q /= np.float32(size)
    s.d["k_cache"].copy_(torch.from_numpy(s.kc.reshape(s.d["k_cache"].shape)))
    s.d["q"].copy_(torch.from_numpy(s.q[:, :16 * HD]))
    K.attn_shared_prefix(**s.d)
    assert relative(s, range(0, n, max(1, n // 5))) < 8e-6


@pytest.mark.parametrize("n", [2, 40])
@pytest.mark.parametrize("size", [1e-6, 1e-3, 300.0])
def test_shared_prefix_values_of_any_size(cuda, n, size):
    """An f32 cache's small or large values keep their precision: hi and lo
    parts to 2^-22, or 2^-36 where that is more; the scores' part as above."""
    s = Shared(cuda, 800, [60] * n, 16, 2, "f32", seed=7)
    s.vc *= np.float32(size)
    s.d["v_cache"].copy_(torch.from_numpy(s.vc.reshape(s.d["v_cache"].shape)))
    K.attn_shared_prefix(**s.d)
    assert relative(s, range(0, n, max(1, n // 5))) < 8e-6 + 2.0 ** -36 / size * 2


@pytest.mark.parametrize("kv,n,prefix,longest", [("f16", 40, 4000, 100), ("f16", 9, 300, 40), ("f32", 30, 1100, 50)])
def test_shared_prefix_captured(cuda, kv, n, prefix, longest):
    """One capture, replayed over other lengths, pages and queries, gives the
    bits of eager calls (each kernel choice: tensor cores, one launch, f32)."""
    lens = [(i * 13) % (longest + 1) for i in range(n)]
    s = Shared(cuda, prefix, lens, 16, 2, kv, seed=3, max_len=longest)
    K.attn_shared_prefix(**s.d)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.attn_shared_prefix(**s.d)
        K.attn_shared_prefix(**s.d)  # the same workspace, one after the other
    for seed in (11, 12):
        o = Shared(cuda, prefix, lens[::-1] if seed == 12 else lens, 16, 2, kv, seed=seed, max_len=longest)
        for k in ("q", "k_cache", "v_cache", "prefix_pages", "pages", "lens"):
            s.d[k].copy_(o.d[k])
        s.d["out"].fill_(5.0)
        g.replay()
        K.attn_shared_prefix(**o.d)
        torch.cuda.synchronize()
        assert torch.equal(s.d["out"], o.d["out"])
        o.check(range(0, n, 5))


def test_shared_prefix_workspace_of_another_size(cuda):
    """Calls of different shapes in turn through one workspace."""
    shapes = [(40, 4000, 60), (3, 100, 20), (12, 1000, 300), (70, 2500, 5)]
    cases = [Shared(cuda, p, [(i * 7) % (m + 1) for i in range(n)], 16, 2, "f16", seed=n, max_len=m) for n, p, m in shapes]
    ws = max((c.d["ws"] for c in cases), key=lambda t: t.numel())
    for _ in range(2):
        for c in cases:
            c.d["out"].fill_(5.0)
            K.attn_shared_prefix(**{**c.d, "ws": ws})
    for c in cases:
        c.check(range(0, len(c.lens), 9))


@pytest.mark.parametrize("prefix", [256, 257, 1535, 1537, 2999, 4097])
def test_shared_prefix_block_ends(cuda, prefix):
    """Prefixes that end at, before and behind the blocks and splits of the tensor-core form, and one bad page in it."""
    n = 65 if prefix > 1000 else 300
    s = Shared(cuda, prefix, [i % 3 for i in range(n)], 16, 2, "f16", seed=prefix)
    K.attn_shared_prefix(**s.d)
    s.check(range(0, n, n // 8))
    assert s.d["err"].item() == 0
    last = (prefix - 1) // PAGE
    s.d["prefix_pages"][last] = 1 << 24
    K.attn_shared_prefix(**s.d)
    s.prefix = last * PAGE
    s.check(range(0, n, n // 8))
    assert s.d["err"].item() == 1


def test_shared_prefix_rising_scores(cuda):
    """Scores that rise along the prefix: the tensor-core form moves its base again and again."""
    n, prefix = 64, 3000
    s = Shared(cuda, prefix, [4] * n, 16, 2, "f16", seed=8)
    rows = R.rows_of(s.ppages, prefix)
    d = np.sign(np.random.default_rng(1).standard_normal(HD)).astype(np.float32)
    s.kc[rows] = (s.kc[rows].astype(np.float32) * 0.3 + np.linspace(0, 4, prefix)[:, None, None] * d / 8).astype(np.float16)
    s.q[:, :16 * HD] = np.tile(d * 12, 16) + s.q[:, :16 * HD] * 0.1
    s.d["k_cache"].copy_(torch.from_numpy(s.kc.reshape(s.d["k_cache"].shape)))
    s.d["q"].copy_(torch.from_numpy(s.q[:, :16 * HD]))
    K.attn_shared_prefix(**s.d)
    s.check(range(0, n, 7))


# ---------------------------------------------------------------- sampling
def rows_for(n, rows, seed, kind):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, n)).astype(np.float32) * 2
    if kind == "peaked":
        for row in x:
            at = rng.choice(n, min(30, n), replace=False)
            row[at] = 5 + 9 * rng.random(len(at))
    elif kind == "bf16":  # logits that were held in bf16: many equal values
        x = (x.view(np.uint32) & 0xFFFF0000).view(np.float32).copy()
    elif kind == "masked":
        x[:, rng.random(n) < 0.7] = -np.inf
        x[:, rng.random(n) < 0.1] = np.nan
        x[0, :] = np.finfo(np.float32).min
        if rows > 1:
            x[1, :] = -1e9
            x[1, n // 2] = 1.0
        if rows > 2:
            x[2, :n // 2] = -1e9
    elif kind == "equal":
        x[:] = 0.25
    return x


def run_sample(cuda, x, t, k, p, m, r):
    rows = len(x)
    f = lambda v: torch.as_tensor(np.broadcast_to(np.asarray(v, np.float32), rows).copy(), device=cuda)  # noqa: E731
    ids = torch.full((rows,), 99, dtype=torch.int32, device=cuda)
    probs = torch.full((rows,), 9.0, device=cuda)
    K.sample_filtered(torch.from_numpy(x).to(cuda), f(r), ids, temp=f(t), top_k=i32(np.broadcast_to(k, rows).copy(), cuda),
                      top_p=f(p), min_p=f(m), probs=probs)
    torch.cuda.synchronize()
    return ids.cpu().numpy().view(np.uint32), probs.cpu().numpy().astype(np.float64)


def check_sample(x, got, probs, t, k, p, m, r):
    for i, row in enumerate(x):
        a = [float(np.float32(np.broadcast_to(v, len(x))[i])) for v in (t, p, m, r)]
        kk = int(np.broadcast_to(k, len(x))[i])
        want, share = R.sample(row, a[0], kk, a[1], a[2], a[3])
        if got[i] != want:
            assert R.sample_near(row, int(got[i]), a[0], kk, a[1], a[2], a[3]), (i, got[i], want, a, kk)
            continue
        # the token's weight (2^-26, or one part of the smallest unit held), the mass kept, the f32 result
        assert abs(probs[i] - share) <= share * (2.0 ** -24 + 2.0 ** -24) + 1e-30, (i, probs[i], share)


@pytest.mark.parametrize("kind", ["flat", "peaked", "bf16", "masked", "equal"])
@pytest.mark.parametrize("n", [1, 2, 33, 5003, 40001])
def test_sample(cuda, kind, n):
    rows = 6
    x = rows_for(n, rows, n, kind)
    r = np.array([0.0, 0.2, 0.5, 0.77, 0.999, 0.9999999], np.float32)
    for t, k, p, m in [(1, 0, 1, 0), (0.7, 40, 1, 0), (1.3, 0, 0.9, 0), (1, 0, 1, 0.05), (0.8, 200, 0.95, 0.01),
                       (1, 1, 1, 0), (1, 0, 0, 0), (0.05, 50, 0.99, 0), (30.0, 0, 0.7, 0), (0, n, 1, 0), (1, n + 5, 0.5, 0.9)]:
        got, probs = run_sample(cuda, x, t, k, p, m, r)
        check_sample(x, got, probs, t, k, p, m, r)


@pytest.mark.parametrize("rows", [1, 3, 12, 13, 40, 70])
def test_sample_full_vocabulary(cuda, rows):
    n = 151936
    x = np.concatenate([rows_for(n, -(-rows // 2), 1, "flat"), rows_for(n, rows // 2, 2, "peaked")])
    rng = np.random.default_rng(3)
    r = rng.random(rows, np.float32)
    t = rng.choice([0.6, 1.0, 1.5], rows)
    k = rng.choice([0, 0, 50, 5000], rows)
    p = rng.choice([1.0, 0.95, 0.5], rows)
    m = rng.choice([0.0, 0.0, 0.1], rows)
    got, probs = run_sample(cuda, x, t, k, p, m, r)
    check_sample(x, got, probs, t, k, p, m, r)


def test_sample_row_without_a_candidate(cuda):
    x = np.full((3, 700), -np.inf, np.float32)
    x[1, 650] = -5.0
    got, probs = run_sample(cuda, x, 1.0, 10, 0.9, 0.1, 0.5)
    assert got.tolist() == [R.EMPTY, 650, R.EMPTY] and probs.tolist() == [0.0, 1.0, 0.0]


def test_sample_infinite_maximum(cuda):
    x = np.zeros((4, 300), np.float32)
    x[:, [7, 200]] = np.inf
    got, probs = run_sample(cuda, x, 1.0, 0, 1.0, 0.0, [0.0, 0.4, 0.6, 1.0])
    assert got.tolist() == [7, 7, 200, 200] and probs.tolist() == [0.5] * 4


def test_sample_strided_rows_and_missing_parameters(cuda):
    x = rows_for(1001, 9, 5, "flat")
    wide = torch.full((9, 1100), 50.0, device=cuda)
    wide[:, 3:1004] = torch.from_numpy(x).to(cuda)
    r = np.linspace(0, 0.99, 9).astype(np.float32)
    ids = torch.zeros(9, dtype=torch.int32, device=cuda)
    K.sample_filtered(wide[:, 3:1004], torch.from_numpy(r).to(cuda), ids)
    torch.cuda.synchronize()
    for i, got in enumerate(ids.tolist()):
        assert R.sample_near(x[i], got, r=float(r[i]))


def test_sample_of_odd_parameters(cuda):
    """NaN and out-of-range parameters read as: temperature 1, filter off, r in [0, 1]."""
    x = rows_for(900, 6, 8, "flat")
    nan = float("nan")
    got, _ = run_sample(cuda, x, [nan, -1, 1, 1, 1, 1], [-3, 0, 0, 0, 0, 0], [1, nan, 2, 1, -1, 1], [0, 0, nan, 2.0, 0, -1],
                        [0.5, 0.5, 0.5, 0.5, 0.5, 7.0])
    best = x.argmax(1)
    for i in range(3):
        assert R.sample_near(x[i], int(got[i]), r=0.5)
    assert got[3] == best[3] and got[4] == best[4]
    assert R.sample_near(x[5], int(got[5]), r=1.0)
    got, _ = run_sample(cuda, x, 1.0, 0, 1.0, 0.0, [nan, -5, 0, 0, 0, 0])
    assert got.tolist() == best.tolist()


def test_sample_agrees_with_topk_and_sample_topk(cuda):
    """With top-k alone it is topk followed by sample_topk, but for r within
    f32's error of a token's border."""
    n = 151936
    x = rows_for(n, 8, 21, "peaked")
    r = np.linspace(0.03, 0.97, 8).astype(np.float32)
    got, _ = run_sample(cuda, x, 0.8, 40, 1.0, 0.0, r)
    for i in range(8):
        ids = torch.zeros(40, dtype=torch.int32, device=cuda)
        vals = torch.zeros(40, device=cuda)
        one = torch.zeros(1, dtype=torch.int32, device=cuda)
        K.topk(torch.from_numpy(x[i]).to(cuda), n, 40, ids, vals)
        K.sample_topk(ids, vals, 40, 0.8, float(r[i]), one)
        torch.cuda.synchronize()
        near = {R.sample(x[i], 0.8, 40, r=float(r[i]) + e)[0] for e in (-1e-5, 0, 1e-5)}
        assert one.item() in near and int(got[i]) in near


@pytest.mark.parametrize("order", ["falling", "rising", "blocks"])
def test_sample_neighbours_in_the_vocabulary(cuda, order):
    """The deciding tokens side by side in the row, or a whole row of a few values."""
    n = 100000
    x = np.sort(rows_for(n, 4, 6, "flat"), 1)
    x = {"falling": x[:, ::-1], "rising": x, "blocks": np.round(x * 4) / 4}[order].astype(np.float32).copy()
    r = np.array([0.1, 0.5, 0.9, 0.99], np.float32)
    for t, k, p, m in [(1, 0, 0.9, 0), (0.7, 3000, 1, 0.01), (1, 0, 1, 0)]:
        got, probs = run_sample(cuda, x, t, k, p, m, r)
        check_sample(x, got, probs, t, k, p, m, r)


def test_sample_extreme_temperatures(cuda):
    x = rows_for(3001, 5, 14, "flat")
    for t in (1e-40, 1e-30, 1e-25, 1e-6, 1e-3, 1e4, 1e28, 1e38, float("inf")):
        r = np.array([0.0, 0.3, 0.6, 0.9, 0.999], np.float32)
        got, probs = run_sample(cuda, x, t, 0, 1.0, 0.0, r)
        if t < 1e-4:
            assert got.tolist() == x.argmax(1).tolist() and (probs > 0.999).all()
        else:
            check_sample(x, got, probs, t, 0, 1.0, 0.0, r)


@pytest.mark.parametrize("spread", [1e-3, 0.3, 4.0, 50.0])
@pytest.mark.parametrize("offset", [0.0, -0.49, 0.02, 100.0, -1e4, 3e5, -2.0 ** 24])
def test_sample_offsets_of_the_logits(cuda, spread, offset):
    """Maxima below, above and near 0, and far above the spread, where neighbouring
    logits are few or one f32 step apart; a bin's middle must not round."""
    rng = np.random.default_rng(31)
    x = (rng.standard_normal((6, 20011)) * spread + offset).astype(np.float32)
    x[3, ::3] = -np.inf
    x[4, 1:] = np.minimum(x[4, 1:], np.float32(offset))
    r = np.array([0.01, 0.3, 0.5, 0.8, 0.97, 0.9999], np.float32)
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (spread, 0, 0.9, 0.0), (0.25 * spread, 300, 0.95, 0.02), (3 * spread, 0, 1.0, 0.3)]:
        got, probs = run_sample(cuda, x, t, k, p, m, r)
        check_sample(x, got, probs, t, k, p, m, r)


def test_sample_extreme_values(cuda):
    big = np.finfo(np.float32).max
    x = np.zeros((6, 500), np.float32)
    x[0, 3] = big
    x[1] = -1e30  # the lowest that is taken
    x[2] = 1e-42  # below f32's normal range, with one above
    x[2, 77] = 1e-38
    x[3, ::2] = -0.0  # equal to +0: ties to the lower id
    x[4] = -5e29
    x[4, 9] = -4e29
    x[5, :499] = np.float32(-1.0000001e30)  # never taken
    r = np.float32(0.5)
    got, probs = run_sample(cuda, x, 1.0, 0, 1.0, 0.0, r)
    assert got[0] == 3 and probs[0] == 1.0
    assert got[4] == 9 and probs[4] == 1.0
    assert got[5] == 499 and probs[5] == 1.0
    for i in (1, 2, 3):
        assert got[i] in (249, 250) and abs(probs[i] - 1 / 500) < 1e-9, (i, got[i], probs[i])
    got, _ = run_sample(cuda, x, 1.0, 7, 1.0, 0.0, np.float32(0.99))
    assert got[3] == 6 and got[1] == 6


def test_sample_two_streams_and_capture(cuda):
    """Two calls at once, and one capture replayed over other inputs (nothing is kept between calls)."""
    n = 30000
    xa, xb = rows_for(n, 7, 1, "flat"), rows_for(n, 40, 2, "peaked")
    f = lambda v, k: torch.full((k,), v, device=cuda)  # noqa: E731
    a = dict(logits=torch.from_numpy(xa).to(cuda), r=f(0.4, 7), ids=i32(np.zeros(7), cuda), top_p=f(0.9, 7))
    b = dict(logits=torch.from_numpy(xb).to(cuda), r=f(0.7, 40), ids=i32(np.zeros(40), cuda), min_p=f(0.02, 40))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        K.sample_filtered(**a, stream=s1)
        K.sample_filtered(**b, stream=s2)
    torch.cuda.synchronize()
    for x, c, kw in ((xa, a, dict(p=float(np.float32(0.9)), r=float(np.float32(0.4)))),
                     (xb, b, dict(minp=float(np.float32(0.02)), r=float(np.float32(0.7))))):
        assert all(R.sample_near(x[i], int(g), **kw) for i, g in enumerate(c["ids"].tolist()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.sample_filtered(**a)
    for seed in (5, 6):
        x = rows_for(n, 7, seed, "peaked")
        a["logits"].copy_(torch.from_numpy(x))
        a["ids"].fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        assert all(R.sample_near(x[i], int(v), p=float(np.float32(0.9)), r=float(np.float32(0.4))) for i, v in enumerate(a["ids"].tolist()))


def test_sample_same_bits_every_time(cuda):
    x = torch.from_numpy(rows_for(151936, 5, 30, "flat")).to(cuda)
    r = torch.rand(5, device=cuda)
    p = torch.full((5,), 0.9, device=cuda)
    out = []
    for _ in range(4):
        ids, probs = torch.zeros(5, dtype=torch.int32, device=cuda), torch.zeros(5, device=cuda)
        K.sample_filtered(x, r, ids, top_p=p, probs=probs)
        out.append((ids.tolist(), probs.tolist()))
    assert all(o == out[0] for o in out)


# ---------------------------------------------------------------- together
def serving_step(s):
    K.kv_append_paged(s["qkv"], s["pos"], s["slot"], s["pages"], s["kc"], s["vc"], s["cos"], s["sin"], 16,
                      q_out=s["q"], prefix_len=s["prefix"], err=s["err"])
    s["lens"] += 1
    K.attn_shared_prefix(s["q"], s["kc"], s["vc"], s["ppages"], s["prefix"], s["pages"], s["lens"], s["max_len"],
                         s["att"], s["ws"], err=s["err"])
    torch.matmul(s["att"], s["head"], out=s["logits"])
    K.sample_filtered(s["logits"], s["r"], s["ids"], temp=s["temp"], top_p=s["p"], probs=s["probs"])
    s["pos"] += 1


@pytest.mark.parametrize("graph", [False, True])
def test_a_serving_loop(cuda, graph):
    """A prefix appended once, then decode steps of a batch: append, attention,
    a head, sampling; each token against the definitions, eagerly and as one
    captured graph replayed for every step."""
    torch.backends.cuda.matmul.allow_tf32 = False
    rng = np.random.default_rng(77)
    n, nh, nkv, prefix, steps, vocab = 5, 16, 2, 37, 20, 300
    cos, sin = tables(prefix + 64)
    d = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(cuda)  # noqa: E731
    f = lambda v: torch.full((n,), v, device=cuda)  # noqa: E731
    perm = rng.permutation(64)
    s = dict(prefix=prefix, ppages=i32(perm[:3], cuda), pages=i32(perm[3:3 + 2 * n].reshape(n, 2), cuda), max_len=32,
             kc=torch.full((64, PAGE, nkv, HD), float("nan"), dtype=torch.float16, device=cuda), cos=d(cos), sin=d(sin),
             slot=i32(np.arange(n), cuda), pos=i32([prefix] * n, cuda), lens=i32([0] * n, cuda),
             qkv=torch.zeros(n, 20 * HD, device=cuda), q=torch.zeros(n, nh * HD, device=cuda),
             att=torch.zeros(n, nh * HD, device=cuda), head=d(rng.standard_normal((nh * HD, vocab)).astype(np.float32) * 0.3),
             logits=torch.zeros(n, vocab, device=cuda), r=f(0.0), temp=f(0.9), p=f(0.95), probs=f(0.0),
             ids=torch.zeros(n, dtype=torch.int32, device=cuda), err=torch.zeros(1, dtype=torch.int32, device=cuda),
             ws=torch.empty(K.attn_shared_prefix_bytes(n, nh, nkv, prefix, 32), dtype=torch.uint8, device=cuda))
    s["vc"] = s["kc"].clone()
    pre = rng.standard_normal((prefix, 20 * HD)).astype(np.float32)
    K.kv_append_paged(d(pre), i32(np.arange(prefix), cuda), i32(np.zeros(prefix), cuda), s["ppages"][None, :].contiguous(),
                      s["kc"], s["vc"], s["cos"], s["sin"], nh, err=s["err"])
    keys = [pre[:, nh * HD:(nh + nkv) * HD].reshape(prefix, nkv, HD)]
    vals = [pre[:, (nh + nkv) * HD:].reshape(prefix, nkv, HD)]
    k_all = [R.rotate(keys[0], cos[:prefix, None], sin[:prefix, None])[0].astype(np.float16)] * n
    v_all = [vals[0].astype(np.float16)] * n
    g = None
    if graph:
        before = {k: s[k].clone() for k in ("pos", "lens", "kc", "vc")}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            serving_step(s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            serving_step(s)
        for k, v in before.items():
            s[k].copy_(v)
    for step in range(steps):
        x = rng.standard_normal((n, 20 * HD)).astype(np.float32)
        r = rng.random(n, np.float32)
        s["qkv"].copy_(d(x))
        s["r"].copy_(d(r))
        g.replay() if graph else serving_step(s)
        torch.cuda.synchronize()
        att, logits = s["att"].cpu().numpy(), s["logits"].cpu().numpy()
        for b in range(n):
            c, sn = cos[prefix + step], sin[prefix + step]
            row = x[b].reshape(20, HD)
            q = R.rotate(row[:nh], c, sn)[0].astype(np.float32)
            k_all[b] = np.concatenate([k_all[b], R.rotate(row[nh:nh + nkv], c, sn)[0].astype(np.float16)[None]])
            v_all[b] = np.concatenate([v_all[b], row[nh + nkv:].astype(np.float16)[None]])
            o, bound = R.attention(q, k_all[b], v_all[b])
            # a key may round to the other f16 neighbour: one step of 2^-10 in one of 128 products, rarely
            slack = 2.0 ** -10 * 4 / HD * abs(o).max() + 2.0 ** -10 * 0.1
            assert (abs(att[b].reshape(nh, HD) - o) <= bound + slack).all()
            assert R.sample_near(logits[b], int(s["ids"][b]), t=float(np.float32(0.9)), p=float(np.float32(0.95)), r=float(r[b]))
    assert s["err"].item() == 0 and s["lens"].tolist() == [steps] * n
