"""Operators on packed sequences and on the paged cache (vaenar_tts_amd/sequence.py) against their definitions in 64 bits.

Tolerances are element by element and come from the arithmetic (before any run), with u = half a step of the operands' type, h = 2^-24:
  logits    e_s = (D + 4) h max_ij sum_d |q||k| scale          products and sums of D terms in 32 bits, the exponential's argument
  out       u |out| + (u + 2 e_s + (n + 16) h) sum_j p|v|       the result's rounding, the probabilities' rounding, 32-bit sums of n terms
  lse       e_s + (n + 16) h + 4 h |lse|
  dS        u |dS| + (2 e_s + 32 h) |dS| + P (e_dP + e_delta), e_dP = (D + 4) h sum|dO||v|,
            e_delta = sum_d |dO| e_out + (D + 4) h sum|dO||out|
  gradients u |g| + scale (sum e_dS |x| + (n + 16) h sum |dS||x|), dV with P in the place of dS"""
import ctypes as C

import numpy as np
import pytest

from vaenar_tts_amd import _lib, sequence
from vaenar_tts_amd.configs import tiny_hps

H24 = 2.0 ** -24
KINDS = {"f32": (np.float32, 2.0 ** -24), "f16": (np.float16, 2.0 ** -11), "bf16": (np.uint16, 2.0 ** -8)}


def store(x, kind):
    return sequence.to_bf16(x) if kind == "bf16" else np.ascontiguousarray(x, KINDS[kind][0])


def value(x):
    return (sequence.from_bf16(x) if x.dtype == np.uint16 else x).astype(np.float64)


def starts(lens, front=0):
    return (np.concatenate([[0], np.cumsum(lens)]) + front).astype(np.int32)


# ---- the definition -------------------------------------------------------------------------------------------------------------------
def definition(q, k, v, cu_q, cu_k, causal, scale, u, dout=None, first=None):
    """out, lse (and the gradients) in 64 bits with their element-wise tolerances: dict name -> (value, tolerance); rows outside the
    sequences are NaN.  ``first``: keys in front of row 0 per sequence (a cache) instead of causal's nk - nq."""
    H, G, D = q.shape[1], k.shape[1], q.shape[2]
    new = lambda *s: [np.full(s, np.nan), np.full(s, np.nan)]
    r = {"out": new(*q.shape), "lse": new(H, len(q))}
    if dout is not None:
        r.update(dq=new(*q.shape), dk=new(*k.shape), dv=new(*k.shape))
    for b in range(len(cu_q) - 1):
        iq, ik = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        nq, nk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if dout is not None:
            for n in ("dk", "dv"):
                for x in r[n]:
                    x[ik] = 0
        for h in range(H):
            g = h // (H // G)
            Q, K, V = q[iq, h], k[ik, g], v[ik, g]
            ahead = nk - nq if first is None else first[b]
            see = np.arange(nk) <= np.arange(nq)[:, None] + ahead if causal else np.ones((nq, nk), bool)
            x = np.where(see, Q @ K.T * scale, -np.inf) if nk else np.zeros((nq, 0))
            e_s = (D + 4) * H24 * scale * (np.where(see, np.abs(Q) @ np.abs(K).T, 0).max(initial=0))
            m = x.max(1, initial=-np.inf)[:, None]
            m = np.where(np.isfinite(m), m, 0)
            with np.errstate(divide="ignore"):
                p = np.exp(x - m)
                s = p.sum(1, keepdims=True)
                p = np.where(s > 0, p / np.where(s > 0, s, 1), 0)
                lse = (m + np.log(s))[:, 0]
            sums = (nk + 16) * H24
            out, A = p @ V, p @ np.abs(V)
            e_out = u * np.abs(out) + (u + 2 * e_s + sums) * A
            r["out"][0][iq, h], r["out"][1][iq, h] = out, e_out
            r["lse"][0][h, iq], r["lse"][1][h, iq] = lse, e_s + sums + 4 * H24 * np.abs(np.where(np.isfinite(lse), lse, 0))
            if dout is None:
                continue
            dO = dout[iq, h]
            dP = dO @ V.T
            delta = (dO * out).sum(1, keepdims=True)
            dS = p * (dP - delta)
            e_dP = (D + 4) * H24 * (np.abs(dO) @ np.abs(V).T)
            e_delta = (np.abs(dO) * e_out).sum(1, keepdims=True) + (D + 4) * H24 * (np.abs(dO) * np.abs(out)).sum(1, keepdims=True)
            e_dS = (u + 2 * e_s + 32 * H24) * np.abs(dS) + p * (e_dP + e_delta) * (1 + u)
            e_p = (u + 2 * e_s + 32 * H24) * p
            n_i = (nq * (H // G) + 16) * H24
            dq = scale * dS @ K
            r["dq"][0][iq, h] = dq
            r["dq"][1][iq, h] = u * np.abs(dq) + scale * (e_dS @ np.abs(K) + sums * np.abs(dS) @ np.abs(K))
            r["dk"][0][ik, g] += scale * dS.T @ Q
            r["dk"][1][ik, g] += scale * (e_dS.T @ np.abs(Q) + n_i * np.abs(dS).T @ np.abs(Q))
            r["dv"][0][ik, g] += p.T @ dO
            r["dv"][1][ik, g] += e_p.T @ np.abs(dO) + n_i * p.T @ np.abs(dO)
    if dout is not None:
        for n in ("dk", "dv"):
            r[n][1] += u * np.abs(r[n][0])
    return r


TINY = 2.0 ** -24          # the smallest step of float16: below its normal range a rounding is absolute


def close(got, want, what, kind="f32"):
    w, tol = want
    live = ~np.isnan(w)
    g = value(got)
    inf = live & np.isinf(w)
    assert (g[inf] == w[inf]).all(), what
    fin = live & ~inf
    off = np.abs(g[fin] - w[fin]) - (tol[fin] + (TINY if kind == "f16" else 1e-30))
    assert off.size == 0 or off.max() <= 0, "%s: %g beyond its tolerance (worst value %g)" % (what, off.max(), np.abs(g[fin] - w[fin]).max())


# ---- CPU ------------------------------------------------------------------------------------------------------------------------------
def test_definition_gradients_match_differences():
    """The gradients the tests hold the kernels to, against central differences of the definition's own output."""
    r = np.random.default_rng(3)
    cu_q, cu_k = starts([3, 4]), starts([5, 2])
    q, k, v, w = r.standard_normal((7, 4, 8)), r.standard_normal((7, 2, 8)), r.standard_normal((7, 2, 8)), r.standard_normal((7, 4, 8))
    f = lambda q, k, v: (definition(q, k, v, cu_q, cu_k, True, 0.4, 0)["out"][0] * w).sum()
    d = definition(q, k, v, cu_q, cu_k, True, 0.4, 0, dout=w)
    eps = 1e-6
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        for at in [(0, 0, 0), (2, 1, 3), (4, 0, 7), (6, 1, 5), (3, 0, 1)]:
            hi, lo = x.copy(), x.copy()
            hi[at] += eps
            lo[at] -= eps
            a = [{"dq": q, "dk": k, "dv": v}[n] for n in ("dq", "dk", "dv")]
            i = ("dq", "dk", "dv").index(name)
            num = (f(*(a[:i] + [hi] + a[i + 1:])) - f(*(a[:i] + [lo] + a[i + 1:]))) / (2 * eps)
            assert abs(num - d[name][0][at]) < 1e-7, (name, at)


def test_bfloat16_bits():
    x = np.array([1, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -2.5, 0, 3e38, np.inf, -np.inf, 1e-40], np.float32)
    y = sequence.from_bf16(sequence.to_bf16(x))
    assert list(y[:5]) == [1, 1, 1 + 2.0 ** -6, -2.5, 0] and np.isinf(y[6]) and np.isinf(y[7])
    assert np.isnan(sequence.from_bf16(sequence.to_bf16(np.float32([np.nan]))))[0]
    assert np.abs(y[5] / x[5] - 1) <= 2.0 ** -8


class Fake:
    """An engine that only lends its name to arrays (nothing is launched: every call below is refused)."""
    handle = None

    def call(self, *a, **k):
        raise AssertionError("a refused call reached the library")


def fake(shape, dtype=np.float16):
    return _lib.DeviceArray(Fake(), shape, dtype, ptr=0x1000, owner=None)


def test_python_refusals():
    e, q, k = Fake(), fake((6, 4, 64)), fake((6, 2, 64))
    cu, lse = fake((3,), np.int32), fake((4, 6), np.float32)
    ok = dict(out=q, lse=lse)
    for bad in (dict(k=fake((5, 2, 32))), dict(v=fake((6, 1, 64))), dict(cu_q=fake((3,), np.float32)), dict(cu_k=fake((4,), np.int32)),
                dict(q=fake((6, 4, 64), np.float64)), dict(k=fake((6, 2, 64), np.float32)), dict(lse=fake((6, 4), np.float32)),
                dict(out=fake((6, 4, 32))), dict(q=fake((6, 256)))):
        a = dict(q=q, k=k, v=k, cu_q=cu, **ok)
        a.update(bad)
        with pytest.raises(_lib.VnrError):
            sequence.packed_attention(e, **a)
    for bad in (dict(dout=fake((6, 4, 32))), dict(dk=fake((6, 4, 64))), dict(dq=fake((6, 4, 64), np.float32))):
        a = dict(dout=q, q=q, k=k, v=k, out=q, lse=lse, cu_q=cu, dq=q, dk=k, dv=k)
        a.update(bad)
        with pytest.raises(_lib.VnrError):
            sequence.packed_attention_grad(e, **a)
    with pytest.raises(_lib.VnrError):
        sequence.PagedCache(e, fake((4, 2, 16, 64)), fake((4, 2, 32, 64)))
    with pytest.raises(_lib.VnrError):
        sequence.PagedCache(e, fake((4, 2, 64)), fake((4, 2, 64)))
    c = sequence.PagedCache(e, fake((4, 2, 16, 64)), fake((4, 2, 16, 64)))
    ctx, table = fake((2,), np.int32), fake((2, 3), np.int32)
    for bad in (dict(k=fake((6, 4, 64))), dict(v=fake((5, 2, 64))), dict(context=fake((3,), np.int32)), dict(table=fake((3, 3), np.int32)),
                dict(q=fake((5, 4, 64))), dict(q_out=q), dict(rotation=fake((48, 64))), dict(k=fake((6, 2, 64), np.float32))):
        a = dict(k=k, v=k, cu=cu, context=ctx, table=table)
        a.update(bad)
        with pytest.raises(_lib.VnrError):
            c.append(**a)
    for bad in (dict(q=fake((6, 4, 32))), dict(out=fake((6, 2, 64))), dict(lse=fake((6, 4), np.float32)), dict(q=fake((6, 4, 64), np.float32))):
        a = dict(q=q, cu=cu, context=ctx, table=table, max_new=4, max_context=40, out=q)
        a.update(bad)
        with pytest.raises(_lib.VnrError):
            c.attend(**a)


def refused(name, *structs):
    lib = _lib.load()
    assert getattr(lib, name)(None, *[C.byref(s) for s in structs]) == -1
    return lib.vnr_last_error(None).decode()


def packed_desc(**kw):
    d = dict(dtype=1, batch=2, heads=4, kv_heads=2, head_dim=64, causal=1, scale=0.125, rows_q=6, rows_k=6, d_cu_q=64, d_cu_k=64, d_q=4096, d_k=4096, d_v=4096,
             ldq=256, ldk=128, ldv=128, d_out=4096, ldo=256, d_lse=None)
    d.update(kw)
    return _lib.vnr_packed_attention_desc(**d)


def test_library_refusals_of_packed_calls():
    """The library's own checks come before any use of the handle: they run here without a GPU, on pointers that nothing touches."""
    for bad, word in ((dict(dtype=3), "dtype"), (dict(batch=0), "batch"), (dict(heads=3), "multiple of kv_heads"), (dict(kv_heads=0), "kv_heads"),
                      (dict(head_dim=60), "head_dim"), (dict(head_dim=136), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(scale=0.0), "scale"),
                      (dict(scale=float("nan")), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(rows_q=-1), "row count"),
                      (dict(d_cu_q=None), "starts"), (dict(d_cu_k=None), "starts"), (dict(d_q=None), "q is null"), (dict(d_k=4104), "aligned"),
                      (dict(ldq=248), "stride"), (dict(ldv=129), "stride"), (dict(ldk=64), "stride"), (dict(d_out=None), "out is null"), (dict(), "null handle")):
        assert word in refused("vnr_op_packed_attention", packed_desc(**bad)), bad
    g = dict(d_dout=4096, lddo=256, d_dq=4096, d_dk=4096, d_dv=4096, lddq=256, lddk=128, lddv=128)
    for bad, word in ((dict(d_dout=None), "dout"), (dict(lddq=128), "dq"), (dict(d_dk=4100), "dk"), (dict(lddv=100), "dv"), (dict(), "null handle")):
        assert word in refused("vnr_op_packed_attention_grad", packed_desc(d_lse=64), _lib.vnr_packed_attention_grad(**{**g, **bad})), bad
    assert "lse" in refused("vnr_op_packed_attention_grad", packed_desc(), _lib.vnr_packed_attention_grad(**g))


def test_library_refusals_of_cache_calls():
    cache = dict(dtype=1, kv_heads=2, head_dim=64, pages=8, page_size=16, d_k=4096, d_v=4096)
    app = dict(batch=2, heads=4, rows=6, d_cu=64, d_context=64, d_table=64, table_width=3, d_k=1 << 20, d_v=1 << 20, ldk=128, ldv=128, d_q=1 << 20, d_q_out=2 << 20,
               ldq=256, ldqo=256, d_rotation=64, rotation_rows=48, rot_dim=64, interleaved=0)
    att = dict(batch=2, heads=4, rows=6, d_cu=64, d_context=64, d_table=64, table_width=3, max_new=4, max_context=40, scale=0.125, d_q=4096, ldq=256, d_out=4096,
               ldo=256, d_lse=None)
    A, P, K = _lib.vnr_kv_append_desc, _lib.vnr_paged_attention_desc, _lib.vnr_kv_cache
    for bad, word in ((dict(page_size=12), "page_size"), (dict(page_size=0), "page_size"), (dict(page_size=8192), "page_size"), (dict(pages=0), "pages"),
                      (dict(d_k=None), "pools"), (dict(d_v=4104), "pools"), (dict(dtype=-1), "dtype"), (dict(head_dim=130), "head_dim")):
        assert word in refused("vnr_op_kv_append", K(**{**cache, **bad}), A(**app)), bad
        assert word in refused("vnr_op_paged_attention", K(**{**cache, **bad}), P(**att)), bad
    for bad, word in ((dict(rows=-1), "row count"), (dict(d_k=None), "k is null"), (dict(ldv=120), "stride"), (dict(d_q_out=None), "together"),
                      (dict(d_q=None), "together"), (dict(d_q_out=1 << 20), "overlaps"), (dict(d_q_out=(1 << 20) + 512), "overlaps"), (dict(rot_dim=72), "rot_dim"),
                      (dict(rot_dim=24), "rot_dim"), (dict(rot_dim=20, interleaved=1), "rot_dim"), (dict(rot_dim=-16), "rot_dim"), (dict(d_rotation=None), "table is null"),
                      (dict(rotation_rows=47), "cover"), (dict(table_width=0), "table_width"), (dict(table_width=1 << 28), "table_width"),
                      (dict(d_cu=None), "starts"), (dict(heads=3), "heads"), (dict(), "null handle"),
                      (dict(d_q=None, d_q_out=None), "null handle"),
                      # q and q_out as two column blocks of one matrix do not overlap
                      (dict(d_q_out=(1 << 20) + 512, ldq=512, ldqo=512), "null handle"), (dict(d_q_out=(1 << 20) + 256, ldq=512, ldqo=512), "overlaps")):
        assert word in refused("vnr_op_kv_append", K(**cache), A(**{**app, **bad})), bad
    for bad, word in ((dict(max_new=0), "max_new"), (dict(max_context=0), "max_context"), (dict(scale=0.0), "scale"), (dict(d_q=None), "q is null"), (dict(heads=5), "heads"),
                      (dict(ldo=200), "stride"), (dict(d_table=None), "table"), (dict(), "null handle")):
        assert word in refused("vnr_op_paged_attention", K(**cache), P(**{**att, **bad})), bad


def test_library_refusals_of_sizes_that_no_launch_holds():
    assert "scale" in refused("vnr_op_packed_attention", packed_desc(scale=3e38))
    assert "heads" in refused("vnr_op_packed_attention", packed_desc(heads=1 << 21, ldq=1 << 27, ldo=1 << 27))
    cache = _lib.vnr_kv_cache(dtype=1, kv_heads=2, head_dim=64, pages=8, page_size=16, d_k=4096, d_v=4096)
    assert "2^24" in refused("vnr_op_kv_append", cache, _lib.vnr_kv_append_desc(batch=1, rows=1 << 24, d_cu=64, d_context=64, d_table=64, table_width=3, d_k=4096, d_v=4096,
                                                                               ldk=128, ldv=128))
    lib = _lib.load()
    assert lib.vnr_op_rotation_table(None, 1 << 30, 128, 1e4, C.c_void_p(4096)) == -1 and "2^31" in lib.vnr_last_error(None).decode()


def test_sequence_structs_match_the_header_layout(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = ["vnr_packed_attention_desc", "vnr_packed_attention_grad", "vnr_kv_cache", "vnr_kv_append_desc", "vnr_paged_attention_desc"]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"vaenar_hip.h\"\nint main(void) {\n"
    want = []
    for n in names:
        s = getattr(_lib, n)
        src += 'printf("%%zu ", sizeof(%s));\n' % n
        want.append(C.sizeof(s))
        for f, _ in s._fields_:
            src += 'printf("%%zu ", offsetof(%s, %s));\n' % (n, f)
            want.append(getattr(s, f).offset)
    open(tmp_path / "t.c", "w").write(src + "return 0; }\n")
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")])
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "t")]).split()] == want


# ---- GPU ------------------------------------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def eng():
    e = _lib.Engine(tiny_hps(), 0)
    yield e
    e.close()


def normal(r, kind, *shape):
    return store(r.standard_normal(shape).astype(np.float32), kind)


PACKED = [
    # lens of queries, lens of keys (None: the same), heads, kv_heads, head_dim, causal
    ([1], None, 1, 1, 64, True),
    ([1, 2, 3, 0, 5], None, 4, 2, 64, True),
    ([33, 64, 65], None, 4, 4, 64, False),
    ([128, 129, 1, 127], None, 2, 1, 128, True),
    ([200, 0, 77], None, 5, 1, 80, True),
    ([31, 32, 100], None, 8, 2, 8, False),
    ([130, 7], None, 3, 3, 104, True),
    ([5, 40, 1, 3], [70, 40, 200, 0], 4, 2, 64, True),            # more keys than rows, and a sequence without keys
    ([70, 150, 12], [5, 131, 12], 2, 1, 128, True),               # more rows than keys: the first rows see nothing
    ([3, 260], [260, 3], 2, 2, 72, False),
    ([0, 0, 9], [4, 0, 9], 2, 1, 64, True),                       # keys that no row sees
    ([300], None, 1, 1, 128, True),
    ([530], None, 2, 1, 64, True),                                # rows enough for the launches of long sequences
    ([400, 633], [633, 400], 4, 2, 128, True),
]
IDS = ["-".join([str(i)]) for i in range(len(PACKED))]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", PACKED, ids=IDS)
def test_packed_attention_and_gradient(eng, case, kind):
    lq, lk, H, G, D, causal = case
    u = KINDS[kind][1]
    r = np.random.default_rng(sum(lq) * 7 + H + D)
    cu_q = starts(lq, 2)
    cu_k = cu_q if lk is None else starts(lk, 3)
    nq, nk = cu_q[-1] + 3, cu_k[-1] + (3 if lk is None else 1)    # rows in front of the first sequence and behind the last
    q, k, v, do = (normal(r, kind, n, h, D) for n, h in ((nq, H), (nk, G), (nk, G), (nq, H)))
    bad = store(np.float32([np.nan]), kind)[0]
    for x, cu in ((q, cu_q), (k, cu_k), (v, cu_k), (do, cu_q)):   # what is in those rows is nobody's business
        x[:cu[0]] = bad
        x[cu[-1]:] = bad
    scale = 1.3 / np.sqrt(D)
    want = definition(value(q), value(k), value(v), cu_q, cu_k, causal, np.float64(np.float32(scale)), u, dout=value(do))
    d = [eng.to_device(x) for x in (q, k, v, do)]
    cq = eng.to_device(cu_q)
    ck = cq if lk is None else eng.to_device(cu_k)
    mark = store(np.full(1, 7.0, np.float32), kind)[0]
    filled = lambda x: eng.to_device(np.full(x.shape, mark, x.dtype))
    out, dq, dk, dv = filled(q), filled(q), filled(k), filled(k)
    lse = eng.to_device(np.full((H, nq), 7.0, np.float32))
    sequence.packed_attention(eng, d[0], d[1], d[2], cq, None if lk is None else ck, causal, scale, out, lse)
    sequence.packed_attention_grad(eng, d[3], d[0], d[1], d[2], out, lse, cq, None if lk is None else ck, causal, scale, dq, dk, dv)
    for name, a in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        got = a.numpy()
        close(got, want[name], name, kind)
        cu = cu_k if name in ("dk", "dv") else cu_q
        assert (got[:cu[0]] == mark).all() and (got[cu[-1]:] == mark).all(), name + ": rows outside the sequences were written"
    got = lse.numpy()
    close(got, want["lse"], "lse")
    assert (got[:, :cu_q[0]] == 7).all() and (got[:, cu_q[-1]:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_packed_attention_on_column_blocks(eng, kind):
    """q, k, v, dout as column blocks of one projection's rows, results as column blocks too: the rest of the rows stays."""
    H, G, D, u = 4, 2, 64, KINDS[kind][1]
    lens = [40, 3, 90]
    cu = starts(lens)
    n, width = cu[-1], (H + 2 * G) * D + 8
    r = np.random.default_rng(9)
    x, do = normal(r, kind, n, width), normal(r, kind, n, H * D + 16)
    cut = lambda a, o, h: value(a[:, o:o + h * D]).reshape(n, h, D)
    q, k, v = cut(x, 0, H), cut(x, H * D, G), cut(x, (H + G) * D, G)
    want = definition(q, k, v, cu, cu, True, D ** -0.5, u, dout=cut(do, 16, H))
    dx, ddo, c = eng.to_device(x), eng.to_device(do), eng.to_device(cu)
    g = eng.to_device(x)                                          # gradients into the same columns of a matrix like it
    o = eng.to_device(np.zeros((n, H * D + 24), x.dtype))
    a = [dx.view(0, (n, H, D)), dx.view(H * D, (n, G, D)), dx.view((H + G) * D, (n, G, D))]
    ov, lse = o.view(8, (n, H, D)), eng.empty((H, n))
    ld = dict(ldq=width, ldk=width, ldv=width, ldo=H * D + 24)
    sequence.packed_attention(eng, *a, c, out=ov, lse=lse, **ld)
    sequence.packed_attention_grad(eng, ddo.view(16, (n, H, D)), *a, ov, lse, c, dq=g.view(0, (n, H, D)), dk=g.view(H * D, (n, G, D)),
                                   dv=g.view((H + G) * D, (n, G, D)), lddout=H * D + 16, lddq=width, lddk=width, lddv=width, **ld)
    oh, gh = o.numpy(), g.numpy()
    shaped = lambda a, o, h: a[:, o:o + h * D].reshape(n, h, D)
    close(shaped(oh, 8, H), want["out"], "out", kind)
    assert (oh[:, :8] == 0).all() and (oh[:, 8 + H * D:] == 0).all() and (gh[:, -8:] == x[:, -8:]).all()
    for name, at, h in (("dq", 0, H), ("dk", H * D, G), ("dv", (H + G) * D, G)):
        close(shaped(gh, at, h), want[name], name, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_with_one_key_add_exactly_nothing_to_dq_and_dk(eng, dim, kind):
    """Their weight is 1 whatever the logit: no rounding of delta may be left over, not even where all of dQ and dK is made of such rows."""
    r = np.random.default_rng(dim)

    def gradients(lq, lk, causal):
        cu_q, cu_k = starts(lq), starts(lk)
        q, k, v, do = (eng.to_device(normal(r, kind, n, h, dim)) for n, h in ((cu_q[-1], 8), (cu_k[-1], 2), (cu_k[-1], 2), (cu_q[-1], 8)))
        cq, ck = eng.to_device(cu_q), eng.to_device(cu_k)
        out, lse = sequence.packed_attention(eng, q, k, v, cq, ck, causal)
        return [value(x.numpy()) for x in sequence.packed_attention_grad(eng, do, q, k, v, out, lse, cq, ck, causal)]

    for lq, lk, causal in (([1] * 7, [1] * 7, True), ([1] * 3, [1] * 3, False), ([40, 1, 300], [1, 1, 1], False), ([40, 300], [1, 1], True)):
        dq, dk, dv = gradients(lq, lk, causal)
        assert (dq == 0).all() and (dk == 0).all() and (dv != 0).any()
    # of longer sequences the first row that sees a key: row 0, and row 20 of the one with more rows than keys
    dq, dk, dv = gradients([50, 300, 120], [50, 300, 100], True)
    assert (dq[[0, 50, 350 + 20]] == 0).all() and (dq[[1, 51, 350 + 21]] != 0).any()


@pytest.mark.gpu
def test_packed_gradient_has_the_same_bits_every_time(eng):
    r = np.random.default_rng(4)
    cu = starts([200, 90, 333])
    q, k, v, do = (eng.to_device(normal(r, "bf16", cu[-1], h, 128)) for h in (8, 2, 2, 8))
    c = eng.to_device(cu)
    out, lse = sequence.packed_attention(eng, q, k, v, c)
    a = [x.numpy() for x in sequence.packed_attention_grad(eng, do, q, k, v, out, lse, c)]
    for _ in range(3):
        assert all((x.numpy() == y).all() for x, y in zip(sequence.packed_attention_grad(eng, do, q, k, v, out, lse, c), a))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_packed_attention_with_broken_starts(eng, kind):
    """Starts that run backwards or leave the tensor: those sequences are empty or cut, the others are right, nothing else is written."""
    H, D = 2, 64
    r = np.random.default_rng(5)
    q, k, v = (normal(r, kind, 50, H, D) for _ in range(3))
    cu = np.int32([0, 20, 10, 1000])                              # 0..20; 20..10 is empty; 10..1000 is cut to 10..50
    d, c = [eng.to_device(x) for x in (q, k, v)], eng.to_device(cu)
    out, lse = sequence.packed_attention(eng, *d, c)
    got = out.numpy()
    assert np.isfinite(value(got)).all()
    want = definition(value(q), value(k), value(v), starts([20]), starts([20]), True, D ** -0.5, KINDS[kind][1])
    close(got[:10], [x[:10] for x in want["out"]], "out", kind)


# ---- the cache ------------------------------------------------------------------------------------------------------------------------
def turned(x, pos, rot, base, interleaved):
    """[n, heads, D] turned by its positions, in 64 bits from the table's 32-bit entries"""
    half = rot // 2
    ang = np.asarray(pos, np.float64)[:, None] * base ** (-2.0 * np.arange(half) / rot)
    cs, sn = (f(ang).astype(np.float32).astype(np.float64)[:, None] for f in (np.cos, np.sin))
    y = x.copy()
    i, j = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(half), np.arange(half, rot))
    y[..., i], y[..., j] = x[..., i] * cs - x[..., j] * sn, x[..., j] * cs + x[..., i] * sn
    return y


def layout(r, totals, P, spare=2):
    """A page table of shuffled pages for sequences of `totals` positions, and the pool's size"""
    held = [-(-t // P) for t in totals]
    pages = sum(held) + spare
    order = r.permutation(pages).astype(np.int32)
    table = np.full((len(totals), max(max(held), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


APPEND = [
    # new, context, page, heads, kv_heads, head_dim, rot_dim, interleaved
    ([1], [0], 16, 1, 1, 64, 64, False),
    ([1, 1, 1], [5, 15, 16], 16, 8, 2, 128, 128, False),
    ([7, 0, 33], [3, 9, 60], 8, 4, 4, 64, 32, False),
    ([20, 5], [0, 100], 1, 3, 1, 80, 48, True),
    ([40], [1000], 64, 5, 5, 8, 8, True),
    ([3, 70], [2, 4000], 128, 4, 2, 104, 16, False),
    ([3, 2], [2, 1], 16, 2, 2, 64, 0, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", APPEND, ids=[str(i) for i in range(len(APPEND))])
def test_append(eng, case, kind):
    new, ctx, P, H, G, D, rot, inter = case
    u = KINDS[kind][1]
    r = np.random.default_rng(sum(new) + P)
    table, pages = layout(r, [n + c for n, c in zip(new, ctx)], P)
    cu = starts(new, 1)
    n = cu[-1] + 2
    k, v, q = normal(r, kind, n, G, D), normal(r, kind, n, G, D), normal(r, kind, n, H, D)
    kc, vc = normal(r, kind, pages, G, P, D), normal(r, kind, pages, G, P, D)
    base = 500.0
    dk, dv = eng.to_device(kc), eng.to_device(vc)
    cache = sequence.PagedCache(eng, dk, dv)
    table_rot = sequence.rotation_table(eng, table.shape[1] * P, rot, base) if rot else None
    mark = store(np.full(1, 7.0, np.float32), kind)[0]
    qo = eng.to_device(np.full(q.shape, mark, q.dtype))
    cache.append(eng.to_device(k), eng.to_device(v), eng.to_device(cu), eng.to_device(np.int32(ctx)), eng.to_device(table), rotation=table_rot,
                 q=eng.to_device(q), q_out=qo, interleaved=inter)
    want_k, want_v, want_q = value(kc), vc.copy(), np.full(q.shape, np.nan)
    touched = np.zeros(kc.shape, bool)
    for b, m in enumerate(new):
        pos = ctx[b] + np.arange(m)
        kt, qt = value(k[cu[b]:cu[b + 1]]), value(q[cu[b]:cu[b + 1]])
        if rot:
            kt, qt = turned(kt, pos, rot, base, inter), turned(qt, pos, rot, base, inter)
        want_q[cu[b]:cu[b + 1]] = qt
        for i, p in enumerate(pos):
            page = table[b, p // P]
            want_k[page, :, p % P], want_v[page, :, p % P] = kt[i], v[cu[b] + i]
            touched[page, :, p % P] = True
    # two products and a sum in 32 bits, one rounding; the table's own rounding of cos / sin is in the reference (h: it may differ by one)
    tol = lambda w: (u + 4 * H24) * np.abs(w) + 12 * H24
    gk, gq = dk.numpy(), qo.numpy()
    assert (dv.numpy() == want_v).all()
    assert (gk[~touched] == kc[~touched]).all()
    close(gk, (want_k, tol(want_k)), "k", kind)
    close(gq, (want_q, np.where(np.isnan(want_q), 0, tol(want_q))), "q", kind)
    assert (gq[0] == mark).all() and (gq[cu[-1]:] == mark).all()


@pytest.mark.gpu
def test_rotation_table_of_far_positions(eng):
    t = sequence.rotation_table(eng, 100003, 64, 10000.0).numpy()
    for p in (0, 1, 4097, 65537, 100002):
        ang = p * 10000.0 ** (-2.0 * np.arange(32) / 64)
        assert np.abs(t[p] - np.concatenate([np.cos(ang), np.sin(ang)])).max() <= 2 * H24
    assert t.shape == (100003, 64)


@pytest.mark.gpu
def test_append_drops_what_has_no_place(eng):
    """Pages outside the pool, positions behind the table: nothing is written for them, the rest is; the queries turn where they have an angle."""
    r = np.random.default_rng(8)
    P, G, D, pages = 4, 2, 64, 5
    k, v = normal(r, "f16", 12, G, D), normal(r, "f16", 12, G, D)
    kc = normal(r, "f16", pages, G, P, D)
    table = np.int32([[3, -1], [1 << 30, 0], [2, 5]])
    cu, ctx = starts([6, 4, 2]), np.int32([0, 6, 3])             # 0: positions 0..5 (page -1 from 4); 1: 6..9 (8, 9 behind the table); 2: 3, 4 (page 5)
    dk, dv = eng.to_device(kc), eng.to_device(kc)
    sequence.PagedCache(eng, dk, dv).append(eng.to_device(k), eng.to_device(v), eng.to_device(cu), eng.to_device(ctx), eng.to_device(table))
    want = kc.copy()
    for row, page, slot in ((0, 3, 0), (1, 3, 1), (2, 3, 2), (3, 3, 3), (6, 0, 2), (7, 0, 3), (10, 2, 3)):
        want[page, :, slot] = k[row]
    assert (dk.numpy() == want).all()


PAGED = [
    # new, context, page, heads, kv_heads, head_dim
    ([1], [0], 16, 1, 1, 64),
    ([1, 1, 0, 1], [1, 63, 7, 64], 16, 4, 4, 64),
    ([1, 1], [1000, 3], 16, 8, 2, 128),
    ([1, 1, 1], [127, 2049, 700], 1, 5, 1, 80),
    ([5, 2, 1], [300, 0, 33], 32, 8, 2, 64),
    ([40, 3], [100, 513], 64, 4, 1, 128),
    ([130, 0, 65], [5, 60, 0], 8, 3, 3, 96),
    ([9, 200], [1500, 1], 128, 4, 2, 64),
    ([1], [5000], 4096, 2, 1, 8),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", PAGED, ids=[str(i) for i in range(len(PAGED))])
def test_paged_attention(eng, case, kind):
    new, ctx, P, H, G, D = case
    u = KINDS[kind][1]
    r = np.random.default_rng(sum(new) + sum(ctx))
    totals = [n + c for n, c in zip(new, ctx)]
    table, pages = layout(r, totals, P)
    # a pool whose unused places hold NaN: behind a sequence's last position, and in pages that are nobody's
    bad = store(np.float32([np.nan]), kind)[0]
    kc, vc = np.full((pages, G, P, D), bad, KINDS[kind][0]), np.full((pages, G, P, D), bad, KINDS[kind][0])
    k, v = normal(r, kind, sum(totals), G, D), normal(r, kind, sum(totals), G, D)
    at = starts(totals)
    for b, n in enumerate(totals):
        for p in range(n):
            kc[table[b, p // P], :, p % P], vc[table[b, p // P], :, p % P] = k[at[b] + p], v[at[b] + p]
    cu = starts(new, 1)
    n = cu[-1] + 2
    q = normal(r, kind, n, H, D)
    q[0], q[cu[-1]:] = bad, bad
    want = definition(value(q), value(k), value(v), cu, at, True, D ** -0.5, u, first=ctx)
    mark = store(np.full(1, 7.0, np.float32), kind)[0]
    out, lse = eng.to_device(np.full(q.shape, mark, q.dtype)), eng.to_device(np.full((H, n), 7.0, np.float32))
    cache = sequence.PagedCache(eng, eng.to_device(kc), eng.to_device(vc))
    cache.attend(eng.to_device(q), eng.to_device(cu), eng.to_device(np.int32(ctx)), eng.to_device(table), max(max(new), 1), max(totals), out=out, lse=lse)
    got, gl = out.numpy(), lse.numpy()
    close(got, want["out"], "out", kind)
    close(gl, want["lse"], "lse")
    assert (got[0] == mark).all() and (got[cu[-1]:] == mark).all() and (gl[:, 0] == 7).all() and (gl[:, cu[-1]:] == 7).all()
    # bounds that are wider than the batch: another launch, the same values
    wide = eng.to_device(np.full(q.shape, mark, q.dtype))
    cache.attend(eng.to_device(q), eng.to_device(cu), eng.to_device(np.int32(ctx)), eng.to_device(table), 10000, 1 << 20, out=wide)
    close(wide.numpy(), want["out"], "out (wide bounds)", kind)


@pytest.mark.gpu
def test_paged_attention_reads_absent_pages_as_zeros(eng):
    r = np.random.default_rng(2)
    P, G, D = 16, 1, 64
    kc, vc = normal(r, "f32", 3, G, P, D), normal(r, "f32", 3, G, P, D)
    q = normal(r, "f32", 2, 2, D)
    table = np.int32([[1, -5, 2], [7, 0, 1 << 30]])
    cu, ctx = starts([1, 1]), np.int32([40, 47])
    full = np.zeros((2, 48, G, D)), np.zeros((2, 48, G, D))
    for b in range(2):
        for j in range(3):
            if 0 <= table[b, j] < 3:
                full[0][b, 16 * j:16 * j + 16], full[1][b, 16 * j:16 * j + 16] = (x[table[b, j]].transpose(1, 0, 2) for x in (kc, vc))
    out = sequence.PagedCache(eng, eng.to_device(kc), eng.to_device(vc)).attend(eng.to_device(q), eng.to_device(cu), eng.to_device(ctx), eng.to_device(table), 1, 48)
    want = definition(value(q), full[0].reshape(96, G, D), full[1].reshape(96, G, D), cu, starts([48, 48]), True, D ** -0.5, 2.0 ** -24, first=[40, 47])
    close(out.numpy(), want["out"], "out")


def prefix(q, k, v, limit, scale):
    """Row by row over the keys it sees and no other: what is behind them may be anything."""
    out = np.zeros((q.shape[0], v.shape[1]))
    with np.errstate(invalid="ignore"):
        for i, n in enumerate(limit):
            if n > 0:
                x = k[:n] @ q[i] * scale
                p = np.exp(x - x.max())
                out[i] = (p / p.sum()) @ v[:n]
    return out


TAINTS = [
    # what, sequence's rows, its keys in front (a cache), head width; places (row or None = all channels, channel)
    ("v", 90, 0, 64, [(40, None)]),
    ("v", 200, 0, 128, [(0, 5), (131, 9), (140, None)]),
    ("v", 70, 0, 64, [(69, None)]),
    ("k", 100, 0, 128, [(33, None), (99, None)]),
    ("v", 130, 70, 64, [(75, 3), (150, None)]),
    ("v", 50, 300, 128, [(320, None), (349, 0)]),
    ("k", 3, 61, 64, [(62, None)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("number", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("case", TAINTS, ids=[str(i) for i in range(len(TAINTS))])
def test_later_keys_that_are_not_finite_reach_no_earlier_row(eng, case, number, kind):
    """An infinity or a NaN in a key or value that a row does not see leaves that row as it is, whichever tile it shares with others that do
    see it; the rows that see it get what the arithmetic gives.  Small and large launches take different kernels: 1 and 80 heads."""
    what, n, ctx, D, places = case
    r = np.random.default_rng(n + ctx)
    total = n + ctx
    k, v = normal(r, kind, total, 1, D), normal(r, kind, total, 1, D)
    for row, ch in places:
        (v if what == "v" else k)[row, 0, slice(None) if ch is None else ch] = store(np.float32([number]), kind)[0]
    for H in (1, 80) if ctx == 0 else (1, 4, 40):
        q = normal(r, kind, n, H, D)
        limit = ctx + np.arange(n) + 1
        if ctx == 0:
            out, _ = sequence.packed_attention(eng, eng.to_device(q), eng.to_device(k), eng.to_device(v), eng.to_device(starts([n])))
        else:
            P = 16
            table, pages = layout(r, [total], P)
            kc, vc = np.zeros((pages, 1, P, D), k.dtype), np.zeros((pages, 1, P, D), k.dtype)
            for p in range(total):
                kc[table[0, p // P], :, p % P], vc[table[0, p // P], :, p % P] = k[p], v[p]
            out = sequence.PagedCache(eng, eng.to_device(kc), eng.to_device(vc)).attend(
                eng.to_device(q), eng.to_device(starts([n])), eng.to_device(np.int32([ctx])), eng.to_device(table), n, total)
        got = value(out.numpy())
        clean_k, clean_v = value(k)[:, 0], value(v)[:, 0]
        for h in (0, H - 1):
            want = prefix(value(q)[:, h], clean_k, clean_v, limit, np.float64(np.float32(D ** -0.5)))
            fine = np.isfinite(want)
            first = min(p for p, _ in places)
            assert np.isfinite(got[:max(0, first - ctx), h]).all()                  # rows in front of all of them
            if what == "v":                                                         # (a logit that is not finite makes its row's sums so, one way or another)
                assert (np.isfinite(got[:, h]) == fine).all()
                # an infinity may come out as NaN: a weight below 2^-25 of the row's largest is 0 in float16 (below 2^-126 in the others),
                # and 0 times infinity is NaN; it comes out as no other infinity
                inf = np.isinf(want) & np.isinf(got[:, h])
                assert (got[:, h][inf] == want[inf]).all()
            u = KINDS[kind][1]
            ok = fine & np.isfinite(got[:, h])
            # (8 u of the values' size is wide of the derived bounds above: what is looked for here is a reach, not a rounding)
            assert np.abs(got[:, h][ok] - want[ok]).max(initial=0) <= 8 * u + 1e-4, (H, h)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_prompt_then_chunks_then_single_rows(eng, kind):
    """The operators as they are used together: prompts through packed attention and append, a chunk, then one row at a time -- every row's
    output has to be what attention over the whole sequence gives."""
    H, G, D, P, u = 4, 2, 64, 16, KINDS[kind][1]
    r = np.random.default_rng(11)
    steps = [[37, 5], [20, 64], [1, 1], [1, 1], [0, 1]]
    total = [sum(s[b] for s in steps) for b in range(2)]
    table, pages = layout(r, total, P)
    cache = sequence.PagedCache.empty(eng, pages, G, P, D, KINDS[kind][0])
    rot, dt = sequence.rotation_table(eng, table.shape[1] * P, D), eng.to_device(table)
    kept = {n: [[], []] for n in ("q", "k", "v", "out")}
    ctx = [0, 0]
    for i, new in enumerate(steps):
        n = sum(new)
        q, k, v = normal(r, kind, n, H, D), normal(r, kind, n, G, D), normal(r, kind, n, G, D)
        dq, dk, dv, cu, c = (eng.to_device(x) for x in (q, k, v, starts(new), np.int32(ctx)))
        qt = cache.append(dk, dv, cu, c, dt, rotation=rot, q=dq)
        kt = eng.empty((n, G, D), KINDS[kind][0])                 # the rotated keys, through the query side of another append
        cache.append(dk, dv, cu, c, dt, rotation=rot, q=dk, q_out=kt)
        if i == 0:
            out, _ = sequence.packed_attention(eng, qt, kt, dv, cu)
        else:
            out = cache.attend(qt, cu, c, dt, max(new), max(x + y for x, y in zip(ctx, new)))
        got, turned_q, turned_k, s = out.numpy(), qt.numpy(), kt.numpy(), starts(new)
        for b in range(2):
            for name, x in (("q", turned_q), ("k", turned_k), ("v", v), ("out", got)):
                kept[name][b].append(x[s[b]:s[b + 1]])
            ctx[b] += new[b]
    cu = starts(total)
    whole = {n: np.concatenate([np.concatenate(kept[n][b]) for b in range(2)]) for n in kept}
    want = definition(value(whole["q"]), value(whole["k"]), value(whole["v"]), cu, cu, True, D ** -0.5, u)
    close(whole["out"], want["out"], "out", kind)


MANY = [
    # sequences, longest, heads, kv_heads, head_dim, causal: more than one look at the starts; more workgroups than the chip holds, in the order of their lengths
    (70, 9, 2, 1, 64, True),
    (150, 40, 1, 1, 64, False),
    (64, 150, 16, 4, 64, True),
    (21, 200, 16, 2, 128, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("case", MANY, ids=[str(i) for i in range(len(MANY))])
def test_many_sequences(eng, case, kind):
    n, longest, H, G, D, causal = case
    u = KINDS[kind][1]
    r = np.random.default_rng(n)
    lens = r.integers(0, longest + 1, n)
    lens[n // 3] = 0
    cu = starts(lens, 1)
    rows = cu[-1] + 1
    q, k, v, do = (normal(r, kind, rows, h, D) for h in (H, G, G, H))
    want = definition(value(q), value(k), value(v), cu, cu, causal, D ** -0.5, u, dout=value(do))
    d, c = [eng.to_device(x) for x in (q, k, v, do)], eng.to_device(cu)
    zeros = lambda x: eng.to_device(np.zeros(x.shape, x.dtype))
    out, lse, grads = zeros(q), eng.to_device(np.zeros((H, rows), np.float32)), [zeros(q), zeros(k), zeros(v)]
    sequence.packed_attention(eng, *d[:3], c, causal=causal, out=out, lse=lse)
    sequence.packed_attention_grad(eng, d[3], *d[:3], out, lse, c, causal=causal, dq=grads[0], dk=grads[1], dv=grads[2])
    for name, a in (("out", out), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        got = a.numpy()
        close(got, want[name], name, kind)
        assert (got[0] == 0).all() and (got[-1] == 0).all()
    if not causal:
        return
    # the same as one chunk of every sequence over a cache
    P = 16
    table, pages = layout(r, lens, P)
    cache = sequence.PagedCache.empty(eng, pages, G, P, D, KINDS[kind][0])
    ctx, t = eng.to_device(np.zeros(n, np.int32)), eng.to_device(table)
    cache.append(d[1], d[2], c, ctx, t)
    chunk = zeros(q)
    cache.attend(d[0], c, ctx, t, max_new=int(lens.max()), max_context=int(lens.max()), out=chunk)
    close(chunk.numpy(), want["out"], "chunk", kind)


@pytest.mark.gpu
@pytest.mark.parametrize("ld", [1 << 23, 1 << 25])              # rows by a lane's 32-bit offset, and by whole addresses
def test_rows_far_apart(eng, ld):
    """Offsets that pass 32 bits in bytes and in elements: 300 / 75 rows of 16 / 64 MB."""
    H, G, D = 4, 2, 64
    lens = [37, 3, 35] if ld > 1 << 24 else [220, 41, 39]
    cu = starts(lens)
    n = cu[-1]
    r = np.random.default_rng(ld)
    x, do = normal(r, "f16", n, (H + 2 * G) * D), normal(r, "f16", n, H, D)
    far = eng.empty((n, ld), np.float16)
    for i in range(n):
        far.view(i * ld, x[i].shape).copy_from(x[i])
    cut = lambda o, h: value(x[:, o:o + h * D]).reshape(n, h, D)
    want = definition(cut(0, H), cut(H * D, G), cut((H + G) * D, G), cu, cu, True, D ** -0.5, KINDS["f16"][1], dout=value(do))
    a = [far.view(0, (n, H, D)), far.view(H * D, (n, G, D)), far.view((H + G) * D, (n, G, D))]
    c, strides = eng.to_device(cu), dict(ldq=ld, ldk=ld, ldv=ld)
    out, lse = sequence.packed_attention(eng, *a, c, **strides)
    grads = sequence.packed_attention_grad(eng, eng.to_device(do), *a, out, lse, c, **strides)
    for name, got in zip(("out", "dq", "dk", "dv"), (out,) + grads):
        close(got.numpy(), want[name], name, "f16")


@pytest.mark.gpu
def test_pages_far_apart(eng):
    """A pool of more than 2^31 elements: its last pages hold the sequences."""
    G, H, P, D, pages = 2, 4, 64, 128, 140000
    lens = [150, 1, 64]
    r = np.random.default_rng(3)
    table, used = layout(r, lens, P, spare=0)
    table[table >= 0] += pages - used
    cu = starts(lens)
    n = cu[-1]
    q, k, v = (normal(r, "bf16", n, h, D) for h in (H, G, G))
    want = definition(value(q), value(k), value(v), cu, cu, True, D ** -0.5, KINDS["bf16"][1])
    cache = sequence.PagedCache(eng, eng.empty((pages, G, P, D), np.uint16), eng.empty((pages, G, P, D), np.uint16))
    c, ctx, t = eng.to_device(cu), eng.to_device(np.zeros(3, np.int32)), eng.to_device(table)
    cache.append(eng.to_device(k), eng.to_device(v), c, ctx, t)
    out = cache.attend(eng.to_device(q), c, ctx, t, max_new=150, max_context=150)
    close(out.numpy(), want["out"], "out", "bf16")
    last = eng.to_device(np.int32([0, 1, 2, 3]))                 # a single row of every sequence
    ql = q[cu[1:] - 1]
    one = cache.attend(eng.to_device(ql), last, eng.to_device(np.int32(lens) - 1), t, max_new=1, max_context=150)
    close(one.numpy(), (want["out"][0][cu[1:] - 1], want["out"][1][cu[1:] - 1]), "single rows", "bf16")


@pytest.mark.gpu
def test_two_engines_in_turn(eng):
    """Calls of two handles on their own streams, in flight at once: neither's workspace is the other's."""
    other = _lib.Engine(tiny_hps(), 0)
    try:
        results = []
        for turn in range(2):
            held = []
            for e, seed in ((eng, 1), (other, 2)):
                r = np.random.default_rng(seed)
                cu = starts([300, 20, 133])
                x = [e.to_device(normal(r, "bf16", cu[-1], h, 64)) for h in (8, 2, 2, 8)]
                kp, vp = (e.to_device(normal(r, "bf16", 40, 2, 64, 64)) for _ in range(2))
                held.append((e, x, e.to_device(cu), sequence.PagedCache(e, kp, vp), e.to_device(starts([1, 1])), e.to_device(np.int32([1100, 900])),
                             e.to_device(np.arange(40, dtype=np.int32).reshape(2, 20)), e.to_device(normal(r, "bf16", 2, 8, 64))))
            got = [[], []]
            for _ in range(3):
                for i, (e, (q, k, v, do), c, cache, one, ctx, table, row) in enumerate(held if turn else held[::-1]):
                    out, lse = sequence.packed_attention(e, q, k, v, c)
                    got[i if turn else 1 - i] = [cache.attend(row, one, ctx, table, 1, 1200), *sequence.packed_attention_grad(e, do, q, k, v, out, lse, c)]
            results.append([[a.numpy() for a in g] for g in got])
        for a, b in zip(*results):
            assert all((x == y).all() for x, y in zip(a, b))
        assert (results[0][0][1] != results[0][1][1]).any()
    finally:
        other.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_batches_without_keys_or_without_rows(eng, kind):
    H, G, D = 4, 2, 64
    r = np.random.default_rng(12)
    x, y = normal(r, kind, 5, H, D), normal(r, kind, 7, G, D)
    fill = lambda *s: eng.to_device(store(np.full(s, 7, np.float32), kind))
    none, five, seven = (eng.to_device(np.int32(c)) for c in ([0, 0, 0], [0, 2, 5], [0, 0, 7]))
    nothing = lambda h: eng.empty((0, h, D), x.dtype)
    q, out, lse, dq = eng.to_device(x), fill(5, H, D), eng.to_device(np.full((H, 5), 7, np.float32)), fill(5, H, D)
    sequence.packed_attention(eng, q, nothing(G), nothing(G), five, none, True, None, out, lse)
    assert (out.numpy() == 0).all() and (lse.numpy() == -np.inf).all()
    sequence.packed_attention_grad(eng, q, q, nothing(G), nothing(G), out, lse, five, none, dq=dq, dk=nothing(G), dv=nothing(G))
    assert (dq.numpy() == 0).all()
    k, dk, dv, empty = eng.to_device(y), fill(7, G, D), fill(7, G, D), eng.empty((H, 0))
    sequence.packed_attention(eng, nothing(H), k, k, none, seven, False, None, nothing(H), empty)
    sequence.packed_attention_grad(eng, nothing(H), nothing(H), k, k, nothing(H), empty, none, seven, False, dq=nothing(H), dk=dk, dv=dv)
    assert (dk.numpy() == 0).all() and (dv.numpy() == 0).all()
    cache = sequence.PagedCache(eng, fill(3, G, 16, D), fill(3, G, 16, D))
    ctx, table = eng.to_device(np.int32([3, 4])), eng.to_device(np.int32([[0], [1]]))
    cache.append(nothing(G), nothing(G), none, ctx, table)
    assert cache.attend(nothing(H), none, ctx, table, 1, 16).numpy().shape == (0, H, D)
    assert (value(cache.k.numpy()) == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 70])
def test_positions_behind_the_bound_are_not_seen(eng, new):
    """max_context below a sequence's length: every row sees the positions in front of the bound; a context that is no length counts as the bound."""
    H, G, D, P, bound = 4, 2, 64, 16, 600
    r = np.random.default_rng(new)
    total = [900, bound + 40]
    table, pages = layout(r, total, P)
    kc, vc = normal(r, "f16", pages, G, P, D), normal(r, "f16", pages, G, P, D)
    ctx = [total[0] - new, total[1] - new]
    held = lambda c: np.concatenate([c[table[b, :-(-bound // P)]].transpose(0, 2, 1, 3).reshape(-1, G, D)[:bound] for b in range(2)])
    cu = starts([new, new])
    q = normal(r, "f16", cu[-1], H, D)
    want = definition(value(q), value(held(kc)), value(held(vc)), cu, starts([bound, bound]), True, D ** -0.5, KINDS["f16"][1], first=ctx)
    cache = sequence.PagedCache(eng, eng.to_device(kc), eng.to_device(vc))
    for contexts in (ctx, [2 ** 31 - 1, ctx[1]]):
        if contexts is not ctx:
            want = definition(value(q), value(held(kc)), value(held(vc)), cu, starts([bound, bound]), True, D ** -0.5, KINDS["f16"][1], first=[bound, ctx[1]])
        out = cache.attend(eng.to_device(q), eng.to_device(cu), eng.to_device(np.int32(contexts)), eng.to_device(table), new, bound)
        close(out.numpy(), want["out"], "out", "f16")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("power", [-14, 12])
@pytest.mark.parametrize("large", ["k", "q"])
def test_gradients_follow_a_power_of_two_on_dout(eng, large, power, dim, kind):
    """The gradient is linear in dout, and a power of two on dout is one on every product and sum of it: where a result is an ordinary number of
    the type both times it is the same but for one step, however small (long rows, dout of 1e-4) or large (beyond float16's 65504) dS is on
    the way.  Large keys and small queries keep dQ inside the type's range, the other way round dK.  Tolerance: half a step for the rounding of either
    result, and for the sums in 32 bits behind each the definition's bound with u = 0 (the matrix instructions round products of subnormal float16
    operands, dout of 1e-4, otherwise than the same products a power of two higher)."""
    r = np.random.default_rng(dim + power)
    cu = starts([700, 65, 3, 2000])
    n, H, G = cu[-1], 4, 2
    up = 2.0 ** (8 if power < 0 else -8)
    fq, fk = (1 / up, up) if large == "k" else (up, 1 / up)
    q, k = (store(value(normal(r, kind, n, h, dim)) * f, kind) for h, f in ((H, fq), (G, fk)))
    v = store(value(normal(r, kind, n, G, dim)) * 8, kind)
    dout = value(store(np.round(r.standard_normal((n, H, dim)).clip(-3.9, 3.9) * 512) / 512, kind))      # exact at both sizes
    d, c = [eng.to_device(x) for x in (q, k, v)], eng.to_device(cu)
    out, lse = sequence.packed_attention(eng, *d, c)
    got = []
    for f in (1.0, 2.0 ** power):
        do = store(dout * f, kind)
        assert (value(do) == dout * f).all()
        got.append([value(x.numpy()) for x in sequence.packed_attention_grad(eng, eng.to_device(do), *d, out, lse, c)])
    least, most = {"f16": (2.0 ** -14, 65504.0)}.get(kind, (2.0 ** -120, 2.0 ** 120))
    sums = None
    for name, one, two in zip(("dq", "dk", "dv"), *got):
        want = one * 2.0 ** power
        size = np.abs(want)
        assert np.isfinite(one).all() and np.isfinite(two[size < 0.99 * most]).all(), name
        both = (np.abs(one) > least) & (size > least) & (size < 0.99 * most)      # (at the least ordinary number a rounding may come from the finer steps below)
        if (two[both] != want[both]).any():
            sums = sums or definition(value(q), value(k), value(v), cu, cu, True, np.float64(np.float32(dim ** -0.5)), 0.0, dout=dout)
            tol = 2 * KINDS[kind][1] * size + 2 * sums[name][1] * 2.0 ** power
            assert (np.abs(two - want)[both] <= tol[both]).all(), name
        if name == {"k": "dq", "q": "dk"}[large]:
            assert both.mean() > 0.8                              # (the case is about these)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_gradients_whose_differences_pass_the_range_of_float16(eng, dim):
    """P (dP - delta) beyond 65504 where dQ, dK and dV are ordinary float16 numbers."""
    r = np.random.default_rng(dim)
    cu = starts([300, 40])
    n, H, G = cu[-1], 4, 2
    u = KINDS["f16"][1]
    q, k, v, do = (store(r.standard_normal((n, h, dim)) * f, "f16") for h, f in ((H, 1), (G, 1), (G, 8), (H, 1500)))
    want = definition(value(q), value(k), value(v), cu, cu, True, np.float64(np.float32(dim ** -0.5)), u, dout=value(do))
    assert max(np.abs(want[x][0]).max() for x in ("dq", "dk", "dv")) < 65000
    d, c = [eng.to_device(x) for x in (q, k, v)], eng.to_device(cu)
    out, lse = sequence.packed_attention(eng, *d, c)
    for name, got in zip(("dq", "dk", "dv"), sequence.packed_attention_grad(eng, eng.to_device(do), *d, out, lse, c)):
        close(got.numpy(), want[name], name, "f16")


FEW = [
    # lens of queries, of keys (None: the same), heads, kv_heads, head_dim
    ([64], None, 8, 2, 128),
    ([65], None, 8, 2, 128),
    ([300, 1, 129, 66], None, 8, 2, 64),
    ([90, 400], [5, 333], 4, 1, 80),                              # rows that see nothing in front of the first ones that see something
    ([700, 650, 700, 700], None, 80, 8, 128),                     # the launch of many rows
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("case", FEW, ids=[str(i) for i in range(len(FEW))])
def test_dq_of_rows_that_see_few_keys(eng, case, kind):
    """delta = sum_d dO out with the rounded `out` reaches every dS of its row, and where few keys share the weight nothing averages it away: rows
    that see up to 64 keys take sum_j P dP, however long their sequence is.  Tolerance: no step of the type but the result's own,
      dS   (u^2 + 2 e_s + 32 h) |dS| + 2^-32 max|dS| + P (e_dP + e_delta),   e_delta = (2 e_s + (n + 48) h) sum P |dP| + sum P e_dP
    (dS goes in two halves: u^2; float16's smallest step against the row's largest; delta is a sum in 32 bits)."""
    lq, lk, H, G, D = case
    u = KINDS[kind][1]
    r = np.random.default_rng(sum(lq))
    cu_q = starts(lq)
    cu_k = cu_q if lk is None else starts(lk)
    q, k, v, do = (normal(r, kind, n, h, D) for n, h in ((cu_q[-1], H), (cu_k[-1], G), (cu_k[-1], G), (cu_q[-1], H)))
    d = [eng.to_device(x) for x in (q, k, v, do)]
    cq, ck = eng.to_device(cu_q), eng.to_device(cu_k)
    out, lse = sequence.packed_attention(eng, *d[:3], cq, ck)
    got = value(sequence.packed_attention_grad(eng, d[3], *d[:3], out, lse, cq, ck)[0].numpy())
    q, k, v, do = (value(x) for x in (q, k, v, do))
    scale, checked = np.float64(np.float32(D ** -0.5)), 0
    for b in range(len(lq)):
        ahead = (cu_k[b + 1] - cu_k[b]) - (cu_q[b + 1] - cu_q[b])
        first = max(0, -ahead)                                    # the first row that sees a key
        rows = cu_q[b] + np.arange(first, min(cu_q[b + 1] - cu_q[b], 64 - ahead))
        nk = min(64, cu_k[b + 1] - cu_k[b])
        if len(rows) == 0:
            continue
        see = np.arange(nk) <= (rows - cu_q[b] + ahead)[:, None]
        for h in range(H):
            K, V = (x[cu_k[b]:cu_k[b] + nk, h // (H // G)] for x in (k, v))
            Q, dO = q[rows, h], do[rows, h]
            x = np.where(see, Q @ K.T * scale, -np.inf)
            e_s = (D + 4) * H24 * scale * np.where(see, np.abs(Q) @ np.abs(K).T, 0).max()
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            dP, e_dP = dO @ V.T, (D + 4) * H24 * (np.abs(dO) @ np.abs(V).T)
            dS = p * (dP - (p * dP).sum(1, keepdims=True))
            e_delta = (2 * e_s + (nk + 48) * H24) * (p * np.abs(dP)).sum(1, keepdims=True) + (p * e_dP).sum(1, keepdims=True)
            e_dS = (u * u + 2 * e_s + 32 * H24) * np.abs(dS) + 2.0 ** -32 * np.abs(dS).max(1, keepdims=True) + p * (e_dP + e_delta)
            want = scale * dS @ K
            tol = u * np.abs(want) + scale * ((e_dS + (nk + 16) * H24 * np.abs(dS)) @ np.abs(K)) + TINY
            off = np.abs(got[rows, h] - want) - tol
            assert off.max() <= 0, (b, h, rows[off.max(1) > 0] - cu_q[b], off.max())
            checked += len(rows)
    assert checked


def tail(n, D, r):
    """One key whose weight is 2^25.5 times that of each of n - 1 others, and a value of zero: the result is made of the others alone."""
    q = np.zeros((1, D))
    q[0, 0] = 1
    k, v = np.zeros((n, D)), 1 + 0.25 * r.standard_normal((n, D))
    k[0, 0], v[0] = np.float16(25.5 * np.log(2)), 0
    return q, k, v


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [1, 160])
def test_small_weights_of_float16_reach_the_result(eng, heads, dim):
    """Weights far below the row's largest are what the row sum counts, so the result has to count them too: in float16 each is rounded by half a step
    of its own, or by 2^-36 of the row's largest."""
    r = np.random.default_rng(dim)
    n, new, u, P = 4096, 130, KINDS["f16"][1], 64
    q1, k1, v1 = tail(n, dim, r)
    q, k, v = store(np.broadcast_to(q1, (n, heads, dim)), "f16"), store(k1[:, None], "f16"), store(v1[:, None], "f16")
    c, ident = eng.to_device(starts([n])), eng.to_device(np.arange(n // P, dtype=np.int32)[None])
    one = definition(value(q)[:1, :1], value(k), value(v), starts([1]), starts([n]), False, 1.0, u)
    w, tol = (x[0, 0] for x in one["out"])
    tol = tol + n * 2.0 ** -36 * np.abs(value(v)).max()
    assert (np.abs(w) > 100 * tol).all() and (np.abs(w) > 2.0 ** -14).all()
    got = {}
    for rows in (1, 40, n) if heads == 1 else (n,):
        cq = eng.to_device(starts([rows]))
        o, _ = sequence.packed_attention(eng, eng.to_device(q[:rows]), eng.to_device(k), eng.to_device(v), cq, c, causal=False, scale=1.0)
        got["packed", rows] = value(o.numpy())
    paged = lambda x: eng.to_device(np.ascontiguousarray(x.reshape(n // P, P, 1, dim).transpose(0, 2, 1, 3)))
    cache = sequence.PagedCache(eng, paged(k), paged(v))
    for rows in (1, new):
        o = cache.attend(eng.to_device(q[:rows]), eng.to_device(starts([rows])), eng.to_device(np.int32([n - 1])), ident, rows, n, scale=1.0)
        got["cache", rows] = value(o.numpy())
    for name, x in got.items():
        assert (np.abs(x - w) <= tol + TINY).all(), (name, x[0, 0, :4], w[:4])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_small_weights_of_float16_reach_dv(eng, dim):
    """512 rows with a weight of 2^-25.5 for each of the later keys: dV of those keys is 2^-25.5 of dout's sum, an ordinary float16 number."""
    r = np.random.default_rng(dim)
    n, rows, u = 600, 512, KINDS["f16"][1]
    q1, k1, v1 = tail(n, dim, r)
    q, k, v = store(np.broadcast_to(q1, (rows, 1, dim)), "f16"), store(k1[:, None], "f16"), store(v1[:, None], "f16")
    do = store(1024 * (1 + 0.25 * r.standard_normal((rows, 1, dim))), "f16")
    cu_q, cu_k = starts([rows]), starts([n])
    want = definition(value(q), value(k), value(v), cu_q, cu_k, False, 1.0, u, dout=value(do))["dv"]
    assert (np.abs(want[0][1:]) > 2.0 ** -14).all() and (np.abs(want[0]) < 65504 * 16).all()
    d, cq, ck = [eng.to_device(x) for x in (q, k, v)], eng.to_device(cu_q), eng.to_device(cu_k)
    out, lse = sequence.packed_attention(eng, *d, cq, ck, causal=False, scale=1.0)
    dv = sequence.packed_attention_grad(eng, eng.to_device(do), *d, out, lse, cq, ck, causal=False, scale=1.0)[2]
    close(dv.numpy()[1:], [x[1:] for x in want], "dv", "f16")


BROKEN = [
    # starts of 50 rows, and which sequence owns each range of them (first row, rows behind the last, place of the first row in its sequence)
    ([0, 50, 20], [(0, 0, 50)]),                                  # 50..20 is empty, 0..50 is not
    ([-7, 12, 30], [(0, 0, 12), (1, 12, 30)]),                    # a start in front of the tensor is its first row
    ([5, 5, 1000], [(1, 5, 50)]),                                 # an end behind it its last
    ([30, 10, 25], [(1, 10, 25)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("bound", [200, 3000])                    # one piece of the keys, and several that are joined
@pytest.mark.parametrize("case", BROKEN, ids=[str(i) for i in range(len(BROKEN))])
def test_cache_calls_with_broken_starts(eng, case, bound, kind):
    """Append and attention agree on who owns which row, whether the keys are cut or not: a broken start takes rows from its own sequences only, and rows
    that are nobody's stay as they were."""
    cu, owned = case
    H, G, D, P, u = 4, 2, 64, 16, KINDS[kind][1]
    r = np.random.default_rng(bound)
    ctx = [70, 110]
    table, pages = layout(r, [bound, bound], P)
    q, k, v = normal(r, kind, 50, H, D), normal(r, kind, 50, G, D), normal(r, kind, 50, G, D)
    kc, vc = normal(r, kind, pages, G, P, D), normal(r, kind, pages, G, P, D)
    cache = sequence.PagedCache(eng, eng.to_device(kc), eng.to_device(vc))
    dcu, dctx, dt = eng.to_device(np.int32(cu)), eng.to_device(np.int32(ctx)), eng.to_device(table)
    mark = store(np.full(1, 7.0, np.float32), kind)[0]
    qo, out = (eng.to_device(np.full(q.shape, mark, q.dtype)) for _ in range(2))
    lse = eng.to_device(np.full((H, 50), 7.0, np.float32))
    cache.append(eng.to_device(k), eng.to_device(v), dcu, dctx, dt, q=eng.to_device(q), q_out=qo)
    wk, wv = kc.copy(), vc.copy()
    nobody = np.ones(50, bool)
    for b, i, j in owned:
        nobody[i:j] = False
        for t in range(i, j):
            p = ctx[b] + t - i
            wk[table[b, p // P], :, p % P], wv[table[b, p // P], :, p % P] = k[t], v[t]
    assert (cache.k.numpy() == wk).all() and (cache.v.numpy() == wv).all()
    gq = qo.numpy()
    assert (gq[~nobody] == q[~nobody]).all() and (gq[nobody] == mark).all()
    cache.attend(eng.to_device(q), dcu, dctx, dt, 50, bound, out=out, lse=lse)
    got, gl = out.numpy(), lse.numpy()
    for b, i, j in owned:
        held = [x[table[b]].transpose(0, 2, 1, 3).reshape(-1, G, D)[:ctx[b] + j - i] for x in (wk, wv)]
        want = definition(value(q[i:j]), value(held[0]), value(held[1]), starts([j - i]), starts([ctx[b] + j - i]), True, D ** -0.5, u, first=[ctx[b]])
        close(got[i:j], want["out"], "out", kind)
        close(gl[:, i:j], want["lse"], "lse")
    assert (got[nobody] == mark).all() and (gl[:, nobody] == 7).all()


def test_library_refusals_of_more_rows_than_a_launch_holds():
    """Before anything is launched -- a gradient's second kernel included -- and as an error of the arguments."""
    far = dict(heads=4096, kv_heads=4096, ldq=4096 * 64, ldk=4096 * 64, ldv=4096 * 64, ldo=4096 * 64)
    most = (1 << 31) - 1
    grad = _lib.vnr_packed_attention_grad(d_dout=4096, lddo=4096 * 64, d_dq=4096, d_dk=4096, d_dv=4096, lddq=4096 * 64, lddk=4096 * 64, lddv=4096 * 64)
    for kw in (dict(rows_q=most), dict(rows_q=1 << 20)):
        assert "launch" in refused("vnr_op_packed_attention", packed_desc(**far, **kw)), kw
        assert "launch" in refused("vnr_op_packed_attention_grad", packed_desc(d_lse=64, **far, **kw), grad), kw
    for kw in (dict(rows_k=most), dict(rows_k=1 << 20), dict(rows_q=0, rows_k=most)):
        assert "null handle" in refused("vnr_op_packed_attention", packed_desc(**far, **kw)), kw      # keys do not make the forward's launch
        assert "launch" in refused("vnr_op_packed_attention_grad", packed_desc(d_lse=64, **far, **kw), grad), kw
    cache = _lib.vnr_kv_cache(dtype=1, kv_heads=2, head_dim=64, pages=8, page_size=16, d_k=4096, d_v=4096)
    att = dict(batch=2, heads=4096, rows=most, d_cu=64, d_context=64, d_table=64, table_width=3, max_new=4, max_context=40, scale=0.125, d_q=4096, ldq=4096 * 64,
               d_out=4096, ldo=4096 * 64, d_lse=None)
    assert "launch" in refused("vnr_op_paged_attention", cache, _lib.vnr_paged_attention_desc(**att))
    assert "launch" in refused("vnr_op_paged_attention", cache, _lib.vnr_paged_attention_desc(**{**att, "rows": 1 << 20}))


class Script:
    """The library as far as the engine's log needs it: notes the calls in order; the checkpoint that follows `trip` finds the range word raised once."""

    def __init__(self, trip):
        self.trip, self.raised, self.calls = trip, False, []

    def vnr_last_error(self, handle):
        return b"range"

    def __getattr__(self, name):
        if not name.startswith("vnr_"):
            raise AttributeError(name)

        def fn(handle, *args):
            self.calls.append(name)
            if name == self.trip:
                self.raised, self.trip = True, None
            if name in ("vnr_synchronize", "vnr_memcpy_d2h", "vnr_memcpy_h2d") and self.raised:
                self.raised = False
                return _lib.VNR_ERR_RANGE
            return 0
        return fn


def test_cache_calls_run_once_whatever_the_range_sentinel_finds(monkeypatch):
    """A module call whose results a raised range word voids is issued again at the next checkpoint.  Calls of this file stand behind such a checkpoint and
    are not issued again themselves: another library may own their arrays and may have moved the context or the table on by then."""
    lib = Script("vnr_prior_sample")
    monkeypatch.setattr(_lib, "load", lambda: lib)
    e = _lib.Engine.__new__(_lib.Engine)
    e.lib, e.handle, e._log, e._log_cap, e._training_mode, e.range_replays = lib, 1, [], 256, False, 0
    e._pool, e._pool_bytes, e._pool_cap = {}, 0, 1 << 30
    array = lambda shape, kind=np.float16: _lib.DeviceArray(e, shape, kind, ptr=4096, owner=lib)
    q, k, cu, cu1, ctx, table = array((6, 4, 64)), array((6, 2, 64)), array((3,), np.int32), array((3,), np.int32), array((2,), np.int32), array((2, 3), np.int32)
    cache = sequence.PagedCache(e, array((4, 2, 16, 64)), array((4, 2, 16, 64)))
    rot, lse = array((48, 64), np.float32), array((4, 6), np.float32)
    e.call("vnr_prior_sample")
    cache.append(k, k, cu, ctx, table, rotation=rot, q=q, q_out=q)
    cache.attend(q, cu, ctx, table, 1, 40, out=q)
    sequence.packed_attention(e, q, k, k, cu, out=q, lse=lse)
    sequence.packed_attention_grad(e, q, q, k, k, q, lse, cu, dq=q, dk=k, dv=k)
    e.synchronize()
    assert lib.calls == ["vnr_prior_sample", "vnr_synchronize", "vnr_prior_sample", "vnr_synchronize", "vnr_op_kv_append", "vnr_op_paged_attention",
                         "vnr_op_packed_attention", "vnr_op_packed_attention_grad", "vnr_synchronize"]
    # a loop of them keeps no log, and the host does not wait for the device in it
    lib.calls.clear()
    for _ in range(300):
        cache.attend(q, cu, ctx, table, 1, 40, out=q)
    assert lib.calls == ["vnr_op_paged_attention"] * 300 and not e._log
    e.handle = None


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", [1, 160])
@pytest.mark.parametrize("size", [10, 12, 14])
def test_logits_far_beyond_their_own_steps(eng, size, heads, kind):
    """Logits of up to 2^29, whose neighbours in 32 bits are tens apart: weights stay weights (the bound that is taken off a row's logits may not be rounded
    below them), and a row whose largest logit leaves the others far behind gets that key's value."""
    r = np.random.default_rng(size)
    n, D, P = 300, 128, 16
    q, k = (store(r.standard_normal((n, h, D)).clip(-3.9, 3.9) * 2.0 ** size, kind) for h in (heads, 1))
    v = normal(r, kind, n, 1, D)
    c, scale = starts([n]), np.float64(np.float32(D ** -0.5))
    dq, dk, dv, dc = (eng.to_device(x) for x in (q, k, v, c))
    out, lse = sequence.packed_attention(eng, dq, dk, dv, dc)
    table, pages = layout(r, [n], P)
    cache = sequence.PagedCache.empty(eng, pages, 1, P, D, KINDS[kind][0])
    zero, dt = eng.to_device(np.int32([0])), eng.to_device(table)
    cache.append(dk, dv, dc, zero, dt)
    outs = [out, cache.attend(dq, dc, zero, dt, n, n), cache.attend(dq, dc, zero, dt, 1, 1 << 20)]
    values = [value(x.numpy()) for x in outs]
    K, V, u = value(k)[:, 0], value(v)[:, 0], KINDS[kind][1]
    for h in (0, heads - 1):
        x = np.where(np.tri(n, dtype=bool), value(q)[:, h] @ K.T * scale, -np.inf)
        off = (D + 4) * H24 * scale * (np.abs(value(q)[:, h]) @ np.abs(K).T).max()      # of a logit in 32 bits
        top = np.argmax(x, 1)
        second = np.where(np.arange(n) == top[:, None], -np.inf, x).max(1)
        clear = x.max(1) - second > 2 * off + 30
        assert clear.mean() > 0.5
        for got in values:
            assert np.isfinite(got[:, h]).all()
            assert (np.abs(got[clear, h] - V[top[clear]]) <= 2 * u * np.abs(V[top[clear]]) + n * 1e-12).all()
    assert np.isfinite(lse.numpy()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [9, 10, 11, 12])
def test_gradients_under_large_logits_stay_finite(eng, size, kind):
    """P is formed anew from lse: with logits of up to 2^24 it may come out as some powers of two above 1, and has to have room for them."""
    r = np.random.default_rng(size)
    n, H, D = 400, 4, 128
    q, k = (store(r.standard_normal((n, H, D)).clip(-3.9, 3.9) * 2.0 ** size, kind) for _ in range(2))
    v, do = normal(r, kind, n, H, D), normal(r, kind, n, H, D)
    q, k, v, do, c = (eng.to_device(x) for x in (q, k, v, do, starts([n])))
    out, lse = sequence.packed_attention(eng, q, k, v, c)
    for name, x in zip(("dq", "dk", "dv"), sequence.packed_attention_grad(eng, do, q, k, v, out, lse, c)):
        got = value(x.numpy())
        assert np.isfinite(got).mean() == 1 if name == "dv" or kind != "f16" else not np.isnan(got).any(), name


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_gradients_of_rows_that_see_no_number_are_none(eng, kind):
    r = np.random.default_rng(8)
    n, H, D = 200, 2, 64
    x = [normal(r, kind, n, H, D) for _ in range(4)]
    x[1][100] = store(np.float32([np.nan]), kind)[0]
    q, k, v, do, c = (eng.to_device(a) for a in (*x, starts([n])))
    out, lse = sequence.packed_attention(eng, q, k, v, c)
    dq, dk, dv = (value(a.numpy()) for a in sequence.packed_attention_grad(eng, do, q, k, v, out, lse, c))
    assert np.isnan(dq[100:]).all() and np.isnan(dk).all() and np.isnan(dv).all()      # every key is seen by a row that sees key 100


def test_cache_calls_behind_fills_do_not_wait_for_the_device(monkeypatch):
    """Zeroed or random arrays raise no range word: calls on them go out at once, and a later replay does not lay the fills over their results."""
    lib = Script("vnr_prior_sample")
    monkeypatch.setattr(_lib, "load", lambda: lib)
    e = _lib.Engine.__new__(_lib.Engine)
    e.lib, e.handle, e._log, e._log_cap, e._training_mode, e.range_replays = lib, 1, [], 256, False, 0
    e._pool, e._pool_bytes, e._pool_cap = {}, 0, 1 << 30
    array = lambda shape, kind=np.float16: _lib.DeviceArray(e, shape, kind, ptr=4096, owner=lib)
    q, cu, ctx, table = array((6, 4, 64)), array((3,), np.int32), array((2,), np.int32), array((2, 3), np.int32)
    cache = sequence.PagedCache(e, array((4, 2, 16, 64)), array((4, 2, 16, 64)))
    e.set_option("n_sample", 1)
    for _ in range(3):
        e.call("vnr_memset", 4096, 0, 64)
        e.call("vnr_random_normal", 1, 0, 1.0, 4096, 16)
        cache.attend(q, cu, ctx, table, 1, 40, out=q)
    assert lib.calls == ["vnr_set_option"] + ["vnr_memset", "vnr_random_normal", "vnr_op_paged_attention"] * 3
    lib.calls.clear()
    e.call("vnr_prior_sample")
    e.synchronize()
    assert lib.calls == ["vnr_prior_sample", "vnr_synchronize", "vnr_set_option", "vnr_prior_sample", "vnr_synchronize"]
    e.handle = None
