"""CPU: what the serving operators (rotary positions, paged KV cache) refuse, through Python and through the C ABI,
and the frequencies of rotary positions."""
import ctypes
import math

import pytest
import torch

BF = torch.bfloat16


def _rotary(M, rot=64, **kw):
    return M.Rotary(M.rotary_frequencies(rot)[0], **kw)


def _paged(B=2, pages=4, page=8, H=2, D=64, dtype=BF, **kw):
    d = dict(cache_k=torch.zeros(pages, page, H, D, dtype=dtype), cache_v=torch.zeros(pages, page, H, D, dtype=dtype),
             block_table=torch.zeros(B, 2, dtype=torch.int32), seq_lens=torch.zeros(B, dtype=torch.int32))
    d.update(kw)
    return d


@pytest.mark.parametrize("kw,error,match", [
    (dict(q=torch.zeros(2, 8, 64, dtype=BF)), AssertionError, "q must be"),
    (dict(G=3), AssertionError, "divisible"),
    (dict(G=0), AssertionError, "divisible"),
    (dict(k=torch.zeros(2, 8, 2, 64, dtype=BF)), AssertionError, "k must be"),
    (dict(k=torch.zeros(2, 4, 3, 64, dtype=BF)), AssertionError, "k must be"),
    (dict(rotary=torch.zeros(3)), TypeError, "Rotary"),
    (dict(rotary=(torch.zeros(32), False, 1.0)), TypeError, "float64"),
    (dict(rotary=(torch.zeros(33, dtype=torch.float64), False, 1.0)), AssertionError, "multiple of 16"),
    (dict(rotary=(torch.zeros(40, dtype=torch.float64), False, 1.0)), AssertionError, "at most head_dim"),
    (dict(rotary=(torch.zeros(64, dtype=torch.float64)[::2], False, 1.0)), AssertionError, "contiguous"),
    (dict(positions=torch.zeros(4)), TypeError, "int32 or int64"),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), AssertionError, "positions must be"),
    (dict(positions=torch.zeros(3, 4, dtype=torch.int64)), AssertionError, "positions must be"),
    (dict(), RuntimeError, "CUDA tensors only"),                    # well-formed: no CPU path
    (dict(positions=torch.zeros(1, 4, dtype=torch.int32)), RuntimeError, "CUDA tensors only"),
    (dict(k=None, positions=7), RuntimeError, "CUDA tensors only"),
])
def test_rotary_refusals(built_library, kw, error, match):
    import moda_b200 as M
    a = dict(q=torch.zeros(2, 8, 2, 64, dtype=BF), k=torch.zeros(2, 4, 2, 64, dtype=BF), rotary=_rotary(M), positions=None, G=2)
    a.update(kw)
    with pytest.raises(error, match=match):
        M.rotary_embedding(a["q"], a["k"], a["rotary"], positions=a["positions"], moda_group_num=a["G"])


@pytest.mark.parametrize("kw,error,match", [
    (dict(k=torch.zeros(2, 3, 64, dtype=BF)), AssertionError, "k and v"),
    (dict(v=torch.zeros(2, 2, 2, 64, dtype=BF)), AssertionError, "k and v"),
    (dict(cache_k=torch.zeros(4, 8, 3, 64, dtype=BF)), AssertionError, "cache_k"),
    (dict(cache_v=torch.zeros(4, 8, 2, 32, dtype=BF)), AssertionError, "cache_v"),
    (dict(cache_k=torch.zeros(0, 8, 2, 64, dtype=BF), cache_v=torch.zeros(0, 8, 2, 64, dtype=BF)), AssertionError, "no pages"),
    (dict(cache_k=torch.zeros(4, 8, 2, 65, dtype=BF)[..., 1:]), AssertionError, "in place"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int64)), TypeError, "int32"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), TypeError, "int32"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32)), AssertionError, "block_table"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), AssertionError, "block_table"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]), AssertionError, "block_table"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), AssertionError, "seq_lens"),
    (dict(seq_lens=torch.zeros(4, dtype=torch.int32)[::2]), AssertionError, "seq_lens"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), TypeError, "lengths"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), AssertionError, "lengths"),
    (dict(), RuntimeError, "CUDA tensors only"),
])
def test_append_refusals(built_library, kw, error, match):
    import moda_b200 as M
    a = dict(k=torch.zeros(2, 3, 2, 64, dtype=BF), v=torch.zeros(2, 3, 2, 64, dtype=BF), lengths=None, rotary=_rotary(M), **_paged())
    a.update(kw)
    with pytest.raises(error, match=match):
        M.paged_moda_append(**a)


def _row(B=2, H=2, D=64):
    return torch.zeros(B, 1, H, D, dtype=BF)


@pytest.mark.parametrize("kw,error,match", [
    (dict(q=torch.zeros(2, 4, 2, 64, dtype=BF)), AssertionError, "moda_group_num"),
    (dict(moda_group_num=0), AssertionError, "moda_group_num"),
    (dict(k=_row()), AssertionError, "together"),
    (dict(k=_row(H=1), v=_row(H=1)), AssertionError, "k and v must be"),
    (dict(record_k=_row(), record_v=_row()), AssertionError, "record_k"),
    (dict(k=_row(), v=_row(), record_k=_row()), AssertionError, "record_k"),
    (dict(k=_row(), v=_row(), record_k=_row(D=72)[..., :64].expand(2, 1, 2, 64)[..., ::1], record_v=_row(B=1).expand(2, 1, 2, 64)), AssertionError, "in place"),
    (dict(cached_k=torch.zeros(2, 3, 2, 64, dtype=BF)), AssertionError, "together"),
    (dict(cached_k=torch.zeros(2, 3, 1, 64, dtype=BF), cached_v=torch.zeros(2, 3, 1, 64, dtype=BF)), AssertionError, "cached_k"),
    (dict(cached_k=torch.zeros(2, 2, 3, 2, 64, dtype=BF), cached_v=torch.zeros(2, 2, 3, 2, 64, dtype=BF)), AssertionError, "depth_positions"),
    (dict(depth_positions=torch.zeros(2, dtype=torch.int32)), AssertionError, "depth_positions"),
    (dict(cached_k=torch.zeros(2, 2, 3, 2, 64, dtype=BF), cached_v=torch.zeros(2, 2, 3, 2, 64, dtype=BF), depth_positions=torch.zeros(2)),
     TypeError, "depth_positions"),
    (dict(seq_lens=torch.zeros(1, dtype=torch.int32)), AssertionError, "seq_lens"),
    (dict(rotary=5), TypeError, "Rotary"),
    (dict(scale="x"), TypeError, "real number"),
    (dict(), RuntimeError, "CUDA tensors only"),
])
def test_decode_refusals(built_library, kw, error, match):
    import moda_b200 as M
    a = dict(q=torch.zeros(2, 2, 2, 64, dtype=BF), moda_group_num=2, **_paged())
    a.update(kw)
    with pytest.raises(error, match=match):
        M.paged_moda_decode(**a)


def test_cache_class_refusals(built_library):
    import moda_b200 as M
    cache = M.PagedKVCache(4, 8, 2, 64, BF, "cpu")
    assert cache.k.shape == (4, 8, 2, 64) and cache.k.stride() == (8 * 2 * 64, 64, 8 * 64, 1)
    p = _paged()
    q, k = torch.zeros(2, 1, 2, 64, dtype=BF), _row()
    chunk = M.DepthKVCache(2, 4, 3, 2, 64, BF, "cpu")
    chunk.L = 1
    with pytest.raises(AssertionError, match="depth_positions"):
        cache.decode(q, p["block_table"], p["seq_lens"], k, k, depth=chunk)
    with pytest.raises(AssertionError, match="record needs"):
        cache.decode(q, p["block_table"], p["seq_lens"], k, k, depth=chunk, depth_positions=p["seq_lens"], record=True)
    with pytest.raises(AssertionError, match="record needs"):
        cache.decode(q, p["block_table"], p["seq_lens"], k, k, record=True)
    own = M.DepthKVCache(2, 1, 3, 2, 64, BF, "cpu")
    own.L = 3
    with pytest.raises(AssertionError, match="full"):
        cache.decode(q, p["block_table"], p["seq_lens"], k, k, depth=own, record=True)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        cache.decode(q, p["block_table"], p["seq_lens"], k, k, depth=own)
    with pytest.raises(AssertionError):
        M.PagedKVCache(4, 0, 2, 64, BF, "cpu")


def test_c_abi_refusals(built_library):
    """Nothing is launched for these: the pointers are not addresses of anything."""
    from moda_b200 import _cabi
    from moda_b200._cabi import DepthRows, PagedCache, Positions, Problem, RotaryArgs, Tensor4
    lib, r = _cabi.load(), ctypes.byref

    def prob(**kw):
        d = dict(B=2, T_kv=1, H=2, D=64, G=2, L=0, mode=0, chunk_rows=64, dtype=0, path=0, scale=0.125, device=0)
        d.update(kw)
        return Problem(**d)

    good = Tensor4(0x1000, 1024, 256, 64)
    null, odd, flat = Tensor4(0, 0, 0, 0), Tensor4(0x1008, 1024, 256, 64), Tensor4(0x1000, 1024, 256, 0)
    rot = RotaryArgs(0x1000, 64, 0, 1.0)

    def rotary(p=prob(), rt=rot, pos=None, q=good, k=good, qo=good, ko=good):
        return lib.moda_b200_rotary(r(p), None if rt is None else r(rt), None if pos is None else r(pos), 0, r(q), r(k), r(qo), r(ko), None)

    assert rotary(p=prob(B=0)) == 2 and rotary(p=prob(T_kv=0)) == 2 and rotary(p=prob(B=65535, T_kv=1 << 20)) == 2
    assert rotary(p=prob(D=96)) == 3 and rotary(p=prob(dtype=2)) == 4
    assert rotary(rt=None) == 1 and rotary(rt=RotaryArgs(0, 64, 0, 1.0)) == 1
    assert rotary(rt=RotaryArgs(0x1004, 64, 0, 1.0)) == 5
    assert rotary(rt=RotaryArgs(0x1000, 24, 0, 1.0)) == 2 and rotary(rt=RotaryArgs(0x1000, 80, 0, 1.0)) == 2 and rotary(rt=RotaryArgs(0x1000, 0, 0, 1.0)) == 2
    assert rotary(pos=Positions(0x1004, 1, 1, 0, 1)) == 5 and rotary(pos=Positions(0x1002, 1, 1, 0, 0)) == 5
    assert rotary(q=null) == 1 and rotary(qo=null) == 1 and rotary(ko=null) == 1 and rotary(q=odd) == 5 and rotary(k=flat) == 5

    def pages(**kw):
        d = dict(k=good, v=good, num_pages=4, page_size=4, block_table=0x2000, table_stride=2, max_pages=2, seq_lens=0x3000)
        d.update(kw)
        return PagedCache(**d)

    def append(p=prob(G=1), c=pages(), k=good, v=good, lengths=None, rt=rot):
        return lib.moda_b200_paged_append(r(p), r(k), r(v), None if c is None else r(c), lengths, None if rt is None else r(rt), None)

    assert append(c=None) == 1 and append(c=pages(block_table=None)) == 1 and append(c=pages(seq_lens=None)) == 1
    assert append(c=pages(num_pages=0)) == 2 and append(c=pages(page_size=0)) == 2 and append(c=pages(max_pages=0)) == 2 and append(c=pages(table_stride=-1)) == 2
    assert append(c=pages(k=null)) == 1 and append(c=pages(v=odd)) == 5 and append(c=pages(block_table=0x2002)) == 5
    assert append(k=null) == 1 and append(v=flat) == 5 and append(lengths=0x2001) == 5 and append(rt=RotaryArgs(0x1000, 8, 0, 1.0)) == 2

    def decode(p=prob(), c=pages(), q=good, k=None, v=None, kc=None, vc=None, depth=None, o=good, lse=0x4000, ws=0x8000, n=0):
        opt = lambda x: None if x is None else r(x)  # noqa: E731
        return lib.moda_b200_paged_decode(r(p), r(q), r(c), opt(k), opt(v), opt(kc), opt(vc), opt(depth), None, r(o), lse, ws, n, None)

    assert decode(p=prob(T_kv=2)) == 2 and decode(p=prob(scale=math.nan)) == 2 and decode(p=prob(G=0)) == 2
    assert decode(q=null) == 1 and decode(o=odd) == 5 and decode(lse=None) == 1 and decode(lse=0x4002) == 5
    assert decode(k=good) == 1 and decode(kc=good, vc=good) == 1 and decode(k=good, v=good, kc=good) == 1
    assert decode(c=pages(page_size=0)) == 2 and decode(p=prob(L=3)) == 1

    def rows(**kw):
        d = dict(k=good, v=good, k_stride_position=4096, v_stride_position=4096, positions_per_sequence=2, positions_seen=None)
        d.update(kw)
        return DepthRows(**d)

    assert decode(p=prob(L=3), depth=rows(positions_per_sequence=0)) == 2 and decode(p=prob(L=3), depth=rows(k=null)) == 1
    assert decode(p=prob(L=3), depth=rows(k_stride_position=0)) == 5 and decode(p=prob(L=3), depth=rows(positions_seen=0x1001)) == 5
    assert decode(p=prob(L=1 << 20), depth=rows(positions_per_sequence=1 << 20)) == 2
    assert lib.moda_b200_paged_decode_workspace_bytes(r(prob()), r(pages()), None) == 1


@pytest.mark.parametrize("rot", [16, 48, 64, 128])
def test_frequencies(built_library, rot):
    import moda_b200 as M
    f, scale = M.rotary_frequencies(rot, base=500.0)
    assert f.dtype == torch.float64 and scale == 1.0
    want = [500.0 ** (-2 * i / rot) for i in range(rot // 2)]
    assert all(math.isclose(a, b, rel_tol=1e-14) for a, b in zip(f.tolist(), want))
    assert torch.allclose(M.rotary_frequencies(rot, 500.0, "linear", 4.0)[0], f / 4, rtol=1e-14)
    ntk = M.rotary_frequencies(rot, 500.0, "ntk", 4.0)[0]
    assert math.isclose(ntk[-1].item(), f[-1].item() / 4, rel_tol=1e-12) and ntk[0] == 1
    yarn, scale = M.rotary_frequencies(rot, 500.0, "yarn", 4.0, original_length=4096)
    assert math.isclose(scale, 0.1 * math.log(4) + 1)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(yarn[turns > 32 * 500 ** (2 / rot)], f[turns > 32 * 500 ** (2 / rot)])       # a pair away from the ramp
    slow = turns < 500 ** (-2 / rot)
    assert torch.allclose(yarn[slow], f[slow] / 4, rtol=1e-14)
    assert ((yarn <= f * (1 + 1e-14)) & (yarn >= f / 4 * (1 - 1e-14))).all() and (yarn.diff() < 0).all()
    for bad in (dict(rotary_dim=24), dict(rotary_dim=rot, scaling="other"), dict(rotary_dim=rot, scaling="yarn"), dict(rotary_dim=rot, factor=0.0)):
        with pytest.raises(AssertionError):
            M.rotary_frequencies(**bad)


def test_strides_of_single_rows_stay_out_of_addresses(tmp_path):
    """A dimension of one element may carry any stride.  The decoding kernel forms addresses of rows behind the last one (of 16 in a tile), which must be
    aligned although they are not read: with one row a page, or one depth layer, that stride is not used."""
    import os
    import shutil
    import subprocess

    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moda_b200", "csrc")
    program = tmp_path / "views.cu"
    program.write_text("""
#include <cstdint>
#include <cstdio>
#include "cabi_common.cuh"
int main() {
  const moda_tensor4 t{reinterpret_cast<void*>(0x1000), 65, 67, 69};
  const int64_t ext[5][3] = {{1, 1, 1}, {2, 1, 3}, {1, 4, 1}, {5, 4, 1}, {2, 3, 4}};
  for (const auto& e : ext) {
    const moda::View v = moda::to_view(&t, e[0], e[1], e[2]);
    std::printf("%d %d %d\\n", (int)v.sb, (int)v.st, (int)v.sh);
  }
  return moda::to_view(nullptr, 1, 1, 1).ptr != nullptr;
}
""")
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", csrc, str(program), "-o", str(tmp_path / "views")], check=True)
    out = subprocess.run([str(tmp_path / "views")], check=True, capture_output=True, text=True).stdout
    assert out.splitlines() == ["0 0 0", "65 0 69", "0 67 0", "65 67 0", "65 67 69"]


def test_what_interleaved_raises_is_not_lost(built_library):
    import moda_b200 as M
    q = torch.zeros(2, 4, 2, 64, dtype=BF)

    class Bad:
        def __bool__(self):
            raise ValueError("no truth in it")

    for bad, error, match in ((torch.zeros(2), RuntimeError, "ambiguous"), (Bad(), ValueError, "no truth in it")):
        rotary = _rotary(M, interleaved=bad)
        with pytest.raises(error, match=match):
            M.rotary_embedding(q, None, rotary)
        with pytest.raises(error, match=match):
            M.paged_moda_append(q, q, rotary=rotary, **_paged())
        with pytest.raises(error, match=match):
            M.paged_moda_decode(q, moda_group_num=4, rotary=rotary, **_paged())


def test_workspace_of_tables_too_large(built_library):
    """What the attention itself refuses has no workspace either (2^62 rows would not fit the division's numbers)."""
    from moda_b200 import _cabi
    from moda_b200._cabi import PagedCache, Problem, Tensor4
    lib, big = _cabi.load(), 2 ** 31 - 1
    t = Tensor4(0x1000, 1024, 256, 64)
    n = ctypes.c_size_t(7)
    for B, pages, page in ((1, big, big), (1, big, 2), (1, 1, big), (65535, 1 << 20, 1)):
        prob = Problem(B=B, T_kv=1, H=2, D=64, G=2, L=0, dtype=0, scale=0.125, device=0)
        cache = PagedCache(k=t, v=t, num_pages=4, page_size=page, block_table=0x2000, table_stride=2, max_pages=pages, seq_lens=0x3000)
        r = ctypes.byref
        assert lib.moda_b200_paged_decode_workspace_bytes(r(prob), r(cache), r(n)) == 11
        assert lib.moda_b200_paged_decode(r(prob), r(t), r(cache), None, None, None, None, None, None, r(t), 0x4000, 0x8000, 0, None) == 11
    assert n.value == 7
