"""What the entry points around 16-bit pages do without a GPU: how the attention's list is cut, the frequencies of
the rotary positions, refusals."""

import ctypes
import math
import os
import subprocess

import pytest
import torch

import flashquant_b200 as fq
from flashquant_b200 import _native as N
from flashquant_b200 import dense
from conftest import ROOT

# Every tile in one run, every piece of a unit group in a slot of its own, as many runs as the workspace has room for.
_DRIVER = r"""
#include <cstdio>
#include <cstdlib>
#include <set>
#include <utility>
#include <vector>
#include "dense_split.h"
using namespace fq;
#define CHECK(x) do { if (!(x)) { std::printf("%s: total %d fixed %d unit [%d, %d)\n", #x, c.total, c.fixed, a, b); return 1; } } while (0)
int main() {
  std::srand(7);
  for (int round = 0; round < 2000; ++round) {
    const int fixed = 1 + std::rand() % (round % 2 ? 1184 : 9);
    std::vector<int> bound{0};
    const int units = 1 + std::rand() % 40, longest = 1 + std::rand() % (round % 3 ? 30 : 30000);
    for (int i = 0; i < units; ++i) bound.push_back(bound.back() + 1 + std::rand() % longest);
    const DenseCut c = dense_cut(bound.back(), fixed, units);
    const int runs = c.fixed + c.taken();
    int a = 0, b = 0;
    CHECK(c.mains + c.tails == c.total && c.taken() <= kDenseTaken * fixed && (c.split || c.tails == 0) && !(c.split && units > kDenseGroups * fixed));
    int next[2] = {0, 0};  // the runs of either kind follow each other
    std::vector<char> seen(c.total);
    for (int r = 0; r < runs; ++r) {
      const bool tail = c.is_tail(r);
      CHECK(c.begin(r) == next[tail] && c.end(r) >= c.begin(r) && (!tail || c.end(r) > c.begin(r)));
      for (int i = c.begin(r); i < c.end(r); ++i) {
        const int x = c.entry(tail, i);
        CHECK(x >= 0 && x < c.total && !seen[x] && c.run_of(tail, i) == r && c.kind_of(tail, x) == i);
        seen[x] = 1;
      }
      next[tail] = c.end(r);
    }
    CHECK(next[0] == c.mains && next[1] == c.tails);
    std::set<int> slots;
    for (int u = 0; u < units; ++u) {
      a = bound[u], b = bound[u + 1];
      const DensePieces p = dense_pieces(c, a, b);
      std::set<int> mine;
      for (int x = a; x < b; ++x) {
        const bool tail = c.main_of(x + 1) == c.main_of(x);
        mine.insert(c.run_of(tail, c.kind_of(tail, x)));
      }
      CHECK(int(mine.size()) == p.count() && p.count() >= 1);
      for (int i = 0; i < p.count(); ++i) {
        CHECK(mine.count(p.run(i)) && dense_whole(c, p.run(i), a, b) == (p.count() == 1));
        const int slot = dense_slot(c, p.run(i), u, units, a);
        if (p.count() > 1) CHECK(slot >= 0 && slot < dense_slots(fixed) && slots.insert(slot).second);
      }
    }
  }
  for (int total : {1, 31 * 1184, 32 * 1184, 1 << 30, (1 << 30) - 1}) {
    const DenseCut c = dense_cut(total, 1184, 8);
    int a = 0, b = total;
    CHECK(c.taken() <= kDenseTaken * 1184 && c.mains + c.tails == total && c.end(c.fixed - 1) == c.mains);
    CHECK(c.tails == 0 || (c.end(c.fixed + c.taken() - 1) == c.tails && c.begin(c.fixed + c.taken() - 1) < c.tails));
  }
  {
    const DenseCut c = dense_cut(0, 148, 3);
    int a = 0, b = 0;
    CHECK(c.taken() == 0 && c.begin(0) == 0 && c.end(0) == 0 && c.end(147) == 0);
  }
  {
    const DenseSpan s = dense_span(2147483647, int64_t(1) << 33, 0), w = dense_span(2147483647, int64_t(1) << 33, 5);
    const DenseCut c = dense_cut(1, 1, 1);
    int a = 0, b = 0;
    CHECK(s.len == 2147483647 && s.tiles == 1 << 27 && s.first_tile == 0);
    CHECK(w.begin == 2147483642 && w.first_tile == (1 << 27) - 1 && w.tiles == 1);
  }
  for (int len = -3; len < 200; ++len)
    for (int window = 0; window < 70; ++window)
      for (int room = 0; room <= 160; room += 16) {
        const DenseSpan s = dense_span(len, room, window);
        const DenseCut c = dense_cut(len < 0 ? 0 : len, 1 + window, 1);
        int a = s.begin, b = s.len;
        CHECK(b >= 0 && b <= room && (len < 0 || b <= len) && a >= 0 && a <= b && s.tiles >= 0);
        CHECK(b == 0 || (b - a == (window && window < b ? window : b)));
        CHECK(16 * s.first_tile <= a && a - 16 * s.first_tile < 16 && 16 * (s.first_tile + s.tiles) >= b);
        CHECK(16 * (s.first_tile + s.tiles) - b < 16 && 16 * (s.first_tile + s.tiles) <= room);
      }
  std::puts("ok");
}
"""


def test_how_the_list_is_cut(tmp_path):
    src = tmp_path / "split.cpp"
    src.write_text(_DRIVER)
    exe = str(tmp_path / "split")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "flashquant_b200", "csrc"), str(src),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.stdout.strip() == "ok", r.stdout


# fp64, a few operations of 2^-53 each on exponents and logarithms of at most 20: 1e-14 covers them
@pytest.mark.parametrize("rd", [2, 64, 128, 10])
def test_frequencies(rd):
    base, factor, length = 500000.0, 8.0, 8192
    want = [base ** (-2.0 * j / rd) for j in range(rd // 2)]
    get = lambda **kw: fq.rotary_frequencies(rd, base, factor=factor, original_length=length, **kw)
    plain, scale = get()
    assert plain.dtype == torch.float64 and scale == 1.0 and plain.tolist() == pytest.approx(want, rel=1e-14)
    assert get(scaling="linear")[0].tolist() == pytest.approx([w / factor for w in want], rel=1e-14)
    blend = []
    for w in want:
        wavelength = 2 * math.pi / w
        if wavelength < length / 4.0:
            blend.append(w)
        elif wavelength > length / 1.0:
            blend.append(w / factor)
        else:
            s = (length / wavelength - 1.0) / (4.0 - 1.0)
            blend.append((1 - s) * w / factor + s * w)
    assert get(scaling="wavelength", low=1.0, high=4.0)[0].tolist() == pytest.approx(blend, rel=1e-13)
    y, scale = get(scaling="yarn", low=1.0, high=32.0)
    assert scale == pytest.approx(0.1 * math.log(factor) + 1.0, rel=1e-15)
    assert all(w / factor * (1 - 1e-14) <= v <= w * (1 + 1e-14) for v, w in zip(y.tolist(), want))
    if rd > 2:
        n = get(scaling="ntk")[0].tolist()
        assert n[0] == 1.0 and n[-1] == pytest.approx(want[-1] / factor, rel=1e-12)


def test_yarn_blends_between_its_two_indices():
    """Frequencies with more than `high` turns are kept, with fewer than `low` divided, and between them falling."""
    f0, _ = fq.rotary_frequencies(128, 10000.0)
    f, _ = fq.rotary_frequencies(128, 10000.0, "yarn", 16.0, 4096, 1.0, 32.0)
    turns = 4096 * f0 / (2 * math.pi)
    ratio = f / f0
    index = lambda n: 64 * math.log(4096 / (n * 2 * math.pi)) / math.log(10000.0)
    first, last = math.floor(index(32.0)), math.ceil(index(1.0))
    assert torch.all(ratio[:first + 1] == 1.0) and torch.allclose(ratio[last:], torch.tensor(1 / 16.0, dtype=torch.float64))
    assert torch.all(ratio[first:last].diff() < 0)
    assert turns[first] >= 32.0 > turns[first + 1] and turns[last] <= 1.0 < turns[last - 1]


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, base=1.0),
                                dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, factor=0.5),
                                dict(rotary_dim=8, scaling="wavelength", low=4.0, high=4.0),
                                dict(rotary_dim=2, scaling="ntk", factor=2.0)])
def test_frequencies_refused(kw):
    with pytest.raises(ValueError):
        fq.rotary_frequencies(**kw)


def test_there_is_no_cpu_path():
    x, pages = torch.zeros(2, 8, 128, dtype=torch.float16), torch.zeros(4, 16, 8, 128, dtype=torch.float16)
    i32 = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 2, dtype=torch.int32)
    freq, _ = fq.rotary_frequencies(128)
    for call in (lambda: fq.rotary_embed(x, x, i32, freq),
                 lambda: fq.rotary_append_dense(x, x, x, pages, pages, i32, i32, freq),
                 lambda: fq.split_k_paged_decode_dense(x, pages, pages, table, i32),
                 lambda: fq.plan_paged_step(i32, i32, table, i32, i32[:1], 16, 8),
                 lambda: fq.release_pages(i32.bool(), i32, table, i32, i32[:1], 16)):
        with pytest.raises(N.FlashQuantNativeError):
            call()
    with pytest.raises(ValueError):
        fq.rotary_embed(x, x, i32, freq, layout="other")


@pytest.mark.parametrize("stride, size, own", [((256, 128, 1), (3, 2, 128), True), ((128, 384, 1), (3, 2, 128), True),
                                               ((0, 128, 1), (3, 2, 128), False), ((128, 128, 1), (3, 2, 128), False),
                                               ((256, 0, 1), (3, 2, 128), False), ((256, 64, 1), (3, 2, 128), False),
                                               ((7, 7, 1), (1, 1, 128), True), ((0, 0, 1), (0, 2, 128), True),
                                               ((256, 128, 2), (3, 2, 128), False), ((1024, 64, 64, 1), (2, 4, 4, 64), False),
                                               ((1024, 256, 64, 1), (2, 4, 4, 64), True), ((1024, 64, 256, 1), (2, 4, 4, 64), True),
                                               ((960, 256, 64, 1), (2, 4, 4, 64), False)])
def test_rows_of_their_own(stride, size, own):
    assert dense._own_rows(torch.empty_strided(size, stride)) is own


# ---- refusals of the C entry points: before any CUDA call ----------------------------------------------
P = ctypes.c_void_p(4096)   # stands for an aligned device pointer; nothing is launched


def _decode(**kw):
    a = dict(q=P, dtype=N.FQ_F16, qs=1024, qh=128, k=P, kb=16384, kt=1024, kh=128, v=P, vb=16384, vt=1024, vh=128, table=P,
             ts=4, width=4, lens=P, seqs=2, hq=8, hkv=8, d=128, bs=16, blocks=8, scale=0.1, window=0, out=P, lse=None,
             ws=P, bytes=1 << 30, stream=None)
    a.update(kw)
    return N.load().fq_dense_paged_decode(*a.values())


@pytest.mark.parametrize("kw, rc", [(dict(q=None), -1), (dict(lens=None), -1), (dict(out=None), -1), (dict(k=None), -1),
                                    (dict(table=None), -1), (dict(window=-1), -1), (dict(seqs=-1), -1),
                                    (dict(hq=12), -1), (dict(hkv=0), -1), (dict(d=80), -2), (dict(seqs=2049), -2),
                                    (dict(bs=24), -2), (dict(bs=0), -2), (dict(dtype=N.FQ_F32), -2),
                                    (dict(kt=1020), -5), (dict(vh=4), -5), (dict(k=ctypes.c_void_p(4104)), -5),
                                    (dict(q=ctypes.c_void_p(4098)), -5), (dict(qs=1023), -5), (dict(out=ctypes.c_void_p(4100)), -5), (dict(ws=None), -3),
                                    (dict(bytes=32768), -3), (dict(width=1 << 29), -2), (dict(seqs=0, q=None), 0)])
def test_decode_refusals(kw, rc):
    assert _decode(**kw) == rc
    if rc:
        assert b"dense decode" in N.load().fq_last_error_string()


def test_decode_workspace_sizes():
    f = N.load().fq_dense_paged_decode_workspace_bytes
    assert f(4, 32, 8, 128) >= 32768 + 148 * 5 * 8 * 4 * 130 * 4
    assert f(4, 32, 8, 80) == 0 and f(4, 12, 8, 128) == 0 and f(-1, 8, 8, 128) == 0
    assert f(1, 32, 8, 128) == f(2048, 32, 8, 128)


def _plan(**kw):
    a = dict(context=P, query=P, n=2, table=P, ts=4, width=4, bs=16, free=P, cap=64, count=P, room=8, lens=P, cu=P, slots=P,
             pos=P, served=P, out=P, stream=None)
    a.update(kw)
    return N.load().fq_plan_paged_step(*a.values())


@pytest.mark.parametrize("kw, rc", [(dict(context=None), -1), (dict(table=None), -1), (dict(count=None), -1),
                                    (dict(out=None), -1), (dict(slots=None), -1), (dict(free=None), -1),
                                    (dict(cu=None), -1), (dict(n=-1), -1), (dict(n=4097), -2), (dict(bs=0), -1),
                                    (dict(ts=3), -1), (dict(room=-1), -1), (dict(cap=1 << 31), -2),
                                    (dict(width=1 << 28, ts=1 << 28), -2)])
def test_plan_refusals(kw, rc):
    assert _plan(**kw) == rc


@pytest.mark.parametrize("kw, rc", [(dict(rd=3), -2), (dict(rd=130), -2), (dict(dtype=7), -1), (dict(layout=2), -1),
                                    (dict(n=-1), -1), (dict(q=None), -1), (dict(freq=None), -1), (dict(pos=None), -1),
                                    (dict(hq=5000), -2), (dict(n=0, q=None), 0)])
def test_rotary_refusals(kw, rc):
    s = (ctypes.c_int64 * 8)(*[1024, 128] * 4)
    a = dict(q=P, k=P, dtype=N.FQ_BF16, n=2, hq=8, hk=8, d=128, rd=128, strides=s, pos=P, p64=1, freq=P, layout=0, scale=1.0,
             inverse=0, qo=P, ko=P, stream=None)
    a.update(kw)
    assert N.load().fq_rotary_embed(*a.values()) == rc


@pytest.mark.parametrize("kw, rc", [(dict(dtype=N.FQ_F32), -2), (dict(bs=0), -1), (dict(slots=None), -1),
                                    (dict(kc=None), -1), (dict(v=None), -1), (dict(pos=None), -1), (dict(num=-1), -1),
                                    (dict(n=0), 0)])
def test_append_refusals(kw, rc):
    s = (ctypes.c_int64 * 14)(*[1024, 128] * 4, *[16384, 1024, 128] * 2)
    a = dict(q=P, k=P, v=P, dtype=N.FQ_BF16, n=2, hq=8, hk=8, d=128, rd=128, strides=s, pos=P, p64=1, freq=P, layout=0,
             scale=1.0, qo=P, kc=P, vc=P, bs=16, num=128, slots=P, s64=1, stream=None)
    a.update(kw)
    assert N.load().fq_rotary_append_dense(*a.values()) == rc
