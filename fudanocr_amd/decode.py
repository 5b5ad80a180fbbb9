"""Autoregressive decoding on the HIP kernels (csrc/paged_attention.hip, csrc/beam.hip): a paged key / value cache, attention
of new tokens over it, beam search's selection and the reordering of the surviving beams' caches.

The recognizers' `beam_search` (fudanocr_amd/sld/beam.py) is built from these; they work on their own as well.  Unlike the
training operators of `kernels` / `sld.ops` they also take bf16 and fp16 tensors, have no backward pass (a tensor that wants a
gradient is refused), and nothing in them waits for the device: lengths, tables and parents stay there.

A cache is four tensors:

* ``k_pages``, ``v_pages``  [num_pages, heads, page, dim]: `page` (a power of two from 8 to 1024) tokens a page;
* ``table``    int32 [seqs, pages per sequence]: row s names the pages of sequence s in order;
* ``kv_lens``  int32 [seqs]: tokens of each sequence in the cache, the new ones of the present call included.

A chunk of new tokens is one packed tensor [tokens, heads, dim]: ``q_start`` (int32 [seqs + 1], non-decreasing) gives the first
row of every sequence, without it each has tokens / seqs rows.  Rows of no sequence (in front of the first, behind the last)
are left as they are: in an output that the call allocates they are whatever the memory held.  The new tokens of a sequence are
its last ones: the first of n has position kv_lens - n.

What comes from the device is checked there: a length beyond the table or `max_kv`, more new tokens than `max_q`, or offsets that
run over the first or the last row make a sequence's output NaN (nothing of it is appended), a page number outside the cache that
of the tokens that need the page (other tokens of the sequence may be NaN then too); nothing outside the given tensors is read or
written.  Offsets that fall are not told apart from right ones: rows that two sequences claim may hold either's results, or none."""
import ctypes
import math

import torch

from . import _lib
from .kernels import _RAW_STREAM

_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_PAGES, _DIMS = frozenset(8 << i for i in range(8)), (64, 128, 256)
_LONGEST = 2 ** 31 - 2 ** 14 - 1          # tokens of a sequence: positions and the steps beyond the last one are 32-bit numbers
_NO_GRAD = "%s wants a gradient, which these operators do not have (torch.no_grad(), or kernels / sld.ops in training)"
_EVEN = "without q_start every sequence has the same number of rows; %d tokens, %d sequences"


def _need(ok, what, *args):
    if not ok:
        raise RuntimeError("fudanocr_amd.decode: " + (what % args if args else what))


def _launch(device, name, *args):
    """the entry point on the current stream of the tensors' device (an index), whatever device is current"""
    if device == _current_device():
        _lib.call(name, *args, _stream(device))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _stream(device))


def _stream(device):
    return _RAW_STREAM(device) if _RAW_STREAM is not None else torch.cuda.current_stream(device).cuda_stream


def _on_gpu(t):
    """the tensors' device as an index (`get_device` -- a device object per check costs more than the rest of it)"""
    dev = t.get_device()
    _need(dev >= 0, "tensors must be on the GPU, got %s", t.device)
    return dev


def _int32(t, shape, dev, what):
    _need(t.dtype is torch.int32 and t.shape == shape and t.is_contiguous() and t.get_device() == dev,
          "%s must be a contiguous int32 tensor %s on the same device as the others", what, tuple(shape))


def _cache(k_pages, v_pages, table, kv_lens, q_start):
    shape, dt, dev = k_pages.shape, k_pages.dtype, k_pages.get_device()
    tshape = table.shape
    # all of it in one condition (a call per check takes longer than the kernel of a small step); what is wrong is said below
    if (len(shape) == 4 and shape == v_pages.shape and dt is v_pages.dtype and dt in _DTYPES and k_pages.is_contiguous()
            and v_pages.is_contiguous() and v_pages.get_device() == dev and shape[2] in _PAGES and shape[3] in _DIMS
            and shape[0] > 0 and shape[1] > 0 and len(tshape) == 2 and tshape[1] > 0 and table.dtype is torch.int32
            and table.is_contiguous() and table.get_device() == dev and kv_lens.dtype is torch.int32
            and kv_lens.shape == (tshape[0],) and kv_lens.is_contiguous() and kv_lens.get_device() == dev
            and (q_start is None or (q_start.dtype is torch.int32 and q_start.shape == (tshape[0] + 1,)
                                     and q_start.is_contiguous() and q_start.get_device() == dev))
            and not k_pages.requires_grad and not v_pages.requires_grad):
        return *shape, *tshape, dt, dev
    _need(len(shape) == 4 and shape == v_pages.shape and dt is v_pages.dtype and dt in _DTYPES,
          "k_pages and v_pages must be two [num_pages, heads, page, dim] tensors of one type (fp32, bf16 or fp16)")
    _need(k_pages.is_contiguous() and v_pages.is_contiguous() and v_pages.get_device() == dev,
          "k_pages and v_pages must be contiguous and on one device")
    num_pages, heads, page, dim = shape
    _need(page in _PAGES, "page must be a power of two from 8 to 1024, got %d", page)
    _need(dim in _DIMS, "head dim must be 64, 128 or 256, got %d", dim)
    _need(num_pages > 0 and heads > 0, "the cache has no pages or no heads")
    _need(len(tshape) == 2 and tshape[1] > 0, "table must be [seqs, pages per sequence]")
    seqs = tshape[0]
    _int32(table, tshape, dev, "table")
    _int32(kv_lens, (seqs,), dev, "kv_lens")
    if q_start is not None:
        _int32(q_start, (seqs + 1,), dev, "q_start")
    _need(not (k_pages.requires_grad or v_pages.requires_grad) or not torch.is_grad_enabled(), _NO_GRAD, "the cache")
    return num_pages, heads, page, dim, seqs, tshape[1], dt, dev


def _rows(t, heads, dim, dt, dev, what):
    """-> tokens, heads and the strides of these two axes"""
    shape, st = t.shape, t.stride()
    if (len(shape) == 3 and shape[2] == dim and (heads is None or shape[1] == heads) and t.dtype is dt and t.get_device() == dev
            and st[2] == 1 and not t.requires_grad):
        return shape[0], shape[1], st[0], st[1]
    _need(len(shape) == 3 and shape[2] == dim and (heads is None or shape[1] == heads) and t.dtype is dt
          and t.get_device() == dev, "%s must be [tokens, %s, %d] %s on the cache's device", what,
          "heads" if heads is None else heads, dim, dt)
    _need(st[2] == 1 or t.numel() == 0, "%s must have contiguous rows of dim", what)
    _need(not t.requires_grad or not torch.is_grad_enabled(), _NO_GRAD, what)
    return shape[0], shape[1], st[0], st[1]


def paged_append(k_new, v_new, k_pages, v_pages, table, kv_lens, q_start=None):
    """writes the new tokens' keys and values [tokens, heads, dim] to their pages (positions kv_lens - n .. kv_lens - 1 of each
    sequence).  A token whose page the table does not name is dropped.  k_pages, v_pages and the new tokens lie apart."""
    num_pages, heads, page, dim, seqs, ld, dt, dev = _cache(k_pages, v_pages, table, kv_lens, q_start)
    tokens, _, kt, kh = _rows(k_new, heads, dim, dt, dev, "k_new")
    v_tokens, _, vt, vh = _rows(v_new, heads, dim, dt, dev, "v_new")
    _need(v_tokens == tokens, "k_new and v_new must have the same tokens")
    if q_start is None and seqs and tokens % seqs:
        _need(False, _EVEN, tokens, seqs)
    if dev < 0:
        _on_gpu(k_pages)
    if tokens == 0 or seqs == 0:
        return
    _launch(dev, "focr_paged_append", k_new.data_ptr(), v_new.data_ptr(), kt, kh, vt, vh, k_pages.data_ptr(), v_pages.data_ptr(),
            table.data_ptr(), kv_lens.data_ptr(), None if q_start is None else q_start.data_ptr(), tokens, seqs, heads, dim, page,
            ld, num_pages, _DTYPES[dt])


def paged_attention(q, k_pages, v_pages, table, kv_lens, q_start=None, causal=True, scale=None, max_q=None, max_kv=None,
                    out=None):
    """softmax(scale q k^T) v of the new tokens q [tokens, heads, dim] over their sequences' caches -> [tokens, heads, dim].

    heads is a multiple of the cache's; head h reads the cache's head h // (heads / cache heads).  causal: a token at position p
    sees the positions 0 .. p, else all kv_lens of them; a token that sees nothing, or scores of -inf alone, gets zeros.  scale:
    1 / sqrt(dim) unless given, positive.  max_q / max_kv: bounds on a sequence's new tokens and on kv_lens that the caller knows
    (they size the launch; the defaults are the most the tensors allow).  out: where to write (apart from q and the cache)."""
    num_pages, kv_heads, page, dim, seqs, ld, dt, dev = _cache(k_pages, v_pages, table, kv_lens, q_start)
    tokens, heads, qt, qh = _rows(q, None, dim, dt, dev, "q")
    _need(heads > 0 and heads % kv_heads == 0, "%d heads over a cache of %d", heads, kv_heads)
    if q_start is None and seqs and tokens % seqs:
        _need(False, _EVEN, tokens, seqs)
    scale = dim ** -0.5 if scale is None else float(scale)
    _need(0.0 < scale < math.inf, "scale must be positive and finite, got %r", scale)
    limit = min(ld * page, _LONGEST)
    max_kv = limit if max_kv is None else min(int(max_kv), limit)
    if q_start is None:
        max_q = tokens // seqs if seqs else 0
    else:
        max_q = tokens if max_q is None else min(int(max_q), tokens)
    _need(max_q >= 0 and max_kv >= 0, "max_q / max_kv out of range")
    if out is not None:
        n, _, ot, oh = _rows(out, heads, dim, dt, dev, "out")
        _need(n == tokens and ((tokens == 1 or ot >= (heads - 1) * oh + dim) and (heads == 1 or oh >= dim)
                               or ot >= dim and oh >= (tokens - 1) * ot + dim), "out must have q's shape and rows of its own")
        _need(not _overlap(out, q), "out must not share q's memory")
    if dev < 0:
        _on_gpu(k_pages)
    if out is None:
        out, ot, oh = torch.empty((tokens, heads, dim), dtype=dt, device=q.device), heads * dim, dim
    if tokens == 0 or seqs == 0:
        return out
    code = _DTYPES[dt]
    n_ws = _lib.load().focr_paged_attention_ws_bytes(tokens, seqs, heads, kv_heads, dim, max_q, max_kv, code)
    _need(n_ws >= 0, "arguments out of range")
    ws = torch.empty(n_ws, dtype=torch.uint8, device=q.device) if n_ws else None
    _launch(dev, "focr_paged_attention_fwd", q.data_ptr(), qt, qh, k_pages.data_ptr(), v_pages.data_ptr(),
            table.data_ptr(), kv_lens.data_ptr(), None if q_start is None else q_start.data_ptr(), out.data_ptr(), ot, oh,
            None if ws is None else ws.data_ptr(), n_ws, tokens, seqs, heads, kv_heads, dim, page, ld, num_pages, max_q, max_kv,
            scale, 1 if causal else 0, code)
    return out


def _overlap(a, b):
    def span(t):
        return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def beam_select(logits, scores, finished=None, eos=None, n=None):
    """the n (default: beams) best continuations of every batch entry over beams and vocabulary, best first.

    logits [batch, beams, vocab] (fp32, bf16 or fp16; rows contiguous), scores fp32 [batch, beams]: the beams' running
    log-probabilities (-inf: no such beam, as for all but the first at a search's first step).  A candidate's score is its beam's
    plus the token's log-softmax; a finished beam (bool [batch, beams]) has the one candidate (itself, eos) at its own score.
    Equal scores go to the lowest (beam, token).  NaN logits and beams whose score or normaliser is not finite rank as -inf.

    -> (scores fp32 [batch, n], parents int32 [batch, n], tokens int64 [batch, n], finished bool [batch, n])"""
    shape, dt, dev = logits.shape, logits.dtype, logits.get_device()
    _need(len(shape) == 3 and dt in _DTYPES, "logits must be [batch, beams, vocab] in fp32, bf16 or fp16")
    batch, beams, vocab = shape
    n = beams if n is None else int(n)
    if not (1 <= beams <= 64 and 1 <= n <= 64 and vocab >= 1 and n <= beams * vocab):
        _need(False, "beams and n must be 1 to 64 and n at most beams * vocab; got %d beams, n = %d, vocab %d", beams, n, vocab)
    ls, rows = logits.stride(), (batch, beams)
    _need(ls[2] == 1 or vocab == 1 or logits.numel() == 0, "logits must have contiguous rows of vocab")
    _need(not (logits.requires_grad or scores.requires_grad) or not torch.is_grad_enabled(), _NO_GRAD, "logits or scores")
    _need(scores.dtype is torch.float32 and scores.shape == rows and scores.is_contiguous() and scores.get_device() == dev,
          "scores must be a contiguous fp32 tensor [batch, beams] on the logits' device")
    if finished is not None:
        _need(finished.dtype is torch.bool and finished.shape == rows and finished.is_contiguous() and finished.get_device() == dev,
              "finished must be a contiguous bool tensor [batch, beams] on the logits' device")
        _need(eos is not None, "finished beams need an eos")
    _need(eos is None or 0 <= int(eos) < vocab, "eos must be inside the vocabulary")
    eos = -1 if eos is None else int(eos)
    if dev < 0:
        _on_gpu(logits)
    device = logits.device
    out_scores = torch.empty_like(scores) if n == beams else torch.empty((batch, n), dtype=torch.float32, device=device)
    out_parents = torch.empty_like(out_scores, dtype=torch.int32)
    out_tokens = torch.empty_like(out_scores, dtype=torch.int64)
    out_finished = torch.empty_like(out_scores, dtype=torch.bool)
    if batch:
        code = _DTYPES[dt]
        n_ws = _lib.load().focr_beam_select_ws_bytes(batch, beams, vocab, n, code)
        ws = torch.empty(n_ws, dtype=torch.uint8, device=device) if n_ws else None
        _launch(dev, "focr_beam_select", logits.data_ptr(), ls[0], ls[1], scores.data_ptr(),
                None if finished is None else finished.data_ptr(), out_scores.data_ptr(), out_parents.data_ptr(),
                out_tokens.data_ptr(), out_finished.data_ptr(), None if ws is None else ws.data_ptr(), n_ws, batch, beams, vocab,
                n, eos, code)
    return out_scores, out_parents, out_tokens, out_finished


def beam_reorder(parents, table, kv_lens, spare, pages, table_out=None, spare_out=None):
    """beam j of every group goes on from its group's beam parents[group, j]: -> (table, spare) of the reordered beams.

    parents int32 [groups, beams]; the cache's sequences are the groups' beams in order, and the beams of a group have the same
    kv_lens (the first one's counts).  Full pages are shared by table entry; the partial last page is copied to the beam's page
    in `spare` (int32 [seqs]), and the one it had becomes its spare.  pages: the page tensors (k_pages and v_pages of every
    layer) that the table stands for.  Before the call, the pages in `spare` and each beam's entries from its partial page on
    must be its own alone (`PagedCache` sees to that).  table_out / spare_out are the inputs or lie apart from them; a parent
    outside the group counts as the beam itself."""
    pshape, dev = parents.shape, parents.get_device()
    _need(len(pshape) == 2, "parents must be [groups, beams]")
    groups, beams = pshape
    slots = groups * beams
    _int32(parents, pshape, dev, "parents")
    _need(1 <= beams <= 64 and slots <= 65535, "beams must be 1 to 64 and groups * beams at most 65535")
    tshape = table.shape
    _need(len(tshape) == 2 and tshape[0] == slots and tshape[1] > 0, "table must be [groups * beams, pages per sequence]")
    _int32(table, tshape, dev, "table")
    _int32(kv_lens, (slots,), dev, "kv_lens")
    _int32(spare, (slots,), dev, "spare")
    pages = list(pages)
    _need(len(pages) > 0, "no page tensors")
    shape, dt = pages[0].shape, pages[0].dtype
    for p in pages:
        if not (len(shape) == 4 and p.shape == shape and p.dtype is dt and dt in _DTYPES and p.is_contiguous()
                and p.get_device() == dev):
            _need(False, "pages must be contiguous [num_pages, heads, page, dim] tensors of one shape and type (fp32, bf16 or "
                  "fp16) on the parents' device")
        _need(not p.requires_grad or not torch.is_grad_enabled(), _NO_GRAD, "a page tensor")
    num_pages, heads, page, dim = shape
    _need(page in _PAGES, "page must be a power of two from 8 to 1024, got %d", page)
    _need(num_pages > 0 and heads > 0 and dim > 0 and dim * pages[0].element_size() % 16 == 0,
          "rows of dim must be whole 16-byte units")
    if table_out is None:
        table_out = torch.empty_like(table)
    else:
        _int32(table_out, tshape, dev, "table_out")
    if spare_out is None:
        spare_out = torch.empty_like(spare)
    else:
        _int32(spare_out, (slots,), dev, "spare_out")
    if dev < 0:
        _on_gpu(parents)
    if slots:
        ptrs = (ctypes.c_void_p * len(pages))(*[p.data_ptr() for p in pages])
        _launch(dev, "focr_beam_reorder", parents.data_ptr(), table.data_ptr(), kv_lens.data_ptr(), spare.data_ptr(),
                table_out.data_ptr(), spare_out.data_ptr(), ptrs, len(pages), groups, beams, heads, dim, page, tshape[1],
                num_pages, _DTYPES[dt])
    return table_out, spare_out


class PagedCache:
    """The caches of a decoder's layers for `seqs` sequences of at most max_len tokens: page tensors per layer, one table, the
    lengths and a spare page per sequence.  Every sequence starts with pages of its own.

    step (n new tokens for every sequence):  cache.advance(n);  per layer: cache.append(layer, k, v), cache.attend(layer, q);
    between the steps of a beam search: cache.reorder(parents).

    A step can be captured into a graph but for `advance`, which counts on the host as well: call it before every replay.  A
    captured `attend` is sized for max_len, an eager one for the tokens that are there."""

    def __init__(self, seqs, max_len, heads, dim, layers=1, page=16, dtype=torch.float32, device="cuda"):
        _need(seqs > 0 and max_len > 0 and heads > 0 and layers > 0, "seqs, max_len, heads and layers must be positive")
        _need(page in _PAGES, "page must be a power of two from 8 to 1024, got %d", page)
        _need(dim in _DIMS and dtype in _DTYPES, "head dim must be 64, 128 or 256, the type fp32, bf16 or fp16")
        per = -(-max_len // page)
        num = seqs * (per + 1)
        _need(num < 2 ** 31, "more pages than int32 numbers")
        self.page, self.max_len, self.length = page, max_len, 0
        self.k = [torch.empty((num, heads, page, dim), dtype=dtype, device=device) for _ in range(layers)]
        self.v = [torch.empty((num, heads, page, dim), dtype=dtype, device=device) for _ in range(layers)]
        ids = torch.arange(num, dtype=torch.int32, device=device)
        self.table, self.spare = ids[:seqs * per].view(seqs, per), ids[seqs * per:].clone()
        self.kv_lens = torch.zeros(seqs, dtype=torch.int32, device=device)

    def advance(self, n):
        """n more tokens for every sequence (their keys and values follow with `append`)"""
        _need(not self._captured(), "advance counts on the host: call it before the replay, outside the graph")
        _need(n >= 0 and self.length + n <= self.max_len, "%d + %d tokens in a cache of %d", self.length, n, self.max_len)
        self.length += n
        self.kv_lens += n

    def _captured(self):
        return self.kv_lens.is_cuda and torch.cuda.is_current_stream_capturing()

    def append(self, layer, k_new, v_new):
        paged_append(k_new, v_new, self.k[layer], self.v[layer], self.table, self.kv_lens)

    def attend(self, layer, q, causal=True, scale=None, out=None):
        return paged_attention(q, self.k[layer], self.v[layer], self.table, self.kv_lens, causal=causal, scale=scale,
                               max_kv=self.max_len if self._captured() else self.length, out=out)

    def reorder(self, parents):
        beam_reorder(parents, self.table, self.kv_lens, self.spare, self.k + self.v, self.table, self.spare)
