"""Soft correspondence: the differentiable counterpart of `correspondence.dense_nn`, and a store of template features.

  soft_match      softmax-weighted transfer of a template's features to query cells, with gradients
  TemplateStore   feature maps of many rendered views in 8 bits: write, read back, and match against them

The reference matches hard (the `KNN` layer of ucn_code/nets/train.prototxt:2116-2141) or hands correlation maps to a
trunk (arch/eccv_net/eccv_net.py:161-231); it looks template views up one at a time (utils/proxy_renderer.py:100-151).
Nothing here has a counterpart in it to be checked against.
"""
import contextlib
import copy
import functools
import math

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _abi, _device as dv

_CODES = {torch.float32: _abi.F32, torch.bfloat16: _abi.BF16}
_COUNTS = {torch.uint8, torch.int8, torch.uint16, torch.int16, torch.uint32, torch.int32, torch.int64}
MAX_CHANNELS = _abi.SOFT_MAX_CHANNELS
_HERE = contextlib.nullcontext()


def _dims(x):
    try:
        return tuple(x.shape)
    except AttributeError:
        return np.shape(x)


def _map(x, name):
    """Dimensions of a feature map given as array or tensor, and its cells; checked before anything touches the device."""
    dims = _dims(x)
    if len(dims) < 3:
        raise ValueError(f"{name} must be (B,C,H,W) or (B,C,n), got {dims}")
    return dims, math.prod(dims[2:])


def _dtype(x, name):
    if not dv.is_tensor(x):
        return torch.float32
    if x.dtype not in _CODES:
        raise ValueError(f"{name} must be float32 or bfloat16, got {x.dtype}")
    return x.dtype


def _place(x):
    """(device of the call, context that makes it the current one): where its first tensor lives, else the current one."""
    if dv.is_tensor(x) and x.is_cuda:
        device = x.device
        return device, _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)
    return dv.device(), _HERE


def _stream(device):
    """Handle of the current stream.  torch.cuda.current_stream() builds an object around it, 2 us of a call of 25."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _on(x, dtype, device):
    """`x` on `device` as a contiguous tensor of `dtype`; itself where it already is one (the usual case, kept short: a call
    for a few queries is bounded by the host)."""
    if x is None:
        return None
    if dv.is_tensor(x) and x.dtype == dtype and x.device == device and x.is_contiguous():
        return x
    return dv.to_dev(x, dtype)


def _aligned(x):
    """The kernels stream maps in 16-byte pieces: a view that starts between them is copied."""
    return x if x is None or x.data_ptr() % 16 == 0 else x.clone()


@functools.lru_cache(maxsize=4096)
def _forward_bytes(*sizes):
    return _abi.lib.ispa_soft_match_workspace_bytes(*sizes)


@functools.lru_cache(maxsize=4096)
def _backward_bytes(*sizes):
    return _abi.lib.ispa_soft_match_backward_workspace_bytes(*sizes)


def _bytes(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _scores(heads, scale, cap, falloff, query_xy, grid, query_shape, batch, n):
    """Checks of what turns products into scores; `grid` is the reference map's (H,W) or None."""
    scale, cap = float(scale), float(cap or 0.0)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    if not (math.isfinite(cap) and cap >= 0):
        raise ValueError(f"cap must be finite and not negative (0 or None: no cap), got {cap}")
    if 0 < cap and (cap < 1e-30 or abs(scale) > 1e30 * cap):   # 0 or an infinite quotient in float32
        raise ValueError(f"cap {cap} is too small for scale {scale}")
    if falloff is not None:
        if grid is None:
            raise ValueError("falloff needs a reference map (B,C,H,W): distances are taken on its grid")
        if query_xy is None and query_shape != grid:
            raise ValueError(f"falloff: queries {query_shape} do not lie on the reference grid {grid}; give query_xy")
        if not np.isscalar(falloff) and _dims(falloff) != (heads,):
            raise ValueError(f"falloff must be a number or hold one value per head ({heads})")
        if not dv.is_tensor(falloff) and not (np.abs(np.asarray(falloff, np.float64)) < 1e38).all():
            raise ValueError(f"falloff must be finite in float32, got {falloff}")
        if query_xy is not None and _dims(query_xy) != (batch, n, 2):
            raise ValueError(f"query_xy must be ({batch},{n},2), got {_dims(query_xy)}")
    return scale, cap


def _score_tensors(heads, falloff, query_xy, device):
    if falloff is None:
        return None, None
    if np.isscalar(falloff):
        f = torch.full((heads,), float(falloff), dtype=torch.float32, device=device)
    else:
        f = _on(falloff, torch.float32, device)
    return f, _on(query_xy, torch.float32, device)


def _counts(num_query, batch):
    if num_query is None:
        return None
    t = num_query if dv.is_tensor(num_query) else np.asarray(num_query)
    if math.prod(t.shape) != batch:
        raise ValueError("num_query must hold one count per batch item")
    if t.dtype not in _COUNTS if dv.is_tensor(t) else t.size and t.dtype.kind not in "iu":
        raise ValueError("num_query must hold integers")
    return t.reshape(-1)


def _count_tensor(num_query, device):
    """Counts as int32; what int32 cannot hold is more than any query map has, or less than none."""
    if num_query is None:
        return None
    low, high = -1, 2 ** 31 - 1
    if not dv.is_tensor(num_query):
        num_query = np.clip(num_query, low, high)
    elif num_query.dtype in (torch.uint32, torch.int64):
        num_query = num_query.to(torch.int64).clamp(low, high)
    return _on(num_query, torch.int32, device)


def _check_mask(mask, batch, size):
    if mask is not None and _dims(mask) not in ((batch,) + size, (batch, 1) + size):
        raise ValueError(f"mask must be {(batch,) + size} or {(batch, 1) + size}, got {_dims(mask)}")


def _mask(mask, device):
    """Bytes, not 0 where the cell takes part.  A bool tensor is the byte array the kernels read."""
    if mask is None:
        return None
    if not dv.is_tensor(mask):
        mask = torch.from_numpy(np.asarray(mask) != 0)
    elif mask.dtype not in (torch.bool, torch.uint8):
        mask = mask != 0
    if mask.dtype == torch.bool:
        mask = mask.contiguous().view(torch.uint8)
    return _on(mask, torch.uint8, device)


def _fixed(x, name):
    """Refuses a scale or cap whose derivative somebody waits for."""
    if dv.is_tensor(x) and x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"no gradient flows to {name}, a number (a learned temperature: multiply query by it; else detach it)")


def _no_tangents(*tensors):
    """Refuses forward-mode derivatives: a dual tensor requires no gradient, and its tangent would be lost."""
    if forward_ad._current_level >= 0 and any(dv.is_tensor(x) and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise ValueError("soft_match has gradients (reverse mode) alone: no forward-mode tangents")


class _Call:
    """One soft_match call: its arguments checked (nothing touches the device), then as device tensors."""

    def __init__(self, query, ref, value, heads, scale, cap, falloff, query_xy, mask, num_query):
        (q_dims, n), (r_dims, cells) = _map(query, "query"), _map(ref, "ref")
        b, c = q_dims[:2]
        dtype = _dtype(query, "query")
        heads = int(heads)
        if r_dims[:2] != (b, c):
            raise ValueError(f"query {q_dims} and ref {r_dims} must share batch and channels")
        if _dtype(ref, "ref") != dtype:
            raise ValueError(f"ref must have query's dtype {dtype}")
        cv = c
        if value is not None:
            v_dims, v_cells = _map(value, "value")
            if v_cells != cells or v_dims[0] != b:
                raise ValueError(f"value {v_dims} must have the batch and cells of ref {r_dims}")
            if _dtype(value, "value") != dtype:
                raise ValueError(f"value must have query's dtype {dtype}")
            cv = v_dims[1]
        if heads < 1 or c < 1 or cv < 1 or c % heads or cv % heads:
            raise ValueError(f"{c} and {cv} channels do not split into {heads} heads")
        if c // heads > MAX_CHANNELS or cv // heads > MAX_CHANNELS:
            raise ValueError(f"at most {MAX_CHANNELS} channels per head")
        if cells < 1:
            raise ValueError("ref has no cells")
        _check_mask(mask, b, r_dims[2:])
        grid = r_dims[2:] if len(r_dims) == 4 else None
        _no_tangents(query, ref, value, scale, cap)
        _fixed(scale, "scale")
        _fixed(cap, "cap")
        if scale is None:
            scale = (c // heads) ** -0.5
        self.scale, self.cap = _scores(heads, scale, cap, falloff, query_xy, grid, q_dims[2:], b, n)
        num_query = _counts(num_query, b)
        self.raw = (query, ref, value, falloff, query_xy, mask, num_query)
        self.code = _CODES[dtype]
        self.dtype, self.b, self.heads, self.d, self.dv, self.n, self.cells = dtype, b, heads, c // heads, cv // heads, n, cells
        self.width = grid[1] if grid else cells
        self.out_shape = (b, cv) + q_dims[2:]

    def upload(self, device):
        query, ref, value, falloff, query_xy, mask, num_query = self.raw
        self.raw = None
        f, xy = _score_tensors(self.heads, falloff, query_xy, device)
        return self.bind(device, query, ref, value, f, xy, _mask(mask, device), _count_tensor(num_query, device))

    def bind(self, device, query, ref, value, falloff, xy, mask, count):
        self.device = device
        self.q, self.r, self.v = (_aligned(_on(x, self.dtype, device)) for x in (query, ref, value))
        self.falloff, self.xy, self.mask, self.count = falloff, xy, mask, count
        return self

    def release(self):
        """The options as device tensors; the call keeps its sizes and settings alone."""
        options = (self.falloff, self.xy, self.mask, self.count)
        self.q = self.r = self.v = self.falloff = self.xy = self.mask = self.count = None
        return options

    def _common(self):
        return (self.code, self.b, self.heads, self.d, self.dv, self.n, self.cells, self.width, self.scale, self.cap,
                dv.ptr(self.falloff), dv.ptr(self.xy), dv.ptr(self.mask), dv.ptr(self.count))

    def forward(self, exact, want_lse):
        """out, its float32 twin (`exact`; the same tensor for float32 maps) and lse.  The workspace is the call's own: calls
        on two streams, or captured in two graphs, share nothing."""
        out = torch.empty(self.out_shape, dtype=self.dtype, device=self.device)
        out32 = out if exact else None
        if exact and self.dtype != torch.float32:
            out32 = torch.empty(self.out_shape, dtype=torch.float32, device=self.device)
        lse = torch.empty((self.b, self.heads, self.n), dtype=torch.float32, device=self.device) if want_lse else None
        need = _forward_bytes(self.code, self.b, self.heads, self.d, self.dv, self.n, 1, self.cells)
        ws = _bytes(need, self.device)
        _abi.check(_abi.lib.ispa_soft_match(dv.ptr(self.q), dv.ptr(self.r), dv.ptr(self.v), *self._common(), dv.ptr(out),
                                            None if out32 is out else dv.ptr(out32), dv.ptr(lse), dv.ptr(ws), need,
                                            _stream(self.device)))
        return out, out32, lse

    def backward(self, out32, lse, d_out, d_lse):
        dq, dr = torch.empty_like(self.q), torch.empty_like(self.r)
        dval = torch.empty_like(self.v) if self.v is not None else None
        if d_out is None:
            d_out = torch.zeros(self.out_shape, dtype=self.dtype, device=self.device)
        d_out, d_lse = _aligned(_on(d_out, self.dtype, self.device)), _on(d_lse, torch.float32, self.device)
        need = _backward_bytes(self.code, self.b, self.heads, self.d, self.dv, self.n, self.cells)
        ws = _bytes(need, self.device)
        _abi.check(_abi.lib.ispa_soft_match_backward(dv.ptr(self.q), dv.ptr(self.r), dv.ptr(self.v), *self._common(),
                                                     dv.ptr(out32), dv.ptr(lse), dv.ptr(d_out), dv.ptr(d_lse), dv.ptr(dq),
                                                     dv.ptr(dr), dv.ptr(dval), dv.ptr(ws), need, _stream(self.device)))
        return dq, dr, dval


class _SoftMatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, ref, value, call):
        device, place = _place(query)
        with place:
            out, out32, lse = call.upload(device).forward(exact=True, want_lse=True)
        ctx.save_for_backward(query, ref, value, out32, lse, *call.release())
        ctx.call = call
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, d_lse):
        if d_out is None and d_lse is None:
            return None, None, None, None
        query, ref, value, out32, lse, *options = ctx.saved_tensors
        device, place = _place(query)
        with place:
            grads = copy.copy(ctx.call).bind(device, query, ref, value, *options).backward(out32, lse, d_out, d_lse)
        return (*(g.reshape(x.shape).to(x.device) if g is not None and need else None
                  for g, x, need in zip(grads, (query, ref, value), ctx.needs_input_grad)), None)


def soft_match(query, ref, value=None, *, heads=1, scale=None, cap=0.0, falloff=None, query_xy=None, mask=None,
               num_query=None, return_lse=False):
    """For every query cell the average of `value` over the reference cells, weighted by the softmax of the match scores.

    query (B,C,Hq,Wq) or (B,C,n); ref (B,C,H,W) or (B,C,cells); value (B,Cv,H,W) over the same cells, or None: ref
    is the value too.  float32 arrays or tensors, or bfloat16 tensors (all of one dtype); channels split into `heads`
    groups of at most 256 that are matched apart.  Scores of query i and cell j, per head:

        x = scale * <q_i, r_j>             scale: 1 / sqrt(C / heads) unless given (features of unit length want 10 to 30)
        y = cap * tanh(x / cap)            cap > 0; 0 or None: y = x
        z = y - falloff * |xy_i - xy_j|^2  falloff: a number or one per head; a prior on where the match lies.  Distances are
                                           in reference cells; queries lie on the reference grid unless query_xy (B,n,2)
                                           gives [x, y]

    mask (B,H,W) or (B,1,H,W): a cell with 0 / False takes no part, whatever its features hold (background of a
    rendered template); all other features are to be finite.  num_query (B,): only the first num_query[b] queries of item
    b are real, as in dense_nn; what lies behind them may be anything.
    Returns out (B,Cv,...) over query's cells in query's dtype, with return_lse also lse (B,heads,n) float32, the log of
    the sum of exp(z): the match's confidence.  A query that is not real, or whose cells are all masked, gets 0 and -inf.

    Tensors that require gradients get them (out and lse, once, in reverse mode; value None: ref's is the sum of both uses); no gradient
    flows to falloff, query_xy or the masks, and a scale or cap that requires one is refused: they are numbers (a learned
    temperature multiplies query).  Scores, sums and log-sums are float32; bfloat16 maps round the weights to
    bfloat16 for the product with the values.  Gradients form their weights from the log-sums, which are off by 2^-24 of
    themselves, as the scores are: scores far beyond 1e5 have no gradients to speak of.  Memory grows with the maps, not with
    their product, and results do not change from run to run."""
    as_tensor = dv.is_tensor(query)
    call = _Call(query, ref, value, heads, scale, cap, falloff, query_xy, mask, num_query)
    if torch.is_grad_enabled() and any(dv.is_tensor(x) and x.requires_grad for x in (query, ref, value)):
        if not all(dv.is_tensor(x) for x in (query, ref, value) if x is not None):
            raise ValueError("query, ref and value must be tensors where one of them requires gradients")
        out, lse = _SoftMatch.apply(query, ref, value, call)
        return (out, lse) if return_lse else out
    device, place = _place(query)
    with place:
        out, _, lse = call.upload(device).forward(exact=False, want_lse=return_lse)
        out = dv.back(out, as_tensor)
        return (out, dv.back(lse, as_tensor)) if return_lse else out


_KINDS = {"int8": (_abi.STORE_INT8, torch.int8), "fp8": (_abi.STORE_FP8, torch.float8_e4m3fn)}


class TemplateStore:
    """Feature maps of rendered views in 8 bits: a quarter of float32's memory for a class's thousands of views, with the
    views that `correspondence.nearest_view` names read back, or matched against, straight from their codes.

    codes (n_view,C,H*W) int8 or float8_e4m3fn, scales (n_view,H*W) float32, mask (n_view,H*W) uint8, on one device.
    A cell's channels share the scale max|x| / 127 ("fp8": / 448); the value is code * scale, so an int8 code is off
    by at most half a scale, an e4m3 one by 2^-4 of x or, below 2^-6 scales, by 2^-10 scales.  Views not yet written have no
    cells.

    Calls run on the current stream; a store that several streams use is ordered by the caller, like any tensor."""

    def __init__(self, n_view, channels, size, kind="int8"):
        self._set(kind, n_view, channels, size)
        cells = self.size[0] * self.size[1]
        device = dv.device()
        self.codes = torch.zeros((self.n_view, self.channels, cells), dtype=torch.uint8, device=device).view(_KINDS[kind][1])
        self.scales = torch.zeros((self.n_view, cells), dtype=torch.float32, device=device)
        self.mask = torch.zeros((self.n_view, cells), dtype=torch.uint8, device=device)

    def _set(self, kind, n_view, channels, size):
        if kind not in _KINDS:
            raise ValueError("kind must be 'int8' or 'fp8'")
        h, w = (int(x) for x in size)
        if n_view < 1 or channels < 1 or h < 1 or w < 1:
            raise ValueError(f"a store of {n_view} views of {channels} x {h} x {w}")
        self.kind, self.n_view, self.channels, self.size = kind, int(n_view), int(channels), (h, w)

    @classmethod
    def from_tensors(cls, codes, scales, mask, size):
        """A store over existing tensors (kept, not copied), e.g. ones that were saved."""
        kind = {torch.int8: "int8", torch.float8_e4m3fn: "fp8"}.get(codes.dtype)
        if kind is None or codes.dim() != 3:
            raise ValueError("codes must be (n_view,C,H*W) int8 or float8_e4m3fn")
        store = cls.__new__(cls)
        store._set(kind, codes.shape[0], codes.shape[1], size)
        flat = (codes.shape[0], codes.shape[2])
        if codes.shape[2] != store.size[0] * store.size[1]:
            raise ValueError(f"codes of {codes.shape[2]} cells are no {store.size} maps")
        if tuple(scales.shape) != flat or scales.dtype != torch.float32:
            raise ValueError(f"scales must be {flat} float32")
        if tuple(mask.shape) != flat or mask.dtype != torch.uint8:
            raise ValueError(f"mask must be {flat} uint8")
        if not (codes.is_cuda and scales.device == codes.device == mask.device):
            raise ValueError("codes, scales and mask must lie on one GPU")
        if not (codes.is_contiguous() and scales.is_contiguous() and mask.is_contiguous()):
            raise ValueError("codes, scales and mask must be contiguous")
        store.codes, store.scales, store.mask = codes, scales, mask
        return store

    def _views(self, views, dims):
        """Host indices are checked here; device ones by the kernels, which take an index outside as no view."""
        if not dv.is_tensor(views) or not views.is_cuda:
            host = np.asarray(views)
            if host.size and not np.issubdtype(host.dtype, np.integer):
                raise ValueError("views must be integers")
            if host.size and (host.min() < -1 or host.max() >= self.n_view):
                raise IndexError(f"view index outside [0, {self.n_view}) (-1: no view)")
            views = host.astype(np.int32)
        elif views.dtype not in (torch.int32, torch.int64):
            raise ValueError("views must be int32 or int64")
        if len(_dims(views)) != dims:
            raise ValueError(f"views must have {dims} dimension{'s' if dims > 1 else ''}, got {_dims(views)}")
        return views

    def _index(self, views):
        # an int64 index that int32 would wrap into the store must stay outside it
        if dv.is_tensor(views) and views.dtype == torch.int64:
            views = views.clamp(-1, 2 ** 31 - 1)
        return _on(views, torch.int32, self.codes.device)

    def write(self, views, features, mask=None):
        """Quantises features (n,C,H,W) (float32, or bfloat16 tensors) into views (n,).  mask (n,H,W) or (n,1,H,W): the cells that hold
        an object, all if None; a cell with a non-finite channel is masked as well.  A view listed twice keeps its
        last entry; -1 skips an entry."""
        views = self._views(views, 1)
        n = _dims(views)[0]
        dtype = _dtype(features, "features")
        if _dims(features) != (n, self.channels) + self.size:
            raise ValueError(f"features must be {(n, self.channels) + self.size}, got {_dims(features)}")
        _check_mask(mask, n, self.size)
        device, place = _place(self.codes)
        with place:
            v, f, m = self._index(views), _on(features, dtype, device), _mask(mask, device)
            _abi.check(_abi.lib.ispa_store_write(dv.ptr(f), _CODES[dtype], dv.ptr(m), dv.ptr(v), n, _KINDS[self.kind][0],
                                                 self.n_view, self.channels, self.codes.shape[2], dv.ptr(self.codes),
                                                 dv.ptr(self.scales), dv.ptr(self.mask), _stream(device)))

    def _read(self, views, dtype, features):
        views = self._views(views, 1)
        device, place = _place(self.codes)
        with place:
            v = self._index(views)
            n = v.shape[0]
            out = torch.empty((n, self.channels) + self.size, dtype=dtype, device=device) if features else None
            mask = None if features else torch.empty((n,) + self.size, dtype=torch.uint8, device=device)
            _abi.check(_abi.lib.ispa_store_read(dv.ptr(self.codes), dv.ptr(self.scales), dv.ptr(self.mask), dv.ptr(v), n,
                                                _KINDS[self.kind][0], self.n_view, self.channels, self.codes.shape[2],
                                                _CODES[dtype], dv.ptr(out), dv.ptr(mask), _stream(device)))
            return out if features else mask

    def read(self, views, dtype=torch.float32):
        """The features of views (n,), (n,C,H,W) of `dtype` (float32 or bfloat16), for dense_nn and the correlation layers.
        Zeros for -1 and views not written."""
        if dtype not in _CODES:
            raise ValueError("dtype must be torch.float32 or torch.bfloat16")
        return self._read(views, dtype, True)

    def read_mask(self, views):
        """The masks of views (n,) as (n,H,W) uint8; zeros for -1 and views not written."""
        return self._read(views, torch.float32, False)

    def soft_match(self, query, views, *, heads=1, scale=None, cap=0.0, falloff=None, query_xy=None, num_query=None,
                   return_lse=False):
        """soft_match of query (B,C,Hq,Wq) or (B,C,n) against the stored views (B,V) of each item: one softmax over the
        cells of all V views, whose features are reference and value, read from their codes.  -1 stands for no
        view, the store's masks apply, and the other arguments are soft_match's.  No gradients flow."""
        dims, n = _map(query, "query")
        b, c = dims[:2]
        dtype = _dtype(query, "query")
        heads = int(heads)
        if c != self.channels:
            raise ValueError(f"query has {c} channels, the store {self.channels}")
        if heads < 1 or c % heads or c // heads > MAX_CHANNELS:
            raise ValueError(f"{c} channels do not split into {heads} heads of at most {MAX_CHANNELS}")
        views = self._views(views, 2)
        if _dims(views)[0] != b:
            raise ValueError(f"views must be ({b},V), got {_dims(views)}")
        if scale is None:
            scale = (c // heads) ** -0.5
        scale, cap = _scores(heads, scale, cap, falloff, query_xy, self.size, dims[2:], b, n)
        count = _counts(num_query, b)
        as_tensor = dv.is_tensor(query)
        device, place = _place(self.codes)
        with place:
            q, v = _on(query.detach() if as_tensor else query, dtype, device), self._index(views)
            f, xy = _score_tensors(heads, falloff, query_xy, device)
            count = _count_tensor(count, device)
            out = torch.empty((b, c) + dims[2:], dtype=dtype, device=device)
            lse = torch.empty((b, heads, n), dtype=torch.float32, device=device) if return_lse else None
            d, cells, code = c // heads, self.codes.shape[2], _CODES[dtype]
            need = _forward_bytes(code, b, heads, d, d, n, v.shape[1], cells)
            ws = _bytes(need, device)
            _abi.check(_abi.lib.ispa_store_match(
                dv.ptr(q), code, dv.ptr(self.codes), dv.ptr(self.scales), dv.ptr(self.mask), _KINDS[self.kind][0], dv.ptr(v),
                v.shape[1], self.n_view, b, heads, d, n, cells, self.size[1], scale, cap, dv.ptr(f), dv.ptr(xy), dv.ptr(count),
                dv.ptr(out), dv.ptr(lse), dv.ptr(ws), need, _stream(device)))
            out = dv.back(out, as_tensor)
            return (out, dv.back(lse, as_tensor)) if return_lse else out
