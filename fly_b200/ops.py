"""Functional layer over the C ABI: builds `SblParams` from torch tensors and
launches on the current CUDA stream.  PyTorch is used only for device memory
and streams; all arithmetic happens in libsblocal_b200.so.
"""
import contextlib
import ctypes
import math
import threading

import torch
from torch.autograd import forward_ad

from . import _cabi

_DTYPES = {torch.float32: _cabi.SBL_DTYPE_F32, torch.bfloat16: _cabi.SBL_DTYPE_BF16}
_ws_lock = threading.Lock()
_workspaces = {}


class _StatusWatch:
    """Device status words of earlier calls, forward and backward, looked at without ever blocking the host.

    The tensor-core kernels leave three int32 words in the workspace (a bounded wait that ran out; an exponential
    that left the fp32 range; a row whose low-rank estimate swamped its exact part).  `post` queues a kernel behind a
    call that brings words other than zero into page-locked host memory, in a captured call with every replay; `poll`
    looks there and raises.  The module and `sblocal_attention` call `poll` at the start of every forward, so a bad
    result is reported by the next call at the latest.  `poll(wait=True)` waits for the devices first: for the end of
    a program, and for graphs, whose replays call nothing that could look."""

    def __init__(self):
        self._lock = threading.Lock()
        self._words = None             # three int32, page-locked
        self._devices = set()          # that have written there

    def post(self, words, device):
        """words: address of the three status words that the current stream's work writes."""
        if self._words is None:
            if torch.cuda.is_current_stream_capturing():
                return                 # (page-locked memory cannot be had in a capture that no call came before)
            with self._lock:
                if self._words is None:
                    self._memory = torch.zeros(3, dtype=torch.int32).pin_memory()
                    self._words = (ctypes.c_int32 * 3).from_address(self._memory.data_ptr())
        self._devices.add(device.index)
        _cabi.check(_cabi.load().sbl_collect_status(words, ctypes.addressof(self._words), _stream(device)))

    def poll(self, wait=False):
        if self._words is None:
            return
        if wait:
            for index in tuple(self._devices):
                torch.cuda.synchronize(index)
        if any(self._words):
            with self._lock:
                words = list(self._words)
                for i, word in enumerate(words):
                    if word:               # (one that arrives meanwhile is left for the next look)
                        self._words[i] = 0
            self._report(words)

    @staticmethod
    def _report(words):
        wait_site, out_of_range, imprecise = words
        if wait_site:
            raise _cabi.SblError(_cabi.SBL_ERR_DEVICE_STATUS,
                                 f'an earlier call gave up on a bounded wait inside a kernel (wait site '
                                 f'{wait_site}); its results are invalid')
        if out_of_range:
            raise _cabi.SblError(_cabi.SBL_ERR_DEVICE_STATUS,
                                 'an earlier forward met logits beyond the range of the bf16 tensor-core kernels '
                                 '(an exponential left the fp32 range); its output is invalid -- use fp32 inputs '
                                 'or Problem(..., generic=True)')
        if imprecise:
            raise _cabi.SblError(_cabi.SBL_ERR_DEVICE_STATUS,
                                 'an earlier forward met query rows whose in-window low-rank estimate is more than '
                                 '16 times their exact softmax mass (logits 3-4 times the unit scale): the bf16 '
                                 'tensor-core kernels lose accuracy there -- use fp32 inputs or '
                                 'Problem(..., generic=True)')


status_watch = _StatusWatch()


def _on(device):
    """`torch.cuda.device(device)`, or nothing where the device is the current one already (some microseconds of a
    small call)."""
    if device.index is not None and device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


# (the current stream's handle without a Stream object around it, where this torch has the call)
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)


def _stream(device):
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


class Problem:
    """One SBLocal problem: parameter block plus the tensors it borrows (kept
    alive for as long as the block is used)."""

    def __init__(self, query, key, value, W, local_context, softmax_temp=None, softmax_eps=0.0,
                 key_lengths=None, out=None, q_pos0=0, k_pos0=0, S_total=None, sum_range=None, generic=False):
        if not (query.is_cuda and key.is_cuda and value.is_cuda):
            raise ValueError('sblocal_b200 runs on CUDA tensors only (there is no CPU path)')
        if key.device != query.device or value.device != query.device:
            raise ValueError('query, key and value must be on one device')
        if query.dim() != 4 or key.dim() != 4 or value.dim() != 4:
            raise ValueError('query/key/value must be (B,T,H,E), (B,S,H,E), (B,S,H,D)')
        if query.dtype not in _DTYPES:
            raise TypeError(f'dtype {query.dtype} is not supported (float32 and bfloat16 are)')
        if key.dtype != query.dtype or value.dtype != query.dtype:
            raise TypeError('query, key and value must share one dtype')
        B, T, H, E = query.shape
        Bk, S, Hk, Ek = key.shape
        Bv, Sv, Hv, D = value.shape
        if (Bk, Hk, Ek) != (B, H, E) or (Bv, Sv, Hv) != (B, S, H):
            raise ValueError(f'shape mismatch: query {tuple(query.shape)}, key {tuple(key.shape)}, '
                             f'value {tuple(value.shape)}')
        if W.dim() != 2 or W.shape[1] != E:
            raise ValueError(f'projection must be (r, {E}), got {tuple(W.shape)}')
        dev = query.device
        # feature axis must be contiguous; the other axes are passed as strides
        query = query if query.stride(-1) == 1 else query.contiguous()
        key = key if key.stride(-1) == 1 else key.contiguous()
        value = value if value.stride(-1) == 1 else value.contiguous()
        W32 = W.detach()
        if W32.device != dev or W32.dtype != torch.float32 or not W32.is_contiguous():
            W32 = W32.to(device=dev, dtype=torch.float32).contiguous()
        if out is None:
            out = torch.empty(B, T, H, D, device=dev, dtype=query.dtype)
        elif (out.shape != (B, T, H, D) or out.dtype != query.dtype or out.stride(-1) != 1 or out.device != dev):
            raise ValueError('out must be (B,T,H,D) in the input dtype with a contiguous last axis, on the device of the '
                             'inputs')
        if key_lengths is not None:
            key_lengths = key_lengths.to(device=dev, dtype=torch.int64).contiguous()
            if key_lengths.shape != (B,):
                raise ValueError(f'key lengths must have shape ({B},)')
        tau = float(softmax_temp) if softmax_temp else 1.0 / math.sqrt(E)
        sum_lo, sum_hi = sum_range if sum_range is not None else (0, S)
        p = _cabi.pack_params(   # in the order of the fields
            _DTYPES[query.dtype], B, H, T, S, E, D, W.shape[0], int(local_context), tau, float(softmax_eps),
            query.data_ptr(), *query.stride()[:3], key.data_ptr(), *key.stride()[:3],
            value.data_ptr(), *value.stride()[:3], out.data_ptr(), *out.stride()[:3], W32.data_ptr(),
            key_lengths.data_ptr() if key_lengths is not None else 0, int(q_pos0), int(k_pos0),
            int(S_total) if S_total is not None else S, sum_lo, sum_hi, _cabi.SBL_FLAG_GENERIC_PATH if generic else 0,
            0, 0, 0)
        self.params = p
        self.device = dev
        self.out = out
        self.m = 2 * W.shape[0]
        self.shape = (B, H, T, S, E, D)
        self._keep = (query, key, value, W32, key_lengths, out)
        lib = _cabi.load()
        nbytes = ctypes.c_size_t(0)
        _cabi.check(lib.sbl_workspace_bytes(ctypes.byref(p), ctypes.byref(nbytes)))
        self.workspace_bytes = nbytes.value
        off = ctypes.c_size_t(0)
        self.status_offset = off.value if lib.sbl_status_words(ctypes.byref(p), ctypes.byref(off)) == 0 else None

    def workspace(self):
        """Grow-only scratch buffer per (device, stream)."""
        stream = torch.cuda.current_stream(self.device)
        key = (self.device.index, stream.cuda_stream)
        with _ws_lock:
            buf = _workspaces.get(key)
            if buf is None or buf.numel() < self.workspace_bytes:
                buf = torch.empty(max(self.workspace_bytes, 1 << 20), dtype=torch.uint8, device=self.device)
                _workspaces[key] = buf
        return buf

    def _call(self, fn, *extra, workspace=None):
        ws = workspace if workspace is not None else self.workspace()
        if ws.device != self.device or not ws.is_contiguous():
            raise ValueError('the workspace must be a contiguous tensor on the problem device')
        with _on(self.device):
            stream = _stream(self.device)
            rc = fn(ctypes.byref(self.params), ws.data_ptr(), ws.numel(), *extra, stream)
        _cabi.check(rc)
        return ws

    # -- entry points -----------------------------------------------------
    def forward(self, workspace=None, watch=False):
        """watch: queue the collection of the kernels' status words (see `status_watch`)."""
        ws = self._call(_cabi.load().sbl_forward, workspace=workspace)
        if watch and self.status_offset is not None:
            with _on(self.device):
                status_watch.post(ws.data_ptr() + self.status_offset, self.device)
        return self.out

    def forward_train(self, workspace):
        """Forward that also returns what `backward` needs of it: two fp32 per query row and one per head."""
        B, H, T = self.shape[:3]
        stats = torch.empty(2 * B * H * T + B * H, device=self.device, dtype=torch.float32)
        self._call(_cabi.load().sbl_forward_train, stats.data_ptr(), workspace=workspace)
        return self.out, stats

    def backward_workspace_bytes(self):
        n = ctypes.c_size_t(0)
        _cabi.check(_cabi.load().sbl_backward_workspace_bytes(ctypes.byref(self.params), ctypes.byref(n)))
        return n.value

    def backward(self, grad_out, row_stats, watch=False, needs=(True, True, True)):
        """(dq, dk, dv) of sum(grad_out * out); the problem's `out` must hold the output of `forward_train`.
        watch: as in `forward`.  needs: which of the three to form, None in the place of the others."""
        query, key, value = self._keep[:3]
        B, H, T, S, E, D = self.shape
        if grad_out.shape != (B, T, H, D) or grad_out.dtype != query.dtype or grad_out.device != self.device:
            raise ValueError('grad_out must be (B,T,H,D) in the input dtype on the problem device')
        if (row_stats.shape != (2 * B * H * T + B * H,) or row_stats.dtype != torch.float32
                or row_stats.device != self.device or not row_stats.is_contiguous()):
            raise ValueError('row_stats must be what forward_train of this problem returned')
        # (the tensor-core kernels read it through tensor maps: no broadcast axes, 16-byte steps)
        tensor = self.status_offset is not None
        if grad_out.stride(-1) != 1 or tensor and (grad_out.data_ptr() % 16 or T > 1 and grad_out.stride(1) < D or any(
                n > 1 and (st <= 0 or st % 8) for n, st in zip(grad_out.shape[:3], grad_out.stride()))):
            # (fresh storage: `contiguous` keeps a dense tensor where it is, and the stride of an axis of one as it is)
            grad_out = torch.empty((B, T, H, D), device=self.device, dtype=query.dtype).copy_(grad_out)
        nbytes = self.backward_workspace_bytes()
        grads = [torch.empty(x.shape, device=self.device, dtype=x.dtype) if need else None
                 for x, need in zip((query, key, value), needs)]
        # of this call alone: a backward pass may run on another stream or be captured while another one is alive
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        places = [n for x in grads for n in ((x.data_ptr(), *x.stride()[:3]) if x is not None else (0, 0, 0, 0))]
        skip = sum(bit for bit, need in zip(_cabi.SBL_SKIP, needs) if not need)
        g = _cabi.pack_grads(grad_out.data_ptr(), *grad_out.stride()[:3], row_stats.data_ptr(), *places, skip, 0, 0, 0)
        with _on(self.device):
            stream = _stream(self.device)
            rc = _cabi.load().sbl_backward(ctypes.byref(self.params), ctypes.byref(g), ws.data_ptr(), nbytes, stream)
            _cabi.check(rc)
            if tensor and watch:
                status_watch.post(ws.data_ptr(), self.device)
        return tuple(grads)

    def check_status(self, workspace=None):
        """Synchronises the stream; raises if a kernel gave up on a bounded wait."""
        self._call(_cabi.load().sbl_check_status, workspace=workspace)

    def key_logscale(self, workspace=None):
        B, H = self.shape[:2]
        beta = torch.empty(B, H, device=self.device, dtype=torch.float32)
        self._call(_cabi.load().sbl_key_logscale, beta.data_ptr(), workspace=workspace)
        return beta

    def key_summary(self, beta, workspace=None, out=None):
        """out: optional (kv, ksum) pair of contiguous fp32 tensors (B,H,m,D) and (B,H,m) to write into (a caller
        that all-reduces both can make them two views of one buffer)."""
        B, H, _, _, _, D = self.shape
        if out is None:
            kv = torch.empty(B, H, self.m, D, device=self.device, dtype=torch.float32)
            ksum = torch.empty(B, H, self.m, device=self.device, dtype=torch.float32)
        else:
            kv, ksum = out
            if (tuple(kv.shape) != (B, H, self.m, D) or tuple(ksum.shape) != (B, H, self.m)
                    or kv.dtype != torch.float32 or ksum.dtype != torch.float32
                    or not kv.is_contiguous() or not ksum.is_contiguous() or kv.device != self.device):
                raise ValueError('out must be contiguous fp32 (B,H,m,D) and (B,H,m) tensors on the problem device')
        beta = beta.contiguous()
        self._call(_cabi.load().sbl_key_summary, beta.data_ptr(), kv.data_ptr(), ksum.data_ptr(),
                   workspace=workspace)
        return kv, ksum

    def band_forward(self, beta, kv, ksum, workspace=None):
        beta, kv, ksum = beta.contiguous(), kv.contiguous(), ksum.contiguous()
        self._call(_cabi.load().sbl_band_forward, beta.data_ptr(), kv.data_ptr(), ksum.data_ptr(),
                   workspace=workspace)
        return self.out

    def attention_weights(self, unnormalized=False, workspace=None):
        """Dense (B,H,T,S) attention matrix (and, with `unnormalized`, the two
        unnormalised matrices) of the forward just run on this workspace; the
        problem must have been created with generic=True."""
        B, H, T, S = self.shape[:4]
        mk = lambda: torch.empty(B, H, T, S, device=self.device, dtype=torch.float32)
        attn = mk()
        un, lr = (mk(), mk()) if unnormalized else (None, None)
        self._call(_cabi.load().sbl_attention_weights, attn.data_ptr(), un.data_ptr() if unnormalized else None,
                   lr.data_ptr() if unnormalized else None, workspace=workspace)
        return (attn, un, lr) if unnormalized else attn

    def query_features(self):
        B, H, T = self.shape[:3]
        qp = torch.empty(B, H, T, self.m, device=self.device, dtype=torch.float32)
        ls = torch.empty(B, H, T, device=self.device, dtype=torch.float32)
        self._call(_cabi.load().sbl_query_features, qp.data_ptr(), ls.data_ptr())
        return qp, ls

    def key_features(self):
        B, H, _, S = self.shape[:4]
        kp = torch.empty(B, H, S, self.m, device=self.device, dtype=torch.float32)
        ls = torch.empty(B, H, device=self.device, dtype=torch.float32)
        self._call(_cabi.load().sbl_key_features, kp.data_ptr(), ls.data_ptr())
        return kp, ls


def sblocal_forward(query, key, value, W, local_context, softmax_temp=None, softmax_eps=0.0,
                    key_lengths=None, out=None, watch=False):
    """out (B,T,H,D) = SBLocal attention of query (B,T,H,E), key (B,S,H,E),
    value (B,S,H,D) with projection W (r,E); one call of `sbl_forward`."""
    return Problem(query, key, value, W, local_context, softmax_temp, softmax_eps, key_lengths,
                   out).forward(watch=watch)


def _refuse_tangents(*tensors):
    """Forward-mode differentiation is not built: without this a call would drop the tangents.  (Outside a dual level,
    where this torch says so, there are none to look for.)"""
    if getattr(forward_ad, '_current_level', 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError('sblocal_b200: forward-mode differentiation is not built')


class _SBLocal(torch.autograd.Function):
    """Differentiable SBLocal attention: saves the inputs, the output and two floats per query row; the gradients
    recompute the weights (sbl_backward)."""

    @staticmethod
    def forward(ctx, query, key, value, W, local_context, softmax_temp, softmax_eps, key_lengths, watch):
        prob = Problem(query, key, value, W, local_context, softmax_temp, softmax_eps, key_lengths)
        ctx.args, ctx.watch = (local_context, softmax_temp, softmax_eps), watch
        if softmax_eps != 0:
            # the forward is built for eps != 0, its gradients are not
            ctx.stats = None
            return prob.forward(watch=watch)
        # a workspace of this call alone, for the reason given in Problem.backward
        ws = torch.empty(prob.workspace_bytes, dtype=torch.uint8, device=prob.device)
        out, stats = prob.forward_train(ws)
        if watch and prob.status_offset is not None:
            with _on(prob.device):
                status_watch.post(ws.data_ptr() + prob.status_offset, prob.device)
        ctx.stats = True
        ctx.save_for_backward(query, key, value, W, key_lengths, out, stats)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        if ctx.stats is None:
            raise NotImplementedError('sblocal_b200: gradients are built for softmax_eps = 0 only')
        query, key, value, W, key_lengths, out, stats = ctx.saved_tensors
        prob = Problem(query, key, value, W, *ctx.args, key_lengths, out=out)
        grads = prob.backward(grad_out, stats, watch=ctx.watch, needs=ctx.needs_input_grad[:3])
        return *grads, None, None, None, None, None, None


def sblocal_attention(query, key, value, W, local_context, softmax_temp=None, softmax_eps=0.0, key_lengths=None,
                      watch=True):
    """`sblocal_forward` that autograd can differentiate in query, key and value (softmax_eps = 0; the projection W
    and the lengths are constants).  Rows of a batch without any real key give an output and gradients of zero, and
    padded keys gradients of zero.  Padded keys and values must hold finite numbers.  A step may be captured into a CUDA
    graph, lengths included, while no eager autograd graph of the same leaves is alive (torch ends the capture).
    watch: report what the kernels of this call, or of its gradients, found wrong to a later call (`status_watch`); a
    replayed step's reports are read by `status_watch.poll(wait=True)`."""
    if watch:
        status_watch.poll()
    _refuse_tangents(query, key, value)
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        return _SBLocal.apply(query, key, value, W, local_context, softmax_temp, softmax_eps, key_lengths, watch)
    return sblocal_forward(query, key, value, W, local_context, softmax_temp, softmax_eps, key_lengths, watch=watch)


# ---- norm and rotation of query and key heads -------------------------------------------------------------------

def _norm_rotary_params(xs, ys, weights, positions, pos0, rotary_dim, theta, interleaved, eps, dys=(None, None),
                        dws=(None, None)):
    """SblNormRotary of the tensors; those it points to must stay alive."""
    w = weights[0] if weights[0] is not None else weights[1]
    B, _, _, E = xs[0].shape
    fields = [_DTYPES[xs[0].dtype], _DTYPES[w.dtype] if w is not None else _cabi.SBL_DTYPE_F32, B, E, rotary_dim,
              1 if interleaved else 0, eps, theta]
    for x, y, dy, w, dw, pos in zip(xs, ys, dys, weights, dws, positions):
        fields += [x.shape[1], x.shape[2], x.data_ptr(), *x.stride()[:3]]
        fields += [y.data_ptr(), *y.stride()[:3]] if y is not None else [0, 0, 0, 0]
        fields += [dy.data_ptr(), *dy.stride()[:3]] if dy is not None else [0, 0, 0, 0]
        fields += [w.data_ptr() if w is not None else 0, dw.data_ptr() if dw is not None else 0]
        fields += ([pos.data_ptr(), pos.stride(0) if pos.dim() == 2 else 0, pos.stride(-1)] if pos is not None
                   else [0, 0, 0])
        fields.append(pos0)
    return _cabi.pack_norm_rotary(*fields, 0, 0, 0, 0)


def _norm_rotary_forward(xs, weights, positions, *args):
    dev = xs[0].device
    ys = tuple(torch.empty(x.shape, dtype=x.dtype, device=dev) for x in xs)
    p = _norm_rotary_params(xs, ys, weights, positions, *args)
    with _on(dev):
        rc = _cabi.load().sbl_norm_rotary_forward(ctypes.byref(p), _stream(dev))
    _cabi.check(rc)
    return ys


class _NormRotary(torch.autograd.Function):
    """Saves the inputs only: the norms are recomputed with the gradients."""

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, positions, key_positions, *args):
        ctx.save_for_backward(query, key, query_weight, key_weight, positions, key_positions)
        ctx.args = args
        return _norm_rotary_forward((query, key), (query_weight, key_weight), (positions, key_positions), *args)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        query, key, query_weight, key_weight, positions, key_positions = ctx.saved_tensors
        weights = (query_weight, key_weight)
        dev = query.device
        dys = [dy if dy.stride(-1) == 1 else dy.contiguous() for dy in (dq_out, dk_out)]
        dws = [torch.empty_like(w) if w is not None and ctx.needs_input_grad[2 + i] else None
               for i, w in enumerate(weights)]
        # (a side of which nothing is needed is left out; one whose weight alone is needed has the place of its dx)
        dxs = [torch.empty(x.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[i] or dws[i] is not None else None
               for i, x in enumerate((query, key))]
        p = _norm_rotary_params((query, key), dxs, weights, (positions, key_positions), *ctx.args, dys, dws)
        lib = _cabi.load()
        ws, nbytes = None, 0
        if dws[0] is not None or dws[1] is not None:
            n = ctypes.c_size_t(0)
            _cabi.check(lib.sbl_norm_rotary_workspace_bytes(ctypes.byref(p), ctypes.byref(n)))
            nbytes = n.value
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        with _on(dev):
            rc = lib.sbl_norm_rotary_backward(ctypes.byref(p), ws.data_ptr() if ws is not None else None, nbytes,
                                              _stream(dev))
        _cabi.check(rc)
        return (*(dx if need else None for dx, need in zip(dxs, ctx.needs_input_grad)), *dws,
                *([None] * (2 + len(ctx.args))))


def qk_norm_rotary(query, key, query_weight=None, key_weight=None, positions=None, key_positions=None, pos0=0,
                   rotary_dim=None, theta=10000.0, interleaved=False, eps=1e-6):
    """Root-mean-square norm of every query and key head, times a weight over the head dim, then the rotation of
    its first `rotary_dim` entries by the row's position, in one kernel for both tensors; autograd differentiates it
    in the inputs and the weights.

    query (B,T,Hq,E), key (B,S,Hk,E), float32 or bfloat16, any strides over the first three axes; weights (E,)
    float32 or bfloat16, or None for ones.  positions: int64 (T,) or (B,T), negative ones too; key_positions the
    same over S, by default `positions` (which then has to fit both).  Without positions row t has position
    pos0 + t.  rotary_dim: even, by default all of an even E; pair i turns by position * theta^(-2i / rotary_dim); pairs are
    (i, i + rotary_dim / 2), or (2i, 2i + 1) with `interleaved`.  Returns new contiguous (query, key)."""
    _refuse_tangents(query, key, query_weight, key_weight)
    if not (query.is_cuda and key.is_cuda):
        raise ValueError('sblocal_b200 runs on CUDA tensors only (there is no CPU path)')
    if query.dim() != 4 or key.dim() != 4 or query.shape[0] != key.shape[0] or query.shape[3] != key.shape[3]:
        raise ValueError(f'query/key must be (B,T,Hq,E), (B,S,Hk,E): got {tuple(query.shape)}, {tuple(key.shape)}')
    if query.dtype not in _DTYPES:
        raise TypeError(f'dtype {query.dtype} is not supported (float32 and bfloat16 are)')
    if key.dtype != query.dtype:
        raise TypeError('query and key must share one dtype')
    dev, E = query.device, query.shape[3]
    if key.device != dev:
        raise ValueError('query and key must be on one device')
    if query.shape[2] == 0 or key.shape[2] == 0 or E == 0:
        raise ValueError('query and key need at least one head and one entry')
    for w in (query_weight, key_weight):
        if w is not None and (w.shape != (E,) or w.device != dev):
            raise ValueError(f'weights must have shape ({E},) on the device of the query')
        if w is not None and w.dtype not in _DTYPES:
            raise TypeError(f'weight dtype {w.dtype} is not supported (float32 and bfloat16 are)')
    if query_weight is not None and key_weight is not None and query_weight.dtype != key_weight.dtype:
        raise TypeError('the two weights must share one dtype')
    if key_positions is None:
        key_positions = positions
    places = []
    for pos, x, name in ((positions, query, 'positions'), (key_positions, key, 'key_positions')):
        if pos is not None:
            if tuple(pos.shape) not in ((x.shape[1],), (x.shape[0], x.shape[1])):
                raise ValueError(f'{name} must be ({x.shape[1]},) or ({x.shape[0]}, {x.shape[1]}), got '
                                 f'{tuple(pos.shape)}')
            if pos.dtype != torch.int64 or pos.device != dev:
                raise ValueError(f'{name} must be int64 on the device of the query')
        places.append(pos)
    rotary_dim = E - E % 2 if rotary_dim is None else int(rotary_dim)
    if rotary_dim < 0 or rotary_dim > E or rotary_dim % 2:
        raise ValueError(f'rotary_dim must be even and in 0..{E}, got {rotary_dim}')
    query = query if query.stride(-1) == 1 else query.contiguous()
    key = key if key.stride(-1) == 1 else key.contiguous()
    query_weight, key_weight = (w if w is None or w.is_contiguous() else w.contiguous()
                                for w in (query_weight, key_weight))
    args = (int(pos0), rotary_dim, float(theta), bool(interleaved), float(eps))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (query, key, query_weight, key_weight)):
        return _NormRotary.apply(query, key, query_weight, key_weight, *places, *args)
    return _norm_rotary_forward((query, key), (query_weight, key_weight), places, *args)
